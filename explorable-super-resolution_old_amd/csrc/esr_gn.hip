// esr_gn.hip — GroupNorm + LeakyReLU on channels-last activations [N][HW][C] fp32: forward, backward and the backward's
// own backward (the WGAN-GP penalty differentiates the discriminator's input gradient once more, loss.py:244-263).
//
// G groups of Cg = C/G channels, M = HW·Cg values of one (sample, group):
//   μ, v = mean / biased variance, r = (v + eps)^-1/2, x̂ = (x − μ)·r, z = γ_c·x̂ + β_c, y = z > 0 ? z : a·z.
// Backward (m = z > 0 ? 1 : a, gz = gy·m, h = γ_c·gz, sums over the group; s1, s2 per (sample, channel)):
//   s1 = Σ gz, s2 = Σ gz·x̂, S1 = Σ h, S2 = Σ h·x̂;  gx = r·(h − S1/M − x̂·S2/M), dβ = Σ_n s1, dγ = Σ_n s2.
// Double backward of (x, γ, gy) -> (gx, dγ, dβ) for upstream (u, ga, gb) (the mask is piecewise constant), with
// U = Σ u, A = Σ u·x̂, Q = Σ u·h:
//   g_gy = m·[γ·r·(u − U/M − x̂·A/M) + ga·x̂ + gb],   g_γ = Σ_n r·(Σ_p u·gz − s1·U/M − s2·A/M)
//   G = −r·(h·A + u·S2)/M + ga·gz                     (∂/∂x̂ at fixed r)
//   g_x = r·(G − mean G − x̂·mean(G·x̂)) − (Q − S1·U/M − S2·A/M)·r²·x̂/M
//   mean G = (−r·(S1·A + U·S2)/M + Σ_c ga·s1)/M,  mean(G·x̂) = (−2r·S2·A/M + Σ_c ga·s2)/M.
//
// Statistics, sums and the pre-activation z are in float64: a z next to 0 decides between a slope of 1 and a, and an
// fp32 z is uncertain there in every 10^7-th value, while HBM still bounds the passes.  All sums run in a fixed order.
// With 8-bit blocks (esr_act8.h) the forward also writes x's codes, and the backward reads them in place of x: μ and r
// stay those of x, everything else is evaluated at the codes' values, and a code that rounding took over the kink goes
// one step back over it, so that every mask bit is the forward's.  (Without that, at a step of max|x|/127 about one
// value in 200 changed its slope: 5 % of the gradient's norm against the codes' own 0.6 %.)
#include "esr_act8.h"
#include "esr_amd.h"
#include "esr_knobs.h"
#include <initializer_list>

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int NT = 256;
constexpr int MAXS = 256;   // row splits of a sample in a reduction
constexpr int UN = 4;       // rows of a thread in flight

// A thread holds V consecutive channels (V = 4: 16-byte accesses; V = 1 where C or a base is not a multiple of 4 values)
// and walks rows; the 32 / V lanes of an 8-bit block sit side by side, a row takes `lanes` threads (its last block padded
// to 32 channels) and a workgroup `rpi` rows at a time.  Rows wider than a workgroup are cut over blockIdx.z.
struct GnP {
    const float *x;              // [N][HW][C], or null: codes / exps
    const int8_t *codes;
    const uint8_t *exps;
    const float *gy, *u;         // [N][HW][C]
    const float *gamma, *beta;   // [C] or null (1, 0)
    const float *gga, *ggb;      // [C] upstream of dγ, dβ, or null
    const double *stat;          // [N][G][2]: μ and r
    const double *grp;           // [N][G][8] per-group coefficients of the pass
    const double *sums, *sums_u; // [N][2][C]: s1, s2; [N][3][C]: Σu, Σu·x̂, Σu·gz
    long long HW;
    int N, C, G, Cg, nb, lanes, rpi, chunks, splits, blocks;
    float slope, eps;
};

// x̂ and z of one value, by the same operations everywhere.  (x − μ)·r rather than x·r − μ·r: the values of a constant
// group are their mean exactly, and their z is β.
__device__ __forceinline__ double xhat(double x, double r, double mu) { return (x - mu) * r; }
__device__ __forceinline__ double preact(double xh, double gamma, double beta) { return fma(gamma, xh, beta); }

template <int V>
__device__ __forceinline__ void load_f(const float *src, long long i, float *v) {
    if constexpr (V == 4) {
        const float4 t = *reinterpret_cast<const float4 *>(src + i);
        v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
    } else {
        v[0] = src[i];
    }
}
// (non-temporal: what a pass writes does not push what the next one reads out of the 256 MB last-level cache)
template <int V>
__device__ __forceinline__ void store_f(float *dst, long long i, const float *v) {
    if constexpr (V == 4) __builtin_nontemporal_store((f32x4){v[0], v[1], v[2], v[3]}, reinterpret_cast<f32x4 *>(dst + i));
    else __builtin_nontemporal_store(v[0], dst + i);
}
// a row's raw input (values, or a word of codes and its exponent byte), loaded ahead of its use
template <int V, bool Q8>
struct Raw {
    float v[V];
    uint32_t w;
    int e;
    __device__ __forceinline__ void load(const GnP &p, long long row, int c) {
        if constexpr (Q8) {
            if constexpr (V == 4) w = *reinterpret_cast<const uint32_t *>(p.codes + row * p.C + c);
            else w = (uint8_t)p.codes[row * p.C + c];
            e = p.exps[row * p.nb + c / act8::BLK];
        } else {
            load_f<V>(p.x, row * p.C + c, v);
        }
    }
    __device__ __forceinline__ float at(int k) const {
        if constexpr (Q8) return act8::value_of(act8::code_at(w, k), e);
        else return v[k];
    }
};
// per-channel constants of a thread
template <int V>
struct Chan {
    double mu[V], r[V], ga[V], be[V];
    __device__ __forceinline__ void load(const GnP &p, int n, int c) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const long long g = (long long)n * p.G + (c + k) / p.Cg;
            mu[k] = p.stat[2 * g];
            r[k] = p.stat[2 * g + 1];
            ga[k] = p.gamma ? (double)p.gamma[c + k] : 1.0;
            be[k] = p.beta ? (double)p.beta[c + k] : 0.0;
        }
    }
};

// partial[n][split][k][c]: MODE 0: Σd, Σd² (d = x − the group's first value); 1: Σgz, Σgz·x̂; 2: Σu, Σu·x̂, Σu·gz
template <int MODE, int V, bool Q8>
__global__ __launch_bounds__(NT) void gn_sums(GnP p, double *partial) {
    constexpr int K = MODE == 2 ? 3 : 2;
    __shared__ double red[K * V][NT];
    const int tid = threadIdx.x, lane = tid % p.lanes, ph = tid / p.lanes, n = blockIdx.y, sp = blockIdx.x;
    const int c = ((int)blockIdx.z * NT + lane) * V;
    const long long r0 = p.HW * sp / p.splits, r1 = p.HW * (sp + 1) / p.splits;
    double s[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) s[k][v] = 0.0;
    if (ph < p.rpi && c < p.C) {
        Chan<V> ch;
        double pivot[V];
        if constexpr (MODE == 0) {
#pragma unroll
            for (int v = 0; v < V; ++v) pivot[v] = p.x[(long long)n * p.HW * p.C + (c + v) / p.Cg * p.Cg];
        } else {
            ch.load(p, n, c);
        }
        for (long long q = r0 + ph; q < r1; q += UN * p.rpi) {
            Raw<V, Q8> raw[UN];
            float gy[UN][V], u[UN][V];
#pragma unroll
            for (int j = 0; j < UN; ++j) {  // rows past the end load the last one and are not added
                const long long row = (long long)n * p.HW + min(q + j * p.rpi, r1 - 1);
                raw[j].load(p, row, c);
                if constexpr (MODE >= 1) load_f<V>(p.gy, row * p.C + c, gy[j]);
                if constexpr (MODE == 2) load_f<V>(p.u, row * p.C + c, u[j]);
            }
#pragma unroll
            for (int j = 0; j < UN; ++j) {
                if (q + j * p.rpi >= r1) break;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const double x = raw[j].at(v);
                    if constexpr (MODE == 0) {
                        const double d = x - pivot[v];
                        s[0][v] += d;
                        s[1][v] = fma(d, d, s[1][v]);
                    } else {
                        const double xh = xhat(x, ch.r[v], ch.mu[v]);
                        const double gz = gy[j][v] * (preact(xh, ch.ga[v], ch.be[v]) > 0.0 ? 1.f : p.slope);
                        if constexpr (MODE == 1) {
                            s[0][v] += gz;
                            s[1][v] = fma(gz, xh, s[1][v]);
                        } else {
                            s[0][v] += u[j][v];
                            s[1][v] = fma((double)u[j][v], xh, s[1][v]);
                            s[K - 1][v] = fma((double)u[j][v], gz, s[K - 1][v]);
                        }
                    }
                }
            }
        }
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) red[k * V + v][tid] = s[k][v];
    __syncthreads();
    for (int i = tid; i < K * V * p.lanes; i += NT) {  // the rows of a workgroup, in order
        const int ln = i / V % p.lanes, k = i / V / p.lanes, v = i % V;
        const int cc = ((int)blockIdx.z * NT + ln) * V + v;
        if (cc >= p.C) continue;
        double t = red[k * V + v][ln];
        for (int q = 1; q < p.rpi; ++q) t += red[k * V + v][q * p.lanes + ln];
        partial[(((long long)n * p.splits + sp) * K + k) * p.C + cc] = t;
    }
}

// One workgroup per sample and set of whole groups (32 channels' worth, or one larger group): the splits' sums per
// channel (sums_out [n][K][C], or null), then each group's: MODE 0: out = μ, r; 1: S1/M, S2/M; 2: the seven coefficients
// of the double backward (partial null: no upstream of gx).
template <int MODE>
__global__ __launch_bounds__(NT) void gn_finish(GnP p, const double *partial, double *sums_out, double *out) {
    constexpr int K = MODE == 2 ? 3 : 2, J = MODE == 2 ? 7 : 2;
    __shared__ double part[8][K][32], chan[J][33], tot[J][32];
    const int tid = threadIdx.x, lane = tid & 31, sl = tid >> 5, n = blockIdx.y;
    const int gpb = p.Cg <= 32 ? 32 / p.Cg : 1, g0 = blockIdx.x * gpb, ng = min(gpb, p.G - g0);
    const int c1 = (g0 + ng) * p.Cg;
    for (int i = tid; i < J * 32; i += NT) tot[i / 32][i % 32] = 0.0;
    for (int c0 = g0 * p.Cg; c0 < c1; c0 += 32) {
        const int c = c0 + lane;
        double s[K] = {};
        if (c < c1 && partial)
#pragma unroll 4
            for (int sp = sl; sp < p.splits; sp += 8)
#pragma unroll
                for (int k = 0; k < K; ++k) s[k] += partial[(((long long)n * p.splits + sp) * K + k) * p.C + c];
#pragma unroll
        for (int k = 0; k < K; ++k) part[sl][k][lane] = s[k];
        __syncthreads();
        if (sl == 0) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                s[k] = part[0][k][lane];
                for (int q = 1; q < 8; ++q) s[k] += part[q][k][lane];
                if (sums_out && c < c1) sums_out[((long long)n * K + k) * p.C + c] = s[k];
            }
            const double ga = MODE && p.gamma && c < c1 ? (double)p.gamma[c] : 1.0;
            if constexpr (MODE < 2) {
                chan[0][lane] = ga * s[0];
                chan[1][lane] = ga * s[1];
            } else {
                const bool in = c < c1;
                const double s1 = in ? p.sums[(long long)n * 2 * p.C + c] : 0.0;
                const double s2 = in ? p.sums[((long long)n * 2 + 1) * p.C + c] : 0.0;
                const double a = in && p.gga ? (double)p.gga[c] : 0.0;
                chan[0][lane] = ga * s1;
                chan[1][lane] = ga * s2;
                chan[2][lane] = s[0];
                chan[3][lane] = s[1];
                chan[4][lane] = ga * s[K - 1];
                chan[5][lane] = p.gga ? a * s1 : 0.0;
                chan[6][lane] = p.gga ? a * s2 : 0.0;
            }
        }
        __syncthreads();
        for (int i = tid; i < J * ng; i += NT) {  // channels of a group, in order
            const int j = i / ng, g = i - j * ng, a = p.Cg <= 32 ? g * p.Cg : 0;
            const int b = p.Cg <= 32 ? a + p.Cg : min(32, c1 - c0);
            double t = tot[j][g];
            for (int k = a; k < b; ++k) t += chan[j][k];
            tot[j][g] = t;
        }
        __syncthreads();
    }
    if (tid >= ng) return;
    const long long i = (long long)n * p.G + g0 + tid;
    const double M = (double)p.HW * p.Cg, t0 = tot[0][tid] / M, t1 = tot[1][tid] / M;
    if constexpr (MODE == 0) {
        const double var0 = t1 - t0 * t0, var = var0 < 0.0 ? 0.0 : var0;  // (a NaN stays one)
        out[2 * i] = p.x[(long long)n * p.HW * p.C + (g0 + tid) * p.Cg] + t0;
        out[2 * i + 1] = 1.0 / sqrt(var + (double)p.eps);
    } else if constexpr (MODE == 1) {
        out[8 * i] = t0;
        out[8 * i + 1] = t1;
    } else {
        const double r = p.stat[2 * i + 1], u = tot[J - 5][tid] / M, a = tot[J - 4][tid] / M;
        out[8 * i] = u;
        out[8 * i + 1] = a;
        out[8 * i + 2] = t0;
        out[8 * i + 3] = t1;
        out[8 * i + 4] = -r * (t0 * a + u * t1) + tot[J - 2][tid] / M;
        out[8 * i + 5] = -2.0 * r * t1 * a + tot[J - 1][tid] / M;
        out[8 * i + 6] = (tot[J - 3][tid] / M - t0 * u - t1 * a) * r * r;
    }
}

// codes of V values of one row in a block whose lanes call together; pre: z of a value
template <int V, typename F>
__device__ __forceinline__ void put_blocks(const GnP &p, const float *v, bool act, long long row, int c, int lane,
                                           int8_t *codes, uint8_t *exps, F pre) {
    constexpr int L = act8::BLK / V;
    unsigned m = 0;
#pragma unroll
    for (int k = 0; k < V; ++k) m = max(m, act8::abs_bits(v[k]));
    const int e = act8::exp_of(act8::block_max<L>(m));
    if (!act) return;
    uint32_t w = 0;
#pragma unroll
    for (int k = 0; k < V; ++k) {
        float code = act8::code_of(v[k], e);
        if (e != 255) {
            const float at = act8::value_of(code, e);
            if (pre(at, k) != pre(v[k], k)) code += at > v[k] ? -1.f : 1.f;
        }
        w |= (uint32_t)(uint8_t)(int8_t)(int)code << (8 * k);
    }
    if constexpr (V == 4) *reinterpret_cast<uint32_t *>(codes + row * p.C + c) = w;
    else codes[row * p.C + c] = (int8_t)w;
    if (lane % L == 0) exps[row * p.nb + c / act8::BLK] = (uint8_t)e;
}

struct GnOut {
    float *o1, *o2;          // MODE 0: y; 1: gx; 2: g_x, g_gy
    float *g_gamma, *g_beta; // [C] or null
    int8_t *codes, *ycodes;  // MODE 0: x's and y's 8-bit blocks, or null
    uint8_t *exps, *yexps;
};

// The elementwise pass.  The first row block of the first sample also sums the parameter gradients over the samples, in
// order.
// BITS: MODE 1, 2: the input is in 8-bit blocks; MODE 0: blocks are written.
template <int MODE, int V, bool BITS>
__global__ __launch_bounds__(NT) void gn_apply(GnP p, GnOut o) {
    constexpr int UA = MODE == 2 ? 2 : UN;
    constexpr bool Q8 = MODE && BITS;
    const int tid = threadIdx.x, lane = tid % p.lanes, ph = tid / p.lanes;
    const int n = blockIdx.y, b = blockIdx.x;
    const int c = ((int)blockIdx.z * NT + lane) * V;
    const bool act = c < p.C;
    if (ph >= p.rpi) return;
    if (MODE && b == 0 && n == 0 && ph == 0 && act) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            double s = 0.0, t = 0.0;
            for (int i = 0; i < p.N; ++i) {
                const double *q = p.sums + (long long)i * 2 * p.C + c + v;
                if constexpr (MODE == 1) {
                    s += q[p.C];
                    t += q[0];
                } else if (p.sums_u) {
                    const long long g = (long long)i * p.G + (c + v) / p.Cg;
                    s += p.stat[2 * g + 1] * (p.sums_u[((long long)i * 3 + 2) * p.C + c + v] - q[0] * p.grp[8 * g] -
                                              q[p.C] * p.grp[8 * g + 1]);
                }
            }
            if (o.g_gamma) o.g_gamma[c + v] = (float)s;
            if (MODE == 1 && o.g_beta) o.g_beta[c + v] = (float)t;
        }
    }
    Chan<V> ch;
    float k0[V], k1[V], k3[V], k4[V], k5[V], k6[V], ua[V], ub[V];
    if (act) {
        ch.load(p, n, c);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if constexpr (MODE >= 1) {
                const double *k = p.grp + 8 * ((long long)n * p.G + (c + v) / p.Cg);
                k0[v] = (float)k[0];
                k1[v] = (float)k[1];
                if constexpr (MODE == 2) {
                    k3[v] = (float)k[3];
                    k4[v] = (float)k[4];
                    k5[v] = (float)k[5];
                    k6[v] = (float)k[6];
                    ua[v] = p.gga ? p.gga[c + v] : 0.f;
                    ub[v] = p.ggb ? p.ggb[c + v] : 0.f;
                }
            }
        }
    }
    const long long r0 = p.HW * b / p.blocks, r1 = p.HW * (b + 1) / p.blocks;
    for (long long q = r0 + ph; q < r1; q += UA * p.rpi) {
        Raw<V, Q8> raw[UA];
        float gy[UA][V], u[UA][V];
        if (act) {
#pragma unroll
            for (int j = 0; j < UA; ++j) {
                const long long row = (long long)n * p.HW + min(q + j * p.rpi, r1 - 1);
                raw[j].load(p, row, c);
                if constexpr (MODE >= 1) load_f<V>(p.gy, row * p.C + c, gy[j]);
                if constexpr (MODE == 2) {
                    if (p.u) load_f<V>(p.u, row * p.C + c, u[j]);
                    else
#pragma unroll
                        for (int v = 0; v < V; ++v) u[j][v] = 0.f;
                }
            }
        }
#pragma unroll
        for (int j = 0; j < UA; ++j) {
            if (q + j * p.rpi >= r1) break;
            const long long row = (long long)n * p.HW + q + j * p.rpi;
            float a[V], d[V];
            if (act) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const double xd = xhat(raw[j].at(v), ch.r[v], ch.mu[v]), z = preact(xd, ch.ga[v], ch.be[v]);
                    if constexpr (MODE == 0) {
                        a[v] = (float)(z * (z > 0.0 ? 1.0 : (double)p.slope));
                    } else {
                        const float m = z > 0.0 ? 1.f : p.slope, xh = (float)xd, rf = (float)ch.r[v], gf = (float)ch.ga[v];
                        const float gz = gy[j][v] * m, h = gf * gz;
                        if constexpr (MODE == 1) {
                            a[v] = rf * (h - k0[v] - xh * k1[v]);
                        } else {
                            const float uu = u[j][v], gg = -rf * (h * k1[v] + uu * k3[v]) + ua[v] * gz;
                            d[v] = m * (gf * rf * (uu - k0[v] - xh * k1[v]) + ua[v] * xh + ub[v]);
                            a[v] = rf * (gg - k4[v] - xh * k5[v]) - k6[v] * xh;
                        }
                    }
                }
                store_f<V>(o.o1, row * p.C + c, a);
                if constexpr (MODE == 2) store_f<V>(o.o2, row * p.C + c, d);
            }
            if constexpr (MODE == 0 && BITS) {
                float t[V];
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    t[v] = act ? raw[j].at(v) : 0.f;
                    a[v] = act ? a[v] : 0.f;
                }
                if (o.codes)
                    put_blocks<V>(p, t, act, row, c, lane, o.codes, o.exps, [&](float x, int v) {
                        return preact(xhat(x, ch.r[v], ch.mu[v]), ch.ga[v], ch.be[v]) > 0.0;
                    });
                if (o.ycodes)
                    put_blocks<V>(p, a, act, row, c, lane, o.ycodes, o.yexps, [](float y, int) { return y > 0.f; });
            }
        }
    }
}

inline int launched() { return hipGetLastError() == hipSuccess ? ESR_OK : ESR_ELAUNCH; }

inline bool shape_ok(int64_t N, int64_t HW, int32_t C, int32_t G) {
    if (N <= 0 || HW <= 0 || C <= 0 || G <= 0 || C % G || C > (1 << 24)) return false;
    if (N > 65535 || (int64_t)N * G > 0x7fffffffLL) return false;
    return HW <= (1LL << 46) / C / N;  // element offsets, with room for the row arithmetic
}
inline bool bits_ok(const void *x, const void *codes, const void *exps) {
    return x ? !codes && !exps : codes && exps;  // exactly one form of the input
}
inline bool aligned(std::initializer_list<const void *> f32, std::initializer_list<const void *> codes) {
    for (const void *q : f32)
        if ((uintptr_t)q % 16) return false;
    for (const void *q : codes)
        if ((uintptr_t)q % 4) return false;
    return true;
}

GnP params(int V, int64_t N, int64_t HW, int32_t C, int32_t G, const float *gamma, const float *beta, float slope) {
    GnP p{};
    p.gamma = gamma; p.beta = beta;
    p.N = (int)N; p.HW = HW; p.C = C; p.G = G; p.Cg = C / G; p.slope = slope;
    p.nb = (C + act8::BLK - 1) / act8::BLK;
    const int lanes = p.nb * (act8::BLK / V);
    p.chunks = (lanes + NT - 1) / NT;
    p.lanes = lanes < NT ? lanes : NT;
    p.rpi = NT / p.lanes;
    // ~4 workgroups per CU for the sums (each leaves K·C float64 partials), 8 for the elementwise pass, of at least UN
    // rows per thread
    const int64_t per = (int64_t)N * p.chunks, rows = (HW + UN * p.rpi - 1) / (UN * p.rpi);
    auto cut = [&](int64_t want, int64_t most) {
        int64_t s = (want + per - 1) / per;
        s = s < rows ? s : rows;
        return (int)(s < most ? s : most);
    };
    p.splits = cut(1024, MAXS);
    p.blocks = cut(2048, 0x7fffffff);
    return p;
}

template <int MODE, bool Q8>
void sums(const GnP &p, int V, double *partial, hipStream_t st) {
    const dim3 grid(p.splits, p.N, p.chunks);
    if (V == 4) hipLaunchKernelGGL((gn_sums<MODE, 4, Q8>), grid, dim3(NT), 0, st, p, partial);
    else hipLaunchKernelGGL((gn_sums<MODE, 1, Q8>), grid, dim3(NT), 0, st, p, partial);
}
template <int MODE>
void finish(const GnP &p, const double *partial, double *sums_out, double *out, hipStream_t st) {
    const int gpb = p.Cg <= 32 ? 32 / p.Cg : 1;
    hipLaunchKernelGGL(gn_finish<MODE>, dim3((p.G + gpb - 1) / gpb, p.N), dim3(NT), 0, st, p, partial, sums_out, out);
}
template <int MODE, bool BITS>
void apply(const GnP &p, int V, const GnOut &o, hipStream_t st) {
    const dim3 grid(p.blocks, p.N, p.chunks);
    if (V == 4) hipLaunchKernelGGL((gn_apply<MODE, 4, BITS>), grid, dim3(NT), 0, st, p, o);
    else hipLaunchKernelGGL((gn_apply<MODE, 1, BITS>), grid, dim3(NT), 0, st, p, o);
}

}  // namespace

extern "C" int64_t esr_gn_workspace_bytes(int64_t N, int64_t HW, int32_t C, int32_t G) {
    if (!shape_ok(N, HW, C, G)) return ESR_EINVAL;
    const int64_t s1 = params(1, N, HW, C, G, nullptr, nullptr, 0.f).splits;
    const int64_t s4 = params(4, N, HW, C, G, nullptr, nullptr, 0.f).splits;
    // split sums [N][splits][3][C], sums of u [N][3][C], group coefficients [N][G][8]
    return 8 * (N * (s1 > s4 ? s1 : s4) * 3 * C + N * 3 * C + N * G * 8);
}

extern "C" int esr_gn_lrelu_fwd(const float *x, int64_t N, int64_t HW, int32_t C, int32_t G, const float *gamma,
                                const float *beta, float eps, float slope, float *y, double *stat, int8_t *codes,
                                uint8_t *exps, int8_t *ycodes, uint8_t *yexps, void *ws, esr_stream_t stream) {
    if (!x || !y || !stat || !ws || !shape_ok(N, HW, C, G) || !(eps >= 0.f) || !codes != !exps || !ycodes != !yexps)
        return ESR_EINVAL;
    const hipStream_t st = (hipStream_t)stream;
    const int V = C % 4 == 0 && aligned({x, y}, {codes, ycodes}) ? 4 : 1;
    GnP p = params(V, N, HW, C, G, gamma, beta, slope);
    p.x = x; p.eps = eps;
    double *partial = (double *)ws;
    sums<0, false>(p, V, partial, st);
    finish<0>(p, partial, nullptr, stat, st);
    p.stat = stat;
    const GnOut o{y, nullptr, nullptr, nullptr, codes, ycodes, exps, yexps};
    if (codes || ycodes) apply<0, true>(p, V, o, st);
    else apply<0, false>(p, V, o, st);
    return launched();
}

extern "C" int esr_gn_lrelu_bwd(const float *x, const int8_t *codes, const uint8_t *exps, const float *gy, int64_t N,
                                int64_t HW, int32_t C, int32_t G, const float *gamma, const float *beta,
                                const double *stat, float slope, float *gx, float *g_gamma, float *g_beta, double *sums_,
                                void *ws, esr_stream_t stream) {
    if (!bits_ok(x, codes, exps) || !gy || !gx || !stat || !sums_ || !ws || !shape_ok(N, HW, C, G)) return ESR_EINVAL;
    const hipStream_t st = (hipStream_t)stream;
    const int V = C % 4 == 0 && aligned({x, gy, gx}, {codes}) ? 4 : 1;
    GnP p = params(V, N, HW, C, G, gamma, beta, slope);
    p.x = x; p.codes = codes; p.exps = exps; p.gy = gy; p.stat = stat;
    double *partial = (double *)ws, *grp = partial + N * p.splits * 3 * C + N * 3 * C;
    if (x) sums<1, false>(p, V, partial, st);
    else sums<1, true>(p, V, partial, st);
    finish<1>(p, partial, sums_, grp, st);
    p.grp = grp; p.sums = sums_;
    const GnOut o{gx, nullptr, g_gamma, g_beta, nullptr, nullptr, nullptr, nullptr};
    if (x) apply<1, false>(p, V, o, st);
    else apply<1, true>(p, V, o, st);
    return launched();
}

extern "C" int esr_gn_lrelu_bwd2(const float *x, const int8_t *codes, const uint8_t *exps, const float *gy,
                                 const float *u, const float *gg_gamma, const float *gg_beta, int64_t N, int64_t HW,
                                 int32_t C, int32_t G, const float *gamma, const float *beta, const double *stat,
                                 float slope, const double *sums_, float *g_x, float *g_gy, float *g_gamma, void *ws,
                                 esr_stream_t stream) {
    if (!bits_ok(x, codes, exps) || !gy || !stat || !sums_ || !g_x || !g_gy || !ws || !shape_ok(N, HW, C, G))
        return ESR_EINVAL;
    const hipStream_t st = (hipStream_t)stream;
    const int V = C % 4 == 0 && aligned({x, gy, u, g_x, g_gy}, {codes}) ? 4 : 1;
    GnP p = params(V, N, HW, C, G, gamma, beta, slope);
    p.x = x; p.codes = codes; p.exps = exps; p.gy = gy; p.u = u; p.gga = gg_gamma; p.ggb = gg_beta; p.stat = stat;
    p.sums = sums_;
    double *partial = (double *)ws, *su = partial + N * p.splits * 3 * C, *grp = su + N * 3 * C;
    if (u) {
        if (x) sums<2, false>(p, V, partial, st);
        else sums<2, true>(p, V, partial, st);
    }
    finish<2>(p, u ? partial : nullptr, su, grp, st);
    p.grp = grp; p.sums_u = u ? su : nullptr;
    const GnOut o{g_x, g_gy, g_gamma, nullptr, nullptr, nullptr, nullptr, nullptr};
    if (x) apply<2, false>(p, V, o, st);
    else apply<2, true>(p, V, o, st);
    return launched();
}
