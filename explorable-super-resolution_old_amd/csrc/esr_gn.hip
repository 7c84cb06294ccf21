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
//
// HBM bounds the large maps: a pass reads its inputs twice (sums, then values) and writes once.  Measured at 16×152×152 ×
// 128 channels (189 MB a tensor): forward 30 + 60 us, backward 59 + 97 us, 5.8 to 6.4 TB/s, where a copy of such a tensor
// reaches 5.35; in float32 arithmetic the four kernels were 1 to 7 % faster.  Working through the samples in halves that
// fit the last-level cache was no faster.  Reading once (a sample's values held in the CUs' registers until its sums are
// known, 20 bytes a value of forward and backward in place of 32) would make workgroups wait for each other.  Small maps
// are bound by launches, hence gn_small.
#include "esr_act8.h"
#include "esr_amd.h"
#include "esr_knobs.h"
#include <initializer_list>

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int NT = 256, NTS = 1024;
constexpr int SMALL_C = 256;  // channels of a chunk of gn_small, at most
constexpr int MAXS = 256;   // row splits of a sample in a reduction
constexpr int UN = 4;       // rows of a thread in flight

// A thread holds V consecutive channels (V = 4: 16-byte accesses; V = 1 where C or a base is not a multiple of 4 values)
// and walks rows; the 32 / V lanes of an 8-bit block sit side by side, a row takes `lanes` threads (its last block padded
// to 32 channels) and a workgroup `rpi` rows at a time.  Rows are cut into chunks of `step` channels over the grid: what a
// workgroup has threads for, or (gn_small) the fewest whole groups and blocks.
//
// Three launches a pass: gn_sums over row splits, gn_finish per sample and set of groups, gn_apply.  Where a chunk of a
// sample has few values, gn_small does the three steps of a pass in one workgroup of 1024 threads.
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
    int N, C, G, Cg, nb, cp, lanes, rpi, step, chunks, splits, blocks;
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
            if constexpr (V == 4) w = *reinterpret_cast<const uint32_t *>(p.codes + row * p.cp + c);
            else w = (uint8_t)p.codes[row * p.cp + c];
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
// per-channel constants of a thread; stat: the statistics from group g0 on of its sample
template <int V>
struct Chan {
    double mu[V], r[V], ga[V], be[V];
    __device__ __forceinline__ void load(const GnP &p, const double *stat, int g0, int c) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int g = (c + k) / p.Cg - g0;
            mu[k] = stat[2 * g];
            r[k] = stat[2 * g + 1];
            ga[k] = p.gamma ? (double)p.gamma[c + k] : 1.0;
            be[k] = p.beta ? (double)p.beta[c + k] : 0.0;
        }
    }
};

// groups of 32 channels, or one
__host__ __device__ __forceinline__ int sets(int Cg) { return Cg <= 32 ? 32 / Cg : 1; }

// Sums over rows r0 .. r1 of a sample's chunk, each handed to put(k, channel, sum): MODE 0: Σd, Σd² (d = x − the group's
// first value); 1: Σgz, Σgz·x̂; 2: Σu, Σu·x̂, Σu·gz.  ch: the thread's channels (MODE 1, 2).
template <int MODE, int V, bool Q8, int NT, typename F>
__device__ __forceinline__ void sums_of(const GnP &p, const Chan<V> &ch, int n, int chunk, long long r0, long long r1, F put) {
    constexpr int K = MODE == 2 ? 3 : 2;
    __shared__ double red[K * V][NT];
    const int tid = threadIdx.x, lane = tid % p.lanes, ph = tid / p.lanes;
    const int c = chunk * p.step + lane * V, c1 = min(p.C, (chunk + 1) * p.step);
    double s[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) s[k][v] = 0.0;
    if (ph < p.rpi && c < c1) {
        double pivot[V];
        if constexpr (MODE == 0)
#pragma unroll
            for (int v = 0; v < V; ++v) pivot[v] = p.x[(long long)n * p.HW * p.C + (c + v) / p.Cg * p.Cg];
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
            const auto add = [&](int j) {
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
            };
            if (q + (UN - 1) * p.rpi < r1) {
#pragma unroll
                for (int j = 0; j < UN; ++j) add(j);
            } else {
#pragma unroll
                for (int j = 0; j < UN - 1; ++j)
                    if (q + j * p.rpi < r1) add(j);
            }
        }
    }
    // the rows of a workgroup, in a fixed order: those of a wave by lane exchanges where a row's lanes divide it, then the
    // waves' (or all rows') through LDS
    const bool fold = p.lanes < 64 && (p.lanes & (p.lanes - 1)) == 0;
    const int parts = fold ? NT / 64 : p.rpi, at = fold ? (tid >> 6) * p.lanes + lane : tid;
    if (fold)
        for (int d = p.lanes; d < 64; d <<= 1)
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int v = 0; v < V; ++v) s[k][v] += __shfl_xor(s[k][v], d);
    if (!fold || (tid & 63) < p.lanes)
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int v = 0; v < V; ++v) red[k * V + v][at] = s[k][v];
    __syncthreads();
    for (int i = tid; i < K * V * p.lanes; i += NT) {
        const int ln = i % p.lanes, kv = i / p.lanes, cc = chunk * p.step + ln * V + kv % V;
        if (cc >= c1) continue;
        double t = red[kv][ln];
#pragma unroll 4
        for (int q = 1; q < parts; ++q) t += red[kv][q * p.lanes + ln];
        put(kv / V, cc, t);
    }
}

// A group's share of channel c, from its sums s: MODE 0, 1: s0, s1 (times γ); 2: S1, S2, U, A, Q, Σ ga·s1, Σ ga·s2
template <int MODE>
__device__ __forceinline__ void shares(const GnP &p, int n, int c, const double *s, double *out) {
    const double ga = MODE && p.gamma ? (double)p.gamma[c] : 1.0;
    if constexpr (MODE < 2) {
        out[0] = ga * s[0];
        out[1] = ga * s[1];
    } else {
        const double s1 = p.sums[(long long)n * 2 * p.C + c], s2 = p.sums[((long long)n * 2 + 1) * p.C + c];
        const double a = p.gga ? (double)p.gga[c] : 0.0;
        out[0] = ga * s1;
        out[1] = ga * s2;
        out[2] = s[0];
        out[3] = s[1];
        out[4] = ga * s[2];
        out[5] = p.gga ? a * s1 : 0.0;
        out[6] = p.gga ? a * s2 : 0.0;
    }
}
// A group's results from the totals of its shares: MODE 0: μ, r; 1: S1/M, S2/M; 2: the seven coefficients of the double
// backward
template <int MODE>
__device__ __forceinline__ void results(const GnP &p, int n, int g, const double *t, double *out) {
    const double M = (double)p.HW * p.Cg, t0 = t[0] / M, t1 = t[1] / M;
    if constexpr (MODE == 0) {
        const double var0 = t1 - t0 * t0, var = var0 < 0.0 ? 0.0 : var0;  // (a NaN stays one)
        out[0] = p.x[(long long)n * p.HW * p.C + g * p.Cg] + t0;
        out[1] = 1.0 / sqrt(var + (double)p.eps);
    } else if constexpr (MODE == 1) {
        out[0] = t0;
        out[1] = t1;
    } else {
        const double r = p.stat[2 * ((long long)n * p.G + g) + 1], u = t[2] / M, a = t[3] / M;
        out[0] = u;
        out[1] = a;
        out[2] = t0;
        out[3] = t1;
        out[4] = -r * (t0 * a + u * t1) + t[5] / M;
        out[5] = -2.0 * r * t1 * a + t[6] / M;
        out[6] = (t[4] / M - t0 * u - t1 * a) * r * r;
    }
}
template <int MODE>
struct Sizes {
    static constexpr int K = MODE == 2 ? 3 : 2, J = MODE == 2 ? 7 : 2, O = MODE ? 8 : 2;  // sums, shares, results
};

// A workgroup per sample and set of whole groups (32 channels' worth, or one larger group): the splits' sums per channel
// (sums_out [n][K][C], or null), then each group's results (partial null: no upstream of gx).
template <int MODE>
__global__ __launch_bounds__(NTS) void gn_finish(GnP p, const double *partial, double *sums_out, double *out) {
    using S = Sizes<MODE>;
    constexpr int W = NTS / 64;
    __shared__ double part[W][S::K][32], chan[S::J][33], tot[S::J][32];
    const int tid = threadIdx.x, lane = tid & 31, sl = tid >> 5, n = blockIdx.y;
    const int gpb = sets(p.Cg), g0 = blockIdx.x * gpb, ng = min(gpb, p.G - g0), c1 = (g0 + ng) * p.Cg;
    if (tid < S::J * 32) tot[tid / 32][tid % 32] = 0.0;
    for (int c0 = g0 * p.Cg; c0 < c1; c0 += 32) {
        const int c = c0 + lane;
        double s[S::K] = {};
        if (c < c1 && partial)
#pragma unroll 4
            for (int sp = sl; sp < p.splits; sp += 2 * W)
#pragma unroll
                for (int k = 0; k < S::K; ++k) s[k] += partial[(((long long)n * p.splits + sp) * S::K + k) * p.C + c];
#pragma unroll
        for (int k = 0; k < S::K; ++k) {
            s[k] += __shfl_xor(s[k], 32);
            if (!(sl & 1)) part[sl >> 1][k][lane] = s[k];
        }
        __syncthreads();
        if (sl == 0 && c < c1) {
            double sh[S::J];
#pragma unroll
            for (int k = 0; k < S::K; ++k) {
                s[k] = part[0][k][lane];
#pragma unroll
                for (int q = 1; q < W; ++q) s[k] += part[q][k][lane];
                if (sums_out) sums_out[((long long)n * S::K + k) * p.C + c] = s[k];
            }
            shares<MODE>(p, n, c, s, sh);
#pragma unroll
            for (int j = 0; j < S::J; ++j) chan[j][lane] = sh[j];
        }
        __syncthreads();
        for (int i = tid; i < S::J * ng; i += NTS) {  // channels of a group, in order
            const int j = i / ng, g = i - j * ng, a = p.Cg <= 32 ? g * p.Cg : 0;
            const int b = p.Cg <= 32 ? a + p.Cg : min(32, c1 - c0);
            double t = tot[j][g];
            for (int k = a; k < b; ++k) t += chan[j][k];
            tot[j][g] = t;
        }
        __syncthreads();
    }
    if (tid >= ng) return;
    double t[S::J];
#pragma unroll
    for (int j = 0; j < S::J; ++j) t[j] = tot[j][tid];
    results<MODE>(p, n, g0 + tid, t, out + S::O * ((long long)n * p.G + g0 + tid));
}

// codes of V values of one row in a block whose lanes call together; up: their sides of the threshold, side: a value's
template <int V, typename F>
__device__ __forceinline__ void put_blocks(const GnP &p, const float *v, const bool *up, bool act, long long row, int c,
                                           int lane, int8_t *codes, uint8_t *exps, F side) {
    constexpr int L = act8::BLK / V;
    unsigned m = 0;
#pragma unroll
    for (int k = 0; k < V; ++k) m = max(m, act8::abs_bits(v[k]));
    const int e = act8::exp_of(act8::block_max<L>(m));
    if (c >= p.cp) return;  // (behind the last channel the code is 0)
    float code[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const float to = act8::code_of(v[k], e), at = ldexpf(to, e - 132);
        // (past the largest float there is no step to go)
        const float back = act8::keep(to + (at > v[k] ? -1.f : 1.f), e);
        code[k] = act & (side(at, k) != up[k]) ? back : to;
    }
    const uint32_t w = act8::word_of<V>(code, e);
    if constexpr (V == 4) *reinterpret_cast<uint32_t *>(codes + row * p.cp + c) = w;
    else codes[row * p.cp + c] = (int8_t)w;
    if (lane % L == 0) exps[row * p.nb + c / act8::BLK] = (uint8_t)e;
}

struct GnOut {
    float *o1, *o2;          // MODE 0: y; 1: gx; 2: g_x, g_gy
    float *g_gamma, *g_beta; // [C] or null
    int8_t *codes, *ycodes;  // MODE 0: x's and y's 8-bit blocks, or null
    uint8_t *exps, *yexps;
};

// dγ and dβ (MODE 1) or g_γ (MODE 2) of a channel: sums over the samples, in order
template <int MODE>
__device__ __forceinline__ void params_of(const GnP &p, int c, float *g_gamma, float *g_beta) {
    double s = 0.0, t = 0.0;
    for (int i = 0; i < p.N; ++i) {
        const double *q = p.sums + (long long)i * 2 * p.C + c;
        if constexpr (MODE == 1) {
            s += q[p.C];
            t += q[0];
        } else if (p.sums_u) {
            const long long g = (long long)i * p.G + c / p.Cg;
            s += p.stat[2 * g + 1] * (p.sums_u[((long long)i * 3 + 2) * p.C + c] - q[0] * p.grp[8 * g] -
                                      q[p.C] * p.grp[8 * g + 1]);
        }
    }
    if (g_gamma) g_gamma[c] = (float)s;
    if (MODE == 1 && g_beta) g_beta[c] = (float)t;
}

// The elementwise pass over rows r0 .. r1 of a sample's chunk; grp: the coefficients from group g0 on of the sample.
// BITS: MODE 1, 2: the input is in 8-bit blocks; MODE 0: blocks are written.
template <int MODE, int V, bool BITS>
__device__ __forceinline__ void apply_of(const GnP &p, const GnOut &o, const Chan<V> &ch, const double *grp, int g0, int n,
                                         int chunk, long long r0, long long r1) {
    constexpr int UA = MODE == 2 ? 2 : UN;
    constexpr bool Q8 = MODE && BITS;
    const int tid = threadIdx.x, lane = tid % p.lanes, ph = tid / p.lanes;
    const int c = chunk * p.step + lane * V;
    const bool act = c < min(p.C, (chunk + 1) * p.step);
    const int cl = act ? c : chunk * p.step;
    if (ph >= p.rpi) return;
    float k0[V], k1[V], k3[V], k4[V], k5[V], k6[V], ua[V], ub[V];
    if (act) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if constexpr (MODE >= 1) {
                const double *k = grp + 8 * ((c + v) / p.Cg - g0);
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
    for (long long q = r0 + ph; q < r1; q += UA * p.rpi) {
        Raw<V, Q8> raw[UA];
        float gy[UA][V], u[UA][V];
#pragma unroll
        for (int j = 0; j < UA; ++j) {  // (lanes behind the last channel load the chunk's first)
            const long long row = (long long)n * p.HW + min(q + j * p.rpi, r1 - 1);
            raw[j].load(p, row, cl);
            if constexpr (MODE >= 1) load_f<V>(p.gy, row * p.C + cl, gy[j]);
            if constexpr (MODE == 2) {
                if (p.u) load_f<V>(p.u, row * p.C + cl, u[j]);
                else
#pragma unroll
                    for (int v = 0; v < V; ++v) u[j][v] = 0.f;
            }
        }
        auto finish = [&](int j) {
            const long long row = (long long)n * p.HW + q + j * p.rpi;
            float a[V], d[V];
            bool up[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const double xd = xhat(raw[j].at(v), ch.r[v], ch.mu[v]), z = preact(xd, ch.ga[v], ch.be[v]);
                if constexpr (MODE == 0) {
                    up[v] = z > 0.0;
                    a[v] = (float)(z * (up[v] ? 1.0 : (double)p.slope));
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
            if (act) {
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
                    put_blocks<V>(p, t, up, act, row, c, lane, o.codes, o.exps, [&](float x, int v) {
                        return preact(xhat(x, ch.r[v], ch.mu[v]), ch.ga[v], ch.be[v]) > 0.0;
                    });
                if (o.ycodes) {
#pragma unroll
                    for (int v = 0; v < V; ++v) up[v] = a[v] > 0.f;
                    put_blocks<V>(p, a, up, act, row, c, lane, o.ycodes, o.yexps, [](float y, int) { return y > 0.f; });
                }
            }
        };
        // (all of the rows without a branch between them, so that they overlap; but for a workgroup's last ones)
        if (q + (UA - 1) * p.rpi < r1) {
#pragma unroll
            for (int j = 0; j < UA; ++j) finish(j);
        } else {
#pragma unroll
            for (int j = 0; j < UA - 1; ++j)
                if (q + j * p.rpi < r1) finish(j);
        }
    }
}

template <int MODE, int V, bool Q8>
__global__ __launch_bounds__(NT) void gn_sums(GnP p, double *partial) {
    constexpr int K = Sizes<MODE>::K;
    const int sp = blockIdx.x, n = blockIdx.y, chunk = blockIdx.z, c = chunk * p.step + (int)threadIdx.x % p.lanes * V;
    Chan<V> ch;
    if constexpr (MODE > 0)
        if (c < p.C) ch.load(p, p.stat + 2LL * n * p.G, 0, c);
    sums_of<MODE, V, Q8, NT>(p, ch, n, chunk, p.HW * sp / p.splits, p.HW * (sp + 1) / p.splits, [&](int k, int cc, double s) {
        partial[(((long long)n * p.splits + sp) * K + k) * p.C + cc] = s;
    });
}
// (the first row block of the first sample also makes the parameter gradients)
template <int MODE, int V, bool BITS>
__global__ __launch_bounds__(NT) void gn_apply(GnP p, GnOut o) {
    const int b = blockIdx.x, n = blockIdx.y, chunk = blockIdx.z, c = chunk * p.step + (int)threadIdx.x % p.lanes * V;
    if constexpr (MODE > 0)
        if (b == 0 && n == 0)
            for (int i = chunk * p.step + threadIdx.x; i < min(p.C, (chunk + 1) * p.step); i += NT)
                params_of<MODE>(p, i, o.g_gamma, o.g_beta);
    Chan<V> ch;
    if (c < p.C) ch.load(p, p.stat + 2LL * n * p.G, 0, c);
    apply_of<MODE, V, BITS>(p, o, ch, p.grp + 8LL * n * p.G, 0, n, chunk, p.HW * b / p.blocks, p.HW * (b + 1) / p.blocks);
}
// A whole pass of one sample's chunk, sums and coefficients in LDS (and in memory what a later launch reads).
template <int MODE, int V, bool BITS>
__global__ __launch_bounds__(NTS) void gn_small(GnP p, GnOut o, double *sums_out, double *out) {
    using S = Sizes<MODE>;
    __shared__ double s_sum[S::K][SMALL_C], s_out[SMALL_C][S::O];
    const int n = blockIdx.y, chunk = blockIdx.x, c0 = chunk * p.step, c1 = min(p.C, c0 + p.step), g0 = c0 / p.Cg;
    const int tid = threadIdx.x, c = c0 + tid % p.lanes * V;
    Chan<V> ch;
    if constexpr (MODE > 0)
        if (c < c1) ch.load(p, p.stat + 2LL * n * p.G, 0, c);
    if (MODE < 2 || p.u) {
        sums_of<MODE, V, MODE && BITS, NTS>(p, ch, n, chunk, 0, p.HW, [&](int k, int cc, double s) {
            s_sum[k][cc - c0] = s;
            if (sums_out) sums_out[((long long)n * S::K + k) * p.C + cc] = s;
        });
    } else {
        for (int i = tid; i < S::K * SMALL_C; i += NTS) s_sum[i / SMALL_C][i % SMALL_C] = 0.0;
    }
    __syncthreads();
    if (tid < (c1 - c0) / p.Cg) {
        const int g = g0 + tid;
        double t[S::J] = {}, sh[S::J], s[S::K], res[S::O] = {};
        for (int i = g * p.Cg; i < (g + 1) * p.Cg; ++i) {  // channels of a group, in order
#pragma unroll
            for (int k = 0; k < S::K; ++k) s[k] = s_sum[k][i - c0];
            shares<MODE>(p, n, i, s, sh);
#pragma unroll
            for (int j = 0; j < S::J; ++j) t[j] += sh[j];
        }
        results<MODE>(p, n, g, t, res);
#pragma unroll
        for (int j = 0; j < S::O; ++j) {
            s_out[tid][j] = res[j];
            out[S::O * ((long long)n * p.G + g) + j] = res[j];
        }
    }
    __syncthreads();
    if constexpr (MODE > 0)
        if (p.N == 1)  // its sums and coefficients are this workgroup's own
            for (int i = c0 + tid; i < c1; i += NTS) params_of<MODE>(p, i, o.g_gamma, o.g_beta);
    if constexpr (MODE == 0)
        if (c < c1) ch.load(p, &s_out[0][0], g0, c);
    apply_of<MODE, V, BITS>(p, o, ch, &s_out[0][0], g0, n, chunk, 0, p.HW);
}
template <int MODE>
__global__ void gn_params(GnP p, float *g_gamma, float *g_beta) {
    const int c = blockIdx.x * NT + threadIdx.x;
    if (c < p.C) params_of<MODE>(p, c, g_gamma, g_beta);
}

inline int launched() { return hipGetLastError() == hipSuccess ? ESR_OK : ESR_ELAUNCH; }

inline bool shape_ok(int64_t N, int64_t HW, int32_t C, int32_t G) {
    if (N <= 0 || HW <= 0 || C <= 0 || G <= 0 || C % G || C > (1 << 24)) return false;
    if (N > 65535 || (int64_t)N * G > 0x7fffffffLL) return false;
    return HW <= (1LL << 46) / C / N;  // element offsets, with room for the row arithmetic
}
inline bool bits_ok(const void *x, const void *codes, const void *exps) {
    return x ? !codes && !exps : codes && exps && (uintptr_t)codes % 16 == 0;  // exactly one form of the input
}
inline bool aligned(std::initializer_list<const void *> ptrs) {  // to 16 bytes
    for (const void *q : ptrs)
        if ((uintptr_t)q % 16) return false;
    return true;
}

// a grid's third dimension (C > 65535·256 without 16-byte accesses exceeds it; gn_small's chunks are its first)
inline bool grid_ok(const GnP &p) { return !p.blocks || p.chunks <= 65535; }

// the fewest channels of whole groups and, unless it is all of them, whole 8-bit blocks
int chunk_of(int32_t C, int32_t Cg) {
    int64_t s = Cg;
    while (s % act8::BLK) s += Cg;  // at most 32 times
    return s < C ? (int)s : C;
}

GnP params(int V, int64_t N, int64_t HW, int32_t C, int32_t G, const float *gamma, const float *beta, float slope) {
    GnP p{};
    p.gamma = gamma; p.beta = beta;
    p.N = (int)N; p.HW = HW; p.C = C; p.G = G; p.Cg = C / G; p.slope = slope;
    p.nb = (C + act8::BLK - 1) / act8::BLK;
    p.cp = act8::pitch(C);
    // One workgroup per sample and chunk where that is at most 64 K values: 46 K (3×40×36×64, chunks of 32 channels) take
    // 15 us forward, as long as three launches, and two launches' host time (7 us) is saved; 96 K (16×31×31×100 in one
    // chunk) take 29 us against 16 us in three.
    const int small = chunk_of(C, p.Cg), ln = (small + act8::BLK - 1) / act8::BLK * (act8::BLK / V);
    const bool one = small <= SMALL_C && HW <= (64 << 10) / small;
    const int threads = one ? NTS : NT, lanes = one ? ln : p.nb * (act8::BLK / V);
    p.lanes = lanes < threads ? lanes : threads;
    p.step = one ? small : p.lanes * V;
    p.chunks = (C + p.step - 1) / p.step;
    p.rpi = threads / p.lanes;
    if (one) {
        p.splits = 1;
        p.blocks = 0;
        return p;
    }
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

// The launches of a pass: sums_out gets the reduction's sums (null: not wanted), out the statistics (MODE 0) or the
// groups' coefficients.
template <int MODE, int V, bool BITS>
void pass(GnP p, const GnOut &o, double *partial, double *sums_out, double *out, hipStream_t st) {
    if constexpr (MODE == 0) p.stat = out;
    else p.grp = out;
    if constexpr (MODE == 1) p.sums = sums_out;
    if constexpr (MODE == 2) p.sums_u = p.u ? sums_out : nullptr;
    if (!p.blocks) {
        hipLaunchKernelGGL((gn_small<MODE, V, BITS>), dim3(p.chunks, p.N), dim3(NTS), 0, st, p, o, sums_out, out);
        if (MODE && p.N > 1 && (o.g_gamma || o.g_beta))
            hipLaunchKernelGGL(gn_params<MODE>, dim3((p.C + NT - 1) / NT), dim3(NT), 0, st, p, o.g_gamma, o.g_beta);
        return;
    }
    const bool reduce = MODE < 2 || p.u;
    const int gpb = sets(p.Cg);
    if (reduce)
        hipLaunchKernelGGL((gn_sums<MODE, V, MODE && BITS>), dim3(p.splits, p.N, p.chunks), dim3(NT), 0, st, p, partial);
    hipLaunchKernelGGL(gn_finish<MODE>, dim3((p.G + gpb - 1) / gpb, p.N), dim3(NTS), 0, st, p, reduce ? partial : nullptr,
                       sums_out, out);
    hipLaunchKernelGGL((gn_apply<MODE, V, BITS>), dim3(p.blocks, p.N, p.chunks), dim3(NT), 0, st, p, o);
}
template <int MODE>
void pass(const GnP &p, int V, bool bits, const GnOut &o, double *partial, double *sums_out, double *out, hipStream_t st) {
    if (V == 4 && bits) pass<MODE, 4, true>(p, o, partial, sums_out, out, st);
    else if (V == 4) pass<MODE, 4, false>(p, o, partial, sums_out, out, st);
    else if (bits) pass<MODE, 1, true>(p, o, partial, sums_out, out, st);
    else pass<MODE, 1, false>(p, o, partial, sums_out, out, st);
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
    if (!x || !y || !stat || !ws || !shape_ok(N, HW, C, G) || !(eps >= 0.f) || !codes != !exps || !ycodes != !yexps ||
        !aligned({codes, ycodes}))
        return ESR_EINVAL;
    const hipStream_t st = (hipStream_t)stream;
    const int V = C % 4 == 0 && aligned({x, y}) ? 4 : 1;
    GnP p = params(V, N, HW, C, G, gamma, beta, slope);
    if (!grid_ok(p)) return ESR_EINVAL;
    p.x = x; p.eps = eps;
    pass<0>(p, V, codes || ycodes, GnOut{y, nullptr, nullptr, nullptr, codes, ycodes, exps, yexps}, (double *)ws, nullptr,
            stat, st);
    return launched();
}

extern "C" int esr_gn_lrelu_bwd(const float *x, const int8_t *codes, const uint8_t *exps, const float *gy, int64_t N,
                                int64_t HW, int32_t C, int32_t G, const float *gamma, const float *beta,
                                const double *stat, float slope, float *gx, float *g_gamma, float *g_beta, double *sums_,
                                void *ws, esr_stream_t stream) {
    if (!bits_ok(x, codes, exps) || !gy || !gx || !stat || !sums_ || !ws || !shape_ok(N, HW, C, G)) return ESR_EINVAL;
    const hipStream_t st = (hipStream_t)stream;
    const int V = C % 4 == 0 && aligned({x, gy, gx}) ? 4 : 1;
    GnP p = params(V, N, HW, C, G, gamma, beta, slope);
    if (!grid_ok(p)) return ESR_EINVAL;
    p.x = x; p.codes = codes; p.exps = exps; p.gy = gy; p.stat = stat;
    double *partial = (double *)ws, *grp = partial + N * p.splits * 3 * C + N * 3 * C;
    pass<1>(p, V, !x, GnOut{gx, nullptr, g_gamma, g_beta, nullptr, nullptr, nullptr, nullptr}, partial, sums_, grp, st);
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
    const int V = C % 4 == 0 && aligned({x, gy, u, g_x, g_gy}) ? 4 : 1;
    GnP p = params(V, N, HW, C, G, gamma, beta, slope);
    if (!grid_ok(p)) return ESR_EINVAL;
    p.x = x; p.codes = codes; p.exps = exps; p.gy = gy; p.u = u; p.gga = gg_gamma; p.ggb = gg_beta; p.stat = stat;
    p.sums = sums_;
    double *partial = (double *)ws, *su = partial + N * p.splits * 3 * C, *grp = su + N * 3 * C;
    pass<2>(p, V, !x, GnOut{g_x, g_gy, g_gamma, nullptr, nullptr, nullptr, nullptr, nullptr}, partial, su, grp, st);
    return launched();
}
