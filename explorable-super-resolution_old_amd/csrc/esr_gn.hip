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

namespace {

constexpr int NT = 256;
constexpr int MAXS = 64;  // row splits of a sample in a reduction

struct GnP {
    const float *x;              // [N][HW][C], or null: codes / exps
    const int8_t *codes;
    const uint8_t *exps;
    const float *gy, *u;         // [N][HW][C]
    const float *gamma, *beta;   // [C] or null (1, 0)
    const float *gga, *ggb;      // [C] upstream of dγ, dβ, or null
    const double *stat;          // [N][G][2]: μ and r
    const double *grp;           // [N][G][8] per-group coefficients of the pass
    long long HW;
    int N, C, G, Cg, splits;
    float slope, eps;
};

__device__ __forceinline__ float load_x(const GnP &p, long long row, int c) {
    if (p.x) return p.x[row * p.C + c];
    const int nb = (p.C + act8::BLK - 1) / act8::BLK;
    return act8::value_of((float)p.codes[row * p.C + c], p.exps[row * nb + c / act8::BLK]);
}
// x̂ and z of one value, by the same operations everywhere.  (x − μ)·r rather than x·r − μ·r: the values of a constant
// group are their mean exactly, and their z is β.
__device__ __forceinline__ double xhat(double x, double r, double mu) { return (x - mu) * r; }
__device__ __forceinline__ double preact(double xh, double gamma, double beta) { return fma(gamma, xh, beta); }

// per-(sample, split, channel) sums: MODE 0: Σd, Σd² (d = x − the group's first value); 1: Σgz, Σgz·x̂; 2: Σu, Σu·x̂, Σu·gz
template <int MODE>
__global__ __launch_bounds__(NT) void gn_colsum(GnP p, double *partial) {
    constexpr int K = MODE == 2 ? 3 : 2;
    const int n = blockIdx.y, sp = blockIdx.x;
    const long long r0 = p.HW * sp / p.splits, r1 = p.HW * (sp + 1) / p.splits;
    __shared__ double red[K][NT];
    const int rpi = p.C <= NT ? NT / p.C : 1;
    for (int cb = 0; cb < p.C; cb += NT) {
        const int c = p.C <= NT ? (int)threadIdx.x % p.C : cb + (int)threadIdx.x;
        const int ph = p.C <= NT ? (int)threadIdx.x / p.C : 0;
        const bool act = c < p.C && ph < rpi;
        double s[K] = {};
        if (act) {
            const int g = c / p.Cg;
            const double pivot = MODE == 0 ? (double)p.x[(long long)n * p.HW * p.C + g * p.Cg] : 0.0;
            const double mu = MODE ? p.stat[((long long)n * p.G + g) * 2] : 0.0;
            const double r = MODE ? p.stat[((long long)n * p.G + g) * 2 + 1] : 0.0;
            const double ga = p.gamma ? p.gamma[c] : 1.0, be = p.beta ? p.beta[c] : 0.0;
            for (long long q = r0 + ph; q < r1; q += rpi) {
                const long long row = (long long)n * p.HW + q, i = row * p.C + c;
                const float x = load_x(p, row, c);
                if (MODE == 0) {
                    const double d = (double)x - pivot;
                    s[0] += d;
                    s[1] = fma(d, d, s[1]);
                } else {
                    const double xh = xhat(x, r, mu);
                    const double gz = (double)(p.gy[i] * (preact(xh, ga, be) > 0.0 ? 1.f : p.slope));
                    if (MODE == 1) {
                        s[0] += gz;
                        s[1] = fma(gz, xh, s[1]);
                    } else {
                        const double u = p.u[i];
                        s[0] += u;
                        s[1] = fma(u, xh, s[1]);
                        s[2] = fma(u, gz, s[2]);
                    }
                }
            }
        }
        for (int k = 0; k < K; ++k) red[k][threadIdx.x] = s[k];
        __syncthreads();
        if (ph == 0 && c < p.C)
            for (int k = 0; k < K; ++k) {
                double v = red[k][threadIdx.x];
                for (int q = 1; q < rpi; ++q) v += red[k][q * p.C + threadIdx.x];
                partial[(((long long)n * p.splits + sp) * K + k) * p.C + c] = v;
            }
        __syncthreads();
        if (p.C <= NT) break;
    }
}

// sums[n][k][c] = Σ over splits, in order
__global__ void gn_splits(const double *partial, int splits, int KC, double *sums) {
    const int n = blockIdx.y, i = blockIdx.x * NT + threadIdx.x;
    if (i >= KC) return;
    double v = 0.0;
    for (int s = 0; s < splits; ++s) v += partial[((long long)n * splits + s) * KC + i];
    sums[(long long)n * KC + i] = v;
}

// MODE 0: stat (μ, r) of each group; 1: grp = S1/M, S2/M; 2: the seven coefficients of the double backward
template <int MODE>
__global__ void gn_groups(GnP p, const double *sums, const double *sums_u, double *out) {
    const int i = blockIdx.x * NT + threadIdx.x;
    if (i >= p.N * p.G) return;
    const int n = i / p.G, g = i - n * p.G;
    const double M = (double)p.HW * p.Cg;
    const double *s = sums + (long long)n * 2 * p.C;
    double t0 = 0, t1 = 0, b0 = 0, b1 = 0, U = 0, A = 0, Q = 0;
    for (int c = g * p.Cg; c < (g + 1) * p.Cg; ++c) {
        const double ga = MODE && p.gamma ? p.gamma[c] : 1.0;
        t0 += ga * s[c];
        t1 += ga * s[p.C + c];
        if (MODE == 2) {
            if (p.gga) {
                b0 += (double)p.gga[c] * s[c];
                b1 += (double)p.gga[c] * s[p.C + c];
            }
            if (sums_u) {
                const double *v = sums_u + (long long)n * 3 * p.C;
                U += v[c];
                A += v[p.C + c];
                Q += ga * v[2 * p.C + c];
            }
        }
    }
    if (MODE == 0) {
        const double pivot = p.x[(long long)n * p.HW * p.C + g * p.Cg];
        const double d = t0 / M, var0 = t1 / M - d * d, var = var0 < 0.0 ? 0.0 : var0;  // (a NaN stays one)
        const double r = 1.0 / sqrt(var + (double)p.eps);
        out[2 * i] = pivot + d;
        out[2 * i + 1] = r;
    } else if (MODE == 1) {
        out[8 * i] = t0 / M;
        out[8 * i + 1] = t1 / M;
    } else {
        const double r = p.stat[2 * i + 1], m1 = t0 / M, m2 = t1 / M, u = U / M, a = A / M;
        out[8 * i] = u;
        out[8 * i + 1] = a;
        out[8 * i + 2] = m1;
        out[8 * i + 3] = m2;
        out[8 * i + 4] = -r * (m1 * a + u * m2) + b0 / M;
        out[8 * i + 5] = -2.0 * r * m2 * a + b1 / M;
        out[8 * i + 6] = (Q / M - m1 * u - m2 * a) * r * r;
    }
}

// dβ, dγ from s1, s2 (MODE 1), or g_γ (MODE 2): sums over the samples, in order
template <int MODE>
__global__ void gn_params(GnP p, const double *sums, const double *sums_u, float *o1, float *o2) {
    const int c = blockIdx.x * NT + threadIdx.x;
    if (c >= p.C) return;
    double a = 0.0, b = 0.0;
    for (int n = 0; n < p.N; ++n) {
        const double *s = sums + (long long)n * 2 * p.C;
        if (MODE == 1) {
            a += s[p.C + c];
            b += s[c];
        } else if (sums_u) {
            const long long i = (long long)n * p.G + c / p.Cg;
            a += p.stat[2 * i + 1] * (sums_u[((long long)n * 3 + 2) * p.C + c] - s[c] * p.grp[8 * i] -
                                      s[p.C + c] * p.grp[8 * i + 1]);
        }
    }
    if (o1) o1[c] = (float)a;
    if (MODE == 1 && o2) o2[c] = (float)b;
}

// MODE 0: y (and x's 8-bit blocks); 1: gx; 2: g_x (o1) and g_gy (o2).  A thread per value, lanes of a 32-channel block
// together (the last block of a row padded to 32 lanes).
template <int MODE>
__global__ __launch_bounds__(NT) void gn_apply(GnP p, float *o1, float *o2, int8_t *codes, uint8_t *exps) {
    const int nb = (p.C + act8::BLK - 1) / act8::BLK, rl = nb * act8::BLK;
    const long long q = (long long)blockIdx.x * NT + threadIdx.x, row = q / rl;
    const int c = (int)(q - row * rl);
    const bool act = row < p.N * p.HW && c < p.C;
    float x = 0.f;
    double r = 0, mu = 0, ga = 1, be = 0, xd = 0, z = 0;
    long long gi = 0;
    if (act) {
        x = load_x(p, row, c);
        gi = row / p.HW * p.G + c / p.Cg;
        mu = p.stat[2 * gi];
        r = p.stat[2 * gi + 1];
        if (p.gamma) ga = p.gamma[c];
        if (p.beta) be = p.beta[c];
        xd = xhat(x, r, mu);
        z = preact(xd, ga, be);
    }
    const long long i = row * p.C + c;
    if (MODE == 0) {
        if (act) o1[i] = (float)(z > 0.0 ? z : (double)p.slope * z);
        if (!codes) return;
        const int e = act8::exp_of(act8::block_max<32>(act8::abs_bits(x)));
        if (!act) return;
        float code = act8::code_of(x, e);
        if (e != 255) {
            const float v = act8::value_of(code, e);
            if ((preact(xhat(v, r, mu), ga, be) > 0.0) != (z > 0.0)) code += v > x ? -1.f : 1.f;
        }
        codes[i] = (int8_t)(int)code;
        if (c % act8::BLK == 0) exps[row * nb + c / act8::BLK] = (uint8_t)e;
        return;
    }
    if (!act) return;
    const float m = z > 0.0 ? 1.f : p.slope, xh = (float)xd, rf = (float)r, gf = (float)ga;
    const double *k = p.grp + 8 * gi;
    const float gz = p.gy[i] * m, h = gf * gz;
    if (MODE == 1) {
        o1[i] = rf * (h - (float)k[0] - xh * (float)k[1]);
        return;
    }
    const float u = p.u ? p.u[i] : 0.f, ua = p.gga ? p.gga[c] : 0.f, ub = p.ggb ? p.ggb[c] : 0.f;
    o2[i] = m * (gf * rf * (u - (float)k[0] - xh * (float)k[1]) + ua * xh + ub);
    const float gg = -rf * (h * (float)k[1] + u * (float)k[3]) + ua * gz;
    o1[i] = rf * (gg - (float)k[4] - xh * (float)k[5]) - (float)k[6] * xh;
}

inline int launched() { return hipGetLastError() == hipSuccess ? ESR_OK : ESR_ELAUNCH; }
inline unsigned blocks_of(long long n) { return (unsigned)((n + NT - 1) / NT); }

inline bool shape_ok(int64_t N, int64_t HW, int32_t C, int32_t G) {
    if (N <= 0 || HW <= 0 || C <= 0 || G <= 0 || C % G) return false;
    if (N > 65535 || (int64_t)N * G > 0x7fffffffLL) return false;
    const int64_t rl = (C + 31) / 32 * 32;
    return HW <= 0x7fffffffLL * NT / rl / N;  // the elementwise grid
}
inline int splits_of(int64_t N, int64_t HW) {
    const int64_t s = HW / 64;
    return (int)(s < 1 ? 1 : (s > MAXS ? MAXS : s));
}
inline bool bits_ok(const void *x, const void *codes, const void *exps) {
    return x ? !codes && !exps : codes && exps;  // exactly one form of the input
}

template <int MODE>
void colsum(const GnP &p, double *partial, double *sums, hipStream_t st) {
    constexpr int K = MODE == 2 ? 3 : 2;
    hipLaunchKernelGGL(gn_colsum<MODE>, dim3(p.splits, p.N), dim3(NT), 0, st, p, partial);
    hipLaunchKernelGGL(gn_splits, dim3(blocks_of((long long)K * p.C), p.N), dim3(NT), 0, st, partial, p.splits, K * p.C,
                       sums);
}

GnP params(const float *x, const int8_t *codes, const uint8_t *exps, int64_t N, int64_t HW, int32_t C, int32_t G,
           const float *gamma, const float *beta, float slope) {
    GnP p{};
    p.x = x; p.codes = codes; p.exps = exps; p.gamma = gamma; p.beta = beta;
    p.N = (int)N; p.HW = HW; p.C = C; p.G = G; p.Cg = C / G; p.slope = slope;
    p.splits = splits_of(N, HW);
    return p;
}

}  // namespace

extern "C" int64_t esr_gn_workspace_bytes(int64_t N, int64_t HW, int32_t C, int32_t G) {
    if (!shape_ok(N, HW, C, G)) return ESR_EINVAL;
    // split sums [N][splits][3][C], sums of u [N][3][C], group coefficients [N][G][8]
    return 8 * (N * splits_of(N, HW) * 3 * C + N * 3 * C + N * G * 8);
}

extern "C" int esr_gn_lrelu_fwd(const float *x, int64_t N, int64_t HW, int32_t C, int32_t G, const float *gamma,
                                const float *beta, float eps, float slope, float *y, double *stat, int8_t *codes,
                                uint8_t *exps, void *ws, esr_stream_t stream) {
    if (!x || !y || !stat || !ws || !shape_ok(N, HW, C, G) || !(eps >= 0.f) || !codes != !exps) return ESR_EINVAL;
    const hipStream_t st = (hipStream_t)stream;
    GnP p = params(x, nullptr, nullptr, N, HW, C, G, gamma, beta, slope);
    p.eps = eps;
    double *partial = (double *)ws, *sums = partial + N * p.splits * 3 * C;
    colsum<0>(p, partial, sums, st);
    hipLaunchKernelGGL(gn_groups<0>, dim3(blocks_of(N * G)), dim3(NT), 0, st, p, sums, nullptr, stat);
    p.stat = stat;
    hipLaunchKernelGGL(gn_apply<0>, dim3(blocks_of(N * HW * ((C + 31) / 32 * 32))), dim3(NT), 0, st, p, y, nullptr,
                       codes, exps);
    return launched();
}

extern "C" int esr_gn_lrelu_bwd(const float *x, const int8_t *codes, const uint8_t *exps, const float *gy, int64_t N,
                                int64_t HW, int32_t C, int32_t G, const float *gamma, const float *beta,
                                const double *stat, float slope, float *gx, float *g_gamma, float *g_beta, double *sums,
                                void *ws, esr_stream_t stream) {
    if (!bits_ok(x, codes, exps) || !gy || !stat || !sums || !ws || !shape_ok(N, HW, C, G)) return ESR_EINVAL;
    const hipStream_t st = (hipStream_t)stream;
    GnP p = params(x, codes, exps, N, HW, C, G, gamma, beta, slope);
    p.gy = gy; p.stat = stat;
    double *partial = (double *)ws, *grp = partial + N * p.splits * 3 * C + N * 3 * C;
    colsum<1>(p, partial, sums, st);
    if (g_gamma || g_beta)
        hipLaunchKernelGGL(gn_params<1>, dim3(blocks_of(C)), dim3(NT), 0, st, p, sums, nullptr, g_gamma, g_beta);
    if (gx) {
        hipLaunchKernelGGL(gn_groups<1>, dim3(blocks_of(N * G)), dim3(NT), 0, st, p, sums, nullptr, grp);
        p.grp = grp;
        hipLaunchKernelGGL(gn_apply<1>, dim3(blocks_of(N * HW * ((C + 31) / 32 * 32))), dim3(NT), 0, st, p, gx, nullptr,
                           nullptr, nullptr);
    }
    return launched();
}

extern "C" int esr_gn_lrelu_bwd2(const float *x, const int8_t *codes, const uint8_t *exps, const float *gy,
                                 const float *u, const float *gg_gamma, const float *gg_beta, int64_t N, int64_t HW,
                                 int32_t C, int32_t G, const float *gamma, const float *beta, const double *stat,
                                 float slope, const double *sums, float *g_x, float *g_gy, float *g_gamma, void *ws,
                                 esr_stream_t stream) {
    if (!bits_ok(x, codes, exps) || !gy || !stat || !sums || !g_x || !g_gy || !ws || !shape_ok(N, HW, C, G))
        return ESR_EINVAL;
    const hipStream_t st = (hipStream_t)stream;
    GnP p = params(x, codes, exps, N, HW, C, G, gamma, beta, slope);
    p.gy = gy; p.u = u; p.gga = gg_gamma; p.ggb = gg_beta; p.stat = stat;
    double *partial = (double *)ws, *su = partial + N * p.splits * 3 * C, *grp = su + N * 3 * C;
    if (u) colsum<2>(p, partial, su, st);
    else su = nullptr;
    hipLaunchKernelGGL(gn_groups<2>, dim3(blocks_of(N * G)), dim3(NT), 0, st, p, sums, su, grp);
    p.grp = grp;
    hipLaunchKernelGGL(gn_apply<2>, dim3(blocks_of(N * HW * ((C + 31) / 32 * 32))), dim3(NT), 0, st, p, g_x, g_gy,
                       nullptr, nullptr);
    if (g_gamma) hipLaunchKernelGGL(gn_params<2>, dim3(blocks_of(C)), dim3(NT), 0, st, p, sums, su, g_gamma, nullptr);
    return launched();
}
