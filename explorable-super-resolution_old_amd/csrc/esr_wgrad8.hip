// esr_wgrad8.hip — a convolution's weight gradient from an input kept in 8-bit blocks (esr_act8.h):
//   gw[co][ci][ky][kx] = Σ_{b, Y, X} x[b, s·Y + ky − p, s·X + kx − p, ci] · dy[b, Y, X, co]   (x zero outside the image)
// as one matrix product per tap (M = ci, N = co, K = pixels), the codes expanded while they are staged.  Split over the
// pixels into partials that a second launch adds in a fixed order into torch's weight layout.
#include "esr_act8.h"
#include "esr_amd.h"
#include "esr_knobs.h"

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
constexpr int NT = 256, KP = 64, PS = 68;

struct WgP {
    const int8_t *codes;
    const uint8_t *exps;
    const float *dy;
    int B, Hs, Ws, cin, MH, MW, cout, k, s, p, nci, nco;
    long long per_split;
    float *partial;  // [splits][taps][nci·64][nco·64]
};

__global__ __launch_bounds__(NT, 2) void wgrad8_kernel(WgP p) {
    __shared__ float s_a[KP * PS], s_b[KP * PS];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hl = lane >> 5, ml = lane & 31;
    const int cob = blockIdx.x % p.nco, cib = blockIdx.x / p.nco % p.nci, t = blockIdx.x / (p.nco * p.nci);
    const int ky = t / p.k, kx = t % p.k, nb = (p.cin + 31) / 32;
    const int per_img = p.MH * p.MW;
    const long long P = (long long)p.B * per_img, k0 = blockIdx.y * p.per_split, k1 = min(P, k0 + p.per_split);
    const int c = tid & 63, ci = cib * 64 + c, co = cob * 64 + c;
    const int mt = wave >> 1, nt = wave & 1;
    f32x16 acc = {};
    for (long long kb = k0; kb < k1; kb += KP) {
        __syncthreads();
        for (int q = wave; q < KP; q += NT / 64) {
            const long long m = kb + q;
            float a = 0.f, b = 0.f;
            if (m < k1) {
                const int img = (int)(m / per_img), r = (int)(m - (long long)img * per_img);
                const int Y = r / p.MW, X = r - Y * p.MW, sy = p.s * Y + ky - p.p, sx = p.s * X + kx - p.p;
                if (ci < p.cin && sy >= 0 && sy < p.Hs && sx >= 0 && sx < p.Ws) {
                    const long long row = ((long long)img * p.Hs + sy) * p.Ws + sx;
                    a = act8::value_of((float)p.codes[row * p.cin + ci], p.exps[row * nb + ci / 32]);
                }
                if (co < p.cout) b = p.dy[m * p.cout + co];
            }
            s_a[q * PS + c] = a;
            s_b[q * PS + c] = b;
        }
        __syncthreads();
        for (int q = 0; q < KP / 2; ++q)
            acc = __builtin_amdgcn_mfma_f32_32x32x2f32(s_a[(2 * q + hl) * PS + 32 * mt + ml],
                                                       s_b[(2 * q + hl) * PS + 32 * nt + ml], acc, 0, 0, 0);
    }
    float *dst = p.partial + (((long long)blockIdx.y * p.k * p.k + t) * p.nci * 64 + cib * 64) * p.nco * 64 + cob * 64;
#pragma unroll
    for (int r = 0; r < 16; ++r)
        dst[(long long)(32 * mt + (r & 3) + 8 * (r >> 2) + 4 * hl) * p.nco * 64 + 32 * nt + ml] = acc[r];
}

// gw[co][ci][t] = Σ over splits, in order
__global__ void wgrad8_reduce(const float *partial, int splits, int T, int cin, int cout, int cip, int cop, float *gw) {
    const long long i = (long long)blockIdx.x * NT + threadIdx.x, n = (long long)T * cin * cout;
    if (i >= n) return;
    const int co = (int)(i % cout), ci = (int)(i / cout % cin), t = (int)(i / ((long long)cout * cin));
    float v = 0.f;
    for (int s = 0; s < splits; ++s) v += partial[(((long long)s * T + t) * cip + ci) * cop + co];
    gw[((long long)co * cin + ci) * T + t] = v;
}

struct Geo {
    int nci, nco, T, splits;
    long long P, per_split;
};
bool geometry(int64_t B, int32_t Hs, int32_t Ws, int32_t cin, int32_t MH, int32_t MW, int32_t cout, int32_t k,
              int32_t s, int32_t pad, Geo &g) {
    if (B <= 0 || Hs <= 0 || Ws <= 0 || cin <= 0 || MH <= 0 || MW <= 0 || cout <= 0 || k <= 0 || s <= 0 || pad < 0)
        return false;
    if (k > 8 || Hs > 65535 || Ws > 65535 || pad > 65535 || s > 65535 || cin > 65536 || cout > 65536) return false;
    if (MH != (Hs + 2 * pad - k) / s + 1 || MW != (Ws + 2 * pad - k) / s + 1 || Hs + 2 * pad < k || Ws + 2 * pad < k)
        return false;
    if (B > 0x7fffffffLL / ((int64_t)MH * MW) || B > 0x7fffffffLL / ((int64_t)Hs * Ws)) return false;
    g.nci = (cin + 63) / 64;
    g.nco = (cout + 63) / 64;
    g.T = k * k;
    g.P = B * MH * MW;
    const long long tiles = (long long)g.nci * g.nco * g.T;
    long long n = (1024 + tiles - 1) / tiles, most = (g.P + 4 * KP - 1) / (4 * KP);
    n = n < most ? n : most;
    g.per_split = ((g.P + n - 1) / n + KP - 1) / KP * KP;
    g.splits = (int)((g.P + g.per_split - 1) / g.per_split);
    return tiles <= 0x7fffffffLL;
}

}  // namespace

extern "C" int64_t esr_dconv_wgrad_act8_workspace_bytes(int64_t B, int32_t Hs, int32_t Ws, int32_t cin, int32_t MH,
                                                        int32_t MW, int32_t cout, int32_t k, int32_t s, int32_t pad) {
    Geo g;
    if (!geometry(B, Hs, Ws, cin, MH, MW, cout, k, s, pad, g)) return ESR_EINVAL;
    return 4LL * g.splits * g.T * g.nci * 64 * g.nco * 64;
}

extern "C" int esr_dconv_wgrad_act8(const int8_t *codes, const uint8_t *exps, int64_t B, int32_t Hs, int32_t Ws,
                                    int32_t cin, const float *dy, int32_t MH, int32_t MW, int32_t cout, int32_t k,
                                    int32_t s, int32_t pad, float *gw, void *ws, esr_stream_t stream) {
    Geo g;
    if (!codes || !exps || !dy || !gw || !ws || !geometry(B, Hs, Ws, cin, MH, MW, cout, k, s, pad, g)) return ESR_EINVAL;
    const hipStream_t st = (hipStream_t)stream;
    WgP p{codes, exps, dy, (int)B, Hs, Ws, cin, MH, MW, cout, k, s, pad, g.nci, g.nco, g.per_split, (float *)ws};
    hipLaunchKernelGGL(wgrad8_kernel, dim3(g.nci * g.nco * g.T, g.splits), dim3(NT), 0, st, p);
    const long long n = (long long)g.T * cin * cout;
    hipLaunchKernelGGL(wgrad8_reduce, dim3((unsigned)((n + NT - 1) / NT)), dim3(NT), 0, st, p.partial, g.splits, g.T,
                       cin, cout, g.nci * 64, g.nco * 64, gw);
    return hipGetLastError() == hipSuccess ? ESR_OK : ESR_ELAUNCH;
}
