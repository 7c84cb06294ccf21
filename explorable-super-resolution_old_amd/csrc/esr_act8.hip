// esr_act8.hip — activations kept in 8 bits between the forward and the backward pass (esr_act8.h: the format).
//
// pack reads 4 B and writes 1 + 1/32 B per value, unpack the reverse: both are bound by HBM.  A thread holds V = 4
// channels (one 16-byte access; V = 1 where C or the base is not a multiple of 4 values), the 32/V lanes of a block take
// its maximum by lane exchanges.  The code keeps x > 0: a positive value that rounds to code 0 takes code 1, so that a
// LeakyReLU mask read from the block is the mask of the values.
#include "esr_act8.h"
#include "esr_amd.h"
#include "esr_knobs.h"

namespace {

constexpr int NT = 256;

// flat index over [P][blocks per row][32 / V]
template <int V>
__global__ __launch_bounds__(NT) void act8_pack_kernel(const float *x, long long P, int C, int8_t *codes, uint8_t *exps) {
    constexpr int L = act8::BLK / V;
    const int nb = (C + act8::BLK - 1) / act8::BLK, rl = nb * L;
    const long long i = (long long)blockIdx.x * NT + threadIdx.x;
    const long long p = i / rl;
    const int q = (int)(i - p * rl), c = q * V;
    const bool act = p < P && c < C;
    float v[V];
    unsigned m = 0;
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = 0.f;
    if (act) {
        if constexpr (V == 4) {
            const float4 t = *reinterpret_cast<const float4 *>(x + p * C + c);
            v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
        } else {
            v[0] = x[p * C + c];
        }
    }
#pragma unroll
    for (int k = 0; k < V; ++k) m = max(m, act8::abs_bits(v[k]));
    const int e = act8::exp_of(act8::block_max<L>(m));
    if (!act) return;
    uint32_t w = 0;
#pragma unroll
    for (int k = 0; k < V; ++k) {
        float code = act8::code_of(v[k], e);
        if (e != 255 && code == 0.f && v[k] > 0.f) code = 1.f;
        w |= (uint32_t)(uint8_t)(int8_t)(int)code << (8 * k);
    }
    if constexpr (V == 4) *reinterpret_cast<uint32_t *>(codes + p * C + c) = w;
    else codes[p * C + c] = (int8_t)w;
    if (q % L == 0) exps[p * nb + q / L] = (uint8_t)e;
}

template <int V>
__global__ __launch_bounds__(NT) void act8_unpack_kernel(const int8_t *codes, const uint8_t *exps, long long P, int C,
                                                         float *x) {
    const int nb = (C + act8::BLK - 1) / act8::BLK, cq = C / V;
    const long long i = (long long)blockIdx.x * NT + threadIdx.x;
    if (i >= P * cq) return;
    const long long p = i / cq;
    const int c = (int)(i - p * cq) * V;
    const int e = exps[p * nb + c / act8::BLK];
    if constexpr (V == 4) {
        const uint32_t w = *reinterpret_cast<const uint32_t *>(codes + p * C + c);
        float4 t;
        t.x = act8::value_of(act8::code_at(w, 0), e);
        t.y = act8::value_of(act8::code_at(w, 1), e);
        t.z = act8::value_of(act8::code_at(w, 2), e);
        t.w = act8::value_of(act8::code_at(w, 3), e);
        *reinterpret_cast<float4 *>(x + p * C + c) = t;
    } else {
        x[p * C + c] = act8::value_of((float)codes[p * C + c], e);
    }
}

inline bool quads(const void *f32, const void *codes, int C) {
    return C % 4 == 0 && (uintptr_t)f32 % 16 == 0 && (uintptr_t)codes % 4 == 0;
}

}  // namespace

extern "C" int esr_act8_pack(const float *x, int64_t P, int32_t C, int8_t *codes, uint8_t *exps, esr_stream_t stream) {
    if (!x || !codes || !exps || P <= 0 || C <= 0) return ESR_EINVAL;
    const int nb = (C + act8::BLK - 1) / act8::BLK;
    const bool v4 = quads(x, codes, C);
    const long long n = (P * nb * (v4 ? 8 : 32) + NT - 1) / NT;
    if (n > 0x7fffffffLL) return ESR_EINVAL;
    const hipStream_t st = (hipStream_t)stream;
    if (v4) hipLaunchKernelGGL(act8_pack_kernel<4>, dim3((unsigned)n), dim3(NT), 0, st, x, P, C, codes, exps);
    else hipLaunchKernelGGL(act8_pack_kernel<1>, dim3((unsigned)n), dim3(NT), 0, st, x, P, C, codes, exps);
    return hipGetLastError() == hipSuccess ? ESR_OK : ESR_ELAUNCH;
}

extern "C" int esr_act8_unpack(const int8_t *codes, const uint8_t *exps, int64_t P, int32_t C, float *x,
                               esr_stream_t stream) {
    if (!x || !codes || !exps || P <= 0 || C <= 0) return ESR_EINVAL;
    const bool v4 = quads(x, codes, C);
    const long long n = (P * (v4 ? C / 4 : C) + NT - 1) / NT;
    if (n > 0x7fffffffLL) return ESR_EINVAL;
    const hipStream_t st = (hipStream_t)stream;
    if (v4) hipLaunchKernelGGL(act8_unpack_kernel<4>, dim3((unsigned)n), dim3(NT), 0, st, codes, exps, P, C, x);
    else hipLaunchKernelGGL(act8_unpack_kernel<1>, dim3((unsigned)n), dim3(NT), 0, st, codes, exps, P, C, x);
    return hipGetLastError() == hipSuccess ? ESR_OK : ESR_ELAUNCH;
}
