// esr_act8.hip — activations kept in 8 bits between the forward and the backward pass (esr_act8.h: the format).
//
// pack reads 4 B and writes 1 + 1/32 B per value, unpack the reverse: both are bound by HBM (16×304×304 × 64 channels: 75
// and 67 us, 6.5 and 7.2 TB/s).  A thread holds V = 4
// channels (one 16-byte access; V = 1 where C or a base is not a multiple of 4 values) of UN rows at a time, the 32/V
// lanes of a block take its maximum by lane exchanges.  Where C is a multiple of 32 the tensor is a flat run of blocks;
// else a row's last block is padded to its lanes.  The fp32 side is non-temporal: it is read or written once, and leaves
// the last-level cache to the codes.  The code keeps x > 0: a positive value that rounds to code 0 takes code 1, so that
// a LeakyReLU mask read from the block is the mask of the values.
#include "esr_act8.h"
#include "esr_amd.h"
#include "esr_knobs.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
constexpr int NT = 256, UN = 4;

struct Rows {
    long long P;
    int C, nb, cp, lanes, rpi;  // cp: codes of a row; lanes: its threads (of this chunk); rpi: rows at a time
};

template <int V>
__device__ __forceinline__ uint32_t codes_of(const float *v, int &e) {
    unsigned m = 0;
#pragma unroll
    for (int k = 0; k < V; ++k) m = max(m, act8::abs_bits(v[k]));
    e = act8::exp_of(act8::block_max<act8::BLK / V>(m));
    float code[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        code[k] = act8::code_of(v[k], e);
        code[k] = v[k] > 0.f ? fmaxf(code[k], 1.f) : code[k];
    }
    return act8::word_of<V>(code, e);
}

template <int V>
__global__ __launch_bounds__(NT) void act8_pack_kernel(const float *x, Rows r, int8_t *codes, uint8_t *exps) {
    constexpr int L = act8::BLK / V;
    const int lane = threadIdx.x % r.lanes, ph = threadIdx.x / r.lanes, c = ((int)blockIdx.y * NT + lane) * V;
    const bool in = c < r.C;  // (behind the last channel the code is 0)
    const long long p0 = (long long)blockIdx.x * r.rpi * UN + ph;
    if (ph >= r.rpi) return;
    float v[UN][V];
#pragma unroll
    for (int j = 0; j < UN; ++j) {
        const long long p = p0 + (long long)j * r.rpi;
#pragma unroll
        for (int k = 0; k < V; ++k) v[j][k] = 0.f;
        if (in && p < r.P) {
            if constexpr (V == 4) {
                const f32x4 t = __builtin_nontemporal_load(reinterpret_cast<const f32x4 *>(x + p * r.C + c));
                v[j][0] = t[0]; v[j][1] = t[1]; v[j][2] = t[2]; v[j][3] = t[3];
            } else {
                v[j][0] = __builtin_nontemporal_load(x + p * r.C + c);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < UN; ++j) {
        const long long p = p0 + (long long)j * r.rpi;
        int e;
        const uint32_t w = codes_of<V>(v[j], e);
        if (c >= r.cp || p >= r.P) continue;
        if constexpr (V == 4) *reinterpret_cast<uint32_t *>(codes + p * r.cp + c) = w;
        else codes[p * r.cp + c] = (int8_t)w;
        if (lane % L == 0) exps[p * r.nb + c / act8::BLK] = (uint8_t)e;
    }
}

template <int V>
__global__ __launch_bounds__(NT) void act8_unpack_kernel(const int8_t *codes, const uint8_t *exps, Rows r, float *x) {
    const int lane = threadIdx.x % r.lanes, ph = threadIdx.x / r.lanes, c = ((int)blockIdx.y * NT + lane) * V;
    const long long p0 = (long long)blockIdx.x * r.rpi * UN + ph;
    if (ph >= r.rpi || c >= r.C) return;
    uint32_t w[UN];
    int e[UN];
#pragma unroll
    for (int j = 0; j < UN; ++j) {  // rows past the end read the last one and are not written
        const long long p = min(p0 + (long long)j * r.rpi, r.P - 1);
        if constexpr (V == 4) w[j] = *reinterpret_cast<const uint32_t *>(codes + p * r.cp + c);
        else w[j] = (uint8_t)codes[p * r.cp + c];
        e[j] = exps[p * r.nb + c / act8::BLK];
    }
#pragma unroll
    for (int j = 0; j < UN; ++j) {
        const long long p = p0 + (long long)j * r.rpi;
        if (p >= r.P) return;
        if constexpr (V == 4) {
            const f32x4 t = {act8::value_of(act8::code_at(w[j], 0), e[j]), act8::value_of(act8::code_at(w[j], 1), e[j]),
                             act8::value_of(act8::code_at(w[j], 2), e[j]), act8::value_of(act8::code_at(w[j], 3), e[j])};
            __builtin_nontemporal_store(t, reinterpret_cast<f32x4 *>(x + p * r.C + c));
        } else {
            __builtin_nontemporal_store(act8::value_of(act8::code_at(w[j], 0), e[j]), x + p * r.C + c);
        }
    }
}

// the rows and the grid; false where the sizes do not fit it
bool plan(int64_t P, int32_t C, int V, Rows &r, dim3 &grid) {
    if (P <= 0 || C <= 0 || P > (1LL << 46) / C) return false;
    const bool flat = C % act8::BLK == 0;  // rows of one block each
    r.P = flat ? P * (C / act8::BLK) : P;
    r.C = flat ? act8::BLK : C;
    r.nb = (r.C + act8::BLK - 1) / act8::BLK;
    r.cp = act8::pitch(r.C);
    const int lanes = r.nb * (act8::BLK / V), chunks = (lanes + NT - 1) / NT;
    r.lanes = lanes < NT ? lanes : NT;
    r.rpi = NT / r.lanes;
    const long long blocks = (r.P + (long long)r.rpi * UN - 1) / (r.rpi * UN);
    if (blocks > 0x7fffffffLL || chunks > 65535) return false;
    grid = dim3((unsigned)blocks, (unsigned)chunks);
    return true;
}

inline bool quads(const void *f32, int C) { return C % 4 == 0 && (uintptr_t)f32 % 16 == 0; }

}  // namespace

extern "C" int esr_act8_pack(const float *x, int64_t P, int32_t C, int8_t *codes, uint8_t *exps, esr_stream_t stream) {
    if (!x || !codes || !exps || C <= 0 || (uintptr_t)codes % 16) return ESR_EINVAL;
    const int V = quads(x, C) ? 4 : 1;
    Rows r;
    dim3 grid;
    if (!plan(P, C, V, r, grid)) return ESR_EINVAL;
    const hipStream_t st = (hipStream_t)stream;
    if (V == 4) hipLaunchKernelGGL(act8_pack_kernel<4>, grid, dim3(NT), 0, st, x, r, codes, exps);
    else hipLaunchKernelGGL(act8_pack_kernel<1>, grid, dim3(NT), 0, st, x, r, codes, exps);
    return hipGetLastError() == hipSuccess ? ESR_OK : ESR_ELAUNCH;
}

extern "C" int esr_act8_unpack(const int8_t *codes, const uint8_t *exps, int64_t P, int32_t C, float *x,
                               esr_stream_t stream) {
    if (!x || !codes || !exps || C <= 0 || (uintptr_t)codes % 16) return ESR_EINVAL;
    const int V = quads(x, C) ? 4 : 1;
    Rows r;
    dim3 grid;
    if (!plan(P, C, V, r, grid)) return ESR_EINVAL;
    const hipStream_t st = (hipStream_t)stream;
    if (V == 4) hipLaunchKernelGGL(act8_unpack_kernel<4>, grid, dim3(NT), 0, st, codes, exps, r, x);
    else hipLaunchKernelGGL(act8_unpack_kernel<1>, grid, dim3(NT), 0, st, codes, exps, r, x);
    return hipGetLastError() == hipSuccess ? ESR_OK : ESR_ELAUNCH;
}
