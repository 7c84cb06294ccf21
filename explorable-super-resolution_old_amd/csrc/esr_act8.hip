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

// the rows; false where the sizes do not fit the kernels
bool plan(int64_t P, int32_t C, int V, Rows &r, int &chunks) {
    if (P <= 0 || C <= 0 || P > (1LL << 46) / C) return false;
    const bool flat = C % act8::BLK == 0;  // rows of one block each
    r.P = flat ? P * (C / act8::BLK) : P;
    r.C = flat ? act8::BLK : C;
    r.nb = (r.C + act8::BLK - 1) / act8::BLK;
    r.cp = act8::pitch(r.C);
    const int lanes = r.nb * (act8::BLK / V);
    chunks = (lanes + NT - 1) / NT;
    r.lanes = lanes < NT ? lanes : NT;
    r.rpi = NT / r.lanes;
    return chunks <= 65535;
}

// launch(grid, part, first row) over all rows: a grid's first dimension ends below 2^32 threads, so that long tensors take
// several launches (of 2^23 workgroups: 2^28 rows of one channel, 2^30 of 32)
template <typename F>
int parts(const Rows &r, int chunks, F launch) {
    const long long per = (long long)r.rpi * UN, most = per << 23;
    for (long long p0 = 0; p0 < r.P; p0 += most) {
        Rows part = r;
        part.P = r.P - p0 < most ? r.P - p0 : most;
        launch(dim3((unsigned)((part.P + per - 1) / per), (unsigned)chunks), part, p0);
        if (hipGetLastError() != hipSuccess) return ESR_ELAUNCH;
    }
    return ESR_OK;
}

inline bool quads(const void *f32, int C) { return C % 4 == 0 && (uintptr_t)f32 % 16 == 0; }

}  // namespace

extern "C" int esr_act8_pack(const float *x, int64_t P, int32_t C, int8_t *codes, uint8_t *exps, esr_stream_t stream) {
    if (!x || !codes || !exps || C <= 0 || (uintptr_t)codes % 16) return ESR_EINVAL;
    const int V = quads(x, C) ? 4 : 1;
    Rows r;
    int chunks;
    if (!plan(P, C, V, r, chunks)) return ESR_EINVAL;
    return parts(r, chunks, [&](dim3 grid, const Rows &t, long long p0) {
        hipLaunchKernelGGL(V == 4 ? act8_pack_kernel<4> : act8_pack_kernel<1>, grid, dim3(NT), 0, (hipStream_t)stream,
                           x + p0 * r.C, t, codes + p0 * r.cp, exps + p0 * r.nb);
    });
}

extern "C" int esr_act8_unpack(const int8_t *codes, const uint8_t *exps, int64_t P, int32_t C, float *x,
                               esr_stream_t stream) {
    if (!x || !codes || !exps || C <= 0 || (uintptr_t)codes % 16) return ESR_EINVAL;
    const int V = quads(x, C) ? 4 : 1;
    Rows r;
    int chunks;
    if (!plan(P, C, V, r, chunks)) return ESR_EINVAL;
    return parts(r, chunks, [&](dim3 grid, const Rows &t, long long p0) {
        hipLaunchKernelGGL(V == 4 ? act8_unpack_kernel<4> : act8_unpack_kernel<1>, grid, dim3(NT), 0, (hipStream_t)stream,
                           codes + p0 * r.cp, exps + p0 * r.nb, t, x + p0 * r.C);
    });
}
