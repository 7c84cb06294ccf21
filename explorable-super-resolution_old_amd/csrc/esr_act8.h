// 8-bit activation blocks (esr_act8.hip, esr_gn.hip, esr_wgrad8.hip; layout in include/esr_amd.h).
//
// A block is 32 consecutive channels of one pixel (the last block of a pixel may be shorter).  Its values share one
// power-of-two step 2^(e - 132), e in [0, 254], the smallest with 127·step >= max|x|; a value is code·step, code in
// [-127, 127] ([-63, 63] at e = 254).  A power of two because code·step is then exact in fp32 (and, with 7 significant
// bits, in f16 / bf16, which is what the matrix-core weight gradient multiplies), and code = rint(x / step) has no
// division error: max error step/2 <= max|x|/127, a whole step where a code is moved to keep x's side of a threshold.
// e = 255 marks a block that holds an infinity or a NaN: all of it reads back as NaN.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>

namespace act8 {

constexpr int BLK = 32;

// codes of a pixel: rows of 16 bytes, so that every pixel's codes start where a 16-byte access may
__host__ __device__ __forceinline__ int pitch(int C) { return (C + 15) & ~15; }

// exponent byte from the bits of max|x| (an unsigned max over abs bits orders finite < inf < NaN)
__device__ __forceinline__ int exp_of(unsigned amax_bits) {
    const int q = (int)(amax_bits >> 23);
    if (q == 0) return 0;  // zero or subnormal: step 2^-132
    if (q == 255) return 255;
    return q - 1 + ((amax_bits & 0x7fffffu) > 0x7e0000u ? 1 : 0);  // mantissa > 127/64: one power more
}
// the largest code (64 · 2^122 is past the largest float), and a code kept to it
__device__ __forceinline__ float most_of(int e) { return e == 254 ? 63.f : 127.f; }
__device__ __forceinline__ float keep(float code, int e) { return __builtin_amdgcn_fmed3f(code, -most_of(e), most_of(e)); }
// (e = 255: anything; word_of drops it)
__device__ __forceinline__ float code_of(float x, int e) { return keep(rintf(ldexpf(x, 132 - e)), e); }
// V codes as bytes, 0 at e = 255: an unsigned byte of code + 128 each, the sign bits turned at the end
template <int V>
__device__ __forceinline__ uint32_t word_of(const float *code, int e) {
    uint32_t w = 0;
#pragma unroll
    for (int k = 0; k < V; ++k) w = __builtin_amdgcn_cvt_pk_u8_f32(code[k] + 128.f, k, w);
    return e == 255 ? 0u : w ^ 0x80808080u;
}
__device__ __forceinline__ float value_of(float code, int e) {
    return e == 255 ? __builtin_nanf("") : ldexpf(code, e - 132);
}
__device__ __forceinline__ unsigned abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// the four codes of a packed word
__device__ __forceinline__ float code_at(uint32_t w, int k) { return (float)(int8_t)(w >> (8 * k)); }

// max over the L lanes (8, 32 or 64, aligned, all active) that hold one block.  The first 16 by data-parallel moves of
// the vector unit (lanes 1, 2 further of four, then the other half of 8 and of 16 mirrored), without LDS's latency.
template <int L>
__device__ __forceinline__ unsigned block_max(unsigned m) {
    const auto with = [&](auto ctrl) {
        m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, decltype(ctrl)::value, 0xf, 0xf, false));
    };
    with(std::integral_constant<int, 0xB1>{});               // quad_perm 1 0 3 2
    with(std::integral_constant<int, 0x4E>{});               // quad_perm 2 3 0 1
    with(std::integral_constant<int, 0x141>{});              // row_half_mirror
    if (L > 8) with(std::integral_constant<int, 0x140>{});   // row_mirror
#pragma unroll
    for (int s = 16; s < L; s <<= 1) m = max(m, (unsigned)__shfl_xor((int)m, s));
    return m;
}

}  // namespace act8
