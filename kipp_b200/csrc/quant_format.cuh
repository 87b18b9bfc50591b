// The quantised cache: how keys and values lie in 8 or 4 bits.  Shared by the kernels that write,
// read back (cache_quant.cu) and attend to it (attention_quant.cu).
//
// One run's cache is four arrays: codes, bytes [page][kv_head][slot][D * bits / 8], and scales,
// bfloat16 [page][kv_head][slot][D / 32], of keys and of values.  The D channels of a head (a
// multiple of 32) form G = D / 32 groups of 32: channel c is in group (c / 4) % G, so a group is
// eight runs of four channels, spread over the whole head.  With L = 2^(bits - 1):
//     m      the group's element of the largest magnitude (the positive one of two alike)
//     scale  bfloat16(m / -L)
//     code   clamp(rint(x / scale), -L, L - 1) + L
//     value  (code - L) * scale
// The scale takes the sign that puts m at the end of the range that reaches further, -L.  Four-bit
// codes lie two to a byte, the even channel in the low half.  (The reference's Q8_0 cache has
// symmetric groups of 32 too, src/kipp.c:2757-2805, with the scale in front of each block's codes.)
//
// Why runs of four: the tensor-core kernel takes the codes from memory in plain channel order, 16 bits
// (a run in 4 bits) at a time, and a product over 16 channels must stay within one group.  Four lanes
// of a warp share a key's row and eight share a value's, each lane a stretch of it; with runs dealt out
// in turn every stretch holds whole runs of every group.  A channel and its rotation partner D / 2
// further are always in the same group.
#pragma once
#include "common.cuh"

// The same condition for every kernel: whole groups, and rows of codes that 16-byte copies can take.
__host__ __device__ inline bool quant_head_ok(int head_dim) { return head_dim > 0 && head_dim % 32 == 0 && head_dim <= 512; }

// What a key or value element is before it gets a code: never an infinity or a NaN (cache_value), and at
// most 2^60, so that scales and the products with them stay far from the ends of float32.
constexpr float QUANT_MOST = 1152921504606846976.f;
__device__ __forceinline__ float quant_input(float v) { return fminf(fmaxf(cache_value(v), -QUANT_MOST), QUANT_MOST); }

// The scale of a group whose largest element is hi and smallest lo, as bfloat16 bits.
template <int BITS> __device__ __forceinline__ uint16_t quant_scale(float hi, float lo) {
    constexpr float INV = BITS == 4 ? -0.125f : -0.0078125f;      // 1 / -L, exact
    const float m = hi >= -lo ? hi : lo;
    return __bfloat16_as_ushort(__float2bfloat16_rn(m * INV));
}
__device__ __forceinline__ float quant_scale_value(uint16_t bits) { return __uint_as_float((uint32_t)bits << 16); }

// The code of x, formed as it is defined; a scale of 0 (a group of zeros) has the code that stands for 0.  Less L, as a number.
template <int BITS> __device__ __forceinline__ float quant_code(float x, float scale) {
    constexpr float L = BITS == 4 ? 8.f : 128.f;
    return scale == 0.f ? 0.f : fminf(fmaxf(rintf(__fdiv_rn(x, scale)), -L), L - 1.f);
}
// 1 / scale, or 0 where that may not be a number: a scale of 0, or a subnormal one.
__device__ __forceinline__ float quant_inverse(float scale) { return fabsf(scale) < 0x1p-126f ? 0.f : __fdiv_rn(1.f, scale); }
// Four codes of one group, side by side in the low 4 BITS bits.  x * inverse is off from x / scale by 2^-22 of it, 2^-15 at most, so its
// rounding to a whole number (an addition of 1.5 * 2^23 and a subtraction: ties to even, no conversion) is the quotient's unless it
// lies as near to the middle between two; `doubt` then grows beyond QUANT_DOUBT and the codes have to be formed as they are defined.
// They are put together as numbers too: whole ones below 2^24 add exactly.
constexpr float QUANT_DOUBT = 0.5f - 0x1p-14f;
template <int BITS> __device__ __forceinline__ uint32_t quant_pack4(float r0, float r1, float r2, float r3) {
    if constexpr (BITS == 4)
        return __float_as_uint(fmaf(r3, 4096.f, fmaf(r2, 256.f, fmaf(r1, 16.f, r0 + (8388608.f + 8.f * 4369.f))))) & 0xffffu;
    return __byte_perm(__float_as_uint(fmaf(r1, 256.f, r0 + (8388608.f + 128.f * 257.f))),
                       __float_as_uint(fmaf(r3, 256.f, r2 + (8388608.f + 128.f * 257.f))), 0x5410);
}
template <int BITS> __device__ __forceinline__ uint32_t quant_codes4(const float* x, float inverse, float& doubt) {
    constexpr float L = BITS == 4 ? 8.f : 128.f, MAGIC = 12582912.f;
    float r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float q = fminf(fmaxf(__fmul_rn(x[i], inverse), -L), L - 1.f);
        r[i] = __fsub_rn(__fadd_rn(q, MAGIC), MAGIC);
        doubt = fmaxf(doubt, fabsf(q - r[i]));
    }
    return quant_pack4<BITS>(r[0], r[1], r[2], r[3]);
}
template <int BITS> __device__ __forceinline__ uint32_t quant_codes4_defined(const float* x, float scale) {
    return quant_pack4<BITS>(quant_code<BITS>(x[0], scale), quant_code<BITS>(x[1], scale), quant_code<BITS>(x[2], scale), quant_code<BITS>(x[3], scale));
}
