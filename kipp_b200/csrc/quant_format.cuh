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

// The code of x as a number, 0 to 2 L - 1; a scale of 0 (a group of zeros) has the code that stands for 0.  `inverse` is 1 / scale,
// rounded: x * inverse is off from x / scale by 2^-22 of it, 2^-15 at most, so the rounding to a whole number is that of the
// quotient unless it lies as near to the middle between two, and then the quotient is formed (one division a group instead of 32; the
// whole number comes out of an addition of 1.5 * 2^23, ties to even, and no conversion).
template <int BITS> __device__ __forceinline__ float quant_code(float x, float scale, float inverse) {
    constexpr float L = BITS == 4 ? 8.f : 128.f, MAGIC = 12582912.f;
    float q = fminf(fmaxf(__fmul_rn(x, inverse), -L), L - 1.f);
    float r = __fsub_rn(__fadd_rn(q, MAGIC), MAGIC);
    if (fabsf(q - r) > 0.5f - 0x1p-14f || inverse == 0.f)
        r = scale == 0.f ? 0.f : fminf(fmaxf(rintf(__fdiv_rn(x, scale)), -L), L - 1.f);
    return r + L;
}
// (0 where it may not be a number: a scale of 0, or a subnormal one)
__device__ __forceinline__ float quant_inverse(float scale) { return fabsf(scale) < 0x1p-126f ? 0.f : __fdiv_rn(1.f, scale); }
// four codes as whole numbers in one: their bits side by side in the low 4 BITS bits (exact: at most 2^24 of 4 bits' worth, or two
// halves of 16)
template <int BITS> __device__ __forceinline__ uint32_t quant_pack4(float c0, float c1, float c2, float c3) {
    constexpr float MAGIC = 8388608.f;
    if constexpr (BITS == 4) return __float_as_uint(fmaf(c3, 4096.f, fmaf(c2, 256.f, fmaf(c1, 16.f, c0))) + MAGIC) & 0xffffu;
    return __byte_perm(__float_as_uint(fmaf(c1, 256.f, c0) + MAGIC), __float_as_uint(fmaf(c3, 256.f, c2) + MAGIC), 0x5410);
}
