// Writing the quantised cache (quant_format.cuh) and reading it back.
//
// Writing: what rope_cache.cu does for a cache in the compute type (per-head RMSNorm of queries and
// keys, rotation, queries to an activation buffer, src/kipp.c:2480-2500, 2368-2382), with keys and
// values rounded to codes on the way into the pages (the reference's Q8_0 cache, src/kipp.c:2757-2805).
//
// Which code an element gets turns on which side of a border it falls, so the arithmetic before it is
// spelled out, and two kernels (and a plain implementation) that see the same head get the same codes:
// the sum of squares is formed in 64 bits and its mean rounded once to 32 (any order of that sum then
// gives the same mean, short of a tie in the 29 bits that are dropped), and the norm and the rotation
// are single operations in 32 bits, each rounded, none fused.  Keys are coded from 32 bits, not
// from a bfloat16 copy.
//
// Reading back: codes -> bfloat16 or float32 rows in pages of the same shape, for a list of pages, or
// for the entries of a step with the block table of the pages made (attention over more than a few tokens reads those); for
// the prompt kernel as float16, by powers of two that bring the largest number of an entry's kv head to 2^15.
#include "quant_format.cuh"
#include "head_math.cuh"
#include <cuda_fp16.h>

namespace {

struct QuantPages {
    uint8_t* k_codes; bf16* k_scales; uint8_t* v_codes; bf16* v_scales;
    int n_pages, page_size, n_kv;
};

struct WriteParams {
    const void* qkv; long long ld;
    void* q_out;
    QuantPages pages;
    const void* q_norm_w; const void* k_norm_w; int norm_dtype; float eps;
    const float2* cos_sin; int rotary_dim;
    const int* positions; const int* entry_of_token; const int* block_table; int table_width;
    int tokens, n_q, head_dim, write_cache;
    int* status;
};

// The cache row (page, kv head, slot) of kv head g of a token, or -1: an unmapped page is refused.
__device__ __forceinline__ long long cache_row(const WriteParams& p, int t, int g) {
    const int pos = p.positions[t], slot = pos / p.pages.page_size;
    const int page = pos >= 0 && slot < p.table_width ? p.block_table[(size_t)p.entry_of_token[t] * p.table_width + slot] : -1;
    if (page < 0 || page >= p.pages.n_pages) return -1;
    return ((long long)page * p.pages.n_kv + g) * p.pages.page_size + (pos - slot * p.pages.page_size);
}

__device__ __forceinline__ float mean_square(double sum, int n) { return (float)(sum / (double)n); }
__device__ __forceinline__ float norm_factor(float mean, float eps) {
    return __fdiv_rn(1.f, __fsqrt_rn(__fadd_rn(mean, eps)));
}
__device__ __forceinline__ void turn(float& a, float& b, float2 cs) {
    const float a0 = a, b0 = b;
    a = __fsub_rn(__fmul_rn(a0, cs.x), __fmul_rn(b0, cs.y));
    b = __fadd_rn(__fmul_rn(b0, cs.x), __fmul_rn(a0, cs.y));
}

// Any head size (a multiple of 32), any rotary size, any alignment: one warp per (token, head), the
// head in shared memory.  A group is a lane per channel.
template <typename T, int BITS>
__global__ void __launch_bounds__(128) quant_write_any_kernel(const WriteParams p) {
    __shared__ float rows[4][512];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, D = p.head_dim, heads = p.n_q + 2 * p.pages.n_kv;
    const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (item >= (long long)p.tokens * heads) return;
    const int t = (int)(item / heads), h = (int)(item - (long long)t * heads);
    const bool is_q = h < p.n_q, is_v = h >= p.n_q + p.pages.n_kv;
    if (!is_q && !p.write_cache) return;
    float* row = rows[threadIdx.x >> 5];
    const T* src = static_cast<const T*>(p.qkv) + (size_t)t * p.ld + (size_t)h * D;
    for (int i = lane; i < D; i += 32) row[i] = to_f32(src[i]);
    __syncwarp();
    if (!is_v) {
        const void* nw = is_q ? p.q_norm_w : p.k_norm_w;
        if (nw != nullptr) {
            double ss = 0.0;
            for (int i = lane; i < D; i += 32) ss += (double)row[i] * (double)row[i];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            const float r = norm_factor(mean_square(ss, D), p.eps);
            for (int i = lane; i < D; i += 32) row[i] = __fmul_rn(__fmul_rn(row[i], r), load_w(nw, p.norm_dtype, i));
            __syncwarp();
        }
        if (p.cos_sin != nullptr) {
            const int half = p.rotary_dim / 2;
            for (int i = lane; i < half; i += 32) turn(row[i], row[i + half], p.cos_sin[(size_t)t * half + i]);
            __syncwarp();
        }
    }
    if (is_q) {
        T* dst = static_cast<T*>(p.q_out) + ((size_t)t * p.n_q + h) * D;
        for (int i = lane; i < D; i += 32) dst[i] = from_f32<T>(row[i]);
        return;
    }
    const long long at = cache_row(p, t, is_v ? h - p.n_q - p.pages.n_kv : h - p.n_q);
    if (at < 0) {
        if (lane == 0) atomicExch(p.status, 2);
        return;
    }
    uint8_t* codes = (is_v ? p.pages.v_codes : p.pages.k_codes) + (size_t)at * (D * BITS / 8);
    bf16* scales = (is_v ? p.pages.v_scales : p.pages.k_scales) + (size_t)at * (D / 32);
    const int G = D / 32;
    for (int g = 0; g < G; ++g) {
        const int c = (lane >> 2) * 4 * G + g * 4 + (lane & 3);
        const float x = quant_input(row[c]);
        const float hi = warp_max(x), lo = -warp_max(-x);
        const uint16_t sb = quant_scale<BITS>(hi, lo);
        const uint32_t code = (uint32_t)(quant_code<BITS>(x, quant_scale_value(sb)) + (BITS == 4 ? 8.f : 128.f));
        if (BITS == 8) {
            codes[c] = (uint8_t)code;
        } else {
            const uint32_t high = __shfl_down_sync(0xffffffffu, code, 1);
            if ((lane & 1) == 0) codes[c >> 1] = (uint8_t)(code | (high << 4));
        }
        if (lane == 0) reinterpret_cast<uint16_t*>(scales)[g] = sb;
    }
}

__device__ __forceinline__ void put8(bf16* p, const float (&x)[8]) { *reinterpret_cast<uint4*>(p) = pack8(x); }
__device__ __forceinline__ void put8(float* p, const float (&x)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
template <int BITS> __device__ __forceinline__ void put_codes(uint8_t* p, uint32_t first, uint32_t second) {
    if constexpr (BITS == 4) *reinterpret_cast<uint32_t*>(p) = first | second << 16;
    else *reinterpret_cast<uint2*>(p) = make_uint2(first, second);
}

// Heads of 64, 128 or 256 channels, rotated whole, by half or not at all, 16-byte aligned: HEAD_DIM / 16 lanes
// share a (token, head), a lane holds 8 channels of the first half and the 8 half a head further, as
// in rope_cache.cu.  A whole rotation's partners are those two; half a rotation's are the first ones of two lanes.  A lane has
// four runs of two groups; the four lanes whose numbers agree modulo HEAD_DIM / 64 hold the same two groups, so a
// group's extremes are two exchanges away.  The 64-bit sum of squares (16 conversions a lane on a pipe of 16 lanes) is
// formed for keys only: queries get no codes, and four in five heads are theirs.
// Bound by its instructions (some 220 a warp and four query heads, three times as many where there are codes to make), at an issue rate of a
// half, and by what its 19 warps an SM wait for between them, their rows first (long scoreboard 2.6 of 9 warps an issue), fixed latencies next
// (1.6), not by memory's rate: 2,048 tokens of 32 and 2 x 8 bfloat16 heads of 128 to 8 bits take 17.4 us
// (46 MB, 2.7 TB/s), 2,513 of 12 and 2 x 2 float32 heads of 64 to 4 bits 8.0 us (18 MB, 2.3 TB/s), eight tokens 2.6 us.  A block is no
// larger than a token's heads need (those float32 heads: 15.8 us with 128 threads of which half are idle, 11.0 with 64); blocks of
// 64, 192 and 384 threads were slower than 128, 8 blocks an SM of 64 registers a thread no faster than 6 of 80.
constexpr int WRITE_THREADS = 128;
__device__ __forceinline__ void fetch8(uint4 (&raw)[1], const bf16* p) { raw[0] = *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ void fetch8(uint4 (&raw)[2], const float* p) {
    raw[0] = reinterpret_cast<const uint4*>(p)[0];
    raw[1] = reinterpret_cast<const uint4*>(p)[1];
}
__device__ __forceinline__ void spread8(float (&x)[8], const uint4 (&raw)[1]) { unpack8(x, raw[0]); }
__device__ __forceinline__ void spread8(float (&x)[8], const uint4 (&raw)[2]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        x[4 * i] = __uint_as_float(raw[i].x); x[4 * i + 1] = __uint_as_float(raw[i].y);
        x[4 * i + 2] = __uint_as_float(raw[i].z); x[4 * i + 3] = __uint_as_float(raw[i].w);
    }
}
template <typename T, int BITS, int HEAD_DIM>
__global__ void __launch_bounds__(WRITE_THREADS, 6) quant_write_kernel(const WriteParams p) {
    constexpr int LPH = HEAD_DIM / 16, HALF = HEAD_DIM / 2, G = HEAD_DIM / 32, RAW = sizeof(T) / 2;
    pdl_launch_dependents();
    const int t = blockIdx.y, sub = threadIdx.x % LPH, PER = blockDim.x / LPH;
    const int n_kv = p.pages.n_kv, heads = p.n_q + (p.write_cache ? 2 * n_kv : 0);
    const T* const row = static_cast<const T*>(p.qkv) + (size_t)t * p.ld + sub * 8;
    int h = blockIdx.x * PER + threadIdx.x / LPH;
    // (the step's lists, before the wait)
    const int pos = p.positions[t], slot = pos / p.pages.page_size;
    int page = -1;
    if (p.write_cache && pos >= 0 && slot < p.table_width) page = p.block_table[(size_t)p.entry_of_token[t] * p.table_width + slot];
    if (page >= p.pages.n_pages) page = -1;
    const bool whole = p.rotary_dim == HEAD_DIM;
    pdl_wait();
    uint4 raw_a[RAW], raw_b[RAW];
    if (h < heads) {
        fetch8(raw_a, row + (size_t)h * HEAD_DIM);
        fetch8(raw_b, row + (size_t)h * HEAD_DIM + HALF);
    }
    float4 cs[4];
    if (p.cos_sin != nullptr) {
        const float4* c = reinterpret_cast<const float4*>(p.cos_sin + (size_t)t * (p.rotary_dim / 2) + (whole ? sub : sub % (LPH / 2)) * 8);
#pragma unroll
        for (int i = 0; i < 4; ++i) cs[i] = c[i];
    }
    if (page < 0 && p.write_cache && blockIdx.x == 0 && threadIdx.x == 0) atomicExch(p.status, 2);      // unmapped page: refused, never written
    // No lane leaves early: a warp holds several heads and all lanes take part in the exchanges.
    for (int first = blockIdx.x * PER; first < heads; first += gridDim.x * PER, h += gridDim.x * PER) {
        const bool active = h < heads, is_q = h < p.n_q, is_k = !is_q && h < p.n_q + n_kv, normed = active && (is_q || is_k);
        float a[8], b[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = b[i] = 0.f;
        if (active) { spread8(a, raw_a); spread8(b, raw_b); }
        if (h + (int)gridDim.x * PER < heads) {
            fetch8(raw_a, row + (size_t)(h + gridDim.x * PER) * HEAD_DIM);
            fetch8(raw_b, row + (size_t)(h + gridDim.x * PER) * HEAD_DIM + HALF);
        }
        if (p.q_norm_w != nullptr) {              // both weights or neither (checked by the host)
            const void* nw = is_q ? p.q_norm_w : p.k_norm_w;
            float mean;
            if (__any_sync(0xffffffffu, is_k)) {
                double ss = 0.0;
#pragma unroll
                for (int i = 0; i < 8; ++i) ss += (double)a[i] * (double)a[i] + (double)b[i] * (double)b[i];
#pragma unroll
                for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                mean = mean_square(ss, HEAD_DIM);
            } else {
                float ss = head_ssq8(a, b);
#pragma unroll
                for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                mean = ss * (1.f / HEAD_DIM);
            }
            if (normed) {
                const float r = norm_factor(mean, p.eps);
                float w[8];
                load_w8(w, nw, p.norm_dtype, sub * 8);
                head_scale8(a, r, w);
                load_w8(w, nw, p.norm_dtype, HALF + sub * 8);
                head_scale8(b, r, w);
            }
        }
        if (p.cos_sin != nullptr) {
            if (whole) {
                if (normed) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        turn(a[2 * i], b[2 * i], make_float2(cs[i].x, cs[i].y));
                        turn(a[2 * i + 1], b[2 * i + 1], make_float2(cs[i].z, cs[i].w));
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float other = __shfl_xor_sync(0xffffffffu, a[i], LPH / 2);
                    if (normed) {
                        const float2 c = i & 1 ? make_float2(cs[i / 2].z, cs[i / 2].w) : make_float2(cs[i / 2].x, cs[i / 2].y);
                        if (sub < LPH / 2) turn(a[i], other, c);
                        else turn(other, a[i], c);
                    }
                }
            }
        }
        if (active && is_q) {
            T* dst = static_cast<T*>(p.q_out) + ((size_t)t * p.n_q + h) * HEAD_DIM + sub * 8;
            put8(dst, a);
            put8(dst + HALF, b);
        }
        if (__all_sync(0xffffffffu, is_q)) continue;
        // (a number that quant_input changes is rare, and looked for all at once: what is not finite makes a sum of zeros a NaN)
        float hi[2], lo[2], zero = 0.f;
        auto extremes = [&] {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                hi[r] = fmaxf(a[4 * r], b[4 * r]);
                lo[r] = fminf(a[4 * r], b[4 * r]);
#pragma unroll
                for (int i = 4 * r + 1; i < 4 * r + 4; ++i) {
                    hi[r] = fmaxf(hi[r], fmaxf(a[i], b[i]));
                    lo[r] = fminf(lo[r], fminf(a[i], b[i]));
                }
            }
        };
        extremes();
#pragma unroll
        for (int i = 0; i < 8; ++i) zero = fmaf(a[i], 0.f, fmaf(b[i], 0.f, zero));
        if (__any_sync(0xffffffffu, zero != 0.f || fmaxf(hi[0], hi[1]) > QUANT_MOST || fminf(lo[0], lo[1]) < -QUANT_MOST)) {
#pragma unroll
            for (int i = 0; i < 8; ++i) { a[i] = quant_input(a[i]); b[i] = quant_input(b[i]); }
            extremes();
        }
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int o = G / 2; o <= G; o <<= 1) {
                hi[r] = fmaxf(hi[r], __shfl_xor_sync(0xffffffffu, hi[r], o));
                lo[r] = fminf(lo[r], __shfl_xor_sync(0xffffffffu, lo[r], o));
            }
        if (page < 0 || !active || is_q) continue;
        const size_t at = ((size_t)page * n_kv + (is_k ? h - p.n_q : h - p.n_q - n_kv)) * p.pages.page_size + (pos - slot * p.pages.page_size);
        const uint16_t b0 = quant_scale<BITS>(hi[0], lo[0]), b1 = quant_scale<BITS>(hi[1], lo[1]);
        const float s0 = quant_scale_value(b0), s1 = quant_scale_value(b1), i0 = quant_inverse(s0), i1 = quant_inverse(s1);
        float doubt = 0.f;
        uint32_t c[4] = {quant_codes4<BITS>(a, i0, doubt), quant_codes4<BITS>(a + 4, i1, doubt), quant_codes4<BITS>(b, i0, doubt),
                         quant_codes4<BITS>(b + 4, i1, doubt)};
        if (doubt > QUANT_DOUBT || i0 == 0.f || i1 == 0.f) {
            c[0] = quant_codes4_defined<BITS>(a, s0); c[1] = quant_codes4_defined<BITS>(a + 4, s1);
            c[2] = quant_codes4_defined<BITS>(b, s0); c[3] = quant_codes4_defined<BITS>(b + 4, s1);
        }
        uint8_t* codes = (is_k ? p.pages.k_codes : p.pages.v_codes) + at * (HEAD_DIM * BITS / 8) + sub * BITS;
        put_codes<BITS>(codes, c[0], c[1]);
        put_codes<BITS>(codes + HALF * BITS / 8, c[2], c[3]);
        if (sub < G / 2)
            reinterpret_cast<uint32_t*>((is_k ? p.pages.k_scales : p.pages.v_scales) + at * G)[sub] = (uint32_t)b0 | (uint32_t)b1 << 16;
    }
}

template <typename T, int BITS> int launch_write(const WriteParams& p, cudaStream_t s) {
    const int heads = p.n_q + 2 * p.pages.n_kv, D = p.head_dim;
    const uintptr_t bits = (uintptr_t)p.qkv | (uintptr_t)p.q_out | (uintptr_t)p.q_norm_w | (uintptr_t)p.k_norm_w | (uintptr_t)p.cos_sin |
                           (uintptr_t)p.pages.k_codes | (uintptr_t)p.pages.v_codes | (uintptr_t)p.pages.k_scales | (uintptr_t)p.pages.v_scales;
    const bool aligned = (bits & 15) == 0 && p.ld * (long long)sizeof(T) % 16 == 0;
    if (aligned && (p.cos_sin == nullptr || p.rotary_dim == D || p.rotary_dim * 2 == D) && p.tokens <= 65535 && (D == 64 || D == 128 || D == 256)) {
        const int lanes = heads * (D / 16), threads = lanes < WRITE_THREADS ? (lanes + 31) / 32 * 32 : WRITE_THREADS, per = threads / (D / 16);
        // A block takes all heads of a token where there are tokens enough: the angles are read once, and the
        // next heads are on their way meanwhile.
        const int shares = (heads + per - 1) / per;
        const dim3 grid((unsigned)(p.tokens >= 4 * kipp_sm_count() ? 1 : shares), (unsigned)p.tokens);
        auto kernel = D == 64 ? quant_write_kernel<T, BITS, 64> : D == 128 ? quant_write_kernel<T, BITS, 128> : quant_write_kernel<T, BITS, 256>;
        return kipp_launch(kernel, grid, dim3((unsigned)threads), 0, s, 1, p);
    }
    const long long blocks = ((long long)p.tokens * heads + 3) / 4;
    if (blocks > 0x7fffffffLL) return KIPP_ERR_ARG;
    return kipp_launch(quant_write_any_kernel<T, BITS>, dim3((unsigned)blocks), dim3(128), 0, s, 1, p);
}

// ------------------------------------------------------------------------------------- reading back
struct ReadParams {
    void* k_out; void* v_out;
    QuantPages pages;
    const int* list;                // [n] pages, or the step's block table
    int n, head_dim;
    int* status;
    // the entries' form: the pages that entries from first_entry on see, and the table of those made
    int* table_out; const int* q_start; const int* context_len;
    int table_width, first_entry, window;
    int at;                         // what the launch begins with, a page's place in the list or among the entries'
    float2* factors;                // float16: [entries][n_kv], what keys and values are multiplied by
    int least;                      // the entries of fewer tokens are left out
};

// The keys of entry e that its tokens see, [first, end): none where it is left out.
__device__ __forceinline__ int2 seen_keys(const ReadParams& p, int e) {
    const int tokens = p.q_start[e + 1] - p.q_start[e];
    if (tokens < p.least) return make_int2(0, 0);
    const int first = min(max(p.context_len[e], 0), 0x7fffffff - tokens);
    return make_int2(p.window > 0 ? max(0, first - p.window + 1) : 0, first + tokens);
}

// The power of two that brings L times the largest scale below 2^15: of the scales of the keys and of the values that an entry's
// tokens see, a block per kv head and entry.  (16 bytes of scales of 144 to 272 a token and head: the lists and two loads in a row
// bound it, 3 us for 6,144 tokens.)
constexpr int FACTOR_THREADS = 1024;
template <int BITS, int G>
__global__ void __launch_bounds__(FACTOR_THREADS) quant_factor_kernel(const ReadParams p) {
    static_assert(G == 2 || G == 4, "the prompt kernel's heads");
    __shared__ uint32_t sh[2][32];
    pdl_launch_dependents();
    pdl_wait();
    const int g = blockIdx.x, e = p.first_entry + blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int2 seen = seen_keys(p, e);
    const int* table = p.list + (size_t)e * p.table_width;
    const int end = min((long long)seen.y, (long long)p.table_width * p.pages.page_size);
    const int begin = min(seen.x, end);           // (a window behind the table's end has nothing, and its keys' numbers may end at 2^31)
    uint32_t most[2] = {0u, 0u};                  // pairs of bfloat16 without signs
    // (what is not there of an entry's keys, behind the table's end too: the prompt kernel takes zeros for both without a word, and a
    // page past the pool is reported by the kernel that reads it; the report made there took 59 registers instead of 48 and 3 % of the time)
    bool missing = seen.y > end;
    for (int base = begin + threadIdx.x; base < end; base += 4 * FACTOR_THREADS) {
        uint32_t k[4][G / 2], v[4][G / 2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = base + i * FACTOR_THREADS, slot = j / p.pages.page_size;
            const int page = j < end ? table[slot] : -1;
            if (page < 0 && j < end) missing = true;
#pragma unroll
            for (int w = 0; w < G / 2; ++w) k[i][w] = v[i][w] = 0u;
            if (page >= 0 && page < p.pages.n_pages) {
                const size_t row = ((size_t)page * p.pages.n_kv + g) * p.pages.page_size + (j - slot * p.pages.page_size);
                const uint32_t* ks = reinterpret_cast<const uint32_t*>(p.pages.k_scales) + row * (G / 2);
                const uint32_t* vs = reinterpret_cast<const uint32_t*>(p.pages.v_scales) + row * (G / 2);
#pragma unroll
                for (int w = 0; w < G / 2; ++w) { k[i][w] = ks[w]; v[i][w] = vs[w]; }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int w = 0; w < G / 2; ++w) {
                most[0] = __vmaxu2(most[0], k[i][w] & 0x7fff7fffu);
                most[1] = __vmaxu2(most[1], v[i][w] & 0x7fff7fffu);
            }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t one = __reduce_max_sync(0xffffffffu, max(most[i] & 0xffffu, most[i] >> 16));
        if (lane == 0) sh[i][warp] = one;
    }
    __syncthreads();
    if (missing) atomicExch(p.status, 3);
    if (warp == 0) {
        float f[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t bits = __reduce_max_sync(0xffffffffu, sh[i][lane]);
            const int exponent = max((int)(bits >> 7) - 127, -100);
            f[i] = __uint_as_float((uint32_t)(127 + 14 - exponent - (BITS == 4 ? 3 : 7)) << 23);
        }
        if (lane == 0) p.factors[(size_t)e * p.pages.n_kv + g] = make_float2(f[0], f[1]);
    }
}

// The eight channels that a word of 4-bit codes, or two of 8-bit, stand for, as bfloat16 pairs of (code - L) * 2^-13: a code in the
// low bits of 16 is the number code * 2^-133 (attention_quant.cu), and one fused multiply-add makes it that, exactly.
template <int BITS> __device__ __forceinline__ void whole_numbers(__nv_bfloat162 (&x)[4], const uint32_t* w) {
    const __nv_bfloat162 up = __float2bfloat162_rn(0x1p120f), less = __float2bfloat162_rn(BITS == 4 ? -0x1p-10f : -0x1p-6f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t v;
        if constexpr (BITS == 4) {
            v = __byte_perm(w[0], w[0] >> 4, i | i << 4 | (4 + i) << 8 | (4 + i) << 12) & 0x000f000fu;       // byte i of both
        } else {
            v = __byte_perm(w[i >> 1], 0u, i & 1 ? 0x4342 : 0x4140);
        }
        x[i] = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&v), up, less);
    }
}
template <int BITS> struct Unit { uint32_t w[BITS / 4]; uint16_t s[2]; };      // eight channels: codes, the scales of their two runs
template <int BITS, bool EVEN> __device__ __forceinline__ Unit<BITS> take_unit(const uint8_t* codes, const uint16_t* scales, int g0, int g1) {
    Unit<BITS> u;
    if constexpr (BITS == 4) u.w[0] = *reinterpret_cast<const uint32_t*>(codes);
    else { const uint2 v = *reinterpret_cast<const uint2*>(codes); u.w[0] = v.x; u.w[1] = v.y; }
    if constexpr (EVEN) {                                 // (an even number of groups: the two lie side by side)
        const uint32_t both = *reinterpret_cast<const uint32_t*>(scales + g0);
        u.s[0] = (uint16_t)both;
        u.s[1] = (uint16_t)(both >> 16);
    } else {
        u.s[0] = scales[g0];
        u.s[1] = scales[g1];
    }
    return u;
}
// (the scale times 2^13, exact, and one rounding; `factor` is float16's)
template <int BITS> __device__ __forceinline__ void put_unit(__half* p, const Unit<BITS>& u, float factor) {
    __nv_bfloat162 x[4];
    whole_numbers<BITS>(x, u.w);
    uint4 out;
    uint32_t* o = reinterpret_cast<uint32_t*>(&out);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float s = quant_scale_value(u.s[i >> 1]) * 8192.f * factor;
        const __half2 r = __floats2half2_rn(__low2float(x[i]) * s, __high2float(x[i]) * s);
        o[i] = *reinterpret_cast<const uint32_t*>(&r);
    }
    *reinterpret_cast<uint4*>(p) = out;
}
template <int BITS> __device__ __forceinline__ void put_unit(bf16* p, const Unit<BITS>& u, float) {
    __nv_bfloat162 x[4];
    whole_numbers<BITS>(x, u.w);
    uint4 out;
    uint32_t* o = reinterpret_cast<uint32_t*>(&out);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 s = __bfloat162bfloat162(__float2bfloat16_rn(quant_scale_value(u.s[i >> 1]) * 8192.f));
        const __nv_bfloat162 r = __hmul2(x[i], s);
        o[i] = *reinterpret_cast<const uint32_t*>(&r);
    }
    *reinterpret_cast<uint4*>(p) = out;
}
template <int BITS> __device__ __forceinline__ void put_unit(float* p, const Unit<BITS>& u, float) {
    __nv_bfloat162 x[4];
    whole_numbers<BITS>(x, u.w);
    float r[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float s = quant_scale_value(u.s[i >> 1]) * 8192.f;
        r[2 * i] = __low2float(x[i]) * s;
        r[2 * i + 1] = __high2float(x[i]) * s;
    }
    put8(p, r);
}

// One block per (share of a page, page); DIM is the head size, or 0 for any.  Every thread has UNROLL units of eight channels of keys
// and of values on their way at once.  A page whose number is negative (unmapped) or past the pool becomes zeros; past the
// pool is also reported.  Bound by HBM, three quarters and more of it writes (8 x 8,100 tokens of 8 heads of 128 from 4 bits: 62 us, 5.5 TB/s).
constexpr int READ_THREADS = 256;
template <typename T> struct IsHalf { static constexpr bool value = false; };
template <> struct IsHalf<__half> { static constexpr bool value = true; };
template <typename T, int BITS, bool ENTRIES, int DIM, int UNROLL>
__global__ void __launch_bounds__(READ_THREADS) quant_read_kernel(const ReadParams p) {
    if constexpr (!ENTRIES) pdl_launch_dependents();      // (a step's table is read before a kernel's wait: this one lets none start early)
    pdl_wait();
    const int i = p.at + blockIdx.y, D = DIM > 0 ? DIM : p.head_dim, G = D / 32;
    const int page = p.list[ENTRIES ? (size_t)(p.first_entry + i / p.table_width) * p.table_width + i % p.table_width : (size_t)i];
    int from = 0, to = 0;                         // the page's slots that a token sees
    const float2* factors = nullptr;
    if constexpr (ENTRIES) {
        const int e = p.first_entry + i / p.table_width, slot = i % p.table_width;
        const int2 seen = seen_keys(p, e);
        const bool used = page >= 0 && (long long)slot * p.pages.page_size < seen.y && (long long)(slot + 1) * p.pages.page_size > seen.x;
        if (blockIdx.x == 0 && threadIdx.x == 0) p.table_out[(size_t)e * p.table_width + slot] = used ? i : -1;
        if (!used) return;
        from = max(0, seen.x - slot * p.pages.page_size);
        to = min(p.pages.page_size, seen.y - slot * p.pages.page_size);
        factors = p.factors + (size_t)e * p.pages.n_kv;
    }
    const bool ok = page >= 0 && page < p.pages.n_pages;
    if (page >= p.pages.n_pages && threadIdx.x == 0) atomicExch(p.status, 3);
    const int per_row = D / 8, rows = p.pages.n_kv * p.pages.page_size, units = rows * per_row;
    const size_t in = (size_t)(ok ? page : 0) * rows, out = (size_t)i * rows;
    const uint8_t *k_codes = p.pages.k_codes + in * (D * BITS / 8), *v_codes = p.pages.v_codes + in * (D * BITS / 8);
    const uint16_t *k_scales = reinterpret_cast<const uint16_t*>(p.pages.k_scales) + in * G, *v_scales = reinterpret_cast<const uint16_t*>(p.pages.v_scales) + in * G;
    T *k_out = static_cast<T*>(p.k_out) + out * D, *v_out = static_cast<T*>(p.v_out) + out * D;
    for (int base = blockIdx.x * READ_THREADS * UNROLL; base < units; base += gridDim.x * READ_THREADS * UNROLL) {
        Unit<BITS> k[UNROLL], v[UNROLL];
#pragma unroll
        for (int j = 0; j < UNROLL; ++j) {
            const int u = base + j * READ_THREADS + threadIdx.x;
            k[j] = v[j] = Unit<BITS>{};
            const int row = u / per_row, at = ENTRIES ? row % p.pages.page_size : 0;
            if (u < units && ok && (!ENTRIES || (at >= from && at < to))) {
                const int c = u - row * per_row, g0 = 2 * c % G, g1 = g0 + 1 == G ? 0 : g0 + 1;
                k[j] = take_unit<BITS, (DIM > 0)>(k_codes + (size_t)u * BITS, k_scales + row * G, g0, g1);
                v[j] = take_unit<BITS, (DIM > 0)>(v_codes + (size_t)u * BITS, v_scales + row * G, g0, g1);
            }
        }
#pragma unroll
        for (int j = 0; j < UNROLL; ++j) {
            const int u = base + j * READ_THREADS + threadIdx.x;
            if (u < units) {
                float2 f = make_float2(1.f, 1.f);
                if constexpr (IsHalf<T>::value) f = factors[u / (per_row * p.pages.page_size)];
                put_unit<BITS>(k_out + (size_t)u * 8, k[j], f.x);
                put_unit<BITS>(v_out + (size_t)u * 8, v[j], f.y);
            }
        }
    }
}

template <typename T, int BITS, bool ENTRIES> auto read_kernel(int head_dim, bool many) {
    if (many) return head_dim == 64 ? quant_read_kernel<T, BITS, ENTRIES, 64, 4> : head_dim == 128 ? quant_read_kernel<T, BITS, ENTRIES, 128, 4>
                   : head_dim == 256 ? quant_read_kernel<T, BITS, ENTRIES, 256, 4> : quant_read_kernel<T, BITS, ENTRIES, 0, 4>;
    return head_dim == 64 ? quant_read_kernel<T, BITS, ENTRIES, 64, 1> : head_dim == 128 ? quant_read_kernel<T, BITS, ENTRIES, 128, 1>
         : head_dim == 256 ? quant_read_kernel<T, BITS, ENTRIES, 256, 1> : quant_read_kernel<T, BITS, ENTRIES, 0, 1>;
}

template <bool ENTRIES> int launch_read(const ReadParams& p, int bits, int out_dtype, cudaStream_t s) {
    const long long units = (long long)p.pages.n_kv * p.pages.page_size * (p.head_dim / 8);
    if (units > 0x3fffffff) return KIPP_ERR_ARG;
    // few pages, or small ones: a unit a thread, on more SMs (77 tokens of 4 heads of 128: 1.4 us, 2.1 with four; 8 x 8,100 of 8 heads:
    // 66 and 63 us)
    const bool many = units >= 4 * READ_THREADS && units * p.n > 32LL * READ_THREADS * kipp_sm_count();
    const int per = READ_THREADS * (many ? 4 : 1);
    const unsigned x = (unsigned)((units + per - 1) / per);
    // (the kernels of one head size take two scales as a word: scales at odd multiples of two bytes go to the one for any size)
    const int dim = (((uintptr_t)p.pages.k_scales | (uintptr_t)p.pages.v_scales) & 3) == 0 ? p.head_dim : 0;
    auto kernel = out_dtype == KIPP_DT_F32 ? (bits == 4 ? read_kernel<float, 4, ENTRIES>(dim, many) : read_kernel<float, 8, ENTRIES>(dim, many))
                                           : (bits == 4 ? read_kernel<bf16, 4, ENTRIES>(dim, many) : read_kernel<bf16, 8, ENTRIES>(dim, many));
    if constexpr (ENTRIES) {
        if (p.factors != nullptr) {
            const bool wide = p.head_dim == 128;
            auto factor = wide ? (bits == 4 ? quant_factor_kernel<4, 4> : quant_factor_kernel<8, 4>) : (bits == 4 ? quant_factor_kernel<4, 2> : quant_factor_kernel<8, 2>);
            const dim3 grid((unsigned)p.pages.n_kv, (unsigned)(p.n / p.table_width));
            if (grid.y > 65535) return KIPP_ERR_ARG;
            if (const int e = kipp_launch(factor, grid, dim3(FACTOR_THREADS), 0, s, 1, p)) return e;
            kernel = bits == 4 ? (wide ? (many ? quant_read_kernel<__half, 4, true, 128, 4> : quant_read_kernel<__half, 4, true, 128, 1>)
                                       : (many ? quant_read_kernel<__half, 4, true, 64, 4> : quant_read_kernel<__half, 4, true, 64, 1>))
                               : (wide ? (many ? quant_read_kernel<__half, 8, true, 128, 4> : quant_read_kernel<__half, 8, true, 128, 1>)
                                       : (many ? quant_read_kernel<__half, 8, true, 64, 4> : quant_read_kernel<__half, 8, true, 64, 1>));
        }
    }
    // (a grid's second dimension ends at 65,535)
    for (ReadParams q = p; q.at < p.n; q.at += 65535) {
        const unsigned y = (unsigned)(p.n - q.at < 65535 ? p.n - q.at : 65535);
        if (const int e = kipp_launch(kernel, dim3(x, y), dim3(READ_THREADS), 0, s, 1, q)) return e;
        if (p.n - q.at <= 65535) break;
    }
    return 0;
}

bool pages_ok(const QuantPages& g, int bits, int head_dim) {
    return (bits == 4 || bits == 8) && quant_head_ok(head_dim) && g.n_pages > 0 && g.page_size > 0 && g.n_kv > 0 &&
           g.k_codes && g.k_scales && g.v_codes && g.v_scales;
}
}  // namespace

// The arguments of the entry points, as one structure each (a caller that packs them spends a quarter of what passing them
// one by one costs it from Python).
struct KippQuantWrite {
    const void* qkv; void* q_out;                       // [tokens][ld_qkv], [tokens][n_q][head_dim], of one type
    void *k_codes, *k_scales, *v_codes, *v_scales;
    const void *q_norm_w, *k_norm_w, *cos_sin;          // or null
    const int *positions, *entry_of_token, *block_table;
    int* status;
    void* stream;
    long long ld_qkv;
    int bits, n_pages, page_size, dtype, norm_dtype, rotary_dim, table_width, tokens, n_q, n_kv, head_dim, write_cache;
    float eps;
};
struct KippQuantRead {
    void *k_out, *v_out;
    const void *k_codes, *k_scales, *v_codes, *v_scales;
    const int* list;                                    // pages
    int* status;
    void* stream;
    int out_dtype, bits, n_pages, page_size, n, n_kv, head_dim;
};
struct KippQuantReadEntries {
    void *k_out, *v_out;
    int* table_out;
    const void *k_codes, *k_scales, *v_codes, *v_scales;
    const int *q_start, *context_len, *block_table;
    int* status;
    void* factors;                                      // or null: float2 [entries of the step][n_kv]
    void* stream;
    int out_dtype, bits, n_pages, page_size, table_width, first_entry, entries, window, n_kv, head_dim;
};

// Norm, rotation and the write of a step's keys and values as codes; queries to q_out in the projection's type.
// write_cache 0: queries only.
extern "C" int kipp_quant_cache_write(const KippQuantWrite* a) {
    if (a->tokens <= 0) return 0;
    const QuantPages pages = {(uint8_t*)a->k_codes, (bf16*)a->k_scales, (uint8_t*)a->v_codes, (bf16*)a->v_scales, a->n_pages, a->page_size, a->n_kv};
    if (!pages_ok(pages, a->bits, a->head_dim) || a->n_q <= 0 || (a->q_norm_w == nullptr) != (a->k_norm_w == nullptr) || a->rotary_dim < 0 ||
        a->rotary_dim > a->head_dim || (a->rotary_dim & 1) || a->table_width <= 0 || a->status == nullptr ||
        a->ld_qkv < (long long)(a->n_q + 2 * a->n_kv) * a->head_dim)
        return KIPP_ERR_ARG;
    if (a->rotary_dim > 0 && ((uintptr_t)a->cos_sin & 7) != 0) return -3;              // (an angle's two numbers are one load)
    if ((a->dtype != KIPP_DT_F32 && a->dtype != KIPP_DT_BF16) || (a->norm_dtype != KIPP_DT_F32 && a->norm_dtype != KIPP_DT_BF16)) return KIPP_ERR_DTYPE;
    const WriteParams p = {a->qkv, a->ld_qkv, a->q_out, pages, a->q_norm_w, a->k_norm_w, a->norm_dtype, a->eps,
                           a->rotary_dim > 0 ? (const float2*)a->cos_sin : nullptr, a->rotary_dim, a->positions, a->entry_of_token,
                           a->block_table, a->table_width, a->tokens, a->n_q, a->head_dim, a->write_cache & 1, a->status};
    cudaStream_t s = (cudaStream_t)a->stream;
    if (a->dtype == KIPP_DT_F32) return a->bits == 4 ? launch_write<float, 4>(p, s) : launch_write<float, 8>(p, s);
    return a->bits == 4 ? launch_write<bf16, 4>(p, s) : launch_write<bf16, 8>(p, s);
}

static bool read_aligned(const QuantPages& g, const void* k_out, const void* v_out) {
    return (((uintptr_t)g.k_codes | (uintptr_t)g.v_codes) & 7) == 0 && (((uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0;
}

// k_out and v_out [n][n_kv][page_size][head_dim] of out_dtype: what pages list[0 .. n) stand for.  A
// negative number gives zeros.
extern "C" int kipp_quant_cache_read(const KippQuantRead* a) {
    if (a->n <= 0) return 0;
    const QuantPages pages = {(uint8_t*)a->k_codes, (bf16*)a->k_scales, (uint8_t*)a->v_codes, (bf16*)a->v_scales, a->n_pages, a->page_size, a->n_kv};
    if (!pages_ok(pages, a->bits, a->head_dim) || a->k_out == nullptr || a->v_out == nullptr || a->list == nullptr || a->status == nullptr)
        return KIPP_ERR_ARG;
    if (a->out_dtype != KIPP_DT_F32 && a->out_dtype != KIPP_DT_BF16) return KIPP_ERR_DTYPE;
    if (!read_aligned(pages, a->k_out, a->v_out)) return -3;
    ReadParams p = {a->k_out, a->v_out, pages, a->list, a->n, a->head_dim, a->status, nullptr, nullptr, nullptr, 0, 0, 0, 0, nullptr, 1};
    return launch_read<false>(p, a->bits, a->out_dtype, (cudaStream_t)a->stream);
}

// The pages that the tokens of entries first_entry .. first_entry + entries - 1 see, read back into pages of
// their own (entry by entry, table_width pages each), and the block table of those: table_out has the
// step's shape and only those entries' rows are written.  The pages no token sees are neither read nor
// written; their table entries are -1.  The slots that no token sees, of pages that some are seen of, become zeros: they may hold
// anything, and the attention over the pages multiplies them by weights of 0.
// With `factors` (heads of 64 and 128) the pages are float16, multiplied by the powers of two that it makes there, and the entries of one
// token, which the kernel over codes serves, count as bringing none.
extern "C" int kipp_quant_cache_read_entries(const KippQuantReadEntries* a) {
    if (a->entries <= 0) return 0;
    const QuantPages pages = {(uint8_t*)a->k_codes, (bf16*)a->k_scales, (uint8_t*)a->v_codes, (bf16*)a->v_scales, a->n_pages, a->page_size, a->n_kv};
    if (!pages_ok(pages, a->bits, a->head_dim) || a->k_out == nullptr || a->v_out == nullptr || a->table_out == nullptr || a->status == nullptr ||
        a->table_width <= 0 || a->first_entry < 0 || a->window < 0 || (long long)a->entries * a->table_width > 0x7fffffffLL)
        return KIPP_ERR_ARG;
    if (a->out_dtype != KIPP_DT_F32 && a->out_dtype != KIPP_DT_BF16) return KIPP_ERR_DTYPE;
    if (a->factors != nullptr && (a->out_dtype != KIPP_DT_BF16 || (a->head_dim != 64 && a->head_dim != 128))) return KIPP_ERR_ARG;
    if (!read_aligned(pages, a->k_out, a->v_out) || ((uintptr_t)a->factors & 7) != 0 ||
        (a->factors != nullptr && (((uintptr_t)a->k_scales | (uintptr_t)a->v_scales) & 3) != 0))
        return -3;
    ReadParams p = {a->k_out, a->v_out, pages, a->block_table, a->entries * a->table_width, a->head_dim, a->status, a->table_out, a->q_start,
                    a->context_len, a->table_width, a->first_entry, a->window, 0, (float2*)a->factors, a->factors != nullptr ? 2 : 1};
    return launch_read<true>(p, a->bits, a->out_dtype, (cudaStream_t)a->stream);
}
