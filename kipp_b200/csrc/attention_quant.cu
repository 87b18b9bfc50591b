// Attention over the quantised cache (quant_format.cuh) for single tokens and short portions, in
// bfloat16: codes go from memory to the tensor cores without ever being written out as numbers.
//
// For a key j and its group scales a[j, g], a query's score is
//     s_j = scale * sum_g a[j, g] * (sum_{c in g} q_c code[j, c]  -  L sum_{c in g} q_c)
// and the result, with weights p_j = exp(s_j - max) and value scales b[j, g],
//     o_c = sum_j (p_j b[j, g(c)]) code[j, c]  -  L sum_j p_j b[j, g(c)],      out = o / sum_j p_j
// so that both products run over bare codes; the scales multiply a score's parts (a number per key, query
// and group) and the weights, and the offset L costs one start value per query and group, and one more
// product of the weights with ones.
//
// A code is a bfloat16 operand as it stands: an integer n of up to 8 bits in the low bits of a 16-bit word
// is the number n * 2^-133 (subnormal up to 127; the exponent's first step goes on in the same line), and
// mma.sync takes subnormals exactly.  Two codes then become an operand register by one mask.  Four-bit
// codes in bits 4 to 7 count sixteenfold: their queries are divided by 16, the results at the end.  Queries
// and weights carry a factor of 2^48, all of these being powers of two: sums of weighted codes then end below float32's upper end with
// every value at the format's limit of 2^60 and every weight at 2^8 (2^48+8+57 a key), and a value of 2^-40 still leaves
// them whole; below, a key loses up to 2^-64 of a result.  A query has to be below 2^80 (beyond it counts as infinite).
//
// A weight is rounded once, to bfloat16 with its value's scale, as the tensor cores take it: it comes there as two bfloat16 words, its upper
// 16 bits and the upper 16 of what they leave, 2^-14 of it at most going lost, and one fused multiply-add rounds the sum of both products.  The
// normaliser sums the weights themselves.  (Rounded by itself first too, a word less: 2 to 3 % faster at 4 bits, level at 8; 8 tokens behind 8,100 keys at 4 bits
// then were off by 0.31 % of the result's norm, now 0.21, 0.16 of it the rounding of the result.)
//
// Products are made the other way round from the kernels of attention_mma.cu, keys (then channels) as
// rows, queries as columns, 8 at a time: mma.m16n8k16 with S^T = K Q^T, O^T = V^T P^T.  The codes are then the
// register operand, and a warp that serves the few queries of a kv head (the heads of its group times
// the tokens) wastes fewer columns.  P^T turns from result to operand by movmatrix.
//
// Up to four columns in 4 bits (the tokens of a decode step): a word of codes has a run of one group in its low half and of the next in its
// high half, and the two would have to be brought together with another word's before they can share a product.  Instead the
// four columns stand twice among the eight, with the first group's queries (weights) in one half of the inner dimension and the
// second's in the other, zeros elsewhere: a word is used as it is, both groups' sums come out of one product, and the accumulators
// are half as many.
//
// What bounds it: at 4 bits a warp executes some 600 instructions for 32 keys of 128 channels (what surrounds its steps counted in), and a
// lone warp needs over 2,000 cycles for them; with three warps a scheduler issue is half busy and the integer pipe 45 % of the time.  8 tokens
// behind 8,100 to 64,800 keys (32 query and 8 key heads) lie on a line of 8 us, the way in and out and the joining of the parts, and 5.3 TB/s: 23.0 us
// and 75 MB behind 8,100.  At 8 bits it is the memory (64 tokens behind 2,048: 55 us, 287 MB).
// Each warp works on its own 32 keys of a step of 128 with its own maximum, fetches its own rows, and meets the other three
// warps only at the end of a piece.  A maximum is raised only when a score passes it by 2^8.
//
// Rows come by cp.async into a ring per warp.  Where the page size is a multiple of 16, 16 keys of one kv head
// lie in one piece and a warp fetches them from one address (bulk copies, eight of 128 to 1,024 bytes for 32 keys,
// cost more: each takes its operands from uniform registers, some 20 instructions a copy); other page
// sizes go row by row.
//
// How the work is cut: every (entry, kv head, block of columns) is a row of steps of 128 keys; all rows
// one behind the other are dealt out in equal runs to one wave of CTAs, whatever the lengths.  A CTA may so
// have the end of one row, some whole ones and the start of another, and each of those costs it a
// queue that fills and drains and a sum over its warps: a row counts for some units more than it has steps.  Parts of a
// row go through scratch and are added in order by a second kernel.  Both make the cut from the step's lists, on
// the device, so a captured graph follows the lengths.
#include "quant_format.cuh"
#include <math.h>

namespace {

constexpr int WARPS = 4, THREADS = WARPS * 32;
constexpr int WARP_KEYS = 32, STEP = WARPS * WARP_KEYS;
constexpr int MOST_CTAS = 148 * 8, MOST_COLUMNS = 16;          // what the scratch has room for

struct Params {
    bf16* out; const bf16* q;
    const uint8_t* k_codes; const uint8_t* k_scales; const uint8_t* v_codes; const uint8_t* v_scales;
    const int* q_start; const int* context_len; const int* block_table;
    int entries, table_width, page_size, page_shift, n_pages, most, n_q, n_kv, group, window;
    float score_scale, query_scale;  // |scale| * log2(e) * 2^85; 2^48 with the scale's sign
    float* part_o; float* part_ml;   // [2 ctas][columns][D], [2 ctas][columns][2]
    // by CTA, the row that it begins and others go on with: (entry, kv head, 2 first column + the slot of its part, the row's last unit,
    // or -1: there is no such row); behind them the cut
    int4* shared;
    int ctas, most_blocks;           // most_blocks: rows of an entry of `most` tokens
    int* status;
};

constexpr int ROW_COST = 1;          // units of a row beside its steps

// One entry's share of the work.
struct Entry {
    int q_len, context, first_step, n_steps, column_blocks, blocks;
    __device__ __forceinline__ int row_units() const { return n_steps + ROW_COST; }
    __device__ __forceinline__ int units() const { return blocks * row_units(); }
};
template <int COLS> __device__ __forceinline__ Entry entry_of(const Params& p, int e) {
    Entry r;
    r.q_len = p.q_start[e + 1] - p.q_start[e];
    r.context = min(p.context_len[e], 0x7fffffff - max(r.q_len, 0));          // (far behind any table: reported, as all that is)
    if (r.q_len <= 0 || r.q_len > p.most || r.context < 0) { r.blocks = r.n_steps = r.column_blocks = 0; return r; }
    const int room = p.table_width * p.page_size;
    const int hi = min(r.context + r.q_len, room) - 1;
    const int lo = p.window > 0 ? max(0, r.context - p.window + 1) : 0;
    r.first_step = min(lo, hi) / STEP;
    r.n_steps = hi / STEP - r.first_step + 1;
    r.column_blocks = (r.q_len * p.group + COLS - 1) / COLS;
    r.blocks = r.column_blocks * p.n_kv;
    return r;
}

// The cut: the first `more` CTAs have `per` + 1 units, the others `per`; there are no more CTAs than units.
struct Cut {
    int ctas, per, more;
    Cut() = default;
    __device__ __forceinline__ Cut(int total, int most_ctas) : ctas(max(min(most_ctas, total), 1)) { per = total / ctas; more = total - per * ctas; }
    __device__ __forceinline__ int start(int cta) const { return per * cta + min(cta, more); }
    __device__ __forceinline__ int cta_of(int unit) const {
        const int first = more * (per + 1);
        return unit < first ? unit / (per + 1) : more + (unit - first) / per;
    }
};

// Where a unit is: the entry, and the units of it that lie before (entry -1: there is no such unit).  One warp, all lanes
// together; `total` comes out as well.  unit_of makes the unit looked for out of the cut (once the total is known).
struct Place { int entry, at; Cut cuts; };
template <int COLS, typename UnitOf> __device__ __forceinline__ Place find_unit(const Params& p, UnitOf unit_of) {
    const int lane = threadIdx.x & 31;
    auto scan = [&](int base, int& mine, int& before) {
        mine = base + lane < p.entries ? entry_of<COLS>(p, base + lane).units() : 0;
        int x = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        before = x - mine;
        return __shfl_sync(0xffffffffu, x, 31);
    };
    int mine, before;
    const int first_sum = scan(0, mine, before);
    int total = first_sum;
    for (int base = 32; base < p.entries; base += 32) {
        int m, b;
        total += scan(base, m, b);
    }
    Place r;
    r.cuts = Cut(total, p.ctas);
    r.entry = -1;
    r.at = 0;
    const int unit = unit_of(total, r.cuts);
    if (unit < 0 || unit >= total) return r;
    int base = 0, passed = 0, sum = first_sum;
    while (passed + sum <= unit) {
        passed += sum;
        base += 32;
        sum = scan(base, mine, before);
    }
    const unsigned here = __ballot_sync(0xffffffffu, passed + before <= unit && unit < passed + before + mine);
    const int who = __ffs(here) - 1;
    r.entry = base + who;
    r.at = unit - passed - __shfl_sync(0xffffffffu, before, who);
    return r;
}

// d = a b + c
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, float c0,
                                    float c1, float c2, float c3) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    mma(c, a0, a1, a2, a3, b0, b1, c[0], c[1], c[2], c[3]);
}
__device__ __forceinline__ uint32_t times2(uint32_t a, uint32_t rest, uint32_t b) {  // two products (a + rest) b, rounded to bfloat16 once
    const __nv_bfloat162 f = *reinterpret_cast<const __nv_bfloat162*>(&b);
    const __nv_bfloat162 v = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&a), f, __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&rest), f));
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float low_f32(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_f32(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ void cp_async_row(uint32_t dst, const void* src, int bytes, int kept) {
    if (bytes == 16) asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(kept) : "memory");
    else if (bytes == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(kept) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(kept) : "memory");
}
template <int BYTES> __device__ __forceinline__ void take(uint32_t (&w)[BYTES / 4], const uint8_t* p) {
    if constexpr (BYTES == 4) w[0] = *reinterpret_cast<const uint32_t*>(p);
    else if constexpr (BYTES == 8) { const uint2 v = *reinterpret_cast<const uint2*>(p); w[0] = v.x; w[1] = v.y; }
    else {
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i) {
            const uint4 v = reinterpret_cast<const uint4*>(p)[i];
            w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
        }
    }
}

template <int D, int BITS> struct Shape {
    static constexpr int G = D / 32;                         // groups
    static constexpr int RB = D * BITS / 8;                  // bytes of a row of codes
    static constexpr int SB = 2 * G;                         // bytes of its scales
    static constexpr int CHUNKS = RB / 16;
    static constexpr int K_BYTES = RB / 4, V_BYTES = RB / 8; // a lane's stretch of a key's row and of a value's
    static constexpr int WARP_STAGE = WARP_KEYS * 2 * (RB + SB);
    // Steps in the ring, and CTAs an SM (ctas_per_sm).  Heads of 128: three CTAs of 168 registers a thread and four steps (at 4 bits four CTAs
    // of 128 registers and three steps took 9 % longer in 8 columns, 1 % in 4).  A step's scores made beside the one before's values, two
    // streams of instructions, gave nothing.
    static constexpr int STAGES = RB == 128 && D == 128 ? 2 : D == 256 ? 3 : 4;
    static constexpr float L = BITS == 4 ? 8.f : 128.f;
};
// NT: tiles of 8 columns, or 0: four columns (4 bits only), each of them twice, for the two groups whose runs share a word.
constexpr int columns_of_tiles(int nt) { return nt == 0 ? 4 : 8 * nt; }
template <int D, int NT> constexpr int q_bytes() { return NT == 0 ? (D / 64) * 32 * 40 : NT * (D / 32) * 32 * 24; }  // a piece's queries as operands
template <int D, int BITS, int NT> constexpr bool q_in_ring() { return q_bytes<D, NT>() <= Shape<D, BITS>::WARP_STAGE; }
template <int D, int BITS, int NT> constexpr int ctas_per_sm() {
    return D == 256 ? (BITS == 4 ? 2 : 1) : NT == 2 ? (D == 64 ? 3 : 2) : D == 128 ? 3 : 4;
}

// Row r of the products (S^T's rows, P^T's and V's inner dimension) is key 4 (2 h + e) + t of a tile of 16, for
// r = 2 t + e + 8 h: a lane (g, t) then meets the values of keys t, 4 + t, 8 + t, 12 + t.
__device__ __forceinline__ int key_of_row(int r) { return 4 * (r & 1) + ((r & 7) >> 1) + (r & 8); }

// Two runs of four codes of a key as four operand registers, two channels of one group in each.  4 bits: `first` and `second` are words,
// `half` which half of them the run is; x[i] has code i of the first run in its low half and of the second in its high half, codes
// 1 and 3 sixteenfold.  8 bits: a run is a word, and has codes 0 and 2, 1 and 3 in the halves of x[0], x[1] (x[2], x[3] the second).
template <int BITS> __device__ __forceinline__ void spread_keys(uint32_t (&x)[4], uint32_t first, uint32_t second, int half) {
    if constexpr (BITS == 4) {
        const uint32_t w = __byte_perm(first, second, half ? 0x7632 : 0x5410), u = w >> 8;
        x[0] = w & 0x000f000fu; x[1] = w & 0x00f000f0u; x[2] = u & 0x000f000fu; x[3] = u & 0x00f000f0u;
    } else {
        x[0] = first & 0x00ff00ffu; x[1] = __byte_perm(first, 0u, 0x4341); x[2] = second & 0x00ff00ffu; x[3] = __byte_perm(second, 0u, 0x4341);
    }
}
// A word of 4-bit codes, a run of two groups: code i of the first group's in the low half of x[i], of the second's in the high half.
__device__ __forceinline__ void spread_word(uint32_t (&x)[4], uint32_t w) {
    const uint32_t u = w >> 8;
    x[0] = w & 0x000f000fu; x[1] = w & 0x00f000f0u; x[2] = u & 0x000f000fu; x[3] = u & 0x00f000f0u;
}
// A run of two values, the first one's codes in the low halves.  (4 bits: x[0] and x[2] could keep both codes of a byte and the even
// channels' sums be made as differences at the end, an instruction in six less and 2 % of the time; but they would then not
// cancel exactly where every value is 0.)
template <int BITS> __device__ __forceinline__ void spread_values(uint32_t (&x)[4], uint32_t first, uint32_t second, int half) {
    if constexpr (BITS == 4) {
        spread_keys<4>(x, first, second, half);
    } else {
        const uint32_t w = __byte_perm(first, second, 0x5410), u = __byte_perm(first, second, 0x7632);
        x[0] = w & 0x00ff00ffu; x[1] = __byte_perm(w, 0u, 0x4341); x[2] = u & 0x00ff00ffu; x[3] = __byte_perm(u, 0u, 0x4341);
    }
}

// TILES: the page size is a multiple of 16.
template <int D, int BITS, int NT, bool TILES>
__global__ void __launch_bounds__(THREADS, ctas_per_sm<D, BITS, NT>()) attn_quant_kernel(const Params p) {
    using S = Shape<D, BITS>;
    constexpr int G = S::G, RB = S::RB, SB = S::SB, COLS = columns_of_tiles(NT), WO = D + 4, STAGES = S::STAGES;
    constexpr bool FOUR = NT == 0;
    constexpr int T = FOUR ? 1 : NT, PAIRS = G / 2, SETS = FOUR ? PAIRS : G;       // operand sets: a pair of groups, or a group
    static_assert(!FOUR || BITS == 4, "two groups share a word in 4 bits only");
    constexpr int RING = WARPS * STAGES * S::WARP_STAGE;
    constexpr bool Q_IN_RING = q_in_ring<D, BITS, NT>();
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Place place;
    __shared__ float part_f[WARPS][COLS];
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g4 = lane >> 2, t4 = lane & 3;
    const int group = p.group;

    // -- the run of this CTA: from the step's lists, which may be read before the wait
    if (warp == 0) {
        const Place found = find_unit<COLS>(p, [&](int total, const Cut& c) { return (int)blockIdx.x < c.ctas && total > 0 ? c.start(blockIdx.x) : -1; });
        if (lane == 0) place = found;
    }
    __syncthreads();
    int entry = place.entry, at = place.at;
    pdl_wait();
    if (threadIdx.x == 0 && p.shared != nullptr) {
        p.shared[blockIdx.x] = make_int4(0, 0, 0, -1);
        if (blockIdx.x == 0) p.shared[p.ctas] = make_int4(place.cuts.ctas, place.cuts.per, place.cuts.more, 0);
    }
    if (entry < 0) return;
    const int run_first = place.cuts.start(blockIdx.x), run_end = place.cuts.start(blockIdx.x + 1);

    uint8_t* const my = smem + warp * (STAGES * S::WARP_STAGE);
    const uint32_t my_s = smem_address(my);
    constexpr int V_AT = WARP_KEYS * RB, KS_AT = 2 * WARP_KEYS * RB, VS_AT = KS_AT + WARP_KEYS * SB;
    // a lane's 16 bytes of a tile's keys, values and scales (the first SB lanes those of the keys, the next SB of the values)
    const uint8_t *const k_lane = p.k_codes + lane * 16, *const v_lane = p.v_codes + lane * 16;
    const uint8_t* const s_lane = lane < SB ? p.k_scales + lane * 16 : p.v_scales + (lane - SB) * 16;
    const int s_to = lane < SB ? KS_AT : VS_AT - 16 * SB;
    int stage = 0;

    for (int x = run_first; x < run_end;) {
        Entry en = entry_of<COLS>(p, entry);
        while (at >= en.units()) { at -= en.units(); en = entry_of<COLS>(p, ++entry); }
        const int block = at / en.row_units(), unit = at - block * en.row_units(), units = min(run_end - x, en.row_units() - unit);
        const int from = max(unit - ROW_COST, 0), n = unit + units - ROW_COST - from;      // steps of the row
        const int slot = 2 * blockIdx.x + (x == run_first ? 0 : 1);
        x += units;
        at += units;
        if (n <= 0) continue;
        const int g = block / en.column_blocks, column0 = (block - g * en.column_blocks) * COLS;
        const int qs = p.q_start[entry], columns = en.q_len * group;
        const int* table = p.block_table + (size_t)entry * p.table_width;
        // the keys that this block's columns see, and what this lane's columns see of them
        const int tok0 = column0 / group, tok1 = min(column0 + COLS - 1, columns - 1) / group;
        const int see_hi = min(en.context + tok1, p.table_width * p.page_size - 1);
        const int see_lo = p.window > 0 ? max(0, en.context + tok0 - p.window + 1) : 0;
        // keys all columns see (a table that ends before a token's position is reported)
        if (en.context + tok1 > see_hi && threadIdx.x == 0) atomicExch(p.status, 3);
        const int all_hi = min(en.context + tok0, see_hi), all_lo = p.window > 0 ? max(0, en.context + tok1 - p.window + 1) : 0;
        const int j_first = (en.first_step + from) * STEP + warp * WARP_KEYS;

        // the row of pages that holds key j (TILES: key j and the 15 behind it); -1: none of it is seen
        auto row_of = [&](int j) {
            int row = -1;
            if (j + (TILES ? 15 : 0) >= see_lo && j <= see_hi) {
                const int slot = p.page_shift >= 0 ? j >> p.page_shift : j / p.page_size;
                const int page = table[slot];
                if (page >= 0 && page < p.n_pages) row = (page * p.n_kv + g) * p.page_size + (j - slot * p.page_size);
                else atomicExch(p.status, 3);
            }
            return row;
        };
        // TILES: the rows of the tiles of 16 steps are looked up at once, a tile a lane, and a batch ahead; otherwise each lane's
        // own key, a step ahead.  (A tile that is not there has scales of 0; its codes are whatever lies in the ring.)
        int rows = -1, rows_next;
        auto look_up = [&](int step) {
            if constexpr (TILES) rows_next = row_of(j_first + (step + (lane >> 1)) * STEP + (lane & 1) * 16);
            else rows_next = row_of(j_first + step * STEP + lane);
        };
        auto fetch = [&](int step, int to_stage) {
            const uint32_t to = my_s + to_stage * S::WARP_STAGE;
            if constexpr (TILES) {
                if ((step & 15) == 0) {
                    rows = rows_next;
                    if (step + 16 < n) look_up(step + 16);
                }
#pragma unroll
                for (int tile = 0; tile < 2; ++tile) {
                    const int row = __shfl_sync(0xffffffffu, rows, 2 * (step & 15) + tile);
                    if (row < 0) {
                        if (lane < 2 * SB) *reinterpret_cast<uint4*>(my + to_stage * S::WARP_STAGE + lane * 16 + s_to + tile * 16 * SB) = make_uint4(0u, 0u, 0u, 0u);
                        continue;
                    }
                    const uint8_t *k = k_lane + (size_t)row * RB, *v = v_lane + (size_t)row * RB;
#pragma unroll
                    for (int i = 0; i < RB / 32; ++i) {
                        cp_async16(to + lane * 16 + tile * 16 * RB + i * 512, k + i * 512, 16);
                        cp_async16(to + lane * 16 + V_AT + tile * 16 * RB + i * 512, v + i * 512, 16);
                    }
                    if (lane < 2 * SB) cp_async16(to + lane * 16 + s_to + tile * 16 * SB, s_lane + (size_t)row * SB, 16);
                }
            } else {
                const int row = rows_next;
                if (step + 1 < n) look_up(step + 1);
                constexpr int ROWS = 32 / S::CHUNKS;               // rows of a pass
                const int c = lane % S::CHUNKS;
#pragma unroll
                for (int i = 0; i < S::CHUNKS; ++i) {
                    const int key = i * ROWS + lane / S::CHUNKS, src = __shfl_sync(0xffffffffu, row, key);
                    const size_t off = (size_t)max(src, 0) * RB + c * 16;
                    cp_async16(to + key * RB + c * 16, p.k_codes + off, src >= 0 ? 16 : 0);
                    cp_async16(to + V_AT + key * RB + c * 16, p.v_codes + off, src >= 0 ? 16 : 0);
                }
                const size_t off = (size_t)max(row, 0) * SB;
                cp_async_row(to + KS_AT + lane * SB, p.k_scales + off, SB, row >= 0 ? SB : 0);
                cp_async_row(to + VS_AT + lane * SB, p.v_scales + off, SB, row >= 0 ? SB : 0);
            }
        };
        look_up(0);
        // -- the queries are asked for first: a warp makes operands of every fourth group's
        constexpr int MINE = (T * SETS + WARPS - 1) / WARPS;
        uint2 q_raw[MINE][2];
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
            const int k = warp + i * WARPS, c = column0 + (FOUR ? g4 & 3 : k / G * 8 + g4);
            q_raw[i][0] = q_raw[i][1] = make_uint2(0u, 0u);
            if (k < T * SETS && c < columns) {
                const int tok = c / group, run = FOUR ? 2 * k + (g4 >> 2) : k % G;
                const bf16* src = p.q + ((size_t)(qs + tok) * p.n_q + g * group + (c - tok * group)) * D + t4 * (D / 4) + 4 * run;
                q_raw[i][0] = *reinterpret_cast<const uint2*>(src);
                q_raw[i][1] = *reinterpret_cast<const uint2*>(src + 4 * G);
            }
        }
#pragma unroll
        for (int s = 0; s < STAGES - 1; ++s) {
            if (s < n) fetch(s, (stage + s) % STAGES);
            cp_async_commit();
        }

        // -- as operands, with what the offset of their codes comes to (through the first warp's free stage, where they have room)
        uint4* const q_operands = reinterpret_cast<uint4*>(Q_IN_RING ? smem + (stage + STAGES - 1) % STAGES * S::WARP_STAGE : smem + RING);
        float2* const q_offsets = reinterpret_cast<float2*>(q_operands + (FOUR ? 2 * PAIRS : NT * G) * 32);
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
            const int k = warp + i * WARPS;
            if (k >= T * SETS) break;
            const uint2 a = q_raw[i][0], b = q_raw[i][1];
            float sum = (low_f32(a.x) + high_f32(a.x)) + (low_f32(a.y) + high_f32(a.y)) + (low_f32(b.x) + high_f32(b.x)) + (low_f32(b.y) + high_f32(b.y));
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            sum *= -S::L * 0x1p-133f * p.query_scale;
            q_offsets[k * 32 + lane] = make_float2(__shfl_sync(0xffffffffu, sum, 8 * t4), __shfl_sync(0xffffffffu, sum, 8 * t4 + 4));
            if constexpr (FOUR) {
                // code 0 .. 3 of the lane's run, in the half of the register that the run's codes come in
                const uint2 run[2] = {a, b};
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    uint32_t w[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const uint32_t pair = c < 2 ? run[n].x : run[n].y;
                        const float f = (c & 1 ? high_f32(pair) * 0.0625f : low_f32(pair)) * p.query_scale;
                        w[c] = g4 < 4 ? pack2(f, 0.f) : pack2(0.f, f);
                    }
                    q_operands[(2 * k + n) * 32 + lane] = make_uint4(w[0], w[1], w[2], w[3]);
                }
                continue;
            }
            const uint32_t mid = BITS == 4 ? b.x : a.y, last = BITS == 4 ? a.y : b.x;              // (as spread_keys pairs the codes)
            const uint32_t raw[4] = {__byte_perm(a.x, mid, 0x5410), __byte_perm(a.x, mid, 0x7632), __byte_perm(last, b.y, 0x5410),
                                     __byte_perm(last, b.y, 0x7632)};
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float f = BITS == 4 && (i & 1) ? p.query_scale * 0.0625f : p.query_scale;
                w[i] = pack2(low_f32(raw[i]) * f, high_f32(raw[i]) * f);
            }
            q_operands[k * 32 + lane] = make_uint4(w[0], w[1], w[2], w[3]);
        }
        __syncthreads();
        uint32_t qf[T][G][4];
        float offset[T][SETS][2];
#pragma unroll
        for (int nt = 0; nt < T; ++nt) {
#pragma unroll
            for (int gi = 0; gi < G; ++gi) {
                const uint4 w = q_operands[(nt * G + gi) * 32 + lane];
                qf[nt][gi][0] = w.x; qf[nt][gi][1] = w.y; qf[nt][gi][2] = w.z; qf[nt][gi][3] = w.w;
            }
#pragma unroll
            for (int k = 0; k < SETS; ++k) {
                const float2 f = q_offsets[(nt * SETS + k) * 32 + lane];
                offset[nt][k][0] = f.x; offset[nt][k][1] = f.y;
            }
        }
        if constexpr (Q_IN_RING) __syncthreads();

        float o[T][2 * SETS][4], ones[T][4], m[T][2], l[T][2];
#pragma unroll
        for (int nt = 0; nt < T; ++nt) {
#pragma unroll
            for (int i = 0; i < 2 * SETS; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[nt][i][k] = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) ones[nt][k] = 0.f;
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
        }

        float s[T][2][4];                                     // scores of a step, to be multiplied by score_scale for units of log2
        uint32_t w[T][2][2], rest[T][2][2];                   // its weights as operands: the upper 16 bits, and what those leave
        // The rows of a step that no column sees may hold anything: their scales become 0 (their codes are numbers anyhow).
        auto arrived = [&](int j0, uint8_t* tile) {
            const int j = j0 + lane;
            if (j > see_hi || j < see_lo) {
#pragma unroll
                for (int k = 0; k < SB / 4; ++k) {
                    *reinterpret_cast<uint32_t*>(tile + KS_AT + lane * SB + 4 * k) = 0u;
                    *reinterpret_cast<uint32_t*>(tile + VS_AT + lane * SB + 4 * k) = 0u;
                }
            }
            __syncwarp();
        };
        auto scores = [&](const uint8_t* tile) {
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
                uint32_t w0[S::K_BYTES / 4], w1[S::K_BYTES / 4];
                const uint8_t* r0 = tile + (mt * 16 + key_of_row(g4)) * RB + t4 * S::K_BYTES;
                take<S::K_BYTES>(w0, r0);
                take<S::K_BYTES>(w1, r0 + 8 * RB);
                uint32_t a0[SB / 4], a1[SB / 4];
                take<SB>(a0, tile + KS_AT + (mt * 16 + key_of_row(g4)) * SB);
                take<SB>(a1, tile + KS_AT + (mt * 16 + key_of_row(g4) + 8) * SB);
#pragma unroll
                for (int nt = 0; nt < T; ++nt) s[nt][mt][0] = s[nt][mt][1] = s[nt][mt][2] = s[nt][mt][3] = 0.f;
                if constexpr (FOUR) {
                    const uint32_t half = t4 < 2 ? 0x1044 : 0x3244;        // this lane's columns are of the first or the second group
#pragma unroll
                    for (int k = 0; k < PAIRS; ++k) {
                        float c[4];
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            const int at = k + n * PAIRS;
                            uint32_t x0[4], x1[4];
                            spread_word(x0, w0[at]);
                            spread_word(x1, w1[at]);
                            if (n == 0) mma(c, x0[0], x1[0], x0[1], x1[1], qf[0][2 * k][0], qf[0][2 * k][1], offset[0][k][0], offset[0][k][1],
                                            offset[0][k][0], offset[0][k][1]);
                            else mma(c, x0[0], x1[0], x0[1], x1[1], qf[0][2 * k + 1][0], qf[0][2 * k + 1][1]);
                            mma(c, x0[2], x1[2], x0[3], x1[3], qf[0][2 * k + n][2], qf[0][2 * k + n][3]);
                        }
                        const float f0 = __uint_as_float(__byte_perm(a0[k], 0u, half)), f1 = __uint_as_float(__byte_perm(a1[k], 0u, half));
                        s[0][mt][0] = fmaf(f0, c[0], s[0][mt][0]);
                        s[0][mt][1] = fmaf(f0, c[1], s[0][mt][1]);
                        s[0][mt][2] = fmaf(f1, c[2], s[0][mt][2]);
                        s[0][mt][3] = fmaf(f1, c[3], s[0][mt][3]);
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) s[0][mt][k] += __shfl_xor_sync(0xffffffffu, s[0][mt][k], 2);
                } else {
#pragma unroll
                    for (int gi = 0; gi < G; ++gi) {
                        uint32_t x0[4], x1[4];
                        constexpr int W = BITS == 4 ? 1 : 0;
                        spread_keys<BITS>(x0, w0[gi >> W], w0[(gi + G) >> W], gi & 1);
                        spread_keys<BITS>(x1, w1[gi >> W], w1[(gi + G) >> W], gi & 1);
                        const float f0 = gi & 1 ? high_f32(a0[gi >> 1]) : low_f32(a0[gi >> 1]);
                        const float f1 = gi & 1 ? high_f32(a1[gi >> 1]) : low_f32(a1[gi >> 1]);
#pragma unroll
                        for (int nt = 0; nt < T; ++nt) {
                            float c[4];
                            mma(c, x0[0], x1[0], x0[1], x1[1], qf[nt][gi][0], qf[nt][gi][1], offset[nt][gi][0], offset[nt][gi][1],
                                offset[nt][gi][0], offset[nt][gi][1]);
                            mma(c, x0[2], x1[2], x0[3], x1[3], qf[nt][gi][2], qf[nt][gi][3]);
                            s[nt][mt][0] = fmaf(f0, c[0], s[nt][mt][0]);
                            s[nt][mt][1] = fmaf(f0, c[1], s[nt][mt][1]);
                            s[nt][mt][2] = fmaf(f1, c[2], s[nt][mt][2]);
                            s[nt][mt][3] = fmaf(f1, c[3], s[nt][mt][3]);
                        }
                    }
                }
            }
        };
        auto weights = [&](int j0, bool cut) {
            bool raise = false;
            float top[T][2];
#pragma unroll
            for (int nt = 0; nt < T; ++nt) {
                if (cut) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int pos = en.context + min(column0 + (FOUR ? (2 * t4 + c) & 3 : nt * 8 + 2 * t4 + c), columns - 1) / group;
                        const int hi = min(pos, see_hi), lo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
#pragma unroll
                        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const int j = j0 + mt * 16 + key_of_row(g4) + h * 8;
                                if (j > hi || j < lo) s[nt][mt][2 * h + c] = -INFINITY;
                            }
                    }
                }
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    top[nt][c] = fmaxf(fmaxf(s[nt][0][c], s[nt][0][2 + c]), fmaxf(s[nt][1][c], s[nt][1][2 + c])) * p.score_scale;
                    raise |= top[nt][c] > m[nt][c] + 8.f;
                }
            }
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int nt = 0; nt < T; ++nt) {
                    float f[2];
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float mx = fmaxf(m[nt][c], top[nt][c]);
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        f[c] = m[nt][c] == -INFINITY ? 0.f : exp2_fast(m[nt][c] - mx);
                        m[nt][c] = mx;
                        l[nt][c] *= f[c];
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        ones[nt][k] *= f[k & 1];
#pragma unroll
                        for (int d = 0; d < 2 * SETS; ++d) o[nt][d][k] *= f[k & 1];
                    }
                }
            }
            // (times 2^48)
#pragma unroll
            for (int nt = 0; nt < T; ++nt) {
                const float back[2] = {(m[nt][0] == -INFINITY ? 0.f : m[nt][0]) - 48.f, (m[nt][1] == -INFINITY ? 0.f : m[nt][1]) - 48.f};
#pragma unroll
                for (int mt = 0; mt < 2; ++mt) {
                    float e[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        e[k] = exp2_fast(fmaf(s[nt][mt][k], p.score_scale, -back[k & 1]));
                        l[nt][k & 1] += e[k];
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t e0 = __float_as_uint(e[2 * h]), e1 = __float_as_uint(e[2 * h + 1]);
                        w[nt][mt][h] = transposed(__byte_perm(e0, e1, 0x7632));
                        rest[nt][mt][h] = transposed(__byte_perm(__float_as_uint(e[2 * h] - high_f32(e0)),
                                                                 __float_as_uint(e[2 * h + 1] - high_f32(e1)), 0x7632));
                    }
                }
            }
        };
        auto add_values = [&](const uint8_t* tile) {
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
                uint32_t v[4][S::V_BYTES / 4], f[4][SB / 4];           // keys t, 4 + t, 8 + t, 12 + t
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    take<S::V_BYTES>(v[k], tile + V_AT + (mt * 16 + 4 * k + t4) * RB + g4 * S::V_BYTES);
                    take<SB>(f[k], tile + VS_AT + (mt * 16 + 4 * k + t4) * SB);
                }
                if constexpr (FOUR) {
                    // a key's weight in the low half for the first group's columns, in the high half for the second's
                    const uint32_t even = g4 < 4 ? 0x4410 : 0x1044, odd = g4 < 4 ? 0x4432 : 0x3244;
                    const uint32_t one_key[4] = {__byte_perm(w[0][mt][0], 0u, even), __byte_perm(w[0][mt][0], 0u, odd),
                                                 __byte_perm(w[0][mt][1], 0u, even), __byte_perm(w[0][mt][1], 0u, odd)};
                    const uint32_t its_rest[4] = {__byte_perm(rest[0][mt][0], 0u, even), __byte_perm(rest[0][mt][0], 0u, odd),
                                                  __byte_perm(rest[0][mt][1], 0u, even), __byte_perm(rest[0][mt][1], 0u, odd)};
#pragma unroll
                    for (int k = 0; k < PAIRS; ++k) {
                        const uint32_t one = g4 == k ? 0x3f803f80u : 0u;
#pragma unroll
                        for (int n = 0; n < 4; n += 2) {
                            uint32_t x0[4], x1[4];
                            spread_word(x0, v[n][k]);
                            spread_word(x1, v[n + 1][k]);
                            const uint32_t b0 = times2(one_key[n], its_rest[n], f[n][k]), b1 = times2(one_key[n + 1], its_rest[n + 1], f[n + 1][k]);
                            mma(o[0][2 * k], x0[0], x0[1], x1[0], x1[1], b0, b1);
                            mma(o[0][2 * k + 1], x0[2], x0[3], x1[2], x1[3], b0, b1);
                            mma(ones[0], one, 0u, one, 0u, b0, b1);
                        }
                    }
                } else {
#pragma unroll
                    for (int gi = 0; gi < G; ++gi) {
                        uint32_t x0[4], x1[4];                             // keys of the first and the second half of the rows
                        constexpr int W = BITS == 4 ? 1 : 0;
                        spread_values<BITS>(x0, v[0][gi >> W], v[1][gi >> W], gi & 1);
                        spread_values<BITS>(x1, v[2][gi >> W], v[3][gi >> W], gi & 1);
                        const uint32_t f0 = __byte_perm(f[0][gi >> 1], f[1][gi >> 1], gi & 1 ? 0x7632 : 0x5410);
                        const uint32_t f1 = __byte_perm(f[2][gi >> 1], f[3][gi >> 1], gi & 1 ? 0x7632 : 0x5410);
                        const uint32_t one = g4 == gi ? 0x3f803f80u : 0u;
#pragma unroll
                        for (int nt = 0; nt < T; ++nt) {
                            const uint32_t b0 = times2(w[nt][mt][0], rest[nt][mt][0], f0), b1 = times2(w[nt][mt][1], rest[nt][mt][1], f1);
                            mma(o[nt][2 * gi], x0[0], x0[1], x1[0], x1[1], b0, b1);
                            mma(o[nt][2 * gi + 1], x0[2], x0[3], x1[2], x1[3], b0, b1);
                            mma(ones[nt], one, 0u, one, 0u, b0, b1);
                        }
                    }
                }
            }
        };
        for (int i = 0; i < n; ++i) {
            if (i + STAGES - 1 < n) fetch(i + STAGES - 1, stage == 0 ? STAGES - 1 : stage - 1);
            cp_async_commit();
            cp_async_wait<STAGES - 1>();
            __syncwarp();
            uint8_t* const tile = my + stage * S::WARP_STAGE;
            const int j0 = j_first + i * STEP;
            // (the warps of a step may all be outside what is seen, but for one)
            if (j0 <= see_hi && j0 + WARP_KEYS > see_lo) {
                const bool cut = j0 + WARP_KEYS - 1 > all_hi || j0 < all_lo;
                if (cut) arrived(j0, tile);
                scores(tile);
                weights(j0, cut);
                add_values(tile);
            }
            __syncwarp();
            stage = stage + 1 == STAGES ? 0 : stage + 1;
        }
        cp_async_wait<0>();

        // -- the four warps' parts together, through shared memory
        __syncthreads();
        float* w_m = reinterpret_cast<float*>(smem);                   // [WARPS][COLS]
        float* w_l = w_m + WARPS * COLS;                               // [WARPS][COLS]
        float* w_o = w_l + WARPS * COLS;                               // [WARPS][COLS][WO]
#pragma unroll
        for (int nt = 0; nt < T; ++nt) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float sum = l[nt][c];
                sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                const int col = FOUR ? (2 * t4 + c) & 3 : nt * 8 + 2 * t4 + c;
                if (g4 == 0) {
                    w_m[warp * COLS + col] = m[nt][c];
                    w_l[warp * COLS + col] = sum * 0x1p-48f;
                }
            }
#pragma unroll
            for (int gi = 0; gi < SETS; ++gi) {
                // (row gi of the product with ones lies with lane 4 gi + t)
                const float less[2] = {__shfl_sync(0xffffffffu, ones[nt][0], 4 * gi + t4) * (S::L * 0x1p-48f),
                                       __shfl_sync(0xffffffffu, ones[nt][1], 4 * gi + t4) * (S::L * 0x1p-48f)};
                constexpr float EVEN = 0x1p85f, ODD = BITS == 4 ? 0x1p81f : 0x1p85f;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float4 r;
                    r.x = fmaf(o[nt][2 * gi][c], EVEN, -less[c]);
                    r.y = fmaf(o[nt][2 * gi][2 + c], ODD, -less[c]);
                    r.z = fmaf(o[nt][2 * gi + 1][c], EVEN, -less[c]);
                    r.w = fmaf(o[nt][2 * gi + 1][2 + c], ODD, -less[c]);
                    const int col = FOUR ? (2 * t4 + c) & 3 : nt * 8 + 2 * t4 + c, run = FOUR ? 2 * gi + (t4 >> 1) : gi;
                    *reinterpret_cast<float4*>(w_o + (size_t)(warp * COLS + col) * WO + g4 * (D / 8) + 4 * run) = r;
                }
            }
        }
        __syncthreads();
        const bool whole = n == en.n_steps;
        const int live = min(COLS, columns - column0);
        if (threadIdx.x < COLS) {
            const int col = threadIdx.x;
            float mx = -INFINITY, sum = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) mx = fmaxf(mx, w_m[w * COLS + col]);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float wm = w_m[w * COLS + col], f = wm == -INFINITY ? 0.f : exp2_fast(wm - mx);
                sum += w_l[w * COLS + col] * f;
                part_f[w][col] = f;
            }
            if (whole) {
#pragma unroll
                for (int w = 0; w < WARPS; ++w) part_f[w][col] = sum == 0.f ? 0.f : part_f[w][col] / sum;
            } else if (col < live) {
                *reinterpret_cast<float2*>(p.part_ml + ((size_t)slot * COLS + col) * 2) = make_float2(mx, sum);
            }
        }
        if (threadIdx.x == THREADS - 1 && p.shared != nullptr && from == 0 && !whole)
            p.shared[blockIdx.x] = make_int4(entry, g, 2 * column0 + (slot & 1), x - 1 + en.n_steps - n);
        __syncthreads();
        for (int i = threadIdx.x * 4; i < live * D; i += THREADS * 4) {
            const int col = i / D, d = i % D;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float f = part_f[w][col];
                const float4 r = *reinterpret_cast<const float4*>(w_o + (size_t)(w * COLS + col) * WO + d);
                acc.x = fmaf(r.x, f, acc.x); acc.y = fmaf(r.y, f, acc.y); acc.z = fmaf(r.z, f, acc.z); acc.w = fmaf(r.w, f, acc.w);
            }
            if (whole) {
                const int c = column0 + col, tok = c / group;
                *reinterpret_cast<uint2*>(p.out + ((size_t)(qs + tok) * p.n_q + g * group + (c - tok * group)) * D + d) =
                    make_uint2(pack2(acc.x, acc.y), pack2(acc.z, acc.w));
            } else {
                *reinterpret_cast<float4*>(p.part_o + ((size_t)slot * COLS + col) * D + d) = acc;
            }
        }
        __syncthreads();
    }
}

// One warp adds the parts first, first + step, .. of a column: D / 32 values a lane and the weights' sum, both of the parts' largest
// maximum `mx`.  A sum of 0 is a row that sees nothing, and gives zeros; one that is no number stays that.  `index` gives the place of a part.  (A batch of parts is on its way at once.  One token behind 60,000 keys, 2 rows of 222
// parts: 11.6 us in all; with a scan of all maxima before them 14.4.)
template <int D, typename Index>
__device__ __forceinline__ void add_parts(const Params& p, int first, int step, int parts, Index index, float (&acc)[D / 32], float& sum, float& mx) {
    constexpr int PER = D / 32, BATCH = 8;
    const int lane = threadIdx.x & 31;
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml);
    mx = -INFINITY;
    sum = 0.f;
#pragma unroll
    for (int k = 0; k < PER; ++k) acc[k] = 0.f;
    for (; first < parts; first += step * BATCH) {
        float r[BATCH][PER];
        float2 f[BATCH];
        float top = mx;
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int part = first + i * step;
            f[i] = make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int k = 0; k < PER; ++k) r[i][k] = 0.f;
            if (part < parts) {
                f[i] = ml[index(part)];
#pragma unroll
                for (int k = 0; k < PER; ++k) r[i][k] = p.part_o[index(part) * D + k * 32 + lane];
            }
        }
#pragma unroll
        for (int i = 0; i < BATCH; ++i) top = fmaxf(top, f[i].x);
        const float before = mx == -INFINITY ? 0.f : exp2_fast(mx - top);
        mx = top;
        sum *= before;
#pragma unroll
        for (int k = 0; k < PER; ++k) acc[k] *= before;
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const float w = f[i].x == -INFINITY ? 0.f : exp2_fast(f[i].x - mx);
            sum = fmaf(f[i].y, w, sum);
#pragma unroll
            for (int k = 0; k < PER; ++k) acc[k] = fmaf(r[i][k], w, acc[k]);
        }
    }
}
template <int D> __device__ __forceinline__ bf16* result_of(const Params& p, int e, int g, int c) {
    const int tok = c / p.group;
    return p.out + ((size_t)(p.q_start[e] + tok) * p.n_q + g * p.group + (c - tok * p.group)) * D;
}

// Adds the parts of the row that CTA x of the first kernel began, in the order of the keys: a warp a column.
constexpr int JOIN_WARPS = 4;
template <int D, int NT>
__global__ void __launch_bounds__(JOIN_WARPS * 32) attn_quant_join_kernel(const Params p) {
    constexpr int COLS = columns_of_tiles(NT);
    pdl_wait();
    const int4 row = p.shared[blockIdx.x], cut = p.shared[p.ctas];
    const int e = row.x, lane = threadIdx.x & 31;
    if (row.w < 0) return;
    Cut cuts;
    cuts.ctas = cut.x;
    cuts.per = cut.y;
    cuts.more = cut.z;
    const int parts = cuts.cta_of(row.w) - (int)blockIdx.x + 1;
    const int columns = (p.q_start[e + 1] - p.q_start[e]) * p.group - (row.z >> 1);
    for (int col = threadIdx.x >> 5; col < min(COLS, columns); col += JOIN_WARPS) {
        auto index = [&](int part) { return (size_t)(2 * ((int)blockIdx.x + part) + (part == 0 ? row.z & 1 : 0)) * COLS + col; };
        float acc[D / 32], sum, mx;
        add_parts<D>(p, 0, 1, parts, index, acc, sum, mx);
        bf16* out = result_of<D>(p, e, row.y, (row.z >> 1) + col);
#pragma unroll
        for (int k = 0; k < D / 32; ++k) out[k * 32 + lane] = __float2bfloat16_rn(sum == 0.f ? 0.f : acc[k] / sum);
    }
}

// The same where there are no more rows than CTAs: a block a row and column, MERGE_WARPS warps that share the parts.  What a block
// is to do it finds from the step's lists before the wait.  (Eight tokens of 8,100 keys, 64 rows of some 7 parts: 1 us less than
// with the kernel above; 64 of 2,048, 512 rows on 444 CTAs: 1.8 us more.)
template <int D, int NT, int MERGE_WARPS>
__global__ void __launch_bounds__(MERGE_WARPS * 32) attn_quant_merge_kernel(const Params p) {
    constexpr int COLS = columns_of_tiles(NT);
    __shared__ float sh_o[MERGE_WARPS][D], sh_l[MERGE_WARPS], sh_m[MERGE_WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = blockIdx.y, e = blockIdx.x / p.most_blocks, block = blockIdx.x - e * p.most_blocks;
    // (every warp for itself, from the step's lists)
    const Entry en = entry_of<COLS>(p, e);
    int total = 0, before = 0;
    for (int i = lane; i < p.entries; i += 32) {
        const int u = entry_of<COLS>(p, i).units();
        total += u;
        if (i < e) before += u;
    }
    const Cut cuts((int)__reduce_add_sync(0xffffffffu, (unsigned)total), p.ctas);
    const int row_start = (int)__reduce_add_sync(0xffffffffu, (unsigned)before) + block * en.row_units();
    pdl_wait();
    if (block >= en.blocks) return;
    const int c0 = cuts.cta_of(row_start + ROW_COST), parts = cuts.cta_of(row_start + en.row_units() - 1) - c0 + 1;
    const int g = block / en.column_blocks, c = (block - g * en.column_blocks) * COLS + col;
    if (parts < 2 || c >= en.q_len * p.group) return;
    // (a CTA's first piece is in slot 0)
    auto index = [&](int part) { return (size_t)(2 * (c0 + part) + (row_start > cuts.start(c0 + part) ? 1 : 0)) * COLS + col; };
    float acc[D / 32], sum, mx;
    add_parts<D>(p, warp, MERGE_WARPS, parts, index, acc, sum, mx);
#pragma unroll
    for (int k = 0; k < D / 32; ++k) sh_o[warp][k * 32 + lane] = acc[k];
    if (lane == 0) { sh_l[warp] = sum; sh_m[warp] = mx; }
    __syncthreads();
    float f[MERGE_WARPS];
    mx = -INFINITY;
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < MERGE_WARPS; ++w) mx = fmaxf(mx, sh_m[w]);
#pragma unroll
    for (int w = 0; w < MERGE_WARPS; ++w) {
        f[w] = sh_m[w] == -INFINITY ? 0.f : exp2_fast(sh_m[w] - mx);
        sum = fmaf(sh_l[w], f[w], sum);
    }
    bf16* out = result_of<D>(p, e, g, c);
    for (int d = threadIdx.x; d < D; d += MERGE_WARPS * 32) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < MERGE_WARPS; ++w) v = fmaf(sh_o[w][d], f[w], v);
        out[d] = __float2bfloat16_rn(sum == 0.f ? 0.f : v / sum);
    }
}

template <int D, int BITS, int NT> constexpr size_t smem_bytes() {
    using S = Shape<D, BITS>;
    constexpr size_t ring = (size_t)WARPS * S::STAGES * S::WARP_STAGE, merge = (size_t)WARPS * columns_of_tiles(NT) * (D + 4 + 2) * 4;
    constexpr size_t all = ring + (q_in_ring<D, BITS, NT>() ? 0 : q_bytes<D, NT>());
    return all > merge ? all : merge;
}
// CTAs of one wave.
template <int D, int BITS, int NT, bool TILES> int wave() {
    static const int ctas = [] {
        int per = 0;
        const size_t smem = smem_bytes<D, BITS, NT>();
        if (kipp_allow_smem(attn_quant_kernel<D, BITS, NT, TILES>, smem) != 0 ||
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, attn_quant_kernel<D, BITS, NT, TILES>, THREADS, smem) != cudaSuccess || per < 1) {
            cudaGetLastError();
            per = 1;
        }
        const int all = per * kipp_sm_count();
        return all < MOST_CTAS ? all : MOST_CTAS;
    }();
    return ctas;
}
template <int D, int BITS, int NT, bool TILES> int launch(Params p, long long steps_of_row, cudaStream_t s) {
    constexpr size_t smem = smem_bytes<D, BITS, NT>();
    constexpr int COLS = columns_of_tiles(NT);
    const int wave_ctas = wave<D, BITS, NT, TILES>();
    const long long rows = (long long)p.entries * p.most_blocks, units = rows * (steps_of_row + ROW_COST);
    p.ctas = (int)(units < wave_ctas ? units : wave_ctas);
    const bool alone = steps_of_row <= 1, by_cta = !alone && rows > p.ctas;            // (alone: every row is one step, none is shared)
    if (!by_cta) p.shared = nullptr;
    if (const int e = kipp_allow_smem(attn_quant_kernel<D, BITS, NT, TILES>, smem)) return e;
    if (const int e = kipp_launch(attn_quant_kernel<D, BITS, NT, TILES>, dim3((unsigned)p.ctas), dim3(THREADS), smem, s, 1, p)) return e;
    if (alone) return 0;
    if (by_cta) return kipp_launch(attn_quant_join_kernel<D, NT>, dim3((unsigned)p.ctas), dim3(JOIN_WARPS * 32), 0, s, 1, p);
    // 16 warps a row and column where there are parts for all of them and an SM for every block (one token behind 8,000 keys, 8 rows: 10.6
    // us in all, 11.9 with 4; 13 entries of two tokens, 26 rows of 12 columns: 17.1 and 12.5)
    const int columns = p.most * p.group, live = columns < COLS ? columns : COLS;
    const dim3 grid((unsigned)rows, (unsigned)live);
    if (rows * 16 <= p.ctas && rows * live <= kipp_sm_count()) return kipp_launch(attn_quant_merge_kernel<D, NT, 16>, grid, dim3(512), 0, s, 1, p);
    return kipp_launch(attn_quant_merge_kernel<D, NT, 4>, grid, dim3(128), 0, s, 1, p);
}

// 4 columns where they hold every query of a kv head in 4 bits (8 tokens behind 8,100 keys, 4 queries each: 23.0 us, with 8 columns 25.0, with
// 16 32.7), 8 where those do, else 16 (12
// queries: 35.5 us, 42.3 with 8); heads of 256 have no room for their sums: always 8
int columns_of(int bits, int head_dim, long long queries) { return bits == 4 && queries <= 4 ? 4 : head_dim == 256 || queries <= 8 ? 8 : 16; }
// The kernel of these heads and columns.
int launch_columns(const Params& p, int bits, int head_dim, long long cols, long long steps, cudaStream_t s) {
    const bool tiles = p.page_size % 16 == 0;
#define KIPP_CASE(d, b)                                                                                            \
    if (head_dim == d && bits == b) {                                                                              \
        if constexpr (b == 4)                                                                                      \
            if (cols == 4) return tiles ? launch<d, b, 0, true>(p, steps, s) : launch<d, b, 0, false>(p, steps, s);                  \
        if (cols == 8) return tiles ? launch<d, b, 1, true>(p, steps, s) : launch<d, b, 1, false>(p, steps, s);                      \
        if constexpr (d != 256) return tiles ? launch<d, b, 2, true>(p, steps, s) : launch<d, b, 2, false>(p, steps, s);             \
    }
    KIPP_CASE(64, 4) KIPP_CASE(64, 8) KIPP_CASE(128, 4) KIPP_CASE(128, 8) KIPP_CASE(256, 4) KIPP_CASE(256, 8)
#undef KIPP_CASE
    return KIPP_ERR_ARG;
}
}  // namespace

// Whether the kernel takes these heads.
extern "C" int kipp_attn_quant_supported(int bits, int head_dim, int n_q, int n_kv) {
    return (bits == 4 || bits == 8) && (head_dim == 64 || head_dim == 128 || head_dim == 256) && n_kv > 0 && n_q > 0 && n_q % n_kv == 0;
}
// Bytes of scratch of a launch (the parts of rows that several CTAs share) whose block table has room for `room` keys an entry,
// whatever the step: none where a row is one step.
extern "C" long long kipp_attn_quant_scratch_bytes(int head_dim, long long room) {
    return room <= STEP ? 0 : 2LL * MOST_CTAS * MOST_COLUMNS * (head_dim + 2) * 4 + (MOST_CTAS + 1) * 16LL;
}

struct KippAttnQuant {
    void* out; const void* q;                           // bf16 [tokens][n_q][head_dim]
    const void *k_codes, *k_scales, *v_codes, *v_scales;
    const int *q_start, *context_len, *block_table;
    void* scratch;
    int* status;
    void* stream;
    long long scratch_bytes;
    int bits, n_pages, page_size, table_width, entries, most, n_q, n_kv, head_dim, window;
    float scale;
};

// The entries that bring 1 to `most` tokens; the others are left alone.
extern "C" int kipp_attn_quant(const KippAttnQuant* a) {
    const int bits = a->bits, head_dim = a->head_dim, n_q = a->n_q, n_kv = a->n_kv, entries = a->entries, most = a->most, page_size = a->page_size;
    if (entries <= 0 || most <= 0) return 0;
    if (!kipp_attn_quant_supported(bits, head_dim, n_q, n_kv) || page_size <= 0 || a->n_pages <= 0 || a->table_width <= 0 || a->window < 0 ||
        a->status == nullptr)
        return KIPP_ERR_ARG;
    const long long need = kipp_attn_quant_scratch_bytes(head_dim, (long long)a->table_width * page_size);
    if (a->scratch_bytes < need || (need > 0 && a->scratch == nullptr)) return -4;
    if ((((uintptr_t)a->q | (uintptr_t)a->out | (uintptr_t)a->k_codes | (uintptr_t)a->v_codes | (uintptr_t)a->k_scales | (uintptr_t)a->v_scales |
          (uintptr_t)a->scratch) & 15) != 0)
        return -3;
    // (row numbers of pages, keys, those of steps that are looked up ahead too, and steps of all rows are 32-bit)
    const long long cols = columns_of(bits, head_dim, (long long)most * (n_q / n_kv));
    const long long room = (long long)a->table_width * page_size, steps = (room + STEP - 1) / STEP;
    const long long blocks = n_kv * (((long long)most * (n_q / n_kv) + cols - 1) / cols), entry_units = blocks * (steps + ROW_COST);
    if ((long long)a->n_pages * n_kv * page_size > 0x7fffffffLL || room > 0x7fffffffLL - 32 * STEP || (long long)most * n_q > 0x3fffffffLL ||
        entry_units > 0x3fffffffLL)
        return KIPP_ERR_ARG;
    // (what every entry may have: a step of many, one of them with many tokens and one with a long table, goes in several launches)
    const int at_once = (int)(0x3fffffffLL / entry_units);
    Params p = {};
    p.out = (bf16*)a->out; p.q = (const bf16*)a->q;
    p.k_codes = (const uint8_t*)a->k_codes; p.k_scales = (const uint8_t*)a->k_scales;
    p.v_codes = (const uint8_t*)a->v_codes; p.v_scales = (const uint8_t*)a->v_scales;
    p.table_width = a->table_width; p.page_size = page_size; p.n_pages = a->n_pages; p.most = most;
    p.page_shift = -1;
    for (int i = 0; i < 31; ++i) if (page_size == 1 << i) p.page_shift = i;
    p.n_q = n_q; p.n_kv = n_kv; p.group = n_q / n_kv; p.window = a->window;
    // (a scale of 0 makes every score 0: by the queries, since a masked score times 0 would be no number)
    p.score_scale = a->scale == 0.f ? 1.f : fabsf(a->scale) * 1.4426950408889634f * 0x1p85f;
    p.query_scale = a->scale == 0.f ? 0.f : a->scale < 0.f ? -0x1p48f : 0x1p48f;
    p.part_o = (float*)a->scratch;
    p.part_ml = p.part_o + 2LL * MOST_CTAS * MOST_COLUMNS * head_dim;
    p.shared = (int4*)(p.part_ml + 2LL * MOST_CTAS * MOST_COLUMNS * 2);
    p.most_blocks = (int)blocks;
    p.status = a->status;
    for (int first = 0; first < entries; first += at_once) {
        p.entries = entries - first < at_once ? entries - first : at_once;
        p.q_start = a->q_start + first; p.context_len = a->context_len + first; p.block_table = a->block_table + (size_t)first * a->table_width;
        if (const int e = launch_columns(p, bits, head_dim, cols, steps, (cudaStream_t)a->stream)) return e;
        if (at_once >= entries - first) break;
    }
    return 0;
}
