// Attention over a cache held in 4 bits, for few query rows per request: decoded tokens, drafted
// ones, short portions of prompts (bfloat16 in and out, head sizes 64, 128 and 256).
//
// The work is reading the pages once, so the kernel is built around what stands between the bytes
// and the tensor cores: widening a code must cost about one instruction.  Keys are the A operand
// (16 keys a tile) and query rows the B operand (8 rows a tile), so a group of up to eight query
// heads costs half the products that 16-row query tiles would.  Both products contract over an
// index whose order is free, so codes are used in the order they lie in:
//   * S^T = K Q^T contracts over channels: a thread takes HD / 4 consecutive channels of two keys, and the queries
//     are laid out to match.  A word of eight codes becomes four half2 (channels i and i + 4) by
//     masking into half-precision numbers whose last bits are the code, (w & 0x000F000F) | 0x48004800 = 8 + c / 128,
//     and one fused multiply-add (8 + c / 128) s - 8.0625 s = (c - 8) s / 128, which is exact (seven significant bits; see
//     kv_q4.cuh).  The 128 goes into the softmax's scale.
//   * O^T = V^T P^T contracts over keys: pairs of keys are put side by side by two byte permutations per pair
//     of words, then widened the same way; P^T is the transpose (movmatrix) of the scores' own registers.
// Halves rather than bfloat16 because the weights P then keep 11 bits; queries are scaled by a power of two
// per row, their largest element into [1, 2): exact down to elements of 2^-17 there, whose eight bits end at the 2^-24 that subnormal
// halves count in, and off by 2^-25 at most below.
//
// A warp works alone: its own ring of shared memory, filled by asynchronous copies of 16 bytes (with pages of 16
// positions a kv head's codes and steps of keys and values are one run of 18 HD bytes), its own running
// maximum and sum.  The maximum lags: O is rescaled only when a score exceeds it by 2^8.  The warps of a CTA take
// tiles of 16 keys in turn and are merged at the end.  (Bulk copies counted by mbarriers were measured first: with them, and
// pieces folded by a second kernel, 64 ragged requests took 62 us where 54 were reached without.)
//
// The grid is as many CTAs as fit at once, and the 16-key tiles of all (item, kv head) pairs, laid
// end to end, are cut into one equal range for each: contexts of any lengths load the GPU evenly, and
// nothing of the launch depends on them.  A CTA works through the pairs of its range, asking for the next pair's
// keys before it merges the warps' results of the last.  A pair that lies in one range whole is written out; the pieces
// of the others go to scratch (at most two per CTA: the one its range begins in and the one it ends in), and the
// CTA whose piece arrives last folds them in ascending order, so results do not depend on the order of arrival.
//
// Measured on a B200 (28 query and 4 kv heads of 128, staged steps in a graph): 64 requests of 300 to 8,192 positions, 157 MB,
// 43.7 us = 3.6 TB/s, 0.55 of the measured copy rate; 8 of 32,768 39.1 us (0.59); 8 of 2,048 8.5 us; one of 519 6.0 us.  Of the
// ragged requests' cycles 55 % issue, at 364 instructions a tile; what warps wait for otherwise is fixed latencies and memory, in
// equal parts.
#include "kv_q4.cuh"

#include <type_traits>

namespace axon {

constexpr int QA_WARPS = 8, QA_THREADS = QA_WARPS * 32;
// Tiles in a warp's ring (8 requests of 32,768 positions: 39.1 us; two 38.7; four 40.6)
constexpr int QA_STAGES = 3;
// A pair counts as its tiles and so many more when ranges are cut: what starting on it and merging the warps'
// results cost the CTA, in tiles.  64 requests of 300 to 8,192 positions: 51.1 us with none (CTAs that met a dozen short
// requests finished last), 48.5 with 8, 45.2 with 16, 43.7 with 24, 43.4 with 40.
constexpr int QA_PAIR_COST = 24;
constexpr int QA_LEAST = QA_WARPS;               // the shortest range: one tile for each warp
constexpr float QA_LAZY = 8.f;                   // log2 units a score may exceed the running maximum

struct QaParams {
    const __nv_bfloat16* q;      // [tokens][heads * HD]
    const uint8_t* pool;
    __nv_bfloat16* out;
    const int32_t* segments;     // [4][n_segments]: slot, q_start, q_len, kv_len
    const int32_t* items;        // [n_items][2]: segment, first row (token * group + head of the group); null: segment i, row 0
    float* part_o;               // [2 * CTA + (0: the pair its range begins in, 1: the one it ends in)][row][HD]
    float2* part_ml;             // the same without the last index: maximum (log2 units) and sum
    unsigned int* arrived;       // [CTA]: pieces written of the pair that begins in the CTA's range and ends in another's; zero between launches
    PagedQ4 kv;
    int n_segments, n_items, heads, group, ctas, window, staged;
    float scale_log2;
};

template <int HD> struct QaTile {
    static constexpr int KC = 8 * HD, KS = HD, BYTES = 2 * (KC + KS);      // codes and steps of 16 keys; a tile with its values
    static constexpr int PIECES = BYTES / 16, LANE_PIECES = (PIECES + 31) / 32;      // 16-byte pieces of a tile, of a lane
    static constexpr int RING = QA_WARPS * QA_STAGES * BYTES;
    static constexpr int PITCH = HD + 8;                                    // floats between rows of the merge buffer
    static constexpr int merge(int nt) { return QA_WARPS * 8 * nt * (PITCH + 2) * 4; }
    static constexpr int queries(int nt) { return nt > 1 ? HD / 16 * nt * 32 * 8 + 8 * nt * 4 : 0; }
    static constexpr int smem(int nt) { return RING + merge(nt) + queries(nt); }
};

__device__ __forceinline__ void qa_copy16(uint32_t smem, const void* gmem) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(gmem) : "memory");
}
__device__ __forceinline__ void qa_copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void qa_copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void qa_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void qa_mma_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t qa_transpose(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float qa_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t qa_pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t qa_fma2(uint32_t a, uint32_t b, uint32_t c) {
    const __half2 r = __hfma2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b), *reinterpret_cast<__half2*>(&c));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t qa_mul2(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
// (w & mask) | magic as one logic operation, `magic` in a register (as an expression of two constants: 49.1 us for the 64 ragged
// requests, 44.0 so).
template <uint32_t MASK> __device__ __forceinline__ uint32_t qa_pick(uint32_t w, uint32_t magic) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "n"(MASK), "r"(magic));
    return r;
}
// The exponents under which a code in bits 0-3 (8 + c / 128) and one in bits 4-7 (0.5 + c / 128) are read, in
// registers the compiler cannot see through.
struct QaMagic {
    uint32_t low, high;
    __device__ __forceinline__ QaMagic() {
        asm volatile("mov.b32 %0, 0x48004800;" : "=r"(low));
        asm volatile("mov.b32 %0, 0x38003800;" : "=r"(high));
    }
};
// Two steps (their bytes << 7, one in each half) with the two addends that take 8 away from a code.
struct QaStep {
    uint32_t s, low, high;       // the steps; -8.0625 s for nibbles in bits 0-3; -0.5625 s for nibbles in bits 4-7
    __device__ __forceinline__ explicit QaStep(uint32_t two) {
        s = two;
        low = qa_mul2(s, 0xC808C808u);
        high = qa_mul2(s, 0xB880B880u);
    }
};
// The codes in bits 0-3, 4-7, 8-11 and 12-15 of both halves of w, times their steps / 128.
__device__ __forceinline__ void qa_widen(uint32_t (&p)[4], uint32_t w, const QaStep& st, const QaMagic& magic) {
    const uint32_t v = w >> 8;
    p[0] = qa_fma2(qa_pick<0x000F000Fu>(w, magic.low), st.s, st.low);
    p[1] = qa_fma2(qa_pick<0x00F000F0u>(w, magic.high), st.s, st.high);
    p[2] = qa_fma2(qa_pick<0x000F000Fu>(v, magic.low), st.s, st.low);
    p[3] = qa_fma2(qa_pick<0x00F000F0u>(v, magic.high), st.s, st.high);
}
template <int N> __device__ __forceinline__ void qa_lds(uint32_t (&r)[N], const uint8_t* p) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const uint4 v = reinterpret_cast<const uint4*>(p)[i];
            r[4 * i] = v.x; r[4 * i + 1] = v.y; r[4 * i + 2] = v.z; r[4 * i + 3] = v.w;
        }
    } else if constexpr (N == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        r[0] = v.x; r[1] = v.y;
    } else {
        r[0] = *reinterpret_cast<const uint32_t*>(p);
    }
}

// One row's share of a query fragment: the HD / 4 channels of this thread (lane % 4) of the row, scaled by
// 2^-e so that the row's largest element lies in [1, 2), and by -1 for a negative scale, as the B operand's
// registers.  Returns the factor that brings scores to log2 units (keys carry a 1 / 128), which is not negative.
template <int HD>
__device__ __forceinline__ float qa_query(uint32_t (&f)[HD / 16][2], const uint4 (&raw)[HD / 32], float scale_log2) {
    constexpr int W = HD / 32;
    uint32_t top = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const uint32_t u[4] = {raw[w].x, raw[w].y, raw[w].z, raw[w].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, max(u[i] & 0x7fffu, (u[i] >> 16) & 0x7fffu));
    }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // (a row of zeros or with a number that is not finite is left as it is)
    int e = (int)(top >> 7) - 127;
    if (top == 0 || top >= 0x7f80u) e = 0;
    e = max(e, -126);                             // (2^126 is the largest power that brings subnormals up)
    const float down = copysignf(e > 126 ? 5.877471754111438e-39f : __uint_as_float((uint32_t)(127 - e) << 23), scale_log2);
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const uint32_t u[4] = {raw[w].x, raw[w].y, raw[w].z, raw[w].w};
        float x[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(u[i] << 16) * down;
            x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u) * down;
        }
        f[2 * w][0] = qa_pack(x[0], x[4]); f[2 * w][1] = qa_pack(x[1], x[5]);
        f[2 * w + 1][0] = qa_pack(x[2], x[6]); f[2 * w + 1][1] = qa_pack(x[3], x[7]);
    }
    return __uint_as_float((uint32_t)(127 + e) << 23) * fabsf(scale_log2) * 128.f;
}

// An item's rows and the keys they see.
struct QaItem {
    int slot, q_start, row0, rows, pos0, pos_first, pos_last, kv_lo, kv_hi, tile0, tiles;
    __device__ __forceinline__ QaItem(const QaParams& p, int item, int most_rows) {
        const int seg = p.items ? p.items[2 * item] : item;
        row0 = p.items ? p.items[2 * item + 1] : 0;
        slot = p.segments[seg];
        q_start = p.segments[p.n_segments + seg];
        const int q_len = p.segments[2 * p.n_segments + seg], kv_len = p.segments[3 * p.n_segments + seg];
        rows = min(most_rows, q_len * p.group - row0);
        pos0 = kv_len - q_len;
        pos_first = pos0;
        pos_last = kv_len - 1;
        if (p.items) {                                             // a part of a segment's rows
            pos_first = pos0 + row0 / p.group;
            pos_last = pos0 + (row0 + rows - 1) / p.group;
        }
        kv_hi = pos_last + 1;
        kv_lo = (p.window > 0 && pos_first - p.window + 1 > 0) ? pos_first - p.window + 1 : 0;
        tile0 = kv_lo / 16;
        tiles = rows > 0 ? max((kv_hi + 15) / 16 - tile0, 0) : 0;
    }
};
// How all pairs, laid end to end (items in order, the kv heads of each in order), fall to the CTAs: a range
// of `per` places each.  Where the pairs cut into pieces of equal length that start at their beginnings make no more
// pieces than there are CTAs, a pair's tiles are padded to whole ranges, so that no CTA has two pieces; else pairs follow one
// another without gaps but for `cost` places before each.  Everything counts in 32 bits: the launcher has seen to it that
// tiles + QA_PAIR_COST * pairs stay below 2^31, there are no more pieces than that, and a padded division, taken for
// no more pieces than CTAs only, has ctas * per places at most, which is within ctas * (QA_LEAST + the shortest range) of the tiles.
struct QaDivision {
    uint32_t total, per, cost;
    bool padded;
    // the length of ranges that pairs are padded to
    __host__ __device__ __forceinline__ QaDivision(uint32_t tiles, uint32_t longest, uint32_t ctas) {
        // one CTA folds a pair's pieces (about 0.12 us each): with few long pairs, ranges as long as the fold of their
        // number, which is about the square root of a pair's tiles (one request of 32,768 positions: 14.5 us; with 1.5 times
        // as long ranges 15.3, twice 16.5, 0.7 times 13.6)
        least = (uint32_t)sqrtf((float)longest);
        least = least > (uint32_t)QA_LEAST ? least : (uint32_t)QA_LEAST;
        const uint32_t even = (tiles + ctas - 1) / ctas;
        padded = true;
        cost = 0;
        total = 0;
        per = ((least > even ? least : even) + QA_LEAST - 1) / QA_LEAST * QA_LEAST;
    }
    __host__ __device__ __forceinline__ uint32_t pieces(uint32_t tiles) const { return (tiles + per - 1) / per; }
    // the choice, once the pieces of all pairs are counted
    __host__ __device__ __forceinline__ void settle(uint32_t all_pieces, uint32_t tiles, uint32_t pairs, uint32_t ctas) {
        if (all_pieces <= ctas) {
            total = all_pieces * per;
            return;
        }
        padded = false;
        cost = QA_PAIR_COST;
        total = tiles + cost * pairs;
        const uint32_t even = (total + ctas - 1) / ctas;
        per = least > even ? least : even;
    }
    // what a pair of `tiles` takes: its cost, then its tiles
    __host__ __device__ __forceinline__ uint32_t weight(uint32_t tiles) const {
        return tiles == 0 ? 0 : padded ? pieces(tiles) * per : tiles + cost;
    }
private:
    uint32_t least;
};
// Every warp works the division out for itself, 32 items at a time.
struct QaPlan : QaDivision {
    // `item`: the one that this CTA's range begins in, `start`: where its first pair begins
    __device__ __forceinline__ QaPlan(const QaParams& p, int most_rows, int* item, uint32_t* start)
        : QaPlan(p, most_rows, (int)(threadIdx.x & 31) < p.n_items ? QaItem(p, (int)(threadIdx.x & 31), most_rows).tiles : 0, item, start) {}
private:
    struct Sums { uint32_t tiles, longest, pairs; };
    // (`mine`: the first 32 items' tiles stay in registers)
    static __device__ __forceinline__ Sums sums(const QaParams& p, int most_rows, uint32_t mine) {
        Sums s{mine, mine, mine != 0};
        for (int i = (int)(threadIdx.x & 31) + 32; i < p.n_items; i += 32) {
            const uint32_t n = QaItem(p, i, most_rows).tiles;
            s.tiles += n;
            s.longest = max(s.longest, n);
            s.pairs += n != 0;
        }
        s.tiles = __reduce_add_sync(0xffffffffu, s.tiles) * p.kv.kv_heads;
        s.longest = __reduce_max_sync(0xffffffffu, s.longest);
        s.pairs = __reduce_add_sync(0xffffffffu, s.pairs) * p.kv.kv_heads;
        return s;
    }
    __device__ __forceinline__ QaPlan(const QaParams& p, int most_rows, uint32_t mine, int* item, uint32_t* start)
        : QaPlan(p, most_rows, mine, sums(p, most_rows, mine), item, start) {}
    __device__ __forceinline__ QaPlan(const QaParams& p, int most_rows, uint32_t mine, const Sums& s, int* item, uint32_t* start)
        : QaDivision(s.tiles, s.longest, p.ctas) {
        const int lane = threadIdx.x & 31;
        uint32_t n_pieces = pieces(mine);
        for (int i = lane + 32; i < p.n_items; i += 32) n_pieces += pieces(QaItem(p, i, most_rows).tiles);
        settle(__reduce_add_sync(0xffffffffu, n_pieces) * p.kv.kv_heads, s.tiles, s.pairs, p.ctas);
        // the item of this CTA's first place
        const uint32_t f = blockIdx.x * per;
        uint32_t base = 0;
        *item = p.n_items;
        for (int i0 = 0; i0 < p.n_items; i0 += 32) {
            const uint32_t n = (i0 == 0 ? weight(mine) : i0 + lane < p.n_items ? weight(QaItem(p, i0 + lane, most_rows).tiles) : 0) * p.kv.kv_heads;
            uint32_t upto = n;                                     // of this item and those before it in the 32
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const uint32_t x = __shfl_up_sync(0xffffffffu, upto, d);
                if (lane >= d) upto += x;
            }
            const unsigned past = __ballot_sync(0xffffffffu, base + upto > f);
            if (past) {
                const int who = __ffs(past) - 1;
                *start = base + __shfl_sync(0xffffffffu, upto - n, who);
                *item = i0 + who;
                break;
            }
            base += __shfl_sync(0xffffffffu, upto, 31);
        }
    }
};

// WHOLE: pages of 16 positions, table entries not checked (a check may store, which keeps the copies behind it apart).
template <int HD, int NT, bool WHOLE>
__global__ void __launch_bounds__(QA_THREADS, (NT == 1 && HD <= 128) ? 2 : 1)
attention_q4_kernel(const QaParams p) {
    using T = QaTile<HD>;
    constexpr int KW = HD / 32, VW = HD / 64, MT = HD / 16;      // words of a key row and of a value row per thread; 16-channel tiles of O
    constexpr int KG = HD / 64;                                   // groups (steps) of a key row per thread
    constexpr int R = 8 * NT;
    extern __shared__ __align__(128) uint8_t qa_smem[];
    __shared__ unsigned int last;
    float* const mo = reinterpret_cast<float*>(qa_smem + T::RING);                // [warp][row][PITCH] results of the warps
    float2* const ml = reinterpret_cast<float2*>(mo + QA_WARPS * R * T::PITCH);   // [warp][row]
    uint2* const q_smem = reinterpret_cast<uint2*>(qa_smem + T::RING + T::merge(NT));         // [HD / 16][NT][lane], several row tiles
    float* const f_smem = reinterpret_cast<float*>(q_smem + HD / 16 * NT * 32);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    uint8_t* const ring = qa_smem + warp * (QA_STAGES * T::BYTES);
    const uint32_t ring_addr = (uint32_t)__cvta_generic_to_shared(ring);
    pdl_launch_dependents();

    // The division of the work and the first table entries do not wait for the kernel before where segments, lists
    // and tables were copied to the device ahead of a step's kernels, none of which writes them.
    if (!p.staged) pdl_wait();
    int item;
    uint32_t start;
    const QaPlan plan(p, R, &item, &start);
    if (item >= p.n_items) {                                       // nothing left for this CTA
        pdl_wait();
        return;
    }
    uint32_t f = blockIdx.x * plan.per;
    const uint32_t f1 = f + min(plan.per, plan.total - f), per = plan.per;
    const QaMagic magic;

    // ---- copies: piece i of a tile is lane i % 32's
    const int ps = p.kv.page_size;
    const uint8_t* head_src;                                       // the pair's record in page 0
    const int32_t* table;
    int tile0, tile1, last_page;
    auto entry_of = [&](int tile) { return tile < tile1 ? table[WHOLE ? tile : tile * 16 / ps] : 0; };     // of its first position
    auto request = [&](int tile, int entry, int stage) {
        if (tile < tile1) {
            const uint32_t dst = ring_addr + stage * T::BYTES + lane * 16;
            if constexpr (WHOLE) {
                const uint8_t* const src = head_src + (long long)entry * p.kv.page_stride + lane * 16;
#pragma unroll
                for (int k = 0; k < T::LANE_PIECES; ++k) if (32 * k + lane < T::PIECES) qa_copy16(dst + k * 512, src + k * 512);
            } else {
                // a tile's four parts lie apart, and with pages that are no multiple of 16 positions its keys do too
                const bool together = ps % 16 == 0;
#pragma unroll
                for (int k = 0; k < T::LANE_PIECES; ++k) {
                    const int i = 32 * k + lane, in_tile = i * 16;                     // (bytes)
                    if (i >= T::PIECES) continue;
                    const int half = in_tile / (T::KC + T::KS), in_half = in_tile % (T::KC + T::KS), steps = in_half >= T::KC;
                    const int in_part = in_half - (steps ? T::KC : 0), row = steps ? HD / 16 : HD / 2;
                    const int key = in_part / row, pos = tile * 16 + key;
                    const int lp = min(pos / ps, last_page), in_page = pos % ps;      // (past the last page: some row of it, hidden later)
                    const int part = half ? (steps ? p.kv.v_steps : p.kv.v_codes) : (steps ? p.kv.k_steps : 0);
                    qa_copy16(dst + k * 512, head_src + (long long)p.kv.page(together ? entry : table[lp]) * p.kv.page_stride + part +
                                                 in_page * row + in_part % row);
                }
            }
        }
        qa_copy_commit();
    };
    int next;                                                      // the table entry of the tile to be asked for next
    QaItem it(p, item, R);
    int off = 0;
    uint32_t pair_weight = plan.weight(it.tiles);                  // (not zero: the plan gives an item that has tiles)
    int kvh = (int)((f - start) / pair_weight);
    uint32_t pair_begin = start + kvh * pair_weight;
    // The next piece of the range: tiles off .. of the pair (it, kvh), f moved to its end; false when there is none.
    auto advance = [&]() {
        while (f < f1) {
            const uint32_t from = f - pair_begin, to = min(pair_weight, f1 - pair_begin);      // within the pair
            if (from >= pair_weight) {
                pair_begin += pair_weight;
                if (++kvh == p.kv.kv_heads) {
                    kvh = 0;
                    do { ++item; it = QaItem(p, min(item, p.n_items - 1), R); } while (it.tiles == 0 && item < p.n_items);
                    if (item >= p.n_items) return false;
                    pair_weight = plan.weight(it.tiles);
                }
                continue;
            }
            f = pair_begin + to;
            if (to <= plan.cost) return false;                     // the range ends before the pair's first tile
            off = max((int)(from - plan.cost), 0);
            tile0 = it.tile0 + off;
            tile1 = it.tile0 + min((int)(to - plan.cost), it.tiles);
            return true;
        }
        return false;
    };
    // ---- a pair's piece begins: table entries, then this thread's share of the queries, are asked for, then the
    // first keys; while they come queries become B fragments, with the factors that bring rows' scores to log2 units
    uint32_t qf[NT == 1 ? HD / 16 : 1][2];
    float factor[NT][2];
    auto begin_pair = [&](auto first_of_all) {
        head_src = p.pool + p.kv.entry_offset + (long long)kvh * p.kv.record;
        table = p.kv.block_table + (long long)it.slot * p.kv.table_stride;
        last_page = (it.kv_hi - 1) / ps;
        int entry[QA_STAGES];
#pragma unroll
        for (int j = 0; j < QA_STAGES; ++j) entry[j] = entry_of(tile0 + warp + j * QA_WARPS);
        next = entry_of(tile0 + warp + QA_STAGES * QA_WARPS);
        if (decltype(first_of_all)::value) pdl_wait();             // keys and queries may be the work of the kernel before
        const int r = NT == 1 ? g : 8 * warp + g, row = it.row0 + r;
        const bool mine = NT == 1 || warp < NT, live = mine && r < it.rows;
        uint4 raw[HD / 32];
        if (live) {
            const int ahead = row < p.group ? 0 : row / p.group;   // tokens of the segment before the row's
            const uint4* const src = reinterpret_cast<const uint4*>(
                p.q + ((long long)(it.q_start + ahead) * p.heads + kvh * p.group + row - ahead * p.group) * HD + t * (HD / 4));
#pragma unroll
            for (int w = 0; w < HD / 32; ++w) raw[w] = src[w];
        } else {
#pragma unroll
            for (int w = 0; w < HD / 32; ++w) raw[w] = make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < QA_STAGES; ++j) request(tile0 + warp + j * QA_WARPS, entry[j], j);
        if constexpr (NT == 1) {
            const float scale = qa_query<HD>(qf, raw, p.scale_log2);
            factor[0][0] = __shfl_sync(0xffffffffu, scale, 8 * t);
            factor[0][1] = __shfl_sync(0xffffffffu, scale, 8 * t + 4);
        } else if (mine) {                                         // (read back after the next barrier)
            uint32_t frag[HD / 16][2];
            const float scale = qa_query<HD>(frag, raw, p.scale_log2);
#pragma unroll
            for (int k = 0; k < HD / 16; ++k) q_smem[(k * NT + warp) * 32 + lane] = make_uint2(frag[k][0], frag[k][1]);
            if (t == 0) f_smem[r] = scale;
        }
    };

    if (!advance()) {
        pdl_wait();
        return;
    }
    begin_pair(std::true_type());
    for (;;) {
    const int rows = it.rows, pos_first = it.pos_first, pos_last = it.pos_last, row0 = it.row0, q_start = it.q_start;
    const int kv_lo = it.kv_lo, kv_hi = it.kv_hi;
    if constexpr (NT > 1) {
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NT; ++n) { factor[n][0] = f_smem[8 * n + 2 * t]; factor[n][1] = f_smem[8 * n + 2 * t + 1]; }
    }

    float o[MT][NT][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) o[j][n][c] = 0.f;
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.f;
    }
    // the position of the query row in column c of row tile n (rows past the last: the last token's)
    auto row_pos = [&](int n, int c) { return it.pos0 + (row0 + min(8 * n + 2 * t + c, rows - 1)) / p.group; };

    // the tiles of this piece that every row sees whole: [clear0, clear1)
    const int clear0 = p.window > 0 ? max(pos_last - p.window + 16, 0) / 16 : 0, clear1 = min(tile1, (pos_first + 1) / 16);
    // One tile; EDGE when it may hold keys that not every row sees.
    auto fold = [&](auto edge, int key0, const uint8_t* tile) {
        constexpr bool EDGE = decltype(edge)::value;
        float s[NT][4];
        {
            float s2[NT][4];                                       // two sums, so that products do not wait for one another
            uint32_t wa[KW], wb[KW];                               // this thread's codes of keys g and g + 8
            qa_lds(wa, tile + g * (HD / 2) + t * (HD / 8));
            qa_lds(wb, tile + (g + 8) * (HD / 2) + t * (HD / 8));
            const uint8_t* const st = tile + T::KC + g * (HD / 16) + t * KG;
#pragma unroll
            for (int w = 0; w < KW; ++w) {
                const QaStep sa(st[w / 2] * 0x00800080u), sb(st[8 * (HD / 16) + w / 2] * 0x00800080u);
                uint32_t a[4], b[4];
                qa_widen(a, wa[w], sa, magic);
                qa_widen(b, wb[w], sb, magic);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    uint2 q0, q1;
                    if constexpr (NT == 1) { q0 = make_uint2(qf[2 * w][0], qf[2 * w][1]); q1 = make_uint2(qf[2 * w + 1][0], qf[2 * w + 1][1]); }
                    else { q0 = q_smem[(2 * w * NT + n) * 32 + lane]; q1 = q_smem[((2 * w + 1) * NT + n) * 32 + lane]; }
                    if (w == 0) {
                        qa_mma_first(s[n], a[0], b[0], a[1], b[1], q0.x, q0.y);
                        qa_mma_first(s2[n], a[2], b[2], a[3], b[3], q1.x, q1.y);
                    } else {
                        qa_mma(s[n], a[0], b[0], a[1], b[1], q0.x, q0.y);
                        qa_mma(s2[n], a[2], b[2], a[3], b[3], q1.x, q1.y);
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 4; ++c) s[n][c] += s2[n][c];
        }
        // scores in log2 units are s * factor; an edge tile's are multiplied out before the mask (0 * infinity is NaN)
        float top[NT][2];
        bool grew = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (EDGE) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int key = key0 + g + (c >> 1) * 8, pos = row_pos(n, c & 1);
                    s[n][c] *= factor[n][c & 1];
                    if (key > pos || (p.window > 0 && key <= pos - p.window)) s[n][c] = -INFINITY;
                }
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                top[n][c] = fmaxf(s[n][c], s[n][c + 2]) * (EDGE ? 1.f : factor[n][c]);
                grew = grew || top[n][c] > m[n][c] + QA_LAZY;
            }
        }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float x = top[n][c];
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                    x = fmaxf(x, m[n][c]);
                    const float f = x == -INFINITY ? 1.f : qa_ex2(m[n][c] - x);
                    m[n][c] = x;
                    l[n][c] *= f;
#pragma unroll
                    for (int k = 0; k < MT; ++k) { o[k][n][c] *= f; o[k][n][c + 2] *= f; }
                }
        }
        uint32_t pf[NT][2];                                        // weights as B fragments
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float w[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float m_c = EDGE && m[n][c & 1] == -INFINITY ? 0.f : m[n][c & 1];
                w[c] = qa_ex2(EDGE ? s[n][c] - m_c : fmaf(s[n][c], factor[n][c & 1], -m_c));
            }
            l[n][0] += w[0] + w[2];
            l[n][1] += w[1] + w[3];
            pf[n][0] = qa_transpose(qa_pack(w[0], w[1]));
            pf[n][1] = qa_transpose(qa_pack(w[2], w[3]));
        }
        const uint8_t* const vt = tile + T::KC + T::KS;
        uint32_t w4[4][VW];                                        // codes of keys 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
        for (int k = 0; k < 4; ++k) qa_lds(w4[k], vt + (2 * t + (k & 1) + (k >> 1) * 8) * (HD / 2) + g * (HD / 16));
#pragma unroll
        for (int u = 0; u < (VW + 1) / 2; ++u) {                   // groups of 16 channels (of 8, the half of one, at head size 64)
            uint32_t by[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) by[k] = vt[T::KC + (2 * t + (k & 1) + (k >> 1) * 8) * (HD / 16) + (g * (HD / 8)) / 16 + u];
            uint32_t nan_keys = 0;
            if (EDGE) {
                // keys that no row sees may hold anything, and a NaN that some rows see must not reach the others (0 * NaN
                // is NaN): both count as zero here, and the rows that see a NaN get theirs below
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int key = 2 * t + (k & 1) + (k >> 1) * 8;
                    const bool in = key0 + key >= kv_lo && key0 + key < kv_hi;
                    if (in && by[k] == Q4_NAN) nan_keys |= 1u << key;
                    if (!in || by[k] == Q4_NAN) by[k] = 0;
                }
            }
            const QaStep s01(by[0] * 0x80u + by[1] * 0x800000u), s89(by[2] * 0x80u + by[3] * 0x800000u);
#pragma unroll
            for (int v = 2 * u; v < VW && v < 2 * u + 2; ++v) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {             // codes 0-3 and 4-7 of the words
                    const uint32_t sel = half ? 0x7632u : 0x5410u;
                    uint32_t a[4], b[4];
                    qa_widen(a, __byte_perm(w4[0][v], w4[1][v], sel), s01, magic);
                    qa_widen(b, __byte_perm(w4[2][v], w4[3][v], sel), s89, magic);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        qa_mma(o[4 * v + 2 * half][n], a[0], a[1], b[0], b[1], pf[n][0], pf[n][1]);
                        qa_mma(o[4 * v + 2 * half + 1][n], a[2], a[3], b[2], b[3], pf[n][0], pf[n][1]);
                    }
                }
            }
            if (EDGE) {
                nan_keys |= __shfl_xor_sync(0xffffffffu, nan_keys, 1);
                nan_keys |= __shfl_xor_sync(0xffffffffu, nan_keys, 2);
                if (nan_keys != 0) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const int pos = row_pos(n, c);
                            bool sees = false;
                            for (int k = 0; k < 16; ++k)
                                sees = sees || ((nan_keys >> k & 1) && key0 + k <= pos && (p.window <= 0 || key0 + k > pos - p.window));
                            if (!sees) continue;
#pragma unroll
                            for (int k = 0; k < (VW == 1 ? 4 : 8); ++k) o[8 * u + k][n][c] = o[8 * u + k][n][c + 2] = __int_as_float(0x7fc00000);
                        }
                }
            }
        }
    };
    // Tiles that every row sees whole go through a loop of their own: it was faster than one loop with the masked
    // code behind a branch.
    for (int tile = tile0 + warp, stage = 0;;) {
        auto take = [&](auto edge) {
            qa_copy_wait<QA_STAGES - 1>();
            __syncwarp();                                          // every lane's pieces are there
            fold(edge, tile * 16, ring + stage * T::BYTES);
            __syncwarp();                                          // every lane is done with the stage
            request(tile + QA_STAGES * QA_WARPS, next, stage);
            next = entry_of(tile + (QA_STAGES + 1) * QA_WARPS);
            tile += QA_WARPS;
            if (++stage == QA_STAGES) stage = 0;
        };
        while (tile >= clear0 && tile < clear1) take(std::false_type());
        if (tile >= tile1) break;
        take(std::true_type());
    }
    qa_copy_wait<0>();

    // ---- the warps' results side by side in shared memory, merged by all threads; the next pair's keys and
    // queries are on their way meanwhile
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], 4);
            l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], 8);
            l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], 16);
            const int r = 8 * n + 2 * t + c;
            float* const dst = mo + (warp * R + r) * T::PITCH + g * (HD / 8);
#pragma unroll
            for (int k = 0; k < MT; ++k) *reinterpret_cast<float2*>(dst + 2 * k) = make_float2(o[k][n][c], o[k][n][c + 2]);
            if (g == 0) ml[warp * R + r] = make_float2(m[n][c], l[n][c]);
        }
    __syncthreads();
    const bool whole_pair = off == 0 && tile1 - tile0 == it.tiles, began_here = off == 0;
    const uint32_t first_place = pair_begin + plan.cost, last_place = first_place + it.tiles - 1;      // of the pair's tiles
    const int head0 = kvh * p.group;
    const bool more = advance();
    if (more) begin_pair(std::false_type());
    auto write_out = [&](int r, int d, const float4& acc, float sum) {
        const float inv = 128.f / sum;                             // (values carry a 1 / 128, as keys do)
        const int row = row0 + r, ahead = row < p.group ? 0 : row / p.group, tok = q_start + ahead, head = head0 + row - ahead * p.group;
        const __nv_bfloat162 a = __floats2bfloat162_rn(acc.x * inv, acc.y * inv), b = __floats2bfloat162_rn(acc.z * inv, acc.w * inv);
        *reinterpret_cast<uint2*>(p.out + ((long long)tok * p.heads + head) * HD + d) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    };
    for (int e = threadIdx.x; e < rows * (HD / 4); e += QA_THREADS) {
        const int r = e / (HD / 4), d = e % (HD / 4) * 4;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < QA_WARPS; ++w) top = fmaxf(top, ml[w * R + r].x);
        const float use = top == -INFINITY ? 0.f : top;
        float sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < QA_WARPS; ++w) {
            const float2 x = ml[w * R + r];
            const float wt = qa_ex2(x.x - use);
            const float4 v = *reinterpret_cast<const float4*>(mo + (w * R + r) * T::PITCH + d);
            sum = fmaf(x.y, wt, sum);
            acc.x = fmaf(v.x, wt, acc.x); acc.y = fmaf(v.y, wt, acc.y); acc.z = fmaf(v.z, wt, acc.z); acc.w = fmaf(v.w, wt, acc.w);
        }
        if (whole_pair) write_out(r, d, acc, sum);
        else {
            const long long at = (2ll * blockIdx.x + began_here) * R + r;
            __stcg(reinterpret_cast<float4*>(p.part_o + at * HD + d), acc);
            if (d == 0) __stcg(p.part_ml + at, make_float2(top, sum));
        }
    }
    if (!whole_pair) {
        const int c0 = (int)(first_place / per), c1 = (int)(last_place / per);
        __syncthreads();                                           // (every thread's share is written; one fence covers them)
        if (threadIdx.x == 0) {
            __threadfence();
            last = atomicAdd(p.arrived + c0, 1u) == (unsigned)(c1 - c0);
            if (last) {
                __threadfence();                                   // the others' pieces, counted by their atomics, are seen from here on
                p.arrived[c0] = 0;                                 // ready for the next launch
            }
        }
        __syncthreads();
        if (last) {
            constexpr int S = 8;                                   // pieces asked for together
            for (int e = threadIdx.x; e < rows * (HD / 4); e += QA_THREADS) {
                const int r = e / (HD / 4), d = e % (HD / 4) * 4;
                float top = -INFINITY, sum = 0.f;
                float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int s0 = c0; s0 <= c1; s0 += S) {
                    float2 x[S];
                    float4 v[S];
#pragma unroll
                    for (int q = 0; q < S; ++q) {
                        const int c = s0 + q;
                        // the pair begins in c0's range, and before all of the others'
                        const long long at = (2ll * c + (c == c0)) * R + r;
                        x[q] = c <= c1 ? __ldcg(p.part_ml + at) : make_float2(-INFINITY, 0.f);
                        v[q] = c <= c1 ? __ldcg(reinterpret_cast<const float4*>(p.part_o + at * HD + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
                    }
                    float up = top;
#pragma unroll
                    for (int q = 0; q < S; ++q) up = fmaxf(up, x[q].x);
                    const float use = up == -INFINITY ? 0.f : up, was = qa_ex2(top - use);
                    top = up;
                    sum *= was; acc.x *= was; acc.y *= was; acc.z *= was; acc.w *= was;
#pragma unroll
                    for (int q = 0; q < S; ++q) {
                        const float wt = qa_ex2(x[q].x - use);
                        sum = fmaf(x[q].y, wt, sum);
                        acc.x = fmaf(v[q].x, wt, acc.x); acc.y = fmaf(v[q].y, wt, acc.y); acc.z = fmaf(v[q].z, wt, acc.z); acc.w = fmaf(v[q].w, wt, acc.w);
                    }
                }
                write_out(r, d, acc, sum);
            }
        }
    }
    if (!more) break;
    __syncthreads();                                               // the next pair's results overwrite what was merged here
    }
}

template <int HD, int NT>
static int launch_q4(const QaParams& p, cudaStream_t stream) {
    constexpr int smem = QaTile<HD>::smem(NT);
    static_assert(smem <= 226 * 1024, "the rings do not fit shared memory");
    if (p.kv.page_size == 16 && p.kv.fault == nullptr) {
        if (int st = ensure_dynamic_smem<attention_q4_kernel<HD, NT, true>>(smem, "axon_attention_q4")) return st;
        launch_pdl(attention_q4_kernel<HD, NT, true>, dim3(p.ctas), dim3(QA_THREADS), smem, stream, p);
    } else {
        if (int st = ensure_dynamic_smem<attention_q4_kernel<HD, NT, false>>(smem, "axon_attention_q4")) return st;
        launch_pdl(attention_q4_kernel<HD, NT, false>, dim3(p.ctas), dim3(QA_THREADS), smem, stream, p);
    }
    return launch_status("axon_attention_q4");
}

}  // namespace axon

using namespace axon;

// How many CTAs an attention launch has (two fit an SM with one tile of 8 rows, up to head size 128).
AXON_API int axon_attention_q4_ctas(int head_dim, int row_tiles) { return (row_tiles == 1 && head_dim <= 128 ? 2 : 1) * 148; }

// How an attention launch of `ctas` CTAs divides items of these many 16-key tiles among them, worked out on the host by the
// kernel's own arithmetic: out = {places in all, places of a CTA, places before each pair, 1 if pairs are padded to whole ranges}.
AXON_API int axon_attention_q4_division(const int32_t* tiles, int n_items, int kv_heads, int ctas, uint32_t* out) {
    uint32_t sum = 0, longest = 0, pairs = 0, n_pieces = 0;
    for (int i = 0; i < n_items; ++i) {
        sum += tiles[i];
        longest = (uint32_t)tiles[i] > longest ? tiles[i] : longest;
        pairs += tiles[i] != 0;
    }
    QaDivision d(sum * kv_heads, longest, ctas);
    for (int i = 0; i < n_items; ++i) n_pieces += d.pieces(tiles[i]);
    d.settle(n_pieces * kv_heads, sum * kv_heads, pairs * kv_heads, ctas);
    out[0] = d.total; out[1] = d.per; out[2] = d.cost; out[3] = d.padded;
    return AXON_OK;
}

// Attention of `n_items` tiles of up to 8 * row_tiles query rows (row_tiles 1, 2 or 4; at head size 256 1).  items null:
// item i is segment i, whose rows all fit one tile.  scratch: 2 * ctas * 8 * row_tiles * (head_dim + 2) + ctas floats, zeroed once:
// launches leave the last ctas of them zero.  staged: segments and the block table were copied to the device before the kernels in
// flight were launched (pdl.cuh).
AXON_API int axon_attention_q4(const void* q, const void* pool, void* out, const int32_t* segments, int n_segments,
                               const int32_t* items, int n_items, const AxonKvLayout* layout, int heads, float scale, int window,
                               int row_tiles, float* scratch, long long scratch_floats, int staged, cudaStream_t stream) {
    if (n_items <= 0) return AXON_OK;
    QaParams p;
    if (int st = to_q4(layout, pool, "axon_attention_q4", &p.kv)) return st;
    const int hd = p.kv.hd;
    if (p.kv.planes != 2 || p.kv.vd != hd) { set_error("axon_attention_q4: takes caches with key and value planes of one width"); return AXON_BAD_ARGUMENT; }
    if (heads < 1 || heads % p.kv.kv_heads) { set_error("axon_attention_q4: %d heads over %d kv heads", heads, p.kv.kv_heads); return AXON_BAD_ARGUMENT; }
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)scratch) & 15) { set_error("axon_attention_q4: operands must be 16-byte aligned"); return AXON_BAD_ARGUMENT; }
    if ((double)n_items * p.kv.kv_heads * ((double)p.kv.table_stride * p.kv.page_size / 16 + 1 + QA_PAIR_COST) > 2147483647.0) { set_error("axon_attention_q4: %d items of %d kv heads at up to %d pages are too many", n_items, p.kv.kv_heads, p.kv.table_stride); return AXON_BAD_ARGUMENT; }
    // a copy moves 16 bytes: at head size 64 the steps of four positions, which have to lie in one page
    if (p.kv.page_size % (hd >= 256 ? 1 : 256 / hd)) { set_error("axon_attention_q4: pages of %d positions of %d values do not fall into pieces it can copy", p.kv.page_size, hd); return AXON_BAD_ARGUMENT; }
    p.ctas = axon_attention_q4_ctas(hd, row_tiles);
    const long long rows = 2ll * p.ctas * 8 * row_tiles;
    if (scratch == nullptr || scratch_floats < rows * (hd + 2) + p.ctas) { set_error("axon_attention_q4: needs %lld floats of zeroed scratch", rows * (hd + 2) + p.ctas); return AXON_BAD_ARGUMENT; }
    p.q = (const __nv_bfloat16*)q; p.pool = (const uint8_t*)pool; p.out = (__nv_bfloat16*)out;
    p.segments = segments; p.items = items;
    p.part_o = scratch; p.part_ml = reinterpret_cast<float2*>(scratch + rows * hd);
    p.arrived = reinterpret_cast<unsigned int*>(scratch + rows * (hd + 2));
    p.n_segments = n_segments; p.n_items = n_items; p.heads = heads; p.group = heads / p.kv.kv_heads; p.window = window; p.staged = staged;
    p.scale_log2 = scale * 1.4426950408889634f;
#define AXON_Q4_CASE(HD, NT) if (hd == HD && row_tiles == NT) return launch_q4<HD, NT>(p, stream)
    AXON_Q4_CASE(64, 1); AXON_Q4_CASE(64, 2); AXON_Q4_CASE(64, 4);
    AXON_Q4_CASE(128, 1); AXON_Q4_CASE(128, 2); AXON_Q4_CASE(128, 4);
    AXON_Q4_CASE(256, 1);
#undef AXON_Q4_CASE
    set_error("axon_attention_q4: no kernel for head size %d with %d tiles of 8 rows", hd, row_tiles);
    return AXON_BAD_ARGUMENT;
}
