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
// per row to the range of halves (exact, but for elements 2^-24 below the row's largest).
//
// A warp works alone: its own ring of shared memory, filled by bulk copies (one per 16-position page
// and kv head: codes and steps of keys and values lie together) that one mbarrier per stage counts, its own running
// maximum and sum.  The maximum lags: O is rescaled only when a score exceeds it by 2^8.  The warps of a CTA take
// chunks of 32 keys in turn and are merged at the end; CTAs split a request's keys, and a second
// kernel folds their shares in ascending order.
#include "kv_q4.cuh"
#include "tcgen05.cuh"

namespace axon {

constexpr int QA_WARPS = 8, QA_THREADS = QA_WARPS * 32;
constexpr int QA_KT = 2, QA_STAGES = 3;          // 16-key tiles per chunk, chunks in a warp's ring
constexpr int QA_MAX_SPLITS = 64;
constexpr float QA_LAZY = 8.f;                   // log2 units a score may exceed the running maximum

struct QaParams {
    const __nv_bfloat16* q;      // [tokens][heads * HD]
    const uint8_t* pool;
    __nv_bfloat16* out;
    const int32_t* segments;     // [4][n_segments]: slot, q_start, q_len, kv_len
    const int32_t* items;        // [n_items][2]: segment, first row (token * group + head of the group); null: segment i, row 0
    float* part_o;               // [item][kv head][split][row][HD], with several splits
    float2* part_ml;             // the same without the last index: maximum (log2 units) and sum
    PagedQ4 kv;
    int n_segments, heads, group, n_splits, window;
    int run;                     // positions of a tile that lie together in a page: gcd(page size, 16)
    float scale_log2;
};

template <int HD> struct QaTile {
    static constexpr int KC = 8 * HD, KS = HD, BYTES = 2 * (KC + KS);      // codes and steps of 16 keys; a tile with its values
    static constexpr int RING = QA_WARPS * QA_STAGES * QA_KT * BYTES;
    static constexpr int PITCH = HD + 8;                                    // floats between rows of the merge buffer
    static constexpr int merge(int nt) { return QA_WARPS * 8 * nt * (PITCH + 2) * 4; }
    static constexpr int queries(int nt) { return nt > 1 ? HD / 16 * nt * 32 * 8 + 8 * nt * 4 : 0; }
    static constexpr int area(int nt) { return RING > merge(nt) ? RING : merge(nt); }
    static constexpr int smem(int nt) { return area(nt) + queries(nt); }
};

__device__ __forceinline__ void qa_bulk_load(uint32_t smem, const void* gmem, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem), "l"(gmem), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void qa_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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
// Two step bytes (in the low byte of each half) with the two addends that take 8 away from a code.
struct QaStep {
    uint32_t s, low, high;       // the steps; -8.0625 s for nibbles in bits 0-3; -0.5625 s for nibbles in bits 4-7
    __device__ __forceinline__ explicit QaStep(uint32_t two) {
        s = two << 7;
        low = qa_mul2(s, 0xC808C808u);
        high = qa_mul2(s, 0xB880B880u);
    }
};
// The codes in bits 0-3, 4-7, 8-11 and 12-15 of both halves of w, times their steps / 128.
__device__ __forceinline__ void qa_widen(uint32_t (&p)[4], uint32_t w, const QaStep& st) {
    const uint32_t v = w >> 8;
    p[0] = qa_fma2((w & 0x000F000Fu) | 0x48004800u, st.s, st.low);
    p[1] = qa_fma2((w & 0x00F000F0u) | 0x38003800u, st.s, st.high);
    p[2] = qa_fma2((v & 0x000F000Fu) | 0x48004800u, st.s, st.low);
    p[3] = qa_fma2((v & 0x00F000F0u) | 0x38003800u, st.s, st.high);
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
// 2^-e so that the row's largest element lies in [1, 2), as the B operand's registers.  Returns 2^e.
template <int HD>
__device__ __forceinline__ float qa_load_query(uint32_t (&f)[HD / 16][2], const __nv_bfloat16* row, int t, bool live) {
    constexpr int W = HD / 32;
    uint4 raw[W];
    uint32_t top = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        raw[w] = live ? reinterpret_cast<const uint4*>(row + t * (HD / 4))[w] : make_uint4(0, 0, 0, 0);
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
    const float down = e > 126 ? 5.877471754111438e-39f : __uint_as_float((uint32_t)(127 - e) << 23);
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
    return __uint_as_float((uint32_t)(127 + e) << 23);
}

template <int HD, int NT>
__global__ void __launch_bounds__(QA_THREADS, (NT == 1 && HD <= 128) ? 2 : 1)
attention_q4_kernel(const QaParams p) {
    using T = QaTile<HD>;
    constexpr int KW = HD / 32, VW = HD / 64, MT = HD / 16;      // words of a key row and of a value row per thread; 16-channel tiles of O
    constexpr int KG = HD / 64;                                   // groups (steps) of a key row per thread
    extern __shared__ __align__(128) uint8_t qa_smem[];
    __shared__ __align__(8) uint64_t qa_bars[QA_WARPS * QA_STAGES];
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    uint8_t* const ring = qa_smem + warp * (QA_STAGES * QA_KT * T::BYTES);
    const uint32_t ring_addr = (uint32_t)__cvta_generic_to_shared(ring);
    const uint32_t bars = (uint32_t)__cvta_generic_to_shared(qa_bars + warp * QA_STAGES);
    if (lane == 0) {
        for (int s = 0; s < QA_STAGES; ++s) mbar_init(bars + 8 * s, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncwarp();
    pdl_wait();

    const int item = blockIdx.x, kvh = blockIdx.y, split = blockIdx.z;
    const int seg = p.items ? p.items[2 * item] : item, row0 = p.items ? p.items[2 * item + 1] : 0;
    const int slot = p.segments[seg], q_start = p.segments[p.n_segments + seg];
    const int q_len = p.segments[2 * p.n_segments + seg], kv_len = p.segments[3 * p.n_segments + seg];
    const int rows = min(8 * NT, q_len * p.group - row0);
    const int pos_first = kv_len - q_len + row0 / p.group, pos_last = kv_len - q_len + (row0 + rows - 1) / p.group;
    const int kv_hi = pos_last + 1, kv_lo = (p.window > 0 && pos_first - p.window + 1 > 0) ? pos_first - p.window + 1 : 0;
    int tile0, tile1;
    {
        const int first = kv_lo / 16, n = (kv_hi + 15) / 16 - first, per = (n + p.n_splits - 1) / p.n_splits;
        tile0 = first + split * per;
        tile1 = min(first + n, tile0 + per);
    }

    // ---- copies.  A lane owns one piece of a chunk: with pages of 16 positions a whole tile, else a run of
    // one of its four parts.
    const bool whole = p.kv.page_size == 16;
    const int pieces = whole ? 1 : 64 / p.run;                    // of a tile
    const int my_tile = lane / pieces, sub = lane % pieces, part = sub & 3, key_off = whole ? 0 : (sub >> 2) * p.run;
    const int row_bytes = (part & 1) ? HD / 16 : HD / 2;
    const uint32_t my_bytes = whole ? T::BYTES : p.run * row_bytes;
    const uint32_t my_dst = my_tile * T::BYTES + (whole ? 0 : (part & 1 ? T::KC : 0) + (part & 2 ? T::KC + T::KS : 0) + key_off * row_bytes);
    const uint8_t* const my_src = p.pool + p.kv.entry_offset + (long long)kvh * p.kv.record +
        (whole || part == 0 ? 0 : part == 1 ? p.kv.k_steps : part == 2 ? p.kv.v_codes : p.kv.v_steps);
    const int32_t* const table = p.kv.block_table + (long long)slot * p.kv.table_stride;
    const int last_page = (kv_hi - 1) / p.kv.page_size;
    auto chunk_tile = [&](int j) { return tile0 + (warp + j * QA_WARPS) * QA_KT; };
    auto my_page = [&](int j) {                                   // the table entry of this lane's piece of its warp's j-th chunk
        const int tile = chunk_tile(j) + my_tile;
        if (my_tile >= QA_KT || tile >= tile1) return 0;
        return (int)table[whole ? tile : min((tile * 16 + key_off) / p.kv.page_size, last_page)];
    };
    auto request = [&](int j, int entry) {
        const int first = chunk_tile(j), n = min(QA_KT, tile1 - first);
        if (n <= 0) return;
        const uint32_t bar = bars + 8 * (j % QA_STAGES);
        if (lane == 0) mbar_expect_tx(bar, n * T::BYTES);
        __syncwarp();
        if (my_tile < n) {
            const int in_page = whole ? 0 : ((first + my_tile) * 16 + key_off) % p.kv.page_size;
            qa_bulk_load(ring_addr + (j % QA_STAGES) * (QA_KT * T::BYTES) + my_dst,
                         my_src + (long long)p.kv.page(entry) * p.kv.page_stride + (long long)in_page * row_bytes, my_bytes, bar);
        }
    };
    int next_entry;
    {
        int e[QA_STAGES];
#pragma unroll
        for (int j = 0; j < QA_STAGES; ++j) e[j] = my_page(j);
        next_entry = my_page(QA_STAGES);
#pragma unroll
        for (int j = 0; j < QA_STAGES; ++j) request(j, e[j]);
    }

    // ---- queries as B fragments, and the factor that brings a row's scores to log2 units
    uint32_t qf[NT == 1 ? HD / 16 : 1][2];
    uint2* const q_smem = reinterpret_cast<uint2*>(qa_smem + T::area(NT));                    // [HD / 16][NT][lane]
    float* const f_smem = reinterpret_cast<float*>(qa_smem + T::area(NT) + HD / 16 * NT * 32 * 8);
    float factor[NT][2];
    auto query_row = [&](int r) {
        const int row = row0 + r, tok = q_start + row / p.group, head = kvh * p.group + row % p.group;
        return p.q + ((long long)tok * p.heads + head) * HD;
    };
    if constexpr (NT == 1) {
        const float f = qa_load_query<HD>(qf, query_row(g < rows ? g : 0), t, g < rows) * p.scale_log2 * 128.f;
        factor[0][0] = __shfl_sync(0xffffffffu, f, 8 * t);
        factor[0][1] = __shfl_sync(0xffffffffu, f, 8 * t + 4);
    } else {
        if (warp < NT) {
            uint32_t f[HD / 16][2];
            const int r = 8 * warp + g;
            const float scale = qa_load_query<HD>(f, query_row(r < rows ? r : 0), t, r < rows) * p.scale_log2 * 128.f;
#pragma unroll
            for (int k = 0; k < HD / 16; ++k) q_smem[(k * NT + warp) * 32 + lane] = make_uint2(f[k][0], f[k][1]);
            if (t == 0) f_smem[r] = scale;
        }
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
    auto row_pos = [&](int n, int c) { return kv_len - q_len + (row0 + min(8 * n + 2 * t + c, rows - 1)) / p.group; };

    for (int j = 0;; ++j) {
        const int first = chunk_tile(j), n_tiles = min(QA_KT, tile1 - first);
        if (n_tiles <= 0) break;
        const uint8_t* const stage = ring + (j % QA_STAGES) * (QA_KT * T::BYTES);
        if (!mbar_wait(bars + 8 * (j % QA_STAGES), (j / QA_STAGES) & 1, 0))
            mbar_wait(bars + 8 * (j % QA_STAGES), (j / QA_STAGES) & 1, 0);      // its copies must not outlive the CTA

        float s[QA_KT][NT][4];
        float top[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) top[n][0] = top[n][1] = -INFINITY;
#pragma unroll
        for (int i = 0; i < QA_KT; ++i) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 4; ++c) s[i][n][c] = i < n_tiles ? 0.f : -INFINITY;
            if (i >= n_tiles) continue;
            const uint8_t* const tile = stage + i * T::BYTES;
            uint32_t wa[KW], wb[KW];                               // this thread's codes of keys g and g + 8
            qa_lds(wa, tile + g * (HD / 2) + t * (HD / 8));
            qa_lds(wb, tile + (g + 8) * (HD / 2) + t * (HD / 8));
            const uint8_t* const st = tile + T::KC + g * (HD / 16) + t * KG;
#pragma unroll
            for (int w = 0; w < KW; ++w) {
                const QaStep sa(st[w / 2] * 0x00010001u), sb(st[8 * (HD / 16) + w / 2] * 0x00010001u);
                uint32_t a[4], b[4];
                qa_widen(a, wa[w], sa);
                qa_widen(b, wb[w], sb);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    uint2 q0, q1;
                    if constexpr (NT == 1) { q0 = make_uint2(qf[2 * w][0], qf[2 * w][1]); q1 = make_uint2(qf[2 * w + 1][0], qf[2 * w + 1][1]); }
                    else { q0 = q_smem[(2 * w * NT + n) * 32 + lane]; q1 = q_smem[((2 * w + 1) * NT + n) * 32 + lane]; }
                    qa_mma(s[i][n], a[0], b[0], a[1], b[1], q0.x, q0.y);
                    qa_mma(s[i][n], a[2], b[2], a[3], b[3], q1.x, q1.y);
                }
            }
            const int key0 = (first + i) * 16;
            const bool partly = key0 + 15 > pos_first || (p.window > 0 && key0 <= pos_last - p.window);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int c = 0; c < 4; ++c) s[i][n][c] *= factor[n][c & 1];
                if (partly) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int key = key0 + g + (c >> 1) * 8, pos = row_pos(n, c & 1);
                        if (key > pos || (p.window > 0 && key <= pos - p.window)) s[i][n][c] = -INFINITY;
                    }
                }
                top[n][0] = fmaxf(top[n][0], fmaxf(s[i][n][0], s[i][n][2]));
                top[n][1] = fmaxf(top[n][1], fmaxf(s[i][n][1], s[i][n][3]));
            }
        }
        bool grew = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) grew = grew || top[n][0] > m[n][0] + QA_LAZY || top[n][1] > m[n][1] + QA_LAZY;
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
        uint32_t pf[QA_KT][NT][2];                                 // weights as B fragments
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float m0 = m[n][0] == -INFINITY ? 0.f : m[n][0], m1 = m[n][1] == -INFINITY ? 0.f : m[n][1];
#pragma unroll
            for (int i = 0; i < QA_KT; ++i) {
                const float p0 = qa_ex2(s[i][n][0] - m0), p1 = qa_ex2(s[i][n][1] - m1), p2 = qa_ex2(s[i][n][2] - m0), p3 = qa_ex2(s[i][n][3] - m1);
                l[n][0] += p0 + p2;
                l[n][1] += p1 + p3;
                pf[i][n][0] = qa_transpose(qa_pack(p0, p1));
                pf[i][n][1] = qa_transpose(qa_pack(p2, p3));
            }
        }
#pragma unroll
        for (int i = 0; i < QA_KT; ++i) {
            if (i >= n_tiles) continue;
            const uint8_t* const tile = stage + i * T::BYTES + T::KC + T::KS;
            const int key0 = (first + i) * 16;
            const bool partly = key0 + 15 > pos_first || (p.window > 0 && key0 <= pos_last - p.window);
            uint32_t w4[4][VW];                                    // codes of keys 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
            for (int k = 0; k < 4; ++k) qa_lds(w4[k], tile + (2 * t + (k & 1) + (k >> 1) * 8) * (HD / 2) + g * (HD / 16));
            uint32_t nan_keys[(VW + 1) / 2];
#pragma unroll
            for (int v = 0; v < VW; ++v) {
                uint32_t by[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) by[k] = tile[T::KC + (2 * t + (k & 1) + (k >> 1) * 8) * (HD / 16) + (g * (HD / 8) + 8 * v) / 16];
                if (partly) {
                    // keys that no row sees may hold anything, and a NaN that some rows see must not reach the others (0 * NaN
                    // is NaN): both count as zero here, and the rows that see a NaN get theirs below
                    if (v % 2 == 0) nan_keys[v / 2] = 0;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int at = 2 * t + (k & 1) + (k >> 1) * 8;
                        const bool in = key0 + at >= kv_lo && key0 + at < kv_hi;
                        if (in && by[k] == Q4_NAN) nan_keys[v / 2] |= 1u << at;
                        if (!in || by[k] == Q4_NAN) by[k] = 0;
                    }
                }
                const QaStep s01(by[0] | by[1] << 16), s89(by[2] | by[3] << 16);
#pragma unroll
                for (int half = 0; half < 2; ++half) {             // codes 0-3 and 4-7 of the words
                    const uint32_t sel = half ? 0x7632u : 0x5410u;
                    uint32_t a[4], b[4];
                    qa_widen(a, __byte_perm(w4[0][v], w4[1][v], sel), s01);
                    qa_widen(b, __byte_perm(w4[2][v], w4[3][v], sel), s89);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        qa_mma(o[4 * v + 2 * half][n], a[0], a[1], b[0], b[1], pf[i][n][0], pf[i][n][1]);
                        qa_mma(o[4 * v + 2 * half + 1][n], a[2], a[3], b[2], b[3], pf[i][n][0], pf[i][n][1]);
                    }
                }
            }
            if (partly) {
#pragma unroll
                for (int v = 0; v < (VW + 1) / 2; ++v) {
                    uint32_t bad = nan_keys[v];
                    bad |= __shfl_xor_sync(0xffffffffu, bad, 1);
                    bad |= __shfl_xor_sync(0xffffffffu, bad, 2);
                    if (bad == 0) continue;
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const int pos = row_pos(n, c);
                            bool sees = false;
                            for (int k = 0; k < 16; ++k)
                                sees = sees || ((bad >> k & 1) && key0 + k <= pos && (p.window <= 0 || key0 + k > pos - p.window));
                            if (!sees) continue;
#pragma unroll
                            for (int k = 0; k < (VW == 1 ? 4 : 8); ++k) o[8 * v + k][n][c] = o[8 * v + k][n][c + 2] = __int_as_float(0x7fc00000);
                        }
                }
            }
        }
        __syncwarp();                                              // every lane is done with the stage
        request(j + QA_STAGES, next_entry);
        next_entry = my_page(j + QA_STAGES + 1);
    }

    // ---- the warps' results side by side in shared memory (the rings are free), merged by all threads
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], 4);
            l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], 8);
            l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], 16);
        }
    __syncthreads();
    constexpr int R = 8 * NT;
    float* const mo = reinterpret_cast<float*>(qa_smem);                       // [warp][row][PITCH]
    float2* const ml = reinterpret_cast<float2*>(mo + QA_WARPS * R * T::PITCH);  // [warp][row]
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int r = 8 * n + 2 * t + c;
            float* const dst = mo + (warp * R + r) * T::PITCH + g * (HD / 8);
#pragma unroll
            for (int k = 0; k < MT; ++k) *reinterpret_cast<float2*>(dst + 2 * k) = make_float2(o[k][n][c], o[k][n][c + 2]);
            if (g == 0) ml[warp * R + r] = make_float2(m[n][c], l[n][c]);
        }
    __syncthreads();
    const long long part0 = (((long long)item * gridDim.y + kvh) * p.n_splits + split) * R;
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
            const float f = qa_ex2(x.x - use);
            const float4 v = *reinterpret_cast<const float4*>(mo + (w * R + r) * T::PITCH + d);
            sum = fmaf(x.y, f, sum);
            acc.x = fmaf(v.x, f, acc.x); acc.y = fmaf(v.y, f, acc.y); acc.z = fmaf(v.z, f, acc.z); acc.w = fmaf(v.w, f, acc.w);
        }
        if (p.n_splits > 1) {
            *reinterpret_cast<float4*>(p.part_o + (part0 + r) * HD + d) = acc;
            if (d == 0) p.part_ml[part0 + r] = make_float2(top, sum);
        } else {
            const float inv = 128.f / sum;                         // (values carry a 1 / 128, as keys do)
            const int row = row0 + r, tok = q_start + row / p.group, head = kvh * p.group + row % p.group;
            const __nv_bfloat162 a = __floats2bfloat162_rn(acc.x * inv, acc.y * inv), b = __floats2bfloat162_rn(acc.z * inv, acc.w * inv);
            *reinterpret_cast<uint2*>(p.out + ((long long)tok * p.heads + head) * HD + d) =
                make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
        }
    }
}

// The shares of each (item, kv head, row), folded in ascending order.  The first eight shares are asked for
// before their weights are known.
constexpr int QA_FOLD_THREADS = 256;
template <int HD, int NT>
__global__ void __launch_bounds__(QA_FOLD_THREADS) attention_q4_fold_kernel(const QaParams p) {
    constexpr int R = 8 * NT, V = HD / 4, S = 8;
    __shared__ float wm[QA_MAX_SPLITS * R], wl[QA_MAX_SPLITS * R];
    pdl_launch_dependents();
    pdl_wait();
    const int item = blockIdx.x, kvh = blockIdx.y;
    const int seg = p.items ? p.items[2 * item] : item, row0 = p.items ? p.items[2 * item + 1] : 0;
    const int q_start = p.segments[p.n_segments + seg], q_len = p.segments[2 * p.n_segments + seg];
    const int rows = min(R, q_len * p.group - row0);
    const long long base = ((long long)item * gridDim.y + kvh) * p.n_splits * R;
    const float4* const po = reinterpret_cast<const float4*>(p.part_o) + base * V;
    for (int e = threadIdx.x; e < p.n_splits * R; e += QA_FOLD_THREADS) {
        if (e % R >= rows) continue;                               // rows past the last are not written
        const float2 x = __ldcg(p.part_ml + base + e);
        wm[e] = x.x;
        wl[e] = x.y;
    }
    __syncthreads();
    if (threadIdx.x < rows) {
        const int r = threadIdx.x;
        float top = -INFINITY, sum = 0.f;
        for (int s = 0; s < p.n_splits; ++s) top = fmaxf(top, wm[s * R + r]);
        const float use = top == -INFINITY ? 0.f : top;
        for (int s = 0; s < p.n_splits; ++s) {
            const float f = qa_ex2(wm[s * R + r] - use);
            sum = fmaf(wl[s * R + r], f, sum);
            wm[s * R + r] = f;
        }
        wl[r] = 128.f / sum;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < rows * V; e += QA_FOLD_THREADS) {
        const int r = e / V, d = e % V * 4;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int s0 = 0; s0 < p.n_splits; s0 += S) {
            float4 v[S];
#pragma unroll
            for (int q = 0; q < S; ++q)
                v[q] = s0 + q < p.n_splits ? __ldcg(po + (long long)(s0 + q) * R * V + e) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int q = 0; q < S; ++q) {
                const float f = s0 + q < p.n_splits ? wm[(s0 + q) * R + r] : 0.f;
                acc.x = fmaf(v[q].x, f, acc.x); acc.y = fmaf(v[q].y, f, acc.y); acc.z = fmaf(v[q].z, f, acc.z); acc.w = fmaf(v[q].w, f, acc.w);
            }
        }
        const float inv = wl[r];
        const int row = row0 + r, tok = q_start + row / p.group, head = kvh * p.group + row % p.group;
        const __nv_bfloat162 a = __floats2bfloat162_rn(acc.x * inv, acc.y * inv), b = __floats2bfloat162_rn(acc.z * inv, acc.w * inv);
        *reinterpret_cast<uint2*>(p.out + ((long long)tok * p.heads + head) * HD + d) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
}

template <int HD, int NT>
static int launch_q4(const QaParams& p, int n_items, cudaStream_t stream) {
    constexpr int smem = QaTile<HD>::smem(NT);
    static_assert(smem <= 226 * 1024, "the rings do not fit shared memory");
    if (int st = ensure_dynamic_smem<attention_q4_kernel<HD, NT>>(smem, "axon_attention_q4")) return st;
    launch_pdl(attention_q4_kernel<HD, NT>, dim3(n_items, p.kv.kv_heads, p.n_splits), dim3(QA_THREADS), smem, stream, p);
    if (int st = launch_status("axon_attention_q4")) return st;
    if (p.n_splits > 1) {
        launch_pdl(attention_q4_fold_kernel<HD, NT>, dim3(n_items, p.kv.kv_heads), dim3(QA_FOLD_THREADS), 0, stream, p);
        return launch_status("axon_attention_q4 fold");
    }
    return AXON_OK;
}

}  // namespace axon

using namespace axon;

// Attention of `n_items` tiles of up to 8 * row_tiles query rows (row_tiles 1, 2 or 4; at head size 256 1 or 2).  items null:
// item i is segment i, whose rows all fit one tile.  With several splits scratch holds
// n_items * kv_heads * splits * 8 * row_tiles * (head_dim + 2) floats.
AXON_API int axon_attention_q4(const void* q, const void* pool, void* out, const int32_t* segments, int n_segments,
                               const int32_t* items, int n_items, const AxonKvLayout* layout, int heads, float scale, int window,
                               int row_tiles, int n_splits, float* scratch, long long scratch_floats, cudaStream_t stream) {
    if (n_items <= 0) return AXON_OK;
    QaParams p;
    if (int st = to_q4(layout, pool, "axon_attention_q4", &p.kv)) return st;
    const int hd = p.kv.hd;
    if (p.kv.planes != 2 || p.kv.vd != hd) { set_error("axon_attention_q4: takes caches with key and value planes of one width"); return AXON_BAD_ARGUMENT; }
    if (heads < 1 || heads % p.kv.kv_heads) { set_error("axon_attention_q4: %d heads over %d kv heads", heads, p.kv.kv_heads); return AXON_BAD_ARGUMENT; }
    if (n_splits < 1 || n_splits > QA_MAX_SPLITS || p.kv.kv_heads > 65535) { set_error("axon_attention_q4: bad split count %d (1..%d)", n_splits, QA_MAX_SPLITS); return AXON_BAD_ARGUMENT; }
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)scratch) & 15) { set_error("axon_attention_q4: operands must be 16-byte aligned"); return AXON_BAD_ARGUMENT; }
    p.run = 1;
    while (p.run < 16 && p.kv.page_size % (2 * p.run) == 0) p.run *= 2;
    // a copy moves whole 16 bytes, and a lane each must do for the pieces of a chunk
    if (p.run * hd / 16 % 16 || QA_KT * (p.kv.page_size == 16 ? 1 : 64 / p.run) > 32) { set_error("axon_attention_q4: pages of %d positions of %d values do not fall into pieces it can copy", p.kv.page_size, hd); return AXON_BAD_ARGUMENT; }
    const long long per = (long long)n_items * p.kv.kv_heads * n_splits * 8 * row_tiles;
    if (n_splits > 1 && (scratch == nullptr || scratch_floats < per * (hd + 2))) { set_error("axon_attention_q4: %d key shares need %lld floats of scratch", n_splits, per * (hd + 2)); return AXON_BAD_ARGUMENT; }
    p.q = (const __nv_bfloat16*)q; p.pool = (const uint8_t*)pool; p.out = (__nv_bfloat16*)out;
    p.segments = segments; p.items = items;
    p.part_o = scratch; p.part_ml = scratch ? reinterpret_cast<float2*>(scratch + per * hd) : nullptr;
    p.n_segments = n_segments; p.heads = heads; p.group = heads / p.kv.kv_heads; p.n_splits = n_splits; p.window = window;
    p.scale_log2 = scale * 1.4426950408889634f;
#define AXON_Q4_CASE(HD, NT) if (hd == HD && row_tiles == NT) return launch_q4<HD, NT>(p, n_items, stream)
    AXON_Q4_CASE(64, 1); AXON_Q4_CASE(64, 2); AXON_Q4_CASE(64, 4);
    AXON_Q4_CASE(128, 1); AXON_Q4_CASE(128, 2); AXON_Q4_CASE(128, 4);
    AXON_Q4_CASE(256, 1); AXON_Q4_CASE(256, 2);
#undef AXON_Q4_CASE
    set_error("axon_attention_q4: no kernel for head size %d with %d tiles of 8 rows", hd, row_tiles);
    return AXON_BAD_ARGUMENT;
}

AXON_API int axon_attention_q4_status() {
    unsigned int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_tc_error, sizeof v) != cudaSuccess) return -1;
    return (int)v;
}
