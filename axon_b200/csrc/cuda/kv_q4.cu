// The 4-bit cache's plain operators: rotating and quantising rows as they are written, reading
// positions back, attention for any sizes, and the fold of partial results of key shares.  The format is in
// kv_layout.h, the arithmetic in kv_q4.cuh.
#include "kv_q4.cuh"

#include <type_traits>

namespace axon {

__device__ __forceinline__ float4 q4_load4(const float* row, const SplitFold& fold, int t, int n) {
    return fold.partial ? fold.at4(t, n) : *reinterpret_cast<const float4*>(row + n);
}

// Rotation and quantised cache write: a warp per (token, head) row, four consecutive channels a
// lane, so that a group of 16 is four neighbouring lanes (two shuffles for its maximum) and a lane's codes are two
// whole bytes.  Rotated values are products and sums rounded to 32 bits one by one (no
// fused multiply-add), so a key's codes do not depend on how a compiler contracts them.  VEC: rows
// and the rotation table are read as float4s (rot % 8 == 0, 16-byte aligned operands).
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
rope_kv_write_q4_kernel(const float* __restrict__ qkv, const float2* __restrict__ table, const int32_t* __restrict__ positions,
                        const int32_t* __restrict__ token_slot, T* __restrict__ q_out, uint8_t* __restrict__ pool, PagedQ4 kv,
                        int heads, int rot, int adjacent, int write_kv, SplitFold fold) {
    pdl_launch_dependents();
    pdl_wait();
    const int t = blockIdx.x, lane = threadIdx.x & 31;
    const int h = blockIdx.y * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int rows = heads + kv.planes * kv.kv_heads;
    if (h >= rows || (h >= heads && !write_kv)) return;
    const bool is_v = h >= heads + kv.kv_heads;
    const int q_dim = heads * kv.hd, k_dim = kv.kv_heads * kv.hd;
    const int width = is_v ? kv.vd : kv.hd;
    const int col = is_v ? q_dim + k_dim + (h - heads - kv.kv_heads) * kv.vd : h * kv.hd;
    const float* row = qkv + (long long)t * (q_dim + k_dim + (kv.planes == 2 ? kv.kv_heads * kv.vd : 0));
    const int rhalf = rot / 2;
    const float2* cs = table + (long long)t * rhalf;
    uint8_t *codes = nullptr, *steps = nullptr;
    if (h >= heads) {
        const int pos = positions[t], lp = pos / kv.page_size, in_page = pos - lp * kv.page_size;
        uint8_t* rec = pool + kv.record_at(token_slot[t], lp, is_v ? h - heads - kv.kv_heads : h - heads);
        codes = rec + (is_v ? kv.v_codes : 0) + (long long)in_page * (width / 2);
        steps = rec + (is_v ? kv.v_steps : kv.k_steps) + (long long)in_page * (width / Q4_GROUP);
    }
    for (int base = 0; base < width; base += 128) {
        const int c0 = base + 4 * lane;
        const bool mine = c0 < width;                          // whole groups of four lanes have or have not
        float x[4] = {0.f, 0.f, 0.f, 0.f};
        if (mine) {
            if (VEC) {
                const float4 own = q4_load4(row, fold, t, col + c0);
                x[0] = own.x; x[1] = own.y; x[2] = own.z; x[3] = own.w;
                if (!is_v && table != nullptr && c0 < rot) {
                    if (adjacent) {
                        const float4 w = *reinterpret_cast<const float4*>(cs + c0 / 2);
                        x[0] = __fsub_rn(__fmul_rn(own.x, w.x), __fmul_rn(own.y, w.y));
                        x[1] = __fadd_rn(__fmul_rn(own.x, w.y), __fmul_rn(own.y, w.x));
                        x[2] = __fsub_rn(__fmul_rn(own.z, w.z), __fmul_rn(own.w, w.w));
                        x[3] = __fadd_rn(__fmul_rn(own.z, w.w), __fmul_rn(own.w, w.z));
                    } else {
                        const bool first = c0 < rhalf;
                        const int i0 = first ? c0 : c0 - rhalf;
                        const float4 other = q4_load4(row, fold, t, col + (first ? c0 + rhalf : i0));
                        const float4 w01 = *reinterpret_cast<const float4*>(cs + i0), w23 = *reinterpret_cast<const float4*>(cs + i0 + 2);
                        const float o[4] = {other.x, other.y, other.z, other.w};
                        const float c[4] = {w01.x, w01.z, w23.x, w23.z}, s[4] = {w01.y, w01.w, w23.y, w23.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            x[j] = first ? __fsub_rn(__fmul_rn(x[j], c[j]), __fmul_rn(o[j], s[j]))
                                         : __fadd_rn(__fmul_rn(o[j], s[j]), __fmul_rn(x[j], c[j]));
                    }
                }
            } else {
                auto at = [&](int n) { return fold.partial ? fold.at(t, col + n) : row[col + n]; };
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int c = c0 + j;
                    x[j] = at(c);
                    if (!is_v && table != nullptr && c < rot) {
                        const bool first = adjacent ? !(c & 1) : c < rhalf;
                        const int i = adjacent ? c >> 1 : first ? c : c - rhalf;
                        const float o = at(adjacent ? c ^ 1 : first ? c + rhalf : c - rhalf);
                        const float2 w = cs[i];
                        x[j] = first ? __fsub_rn(__fmul_rn(x[j], w.x), __fmul_rn(o, w.y))
                                     : __fadd_rn(__fmul_rn(o, w.y), __fmul_rn(x[j], w.x));
                    }
                }
            }
        }
        if (h < heads) {
            if (mine) {
                T* dst = q_out + (long long)t * q_dim + col + c0;
                stf(dst, x[0]); stf(dst + 1, x[1]); stf(dst + 2, x[2]); stf(dst + 3, x[3]);
            }
            continue;
        }
        // magnitudes compare as integers, and what is not finite is larger than all that is
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) top = max(top, __float_as_uint(x[j]) & 0x7fffffffu);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int byte = q4_step_byte(top);
        const float inv = q4_inverse(byte);
        const uint32_t two = q4_codes4(x[0], x[1], x[2], x[3], byte, inv);
        if (mine) {
            *reinterpret_cast<uint16_t*>(codes + c0 / 2) = (uint16_t)two;
            if ((lane & 3) == 0) steps[c0 / Q4_GROUP] = (uint8_t)byte;
        }
    }
}

// The same for the common layout (pairs (i, i + hd / 2) over the whole head, hd % 32 == 0, keys and values of one
// width, 16-byte aligned operands): a thread owns four channels of each half of a row, so that nothing is read twice
// and the groups of both halves are again four neighbouring lanes.  2,048 tokens at 28 + 4 + 4 heads of 128 move
// 57 MB in 12.3 us (0.71 of the measured copy rate), 12.9 where the step is not staged; one token takes 1.9 and 2.2 us.
template <typename T>
__device__ __forceinline__ void q4_store4(T* dst, const float (&x)[4]);
template <>
__device__ __forceinline__ void q4_store4<float>(float* dst, const float (&x)[4]) {
    *reinterpret_cast<float4*>(dst) = make_float4(x[0], x[1], x[2], x[3]);
}
template <>
__device__ __forceinline__ void q4_store4<__nv_bfloat16>(__nv_bfloat16* dst, const float (&x)[4]) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
    *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}
constexpr int Q4_WRITE_THREADS = 192;
template <typename T>
__global__ void __launch_bounds__(Q4_WRITE_THREADS)
rope_kv_write_q4_vec_kernel(const float* __restrict__ qkv, const float2* __restrict__ table, const int32_t* __restrict__ positions,
                            const int32_t* __restrict__ token_slot, T* __restrict__ q_out, uint8_t* __restrict__ pool, PagedQ4 kv,
                            int heads, int write_kv, int staged, SplitFold fold) {
    pdl_launch_dependents();
    if (!staged) pdl_wait();
    const int t = blockIdx.x, half = kv.hd / 2, lanes = half / 4;                  // threads of a row
    const int items = (heads + (write_kv ? 2 * kv.kv_heads : 0)) * lanes;
    const float* row = qkv + (long long)t * ((heads + 2 * kv.kv_heads) * kv.hd);
    // (staged positions, slots and tables are no work of the kernel before: no need to wait for it)
    const int pos = positions[t], lp = pos / kv.page_size, in_page = pos - lp * kv.page_size;
    const int entry = write_kv ? kv.block_table[(long long)token_slot[t] * kv.table_stride + lp] : 0;
    pdl_wait();
    const long long page = (long long)kv.page(entry) * kv.page_stride + kv.entry_offset;
    // (the items of a row are a multiple of four, so the lanes of a group are all here or all beyond the last item)
    for (int it = blockIdx.y * Q4_WRITE_THREADS + threadIdx.x; it < items; it += gridDim.y * Q4_WRITE_THREADS) {
        const int h = it / lanes, i0 = (it - h * lanes) * 4, col = h * kv.hd;
        const float4 a4 = q4_load4(row, fold, t, col + i0), b4 = q4_load4(row, fold, t, col + half + i0);
        float a[4] = {a4.x, a4.y, a4.z, a4.w}, b[4] = {b4.x, b4.y, b4.z, b4.w};
        if (h < heads + kv.kv_heads) {
            const float4 w01 = *reinterpret_cast<const float4*>(table + (long long)t * half + i0), w23 = *reinterpret_cast<const float4*>(table + (long long)t * half + i0 + 2);
            const float c[4] = {w01.x, w01.z, w23.x, w23.z}, s[4] = {w01.y, w01.w, w23.y, w23.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float x = a[j], y = b[j];
                a[j] = __fsub_rn(__fmul_rn(x, c[j]), __fmul_rn(y, s[j]));
                b[j] = __fadd_rn(__fmul_rn(x, s[j]), __fmul_rn(y, c[j]));
            }
        }
        if (h < heads) {
            T* dst = q_out + (long long)t * (heads * kv.hd) + col + i0;
            q4_store4<T>(dst, a);
            q4_store4<T>(dst + half, b);
            continue;
        }
        const bool is_v = h >= heads + kv.kv_heads;
        uint8_t* rec = pool + page + (long long)(is_v ? h - heads - kv.kv_heads : h - heads) * kv.record;
        uint8_t* codes = rec + (is_v ? kv.v_codes : 0) + (long long)in_page * (kv.hd / 2) + i0 / 2;
        uint8_t* steps = rec + (is_v ? kv.v_steps : kv.k_steps) + (long long)in_page * (kv.hd / Q4_GROUP) + i0 / Q4_GROUP;
        const unsigned group = 0xFu << (threadIdx.x & 28);
#pragma unroll
        for (int part = 0; part < 2; ++part) {
            const float x[4] = {part ? b[0] : a[0], part ? b[1] : a[1], part ? b[2] : a[2], part ? b[3] : a[3]};
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) top = max(top, __float_as_uint(x[j]) & 0x7fffffffu);
            top = max(top, __shfl_xor_sync(group, top, 1));
            top = max(top, __shfl_xor_sync(group, top, 2));
            const int byte = q4_step_byte(top);
            const float inv = q4_inverse(byte);
            const uint32_t two = q4_codes4(x[0], x[1], x[2], x[3], byte, inv);
            *reinterpret_cast<uint16_t*>(codes + part * (half / 2)) = (uint16_t)two;
            if ((threadIdx.x & 3) == 0) steps[part * (half / Q4_GROUP)] = (uint8_t)byte;
        }
    }
}

// Positions back as rows of T.  A CTA owns up to 32 consecutive rows of the output: its first
// threads find each row's span and page once, then every thread takes one word of eight codes of a row through all heads
// and both planes, several loads at a time; neighbouring threads go along a row and then along positions,
// which is how both sides lie in memory.  Output row r of plane p and kv head h starts at
//   (r / block) * block_stride + (r % block) * row_stride + h * head_stride,   block = 2^block_shift.
// 32,700 positions of 4 heads of 128 in bfloat16, 19 MB read and 67 MB written: 21.7 us (0.6 of the measured copy rate).
struct Q4Out {
    void *k, *v;
    long long block_stride, row_stride, head_stride;
    int block_shift;
};
template <typename T>
__device__ __forceinline__ void q4_store8(T* dst, uint32_t word, int byte);
template <>
__device__ __forceinline__ void q4_store8<float>(float* dst, uint32_t word, int byte) {
    const float s = q4_step(byte);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = q4_digit(word, i) * s;
    reinterpret_cast<float4*>(dst)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(dst)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
// In bfloat16 a code in the last four bits of 128 + code, and one fused multiply-add that takes 136 s away: (c - 8) s
// has seven significant bits and 136 s eight, so nothing is rounded.
template <>
__device__ __forceinline__ void q4_store8<__nv_bfloat16>(__nv_bfloat16* dst, uint32_t word, int byte) {
    const __nv_bfloat162 s = __float2bfloat162_rn(q4_step(byte)), less = __hmul2(s, __float2bfloat162_rn(-136.f));
    uint32_t v[4];                                             // codes (i, i + 4)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t c = ((word >> (4 * i)) & 0x000F000Fu) | 0x43004300u;
        const __nv_bfloat162 x = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&c), s, less);
        v[i] = *reinterpret_cast<const uint32_t*>(&x);
    }
    *reinterpret_cast<uint4*>(dst) = make_uint4(__byte_perm(v[0], v[1], 0x5410), __byte_perm(v[2], v[3], 0x5410),
                                                __byte_perm(v[0], v[1], 0x7632), __byte_perm(v[2], v[3], 0x7632));
}

constexpr int Q4_READ_ROWS = 32, Q4_READ_THREADS = 256, Q4_READ_BATCH = 4;      // (threads: for one plane, or half for each of two)
// Writes a CTA's rows r0 .. once `rec` (a row's record of kv head 0; -1: not written, -2: zeros) and `at` (its place in
// the page) are known.  ATTEND (both planes, of one width): rows for an attention that multiplies values with weights of zero
// where a token does not see them.  Values of a group that is not finite become zeros, and the same channels of their key NaN
// instead: a score that a mask hides is hidden whatever it is, so such a value reaches the tokens that see it (all
// channels of the head) and no others.
template <typename T, bool ATTEND>
__device__ __forceinline__ void q4_read_rows(const uint8_t* __restrict__ pool, const PagedQ4& kv, const long long* rec, const int* at,
                                             long long r0, int rows_per_cta, const Q4Out& out) {
    // with both planes to write the first half of the threads takes keys, the second values
    const bool both = out.k != nullptr && out.v != nullptr, is_v = both ? threadIdx.x >= Q4_READ_THREADS / 2 : out.v != nullptr;
    const int threads = both ? Q4_READ_THREADS / 2 : Q4_READ_THREADS, tid = both ? threadIdx.x % (Q4_READ_THREADS / 2) : threadIdx.x;
    T* const base = (T*)(is_v ? out.v : out.k);
    const int words = (is_v ? kv.vd : kv.hd) / 8, codes = is_v ? kv.v_codes : 0, steps = is_v ? kv.v_steps : kv.k_steps;
    const int r_step = max(threads / words, 1), to_value = is_v ? 0 : kv.v_steps - kv.k_steps;
    for (int i = tid; i < (threads / words > 0 ? r_step * words : words); i += threads) {      // (a row of more words than threads: several of them)
        const int w = i % words;
        constexpr int ROWS = 2;                                // a thread's rows whose loads are in flight together
        for (int ra = i / words; ra < rows_per_cta; ra += ROWS * r_step) {
            long long where[ROWS];
            const uint8_t *word_at[ROWS], *step_at[ROWS];
            T* dst[ROWS];
#pragma unroll
            for (int q = 0; q < ROWS; ++q) {
                const int r = ra + q * r_step;
                where[q] = r < rows_per_cta ? rec[r] : -1;
                const long long row = r0 + r;
                const int place = where[q] >= 0 ? at[r] : 0;
                // (rows that hold nothing load from the pool's start and store zeros, or store nothing)
                word_at[q] = pool + (where[q] >= 0 ? where[q] : 0) + codes + (place * words + w) * 4;
                step_at[q] = pool + (where[q] >= 0 ? where[q] : 0) + steps + place * (words / 2) + w / 2;
                dst[q] = base + (row >> out.block_shift) * out.block_stride + (row & ((1 << out.block_shift) - 1)) * out.row_stride + w * 8;
            }
            auto batch = [&](auto n) {                         // `n` heads
                uint32_t word[ROWS][decltype(n)::value];
                int byte[ROWS][decltype(n)::value], of_value[ROWS][decltype(n)::value];
#pragma unroll
                for (int q = 0; q < ROWS; ++q)
#pragma unroll
                    for (int k = 0; k < decltype(n)::value; ++k) {
                        word[q][k] = *reinterpret_cast<const uint32_t*>(word_at[q] + k * kv.record);
                        byte[q][k] = step_at[q][k * kv.record];
                        if (ATTEND) of_value[q][k] = step_at[q][k * kv.record + to_value];
                    }
#pragma unroll
                for (int q = 0; q < ROWS; ++q)
#pragma unroll
                    for (int k = 0; k < decltype(n)::value; ++k)
                        if (ATTEND && of_value[q][k] == Q4_NAN) byte[q][k] = is_v ? 0 : Q4_NAN;
#pragma unroll
                for (int q = 0; q < ROWS; ++q) {
                    if (where[q] != -1) {
#pragma unroll
                        for (int k = 0; k < decltype(n)::value; ++k)
                            q4_store8<T>(dst[q] + k * out.head_stride, where[q] >= 0 ? word[q][k] : 0x88888888u, where[q] >= 0 ? byte[q][k] : 0);
                    }
                    word_at[q] += decltype(n)::value * kv.record;
                    step_at[q] += decltype(n)::value * kv.record;
                    dst[q] += decltype(n)::value * out.head_stride;
                }
            };
            int h = 0;
            for (; h + Q4_READ_BATCH <= kv.kv_heads; h += Q4_READ_BATCH) batch(std::integral_constant<int, Q4_READ_BATCH>());
            for (; h < kv.kv_heads; ++h) batch(std::integral_constant<int, 1>());
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(Q4_READ_THREADS)
kv_read_q4_kernel(const uint8_t* __restrict__ pool, PagedQ4 kv, const int32_t* __restrict__ spans, int n_spans, int n_slots,
                  long long n_rows, int rows_per_cta, Q4Out out) {
    __shared__ long long rec[Q4_READ_ROWS];
    __shared__ int at[Q4_READ_ROWS];
    __shared__ int owner[Q4_READ_ROWS];                        // the first span that covers it
    if (threadIdx.x < Q4_READ_ROWS) owner[threadIdx.x] = n_spans;
    pdl_launch_dependents();
    pdl_wait();
    const long long r0 = (long long)blockIdx.x * rows_per_cta, r1 = min(r0 + rows_per_cta, n_rows);
    __syncthreads();
    for (int s = threadIdx.x; s < n_spans; s += Q4_READ_THREADS) {
        const long long out0 = spans[3 * n_spans + s], count = max(spans[2 * n_spans + s], 0);
        const long long a = max(out0, r0), b = min(out0 + count, r1);
        for (long long r = a; r < b; ++r) atomicMin(&owner[r - r0], s);
    }
    __syncthreads();
    if (threadIdx.x < rows_per_cta) {
        const int s = owner[threadIdx.x];
        long long where = -1;
        int in_page = 0;
        if (s < n_spans) {
            const long long i = r0 + threadIdx.x - spans[3 * n_spans + s];
            const int slot = spans[s];
            const long long pos = spans[n_spans + s] + i, lp = pos / kv.page_size;
            if (slot >= 0 && slot < n_slots && pos >= 0 && lp < kv.table_stride) {
                where = kv.record_at(slot, (int)lp, 0);
                in_page = (int)(pos - lp * kv.page_size);
            }
        }
        rec[threadIdx.x] = where;
        at[threadIdx.x] = in_page;
    }
    __syncthreads();
    q4_read_rows<T, false>(pool, kv, rec, at, r0, rows_per_cta, out);
}

// Keys and values of whole prompts for the attention that takes bfloat16 pages: of each of the n_long segments named in `which`
// the positions that its rows see, from a multiple of 64 on, one segment after another in pages of 64 positions
// (two CTAs a page; rows behind a segment's last position are zeros).  The CTA at a segment's first page also writes what
// that attention needs to find them: the segment counted from its first position here (`seg_out` [4][n_long]) and its row of
// `table` [n_long][stride].  What `pages` and `stride` do not hold is left out (the host sizes both from the same lengths).
template <typename T>
__global__ void __launch_bounds__(Q4_READ_THREADS)
kv_read_q4_pages_kernel(const uint8_t* __restrict__ pool, PagedQ4 kv, const int32_t* __restrict__ segments, int n_segments,
                        const int32_t* __restrict__ which, int n_long, int window, int pages, int stride, int staged,
                        int32_t* __restrict__ seg_out, int32_t* __restrict__ table, Q4Out out) {
    __shared__ long long rec[Q4_READ_ROWS];
    __shared__ int at[Q4_READ_ROWS];
    __shared__ int who, first_page, lo, count;
    pdl_launch_dependents();
    if (!staged) pdl_wait();
    const int page = blockIdx.x / 2;
    if (threadIdx.x == 0) who = -1;
    __syncthreads();
    if (threadIdx.x < 32) {
        int base = 0;
        for (int i0 = 0; i0 < n_long; i0 += 32) {
            const int i = i0 + threadIdx.x;
            int from = 0, keys = 0, n = 0;
            if (i < n_long) {
                const int q_len = segments[2 * n_segments + which[i]], kv_len = segments[3 * n_segments + which[i]];
                from = window > 0 ? max(kv_len - q_len - window + 1, 0) / 64 * 64 : 0;
                keys = kv_len - from;
                n = min((keys + 63) / 64, stride);
            }
            int upto = n;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, upto, d);
                if ((int)threadIdx.x >= d) upto += x;
            }
            if (page >= base + upto - n && page < base + upto) { who = i; first_page = base + upto - n; lo = from; count = min(keys, n * 64); }
            base += __shfl_sync(0xffffffffu, upto, 31);
            if (base > page) break;
        }
    }
    pdl_wait();
    __syncthreads();
    if (who < 0) return;
    const int seg = which[who], slot = segments[seg];
    if (page == first_page && blockIdx.x % 2 == 0) {
        if (threadIdx.x == 0) {
            seg_out[who] = who;
            seg_out[n_long + who] = segments[n_segments + seg];
            seg_out[2 * n_long + who] = segments[2 * n_segments + seg];
            seg_out[3 * n_long + who] = count;
        }
        for (int j = threadIdx.x; j < stride; j += Q4_READ_THREADS) table[(long long)who * stride + j] = min(first_page + j, pages - 1);
    }
    const long long r0 = (long long)page * 64 + blockIdx.x % 2 * Q4_READ_ROWS;
    if (threadIdx.x < Q4_READ_ROWS) {
        const int i = (int)(r0 - (long long)first_page * 64) + threadIdx.x, pos = lo + i, lp = pos / kv.page_size;
        const bool held = i < count && lp < kv.table_stride;
        rec[threadIdx.x] = held ? kv.record_at(slot, lp, 0) : -2;
        at[threadIdx.x] = held ? pos - lp * kv.page_size : 0;
    }
    __syncthreads();
    q4_read_rows<T, true>(pool, kv, rec, at, r0, Q4_READ_ROWS, out);
}

// ---------------------------------------------------------------------------
// Causal attention for any sizes (and the 32-bit model): a CTA per (token, up to eight heads of
// a kv head, share of the keys).  64 keys at a time are widened to float in shared memory, scored by FFMA
// (a thread per key and four heads), folded with a running maximum and sum, then the same
// tile holds the values (a thread per channel and eight heads).  Scores are in log2 units.
constexpr int Q4P_KEYS = 64, Q4P_HEADS = 8, Q4P_THREADS = 128;

template <typename T>
__global__ void __launch_bounds__(Q4P_THREADS)
attention_q4_plain_kernel(const T* __restrict__ q, const uint8_t* __restrict__ pool, const int32_t* __restrict__ positions,
                          const int32_t* __restrict__ token_slot, T* __restrict__ out, PagedQ4 kv, int heads, float scale_log2,
                          int window, float* __restrict__ part_o, float2* __restrict__ part_ml, unsigned int* __restrict__ arrived) {
    extern __shared__ float q4p_smem[];
    const int hd = kv.hd, vd = kv.vd, group = heads / kv.kv_heads, blocks = (group + Q4P_HEADS - 1) / Q4P_HEADS;
    const int t = blockIdx.x, kh = blockIdx.y / blocks, h0 = kh * group + blockIdx.y % blocks * Q4P_HEADS;
    const int n_heads = min(Q4P_HEADS, (kh + 1) * group - h0);
    const int pitch = max(hd, vd) + 1;                         // odd: a column of the tile falls into 32 banks
    float* qs = q4p_smem;                                      // [hd][8]
    float* tile = qs + Q4P_HEADS * hd;                         // [64][pitch]
    float* sc = tile + Q4P_KEYS * pitch;                       // [64][8] scores, then weights
    __shared__ float m_run[Q4P_HEADS], l_run[Q4P_HEADS], corr[Q4P_HEADS];
    __shared__ long long rec[Q4P_KEYS];
    __shared__ int at[Q4P_KEYS];
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, pos = positions[t], slot = token_slot[t];
    const int lo_all = (window > 0 && pos - window + 1 > 0) ? pos - window + 1 : 0;
    const int tiles = (pos + 1 - lo_all + Q4P_KEYS - 1) / Q4P_KEYS, per = (tiles + gridDim.z - 1) / gridDim.z;
    const int lo = lo_all + (int)blockIdx.z * per * Q4P_KEYS, hi = min(pos + 1, lo + per * Q4P_KEYS);
    for (int i = tid; i < Q4P_HEADS * hd; i += Q4P_THREADS)
        qs[i % hd * Q4P_HEADS + i / hd] = i / hd < n_heads ? ldf(q + ((long long)t * heads + h0) * hd + i) * scale_log2 : 0.f;
    if (tid < Q4P_HEADS) { m_run[tid] = -INFINITY; l_run[tid] = 0.f; }
    float acc[2][Q4P_HEADS];
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < Q4P_HEADS; ++i) acc[c][i] = 0.f;
    const int key = tid & 63, half = tid >> 6;

    for (int p0 = lo; p0 < hi; p0 += Q4P_KEYS) {
        const int cnt = min(Q4P_KEYS, hi - p0);
        __syncthreads();                                       // the tile before has been used
        if (tid < cnt) {
            const int lp = (p0 + tid) / kv.page_size;
            rec[tid] = kv.record_at(slot, lp, kh);
            at[tid] = p0 + tid - lp * kv.page_size;
        }
        __syncthreads();
        auto widen = [&](int codes, int steps, int width) {
            constexpr int BATCH = 4;                           // words of a thread in flight together
            const int words = width / 8;
            for (int i0 = tid; i0 < cnt * words; i0 += BATCH * Q4P_THREADS) {
                uint32_t word[BATCH];
                int byte[BATCH];
#pragma unroll
                for (int k = 0; k < BATCH; ++k) {
                    const int i = i0 + k * Q4P_THREADS, r = i / words, w = i - r * words;
                    if (i >= cnt * words) continue;
                    const uint8_t* from = pool + rec[r];
                    word[k] = *reinterpret_cast<const uint32_t*>(from + codes + ((long long)at[r] * words + w) * 4);
                    byte[k] = from[steps + (long long)at[r] * (words / 2) + w / 2];
                }
#pragma unroll
                for (int k = 0; k < BATCH; ++k) {
                    const int i = i0 + k * Q4P_THREADS, r = i / words, w = i - r * words;
                    if (i >= cnt * words) continue;
                    const float s = q4_step(byte[k]);
#pragma unroll
                    for (int j = 0; j < 8; ++j) tile[r * pitch + w * 8 + j] = q4_digit(word[k], j) * s;
                }
            }
        };
        widen(0, kv.k_steps, hd);
        __syncthreads();
        {
            float s[4] = {0.f, 0.f, 0.f, 0.f};
            if (key < cnt) {
                const float* kr = tile + key * pitch;
                for (int d = 0; d < hd; ++d) {
                    const float k = kr[d];
                    const float4 x = *reinterpret_cast<const float4*>(qs + d * Q4P_HEADS + half * 4);
                    s[0] = fmaf(x.x, k, s[0]); s[1] = fmaf(x.y, k, s[1]); s[2] = fmaf(x.z, k, s[2]); s[3] = fmaf(x.w, k, s[3]);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[key * Q4P_HEADS + half * 4 + i] = key < cnt ? s[i] : -INFINITY;
        }
        __syncthreads();
        // a warp per two heads: maximum, weights and sum of the tile's 64 scores
        {
            const int warp = tid >> 5, lane = tid & 31;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int h = warp * 2 + i;
                const float a = sc[lane * Q4P_HEADS + h], b = sc[(lane + 32) * Q4P_HEADS + h];
                const float m_old = m_run[h], m_new = fmaxf(m_old, warp_max(fmaxf(a, b)));
                const float use = m_new == -INFINITY ? 0.f : m_new;
                const float pa = exp2f(a - use), pb = exp2f(b - use);
                const float l = warp_sum(pa + pb);
                sc[lane * Q4P_HEADS + h] = pa;
                sc[(lane + 32) * Q4P_HEADS + h] = pb;
                __syncwarp();
                if (lane == 0) {
                    const float f = exp2f(m_old - use);
                    corr[h] = f;
                    l_run[h] = l_run[h] * f + l;
                    m_run[h] = m_new;
                }
            }
        }
        widen(kv.v_codes, kv.v_steps, vd);
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < Q4P_HEADS; ++i) acc[c][i] *= corr[i];
        for (int j = 0; j < cnt; ++j) {
            const float4 a = *reinterpret_cast<const float4*>(sc + j * Q4P_HEADS), b = *reinterpret_cast<const float4*>(sc + j * Q4P_HEADS + 4);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int d = tid + c * Q4P_THREADS;
                if (d < vd) {
                    const float v = tile[j * pitch + d];
                    acc[c][0] = fmaf(a.x, v, acc[c][0]); acc[c][1] = fmaf(a.y, v, acc[c][1]);
                    acc[c][2] = fmaf(a.z, v, acc[c][2]); acc[c][3] = fmaf(a.w, v, acc[c][3]);
                    acc[c][4] = fmaf(b.x, v, acc[c][4]); acc[c][5] = fmaf(b.y, v, acc[c][5]);
                    acc[c][6] = fmaf(b.z, v, acc[c][6]); acc[c][7] = fmaf(b.w, v, acc[c][7]);
                }
            }
        }
    }
    __syncthreads();
    const long long part = (((long long)t * gridDim.y + blockIdx.y) * gridDim.z + blockIdx.z) * Q4P_HEADS;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const int d = tid + c * Q4P_THREADS;
        if (d >= vd) continue;
#pragma unroll
        for (int i = 0; i < Q4P_HEADS; ++i) {
            if (i >= n_heads) continue;
            if (part_o == nullptr) stf(out + ((long long)t * heads + h0 + i) * vd + d, acc[c][i] / l_run[i]);
            else part_o[(part + i) * vd + d] = acc[c][i];
        }
    }
    if (part_o == nullptr) return;
    if (tid < Q4P_HEADS) part_ml[part + tid] = make_float2(m_run[tid], l_run[tid]);
    // the share that arrives last folds all of them, in ascending order
    __shared__ bool last;
    __syncthreads();
    if (tid == 0) {
        unsigned int* const counter = arrived + (long long)t * gridDim.y + blockIdx.y;
        __threadfence();
        last = atomicAdd(counter, 1u) == gridDim.z - 1;
        __threadfence();
        if (last) *counter = 0;                                // ready for the next launch
    }
    __syncthreads();
    if (!last) return;
    const long long first = part - (long long)blockIdx.z * Q4P_HEADS;
    const int splits = gridDim.z;
    for (int i = tid; i < n_heads * vd; i += Q4P_THREADS) {
        const int h = i / vd, d = i % vd;
        constexpr int S = 8;                                   // shares asked for together
        float top = -INFINITY, l = 0.f, o = 0.f;
        for (int s0 = 0; s0 < splits; s0 += S) {
            float2 ml[S];
            float v[S];
#pragma unroll
            for (int k = 0; k < S; ++k) {
                const bool there = s0 + k < splits;
                const long long at_s = first + (long long)(s0 + k) * Q4P_HEADS + h;
                ml[k] = there ? __ldcg(part_ml + at_s) : make_float2(-INFINITY, 0.f);
                v[k] = there ? __ldcg(part_o + at_s * vd + d) : 0.f;
            }
            float up = top;
#pragma unroll
            for (int k = 0; k < S; ++k) up = fmaxf(up, ml[k].x);
            const float use = up == -INFINITY ? 0.f : up, kept = exp2f(top - use);
            top = up;
            l *= kept;
            o *= kept;
#pragma unroll
            for (int k = 0; k < S; ++k) {
                const float f = exp2f(ml[k].x - use);
                l = fmaf(ml[k].y, f, l);
                o = fmaf(v[k], f, o);
            }
        }
        stf(out + ((long long)t * heads + h0 + h) * vd + d, o / l);
    }
}

template <typename T>
static int attention_q4_plain_launch(const T* q, const uint8_t* pool, const int32_t* positions, const int32_t* token_slot, T* out,
                                     const PagedQ4& kv, int n, int heads, float scale_log2, int window, int splits, float* scratch,
                                     int32_t* counters, cudaStream_t stream) {
    const int group = heads / kv.kv_heads, gy = kv.kv_heads * ((group + Q4P_HEADS - 1) / Q4P_HEADS);
    const size_t smem = (Q4P_HEADS * kv.hd + Q4P_KEYS * ((kv.hd > kv.vd ? kv.hd : kv.vd) + 1) + Q4P_KEYS * Q4P_HEADS) * sizeof(float);
    constexpr size_t most = (Q4P_HEADS * 256 + Q4P_KEYS * 257 + Q4P_KEYS * Q4P_HEADS) * sizeof(float);
    if (int st = ensure_dynamic_smem<attention_q4_plain_kernel<T>>(most, "axon_attention_q4_plain")) return st;
    float* po = splits > 1 ? scratch : nullptr;
    float2* ml = splits > 1 ? reinterpret_cast<float2*>(scratch + (long long)n * gy * splits * Q4P_HEADS * kv.vd) : nullptr;
    unsigned int* arrived = splits > 1 ? reinterpret_cast<unsigned int*>(counters) : nullptr;
    launch_pdl(attention_q4_plain_kernel<T>, dim3(n, gy, splits), dim3(Q4P_THREADS), smem, stream, q, pool, positions, token_slot, out, kv,
               heads, scale_log2, window, po, ml, arrived);
    return launch_status("axon_attention_q4_plain");
}

}  // namespace axon

using namespace axon;

enum { AXON_Q4_F32 = 0, AXON_Q4_BF16 = 1 };          // the dtype codes of generic.cu

// Rotates q and k (as axon_rope_kv_write), writes q in `dtype` and k and v quantised into the pool.  staged: positions, slots and
// the block table were copied to the device before the kernels in flight were launched (pdl.cuh).
AXON_API int axon_rope_kv_write_q4(const float* qkv, const float* table, const int32_t* positions, const int32_t* token_slot,
                                   void* q_out, void* pool, int dtype, const AxonKvLayout* layout, int n, int heads, int rot,
                                   int adjacent, int write_kv, const float* partial, int splits, int ntok, const float* bias,
                                   int staged, cudaStream_t stream) {
    if (n <= 0) return AXON_OK;
    if (partial != nullptr && (splits < 1 || ntok < n)) { set_error("axon_rope_kv_write_q4: bad partial sums (splits %d, tokens %d of %d)", splits, n, ntok); return AXON_BAD_ARGUMENT; }
    PagedQ4 kv;
    if (int st = to_q4(layout, pool, "axon_rope_kv_write_q4", &kv)) return st;
    if (rot % 2 || rot > kv.hd || rot < 0) { set_error("axon_rope_kv_write_q4: rotated size %d must be even and at most the head size %d", rot, kv.hd); return AXON_BAD_ARGUMENT; }
    if (dtype != AXON_Q4_F32 && dtype != AXON_Q4_BF16) { set_error("axon_rope_kv_write_q4: unknown dtype %d", dtype); return AXON_BAD_ARGUMENT; }
    const SplitFold fold{partial, partial ? bias : nullptr, splits, ntok};
    if (table != nullptr && !adjacent && rot == kv.hd && kv.hd % 32 == 0 && kv.planes == 2 && kv.vd == kv.hd &&
        (((uintptr_t)qkv | (uintptr_t)table | (uintptr_t)partial | (uintptr_t)bias | (uintptr_t)q_out) & 15) == 0) {
        const int items = (heads + (write_kv ? 2 * kv.kv_heads : 0)) * (kv.hd / 8);
        // few tokens: a CTA per 192 of a token's items; many: a CTA per token
        const dim3 vgrid(n, n >= 4 * 148 ? 1 : (items + Q4_WRITE_THREADS - 1) / Q4_WRITE_THREADS);
        if (dtype == AXON_Q4_F32)
            launch_pdl(rope_kv_write_q4_vec_kernel<float>, vgrid, dim3(Q4_WRITE_THREADS), 0, stream, qkv, (const float2*)table, positions, token_slot, (float*)q_out, (uint8_t*)pool, kv, heads, write_kv, staged, fold);
        else
            launch_pdl(rope_kv_write_q4_vec_kernel<__nv_bfloat16>, vgrid, dim3(Q4_WRITE_THREADS), 0, stream, qkv, (const float2*)table, positions, token_slot, (__nv_bfloat16*)q_out, (uint8_t*)pool, kv, heads, write_kv, staged, fold);
        return launch_status("axon_rope_kv_write_q4");
    }
    const int rows = heads + kv.planes * kv.kv_heads;
    const dim3 grid(n, (rows + 7) / 8);
    const bool vec = rot % 8 == 0 && (((uintptr_t)qkv | (uintptr_t)table | (uintptr_t)partial | (uintptr_t)bias) & 15) == 0;
#define AXON_Q4_WRITE(T, VEC) launch_pdl(rope_kv_write_q4_kernel<T, VEC>, grid, dim3(256), 0, stream, qkv, (const float2*)table, positions, token_slot, (T*)q_out, (uint8_t*)pool, kv, heads, rot, adjacent, write_kv, fold)
    if (dtype == AXON_Q4_F32) { if (vec) AXON_Q4_WRITE(float, true); else AXON_Q4_WRITE(float, false); }
    else { if (vec) AXON_Q4_WRITE(__nv_bfloat16, true); else AXON_Q4_WRITE(__nv_bfloat16, false); }
#undef AXON_Q4_WRITE
    return launch_status("axon_rope_kv_write_q4");
}

static int kv_read_launch(const void* pool, const PagedQ4& kv, const int32_t* spans, int n_spans, int n_slots, int dtype, long long n_rows,
                          const Q4Out& out, cudaStream_t stream) {
    int rows = Q4_READ_ROWS;
    while (rows > 1 && (n_rows + rows - 1) / rows < 2 * 148) rows /= 2;      // few rows: more CTAs rather than longer ones
    const long long ctas = (n_rows + rows - 1) / rows;
    if (ctas > 0x7fffffffLL) { set_error("axon_kv_read_q4: %lld rows are too many", n_rows); return AXON_BAD_ARGUMENT; }
    if (dtype == AXON_Q4_F32)
        launch_pdl(kv_read_q4_kernel<float>, dim3((unsigned)ctas), dim3(Q4_READ_THREADS), 0, stream, (const uint8_t*)pool, kv, spans, n_spans, n_slots, n_rows, rows, out);
    else if (dtype == AXON_Q4_BF16)
        launch_pdl(kv_read_q4_kernel<__nv_bfloat16>, dim3((unsigned)ctas), dim3(Q4_READ_THREADS), 0, stream, (const uint8_t*)pool, kv, spans, n_spans, n_slots, n_rows, rows, out);
    else { set_error("axon_kv_read_q4: unknown dtype %d", dtype); return AXON_BAD_ARGUMENT; }
    return launch_status("axon_kv_read_q4");
}

// Output rows 0 .. n_rows - 1 ([kv_heads][width] each) from the spans [4][n_spans]: slot, first
// position, count, first output row.  Rows of no span, and rows of a span that lies outside the block
// table (n_slots rows), stay as they are.  keys or values may be null.
AXON_API int axon_kv_read_q4(const void* pool, const AxonKvLayout* layout, const int32_t* spans, int n_spans, int n_slots,
                             void* keys, void* values, int dtype, long long n_rows, cudaStream_t stream) {
    if (n_rows <= 0 || n_spans <= 0) return AXON_OK;
    PagedQ4 kv;
    if (int st = to_q4(layout, pool, "axon_kv_read_q4", &kv)) return st;
    if (((uintptr_t)keys | (uintptr_t)values) & 15) { set_error("axon_kv_read_q4: outputs must be 16-byte aligned"); return AXON_BAD_ARGUMENT; }
    // planes of different widths have strides of their own: one launch each
    const bool apart = keys != nullptr && values != nullptr && kv.vd != kv.hd;
    for (int part = 0; part < (apart ? 2 : 1); ++part) {
        void* const k = apart && part ? nullptr : keys;
        void* const v = apart && !part ? nullptr : values;
        const long long width = k != nullptr ? kv.hd : kv.vd;
        const Q4Out out{k, v, kv.kv_heads * width, 0, width, 0};
        if (int st = kv_read_launch(pool, kv, spans, n_spans, n_slots, dtype, n_rows, out, stream)) return st;
    }
    return AXON_OK;
}

// See kv_read_q4_pages_kernel.  staged: segments and the block table were copied to the device before the kernels in flight
// were launched (the list `which` has to be in any case).  pages_out: bfloat16 [pages][2][kv_heads][64][head_dim].
AXON_API int axon_kv_read_q4_pages(const void* pool, const AxonKvLayout* layout, const int32_t* segments, int n_segments, const int32_t* which,
                                   int n_long, int window, int pages, int stride, int32_t* seg_out, int32_t* table, void* pages_out,
                                   int staged, cudaStream_t stream) {
    if (n_long <= 0) return AXON_OK;
    PagedQ4 kv;
    if (int st = to_q4(layout, pool, "axon_kv_read_q4_pages", &kv)) return st;
    if (kv.planes != 2 || kv.vd != kv.hd) { set_error("axon_kv_read_q4_pages: takes caches with key and value planes of one width"); return AXON_BAD_ARGUMENT; }
    if (pages < 1 || stride < 1 || pages > (1 << 29)) { set_error("axon_kv_read_q4_pages: no room (%d pages, %d per request)", pages, stride); return AXON_BAD_ARGUMENT; }
    if ((uintptr_t)pages_out & 15) { set_error("axon_kv_read_q4_pages: outputs must be 16-byte aligned"); return AXON_BAD_ARGUMENT; }
    const long long plane = (long long)kv.kv_heads * 64 * kv.hd;
    const Q4Out out{pages_out, (uint8_t*)pages_out + plane * 2, 2 * plane, kv.hd, 64ll * kv.hd, 6};
    launch_pdl(kv_read_q4_pages_kernel<__nv_bfloat16>, dim3(2 * pages), dim3(Q4_READ_THREADS), 0, stream, (const uint8_t*)pool, kv, segments,
               n_segments, which, n_long, window, pages, stride, staged, seg_out, table, out);
    return launch_status("axon_kv_read_q4_pages");
}

// Floats of scratch that axon_attention_q4_plain needs for its key shares (0 for one share).
AXON_API long long axon_attention_q4_plain_scratch(int n, int heads, int kv_heads, int v_dim, int splits) {
    if (splits <= 1 || kv_heads < 1) return 0;
    const int group = heads / kv_heads;
    return (long long)n * kv_heads * ((group + Q4P_HEADS - 1) / Q4P_HEADS) * splits * Q4P_HEADS * (v_dim + 2);
}

AXON_API int axon_attention_q4_plain(const void* q, const void* pool, int dtype, const int32_t* positions, const int32_t* token_slot,
                                     void* out, const AxonKvLayout* layout, int n, int heads, float scale, int window, int splits,
                                     float* scratch, long long scratch_floats, int32_t* counters, long long n_counters, cudaStream_t stream) {
    // counters: one for each (token, eight heads of a kv head), zeroed once; launches leave them zero
    if (n <= 0) return AXON_OK;
    PagedQ4 kv;
    if (int st = to_q4(layout, pool, "axon_attention_q4_plain", &kv)) return st;
    if (kv.hd > 256 || kv.vd > 256) { set_error("axon_attention_q4_plain: rows of %d and %d values exceed 256", kv.hd, kv.vd); return AXON_BAD_ARGUMENT; }
    if (heads < 1 || heads % kv.kv_heads) { set_error("axon_attention_q4_plain: %d heads over %d kv heads", heads, kv.kv_heads); return AXON_BAD_ARGUMENT; }
    if (splits < 1 || splits > 65535) { set_error("axon_attention_q4_plain: bad split count %d", splits); return AXON_BAD_ARGUMENT; }
    if ((long long)kv.kv_heads * ((heads / kv.kv_heads + Q4P_HEADS - 1) / Q4P_HEADS) > 65535) { set_error("axon_attention_q4_plain: %d heads are too many", heads); return AXON_BAD_ARGUMENT; }
    const long long need = axon_attention_q4_plain_scratch(n, heads, kv.kv_heads, kv.vd, splits);
    if (need > 0 && (scratch == nullptr || scratch_floats < need || ((uintptr_t)scratch & 15))) { set_error("axon_attention_q4_plain: %d key shares need %lld floats of 16-byte aligned scratch", splits, need); return AXON_BAD_ARGUMENT; }
    if (need > 0 && (counters == nullptr || n_counters < (long long)n * kv.kv_heads * ((heads / kv.kv_heads + Q4P_HEADS - 1) / Q4P_HEADS))) { set_error("axon_attention_q4_plain: %lld counters are too few", n_counters); return AXON_BAD_ARGUMENT; }
    const float scale_log2 = scale * 1.4426950408889634f;
    if (dtype == AXON_Q4_F32)
        return attention_q4_plain_launch<float>((const float*)q, (const uint8_t*)pool, positions, token_slot, (float*)out, kv, n, heads, scale_log2, window, splits, scratch, counters, stream);
    if (dtype == AXON_Q4_BF16)
        return attention_q4_plain_launch<__nv_bfloat16>((const __nv_bfloat16*)q, (const uint8_t*)pool, positions, token_slot, (__nv_bfloat16*)out, kv, n, heads, scale_log2, window, splits, scratch, counters, stream);
    set_error("axon_attention_q4_plain: unknown dtype %d", dtype);
    return AXON_BAD_ARGUMENT;
}
