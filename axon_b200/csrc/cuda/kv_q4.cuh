// The 4-bit cache on the device: where a row's codes and steps lie, and how sixteen values
// become a step byte and codes.
//
// Sixteen consecutive values x of a row share a step s, the smallest step that is not below
// max|x| * (2 / 15), and each is held as c = rint(x / s) in -7 .. 7 (nibble c + 8).  As 7.5 s
// reaches the largest, |x - c s| <= s / 2 always, up to max|x| = 57,600 (the largest step is 7,680);
// larger ones saturate at 53,760.  A step has four significant bits and a code three, so c s
// has seven: it is exact in bfloat16 and in float, and every kernel that reads the cache sees the
// same values.  A group with a value that is not finite is held as NaN (step byte 255).
// 16 values a step rather than 32 or a whole row: keys have channels ten times larger than
// the rest, and a step confines each to its neighbours; the price is half a bit a value (4.5 in all).
#pragma once

#include "common.cuh"

#include <cuda_fp16.h>

namespace axon {

constexpr int Q4_GROUP = 16;
constexpr int Q4_TOP = 223, Q4_NAN = 255;       // the largest step byte written, and the one of a group that is not finite

struct PagedQ4 {
    const int32_t* block_table;
    uint32_t* fault;
    long long page_stride, entry_offset;         // bytes
    int table_stride, page_size, kv_heads, hd, vd, planes, n_pages;
    int record, k_steps, v_codes, v_steps;       // bytes of a head's record, and its parts' offsets (values: the keys with one plane)

    __device__ __forceinline__ int page(int entry) const {
        if (fault != nullptr && (unsigned)entry > (unsigned)n_pages) {
            fault[1] = (uint32_t)entry;
            fault[0] = 1u;
            return n_pages;
        }
        return entry;
    }
    // a kv head's record in the page of logical index lp
    __device__ __forceinline__ long long record_at(int slot, int lp, int kv_head) const {
        return (long long)page(block_table[(long long)slot * table_stride + lp]) * page_stride + entry_offset + (long long)kv_head * record;
    }
};

inline int to_q4(const AxonKvLayout* l, const void* pool, const char* what, PagedQ4* out) {
    if (l == nullptr || l->bits != 4) { set_error("%s: takes a cache of 4-bit rows", what); return AXON_BAD_ARGUMENT; }
    const int vd = l->planes == 1 || l->v_dim <= 0 ? l->head_dim : l->v_dim;
    if (l->head_dim < 16 || l->head_dim % 16 || vd % 16) { set_error("%s: 4-bit rows are multiples of 16 values, not %d and %d", what, l->head_dim, vd); return AXON_BAD_ARGUMENT; }
    if (l->page_size < 1 || l->kv_heads < 1 || l->table_stride < 1) { set_error("%s: bad layout (page size %d, %d kv heads, table stride %d)", what, l->page_size, l->kv_heads, l->table_stride); return AXON_BAD_ARGUMENT; }
    if (((uintptr_t)pool | (uintptr_t)l->page_stride | (uintptr_t)l->entry_offset) & 15) { set_error("%s: a 4-bit pool and its pages and entries are 16-byte aligned", what); return AXON_BAD_ARGUMENT; }
    auto up = [](long long n) { return (n + 15) / 16 * 16; };
    const long long kc = up((long long)l->page_size * l->head_dim / 2), ks = up((long long)l->page_size * l->head_dim / 16);
    const long long vc = up((long long)l->page_size * vd / 2), vs = up((long long)l->page_size * vd / 16);
    const long long record = kc + ks + (l->planes == 1 ? 0 : vc + vs);
    if (record > (1 << 28)) { set_error("%s: pages of %d positions are too large", what, l->page_size); return AXON_BAD_ARGUMENT; }
    PagedQ4 q;
    q.block_table = l->block_table; q.fault = l->fault;
    q.page_stride = l->page_stride; q.entry_offset = l->entry_offset;
    q.table_stride = l->table_stride; q.page_size = l->page_size; q.kv_heads = l->kv_heads;
    q.hd = l->head_dim; q.vd = vd; q.planes = l->planes == 1 ? 1 : 2; q.n_pages = l->n_pages;
    q.record = (int)record; q.k_steps = (int)kc;
    q.v_codes = l->planes == 1 ? 0 : (int)(kc + ks);
    q.v_steps = l->planes == 1 ? (int)kc : (int)(kc + ks + vc);
    *out = q;
    return AXON_OK;
}

// The step byte of a group whose largest magnitude has the float bits `top` (sign cleared).
__device__ __forceinline__ int q4_step_byte(uint32_t top) {
    if (top >= 0x7f800000u) return Q4_NAN;
    const float t = __fmul_rn(__uint_as_float(top), 2.0f / 15.0f);
    // below 2^-14 steps are multiples of 2^-17 (subnormal halves); above, round the mantissa up to three bits
    const int b = t < 6.103515625e-05f ? (int)ceilf(t * 131072.0f) : (int)((__float_as_uint(t) + 0xFFFFFu) >> 20) - (112 << 3);
    return min(b, Q4_TOP);
}
__device__ __forceinline__ float q4_step(int byte) { return __half2float(__ushort_as_half((unsigned short)(byte << 7))); }
__device__ __forceinline__ float q4_inverse(int byte) { return byte == 0 || byte == Q4_NAN ? 0.f : __frcp_rn(q4_step(byte)); }
// The nibbles of four values of a group with this step byte; `inv` is 1 / step rounded to 32 bits (0 for a step of 0 or NaN).
// Adding 1.5 * 2^23 + 8 rounds to whole numbers as rint does and leaves code + 8 in the last four bits.
__device__ __forceinline__ uint32_t q4_codes4(float x0, float x1, float x2, float x3, int byte, float inv) {
    auto code = [&](float x) { return __float_as_uint(__fadd_rn(fminf(fmaxf(__fmul_rn(x, inv), -7.f), 7.f), 12582920.0f)) & 15u; };
    return byte == Q4_NAN ? 0x8888u : code(x0) | code(x1) << 4 | code(x2) << 8 | code(x3) << 12;
}
// nibble i of a word of eight codes, as a float without its step
__device__ __forceinline__ float q4_digit(uint32_t word, int i) {
    return __uint_as_float(0x4B000000u | ((word >> (4 * i)) & 15u)) - 8388616.0f;      // 2^23 + code, exactly
}

}  // namespace axon
