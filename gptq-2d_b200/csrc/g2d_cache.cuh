// Shared by the kernels of the packed key / value cache: its addressing, and the sequences of a step.
#pragma once
#include "g2d_common.cuh"

namespace g2d {

constexpr int CACHE_BLOCK = 64;  // keys per step of the attention kernels

// What a step says about its sequences.  Lengths, offsets and page numbers live on the device and are taken as they are: everything that is
// derived from them is brought into range here, so that no value of theirs leads out of a buffer.
struct CacheView {
    uint8_t *k_codes, *v_codes;  // [pages, kv_heads, page_size, head_dim / 2]
    __half *k_scale, *v_scale;   // [pages, kv_heads, page_size]
    const int32_t *table;        // [batch, table_width], rows of table_stride
    const int32_t *lengths;      // [batch], this step's tokens included
    const int32_t *offsets;      // [batch + 1] or null: the same number of tokens for every sequence
    int64_t table_stride, pages;
    int batch, tokens, kv_heads, head_dim;
    int page_size, page_shift, table_width;
    int bf16;
};

// first token of sequence b, and their number
__device__ __forceinline__ void tokens_of(const CacheView &c, int b, int &first, int &count) {
    if (c.offsets) {
        const int lo = min(max(c.offsets[b], 0), c.tokens), hi = min(max(c.offsets[b + 1], lo), c.tokens);
        first = lo;
        count = hi - lo;
    } else {
        count = c.tokens / c.batch;
        first = b * count;
    }
}
__device__ __forceinline__ int capacity_of(const CacheView &c) { return (int)min((int64_t)c.table_width << c.page_shift, (int64_t)0x7fffffff); }
// keys of sequence b that the cache can hold
__device__ __forceinline__ int keys_of(const CacheView &c, int length) { return min(max(length, 0), capacity_of(c)); }

// The sequence of a token: the last one that starts at or before it.  -1 for a token of none.
__device__ __forceinline__ int sequence_of(const CacheView &c, int token, int &first, int &count) {
    if (!c.offsets) {
        const int b = token / max(c.tokens / c.batch, 1);
        if (b >= c.batch) return -1;
        tokens_of(c, b, first, count);
        return b;
    }
    int lo = 0, hi = c.batch;  // offsets[lo] <= token < offsets[hi]
    if (token < c.offsets[0] || token >= c.offsets[c.batch]) return -1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (c.offsets[mid] <= token) lo = mid;
        else hi = mid;
    }
    tokens_of(c, lo, first, count);
    return token >= first && token < first + count ? lo : -1;
}

// Row (page, head, place) of a position among all rows of the cache, or -1 where the table has no such page.
__device__ __forceinline__ int64_t cache_row(const CacheView &c, int b, int position, int head) {
    if (position < 0 || position >= capacity_of(c)) return -1;
    const int page = c.table[b * c.table_stride + (position >> c.page_shift)];
    if (page < 0 || page >= c.pages) return -1;
    return (((int64_t)page * c.kv_heads + head) << c.page_shift) + (position & (c.page_size - 1));
}

// pairs of floats: one instruction each
__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
    return r;
}
__device__ __forceinline__ uint64_t pack2(float lo, float hi) { return pack2(__float_as_uint(lo), __float_as_uint(hi)); }
__device__ __forceinline__ void unpack2(uint64_t v, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ float half_bits_to_float(uint32_t bits, int bf16) {
    return bf16 ? __uint_as_float(bits << 16) : __half2float(__ushort_as_half((unsigned short)bits));
}
__device__ __forceinline__ uint32_t float_to_half_bits(float v, int bf16) {
    return bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}
__device__ __forceinline__ uint32_t pack_halves(float lo, float hi, int bf16) {
    uint32_t r;
    if (bf16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

}  // namespace g2d
