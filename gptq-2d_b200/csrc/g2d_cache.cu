// Keys and values of a paged cache in 4-bit codes: writing new rows and reading rows back.
//
// A row is the head_dim values of one token and one kv head.  It is rounded as the dynamic abs-max quantizer rounds a row of a super-entry
// (quantizer_int.py:120-134 of the reference) to the codes -8 .. 7: scale = absmax / 7.5 rounded to fp16 through fp32 (1 for zeros), code =
// clamp(rint(v / scale), -8, 7), all in fp32, and stored as g2d_pack_codes stores a row with qmin = -8.  A row with an infinity or a NaN gets a
// scale that is not finite, so that it reads back as NaN: absmax is taken over the bits of |v|, where both are larger than any number.
//
// Bound: HBM, 2 bytes read per value and half a byte written (the other way round for reading).  A lane takes eight values (16 bytes), so a row is that
// of 16 or 8 neighbouring lanes and its absmax 3 or 4 shuffles.  Offsets are searched once per row, from the L1.
#include "g2d_cache.cuh"

namespace g2d {

constexpr int CACHE_THREADS = 256;

template <int LANES>
__device__ __forceinline__ unsigned lanes_max(unsigned v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// rows: (token, head, key or value), the last fastest
template <int LANES>
__global__ void __launch_bounds__(CACHE_THREADS) cache_append_kernel(const CacheView c, const uint16_t *__restrict__ k, const uint16_t *__restrict__ v, int64_t k_token, int64_t k_head,
                                                                     int64_t v_token, int64_t v_head) {
    constexpr int PER_CTA = CACHE_THREADS / LANES;
    const int64_t rows = (int64_t)c.tokens * c.kv_heads * 2;
    const int part = threadIdx.x % LANES;
    for (int64_t r0 = (int64_t)blockIdx.x * PER_CTA; r0 < rows; r0 += (int64_t)gridDim.x * PER_CTA) {  // the same trips for all lanes of a warp
        const int64_t r = r0 + threadIdx.x / LANES;
        uint4 raw = make_uint4(0u, 0u, 0u, 0u);
        int64_t at = -1;
        const bool value = r & 1;
        if (r < rows) {
            const int token = (int)((r >> 1) / c.kv_heads), head = (int)((r >> 1) % c.kv_heads);
            raw = *reinterpret_cast<const uint4 *>((value ? v + token * v_token + head * v_head : k + token * k_token + head * k_head) + part * 8);
            int first, count;
            const int b = sequence_of(c, token, first, count);
            if (b >= 0) {
                const int64_t p = (int64_t)c.lengths[b] - count + (token - first);
                at = cache_row(c, b, (int)max(min(p, (int64_t)0x7fffffff), (int64_t)-1), head);
            }
        }
        float x[8];
        const uint32_t word[4] = {raw.x, raw.y, raw.z, raw.w};
        unsigned largest = 0u;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] = half_bits_to_float((word[e >> 1] >> (16 * (e & 1))) & 0xffffu, c.bf16);
            largest = max(largest, __float_as_uint(x[e]) & 0x7fffffffu);
        }
        const float scale = absmax_scale_value(__uint_as_float(lanes_max<LANES>(largest)), 7.5f, G2D_FP16);
        const bool finite = scale <= 65504.f;
        uint32_t codes = 0u;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float t = fminf(fmaxf(rintf(div_rn(x[e], scale)), -8.f), 7.f);
            codes |= (finite ? (uint32_t)(__float2int_rn(t) + 8) : 8u) << (4 * e);  // a row that is not finite: zeros under a scale that is not
        }
        if (at >= 0) {
            uint8_t *const to = (value ? c.v_codes : c.k_codes) + at * (LANES * 4);
            reinterpret_cast<uint32_t *>(to)[part] = codes;
            if (part == 0) (value ? c.v_scale : c.k_scale)[at] = __float2half_rn(scale);
        }
    }
}

template <int LANES>
__global__ void __launch_bounds__(CACHE_THREADS) cache_read_kernel(const CacheView c, uint16_t *__restrict__ k, uint16_t *__restrict__ v) {
    constexpr int PER_CTA = CACHE_THREADS / LANES;
    const int64_t rows = (int64_t)c.tokens * c.kv_heads * 2;
    const int part = threadIdx.x % LANES;
    for (int64_t r = (int64_t)blockIdx.x * PER_CTA + threadIdx.x / LANES; r < rows; r += (int64_t)gridDim.x * PER_CTA) {
        const bool value = r & 1;
        const int token = (int)((r >> 1) / c.kv_heads), head = (int)((r >> 1) % c.kv_heads);
        int first, count;
        const int b = sequence_of(c, token, first, count);
        if (b < 0) continue;  // a row of no sequence stays as it is
        const int64_t p = (int64_t)c.lengths[b] - count + (token - first);
        const int64_t at = cache_row(c, b, (int)max(min(p, (int64_t)0x7fffffff), (int64_t)-1), head);
        uint32_t codes = 0x88888888u;  // a position that the cache does not hold reads as zeros
        float scale = 0.f;
        if (at >= 0) {
            codes = reinterpret_cast<const uint32_t *>((value ? c.v_codes : c.k_codes) + at * (LANES * 4))[part];
            scale = __half2float((value ? c.v_scale : c.k_scale)[at]);
        }
        uint32_t word[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float lo = (float)((int)((codes >> (8 * e)) & 15u) - 8) * scale, hi = (float)((int)((codes >> (8 * e + 4)) & 15u) - 8) * scale;
            word[e] = pack_halves(lo, hi, c.bf16);
        }
        reinterpret_cast<uint4 *>((value ? v : k) + ((int64_t)token * c.kv_heads + head) * (LANES * 8))[part] = make_uint4(word[0], word[1], word[2], word[3]);
    }
}

// G2D_OK and the view, or what is wrong with the descriptor
int cache_view(const g2d_cache_desc *d, CacheView *c) {
    if (!d || (d->half != G2D_FP16 && d->half != G2D_BF16) || d->pages < 0 || d->batch < 0 || d->table_width < 0 || d->tokens < 0 || d->kv_heads < 1) return G2D_ERR_BAD_ARGUMENT;
    if (d->head_dim != 64 && d->head_dim != 128) return G2D_ERR_UNSUPPORTED;
    if (d->page_size < 16 || d->page_size > (1 << 20) || (d->page_size & (d->page_size - 1)) != 0) return G2D_ERR_UNSUPPORTED;
    if (d->tokens > 0x3fffffff || d->batch > 0x3fffffff || d->table_width > 0x3fffffff || d->pages > 0x7fffffff || d->kv_heads > 65536) return G2D_ERR_TOO_LARGE;
    if (d->batch > 0 && !d->offsets && d->tokens % d->batch != 0) return G2D_ERR_BAD_ARGUMENT;
    if (d->batch == 0 && d->tokens > 0 && !d->offsets) return G2D_ERR_BAD_ARGUMENT;
    if (d->pages > 0 && (!d->k_codes || !d->k_scale || !d->v_codes || !d->v_scale)) return G2D_ERR_BAD_ARGUMENT;
    if ((((uintptr_t)d->k_codes | (uintptr_t)d->v_codes | (uintptr_t)d->k_scale | (uintptr_t)d->v_scale) & 15) != 0) return G2D_ERR_BAD_ARGUMENT;
    if (d->batch > 0 && (!d->lengths || (d->table_width > 0 && !d->table) || d->table_stride < 0)) return G2D_ERR_BAD_ARGUMENT;
    c->k_codes = d->k_codes;
    c->v_codes = d->v_codes;
    c->k_scale = (__half *)d->k_scale;
    c->v_scale = (__half *)d->v_scale;
    c->table = d->table;
    c->lengths = d->lengths;
    c->offsets = d->offsets;
    c->table_stride = d->table_stride;
    c->pages = d->pages;
    c->batch = (int)d->batch;
    c->tokens = (int)d->tokens;
    c->kv_heads = d->kv_heads;
    c->head_dim = d->head_dim;
    c->page_size = d->page_size;
    c->page_shift = 0;
    while ((1 << c->page_shift) < d->page_size) ++c->page_shift;
    c->table_width = (int)d->table_width;
    c->bf16 = d->half == G2D_BF16;
    return G2D_OK;
}

static unsigned cache_grid(const CacheView &c) {
    const int64_t blocks = ceil_div((int64_t)c.tokens * c.kv_heads * 2 * (c.head_dim / 8), (int64_t)CACHE_THREADS);
    return (unsigned)(blocks < 148 * 32 ? blocks : 148 * 32);
}

}  // namespace g2d

using namespace g2d;

extern "C" int g2d_cache_append(const g2d_cache_desc *desc, const void *k, int64_t k_token_stride, int64_t k_head_stride, const void *v, int64_t v_token_stride, int64_t v_head_stride,
                                void *stream) {
    CacheView c;
    const int status = cache_view(desc, &c);
    if (status != G2D_OK) return status;
    if (c.tokens == 0 || c.batch == 0) return G2D_OK;
    if (!k || !v || (((uintptr_t)k | (uintptr_t)v) & 15) != 0 || ((k_token_stride | k_head_stride | v_token_stride | v_head_stride) & 7) != 0) return G2D_ERR_BAD_ARGUMENT;
    const auto kernel = c.head_dim == 128 ? cache_append_kernel<16> : cache_append_kernel<8>;
    kernel<<<cache_grid(c), CACHE_THREADS, 0, (cudaStream_t)stream>>>(c, (const uint16_t *)k, (const uint16_t *)v, k_token_stride, k_head_stride, v_token_stride, v_head_stride);
    return check_launch();
}

extern "C" int g2d_cache_read(const g2d_cache_desc *desc, void *k, void *v, void *stream) {
    CacheView c;
    const int status = cache_view(desc, &c);
    if (status != G2D_OK) return status;
    if (c.tokens == 0 || c.batch == 0) return G2D_OK;
    if (!k || !v || (((uintptr_t)k | (uintptr_t)v) & 15) != 0) return G2D_ERR_BAD_ARGUMENT;
    const auto kernel = c.head_dim == 128 ? cache_read_kernel<16> : cache_read_kernel<8>;
    kernel<<<cache_grid(c), CACHE_THREADS, 0, (cudaStream_t)stream>>>(c, (uint16_t *)k, (uint16_t *)v);
    return check_launch();
}
