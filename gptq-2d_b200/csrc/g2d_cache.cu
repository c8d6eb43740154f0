// Keys and values of a paged cache in 4-bit codes: writing new rows and reading rows back.
//
// A row is the head_dim values of one token and one kv head.  It is rounded as the dynamic abs-max quantizer rounds a row of a super-entry
// (quantizer_int.py:120-134 of the reference) to the codes -8 .. 7: scale = absmax / 7.5 rounded to fp16 through fp32 (1 for zeros), code =
// clamp(rint(v / scale), -8, 7), all in fp32, and stored as g2d_pack_codes stores a row with qmin = -8.  A row with an infinity or a NaN gets a
// scale that is not finite, so that it reads back as NaN: absmax is taken over the bits of |v|, where both are larger than any number.
//
// Bound: HBM, 2 bytes read per value and half a byte written (the other way round for reading).  A lane takes eight values (16 bytes), so a row is that
// of 16 or 8 neighbouring lanes and its absmax 3 or 4 shuffles.  6293 tokens of 8 heads, 128 channels, written and read back: 25.3 us (2.6 TB/s of what has to move); one token of 8 sequences 6.5.
#include "g2d_cache.cuh"

namespace g2d {

constexpr int CACHE_THREADS = 256;

template <int LANES>
__device__ __forceinline__ unsigned lanes_max(unsigned v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
// A warp takes tokens that stand together, a token at a time: where it goes is found once for all of its rows, and its sequence once for as long as it lasts.
struct CachePlace {
    int b = -1, first = 0, count = 0, length = 0;
    // row of the cache of kv head 0 of the token's position (heads lie page_size rows apart), -1 where there is none
    __device__ __forceinline__ int64_t of(const CacheView &c, int token) {
        if (b < 0 || token < first || token >= first + count) {
            b = sequence_of(c, token, first, count);
            if (b >= 0) length = max(c.lengths[b], -0x40000000);
        }
        return b < 0 ? -1 : cache_row(c, b, length - count + (token - first), 0);
    }
};
__device__ __forceinline__ void tokens_of_warp(const CacheView &c, int &t0, int &t1) {
    const int64_t warps = (int64_t)gridDim.x * (CACHE_THREADS / 32), w = (int64_t)blockIdx.x * (CACHE_THREADS / 32) + (threadIdx.x >> 5);
    t0 = (int)(w * c.tokens / warps);
    t1 = (int)((w + 1) * c.tokens / warps);
}

// Quotients by one reciprocal (within two units of its last bit) and one correction, which leaves them within theirs.  That is enough: the quotient of an x of 11 bits at most by a scale of 11
// bits (or by 7.5) is either a half-integer (or halfway between two halves) exactly, and then both steps are exact as well, or more than 2^-16 of itself away from one.
__device__ __forceinline__ float reciprocal(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float scale_of(float absmax) {  // absmax / 7.5 as a half, 1 for zero
    constexpr float RC = 1.f / 7.5f;
    const float q0 = absmax * RC, q = __half2float(__float2half_rn(absmax < INFINITY ? fmaf(fmaf(-q0, 7.5f, absmax), RC, q0) : absmax));
    return q == 0.f ? 1.f : q;
}
// two values over the scale, rounded to the nearest of -8 .. 7, plus 8: by the addition of 1.5 2^23 + 8, in the lowest bits of what is returned
__device__ __forceinline__ void codes_of(uint64_t x, uint64_t minus_scale, uint64_t rc, uint32_t &lo, uint32_t &hi) {
    const uint64_t q0 = mul2(x, rc);
    float a, b;
    unpack2(fma2(fma2(q0, minus_scale, x), rc, q0), a, b);
    lo = __float_as_uint(fminf(fmaxf(a, -8.f), 7.f) + 12582920.f);
    hi = __float_as_uint(fminf(fmaxf(b, -8.f), 7.f) + 12582920.f);
}

// rows of a token: (head, key or value), the latter fastest; LANES lanes each
template <int LANES>
__global__ void __launch_bounds__(CACHE_THREADS) cache_append_kernel(const CacheView c, const uint16_t *__restrict__ k, const uint16_t *__restrict__ v, int64_t k_token, int64_t k_head,
                                                                     int64_t v_token, int64_t v_head) {
    constexpr int ROWS = 32 / LANES, BATCH = 4;  // rows of a warp at once, and so many times; a CTA along y takes so many of each token's
    const int lane = threadIdx.x & 31, part = lane % LANES, sub = lane / LANES, rows = 2 * c.kv_heads, r0 = blockIdx.y * (ROWS * BATCH);
    int t0, t1;
    tokens_of_warp(c, t0, t1);
    CachePlace place;
    for (int token = t0; token < t1; ++token) {
        const int64_t at = place.of(c, token);
        if (at < 0) continue;
        {
            uint4 raw[BATCH];
#pragma unroll
            for (int n = 0; n < BATCH; ++n) {
                const int r = r0 + n * ROWS + sub, head = r >> 1;
                raw[n] = r < rows ? __ldg(reinterpret_cast<const uint4 *>((r & 1 ? v + token * v_token + head * v_head : k + token * k_token + head * k_head) + part * 8)) : make_uint4(0u, 0u, 0u, 0u);
            }
#pragma unroll
            for (int n = 0; n < BATCH; ++n) {
                const int r = r0 + n * ROWS + sub, head = r >> 1;
                if (r0 + n * ROWS >= rows) break;  // for the whole warp
                const uint32_t word[4] = {raw[n].x, raw[n].y, raw[n].z, raw[n].w};
                // the largest as the bits of a half, whose order is that of the values (NaN above infinity)
                const uint32_t pair = __vmaxu2(__vmaxu2(word[0] & 0x7fff7fffu, word[1] & 0x7fff7fffu), __vmaxu2(word[2] & 0x7fff7fffu, word[3] & 0x7fff7fffu));
                const float scale = scale_of(half_bits_to_float(lanes_max<LANES>(max(pair & 0xffffu, pair >> 16)), c.bf16));
                uint32_t codes = 0x88888888u;  // a row that is not finite: zeros under a scale that is not
                if (scale <= 65504.f) {
                    const uint64_t minus = pack2(-scale, -scale);
                    const float r1 = reciprocal(scale);
                    const uint64_t rc = pack2(r1, r1);
                    codes = 0u;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint32_t lo, hi;
                        codes_of(pack2(half_bits_to_float(word[e] & 0xffffu, c.bf16), half_bits_to_float(word[e] >> 16, c.bf16)), minus, rc, lo, hi);
                        codes |= (lo & 15u) << (8 * e) | (hi & 15u) << (8 * e + 4);
                    }
                }
                if (r < rows) {
                    const int64_t row = at + ((int64_t)head << c.page_shift);
                    reinterpret_cast<uint32_t *>((r & 1 ? c.v_codes : c.k_codes) + row * (LANES * 4))[part] = codes;
                    if (part == 0) (r & 1 ? c.v_scale : c.k_scale)[row] = __float2half_rn(scale);
                }
            }
        }
    }
}

template <int LANES>
__global__ void __launch_bounds__(CACHE_THREADS) cache_read_kernel(const CacheView c, uint16_t *__restrict__ k, uint16_t *__restrict__ v) {
    constexpr int ROWS = 32 / LANES, BATCH = 4;
    const int lane = threadIdx.x & 31, part = lane % LANES, sub = lane / LANES, rows = 2 * c.kv_heads, r0 = blockIdx.y * (ROWS * BATCH);
    int t0, t1;
    tokens_of_warp(c, t0, t1);
    CachePlace place;
    for (int token = t0; token < t1; ++token) {
        const int64_t at = place.of(c, token);
        {
            uint32_t codes[BATCH];
            float scale[BATCH];
#pragma unroll
            for (int n = 0; n < BATCH; ++n) {
                const int r = r0 + n * ROWS + sub;
                const int64_t row = at + ((int64_t)(r >> 1) << c.page_shift);
                codes[n] = 0x88888888u;  // a row of no sequence and a position that the cache does not hold read as zeros
                scale[n] = 0.f;
                if (at >= 0 && r < rows) {
                    codes[n] = reinterpret_cast<const uint32_t *>((r & 1 ? c.v_codes : c.k_codes) + row * (LANES * 4))[part];
                    scale[n] = __half2float((r & 1 ? c.v_scale : c.k_scale)[row]);
                }
            }
#pragma unroll
            for (int n = 0; n < BATCH; ++n) {
                const int r = r0 + n * ROWS + sub;
                if (r >= rows) continue;
                uint32_t word[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float lo = (float)((int)((codes[n] >> (8 * e)) & 15u) - 8) * scale[n], hi = (float)((int)((codes[n] >> (8 * e + 4)) & 15u) - 8) * scale[n];
                    word[e] = pack_halves(lo, hi, c.bf16);
                }
                reinterpret_cast<uint4 *>((r & 1 ? v : k) + ((int64_t)token * c.kv_heads + (r >> 1)) * (LANES * 8))[part] = make_uint4(word[0], word[1], word[2], word[3]);
            }
        }
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

static dim3 cache_grid(const CacheView &c) {  // a token and four times a warp's rows per warp; more tokens where that is more than 32 CTAs per SM (6293 tokens of 8 heads, written and read: 29.8 us, with 8 CTAs 31.0, both with 8 for clearing the results first)
    const int64_t blocks = ceil_div((int64_t)c.tokens, (int64_t)(CACHE_THREADS / 32)), groups = ceil_div((int64_t)2 * c.kv_heads * (c.head_dim / 8), (int64_t)(32 * 4));
    const int64_t most = groups < 148 * 32 ? 148 * 32 / groups : 1;
    return dim3((unsigned)(blocks < most ? blocks : most), (unsigned)groups);
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
