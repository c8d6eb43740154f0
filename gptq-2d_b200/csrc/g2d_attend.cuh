// Shared by the attention kernels over the packed cache.
#pragma once
#include "g2d_cache.cuh"
#include "g2d_tc.cuh"

namespace g2d {

int cache_view(const g2d_cache_desc *d, CacheView *c);

// ---- attention: what its kernels share ----
struct AttendArgs {
    CacheView c;
    const void *q;
    void *out;  // [tokens, heads, head_dim]
    int64_t q_token_stride, q_head_stride;
    int heads, group;
    int causal;
    float scale;             // of the scores
    float softcap;           // 0: none
    const float *slopes;     // per head, or null
    const int32_t *prefix;   // per sequence, or null
    int rows_from, rows_to;  // the kernel's sequences: those with rows_from <= queries x group < rows_to
    float *partial;
    int *status;
    long long wait_cycles;
};
struct AttendSequence {
    int first, count, length, keys, prefix;
};
__device__ __forceinline__ AttendSequence attend_sequence(const AttendArgs &a, int b) {
    AttendSequence s;
    tokens_of(a.c, b, s.first, s.count);
    s.length = max(a.c.lengths[b], -0x40000000);  // so that positions stay in 32 bits
    s.keys = keys_of(a.c, s.length);
    s.prefix = a.prefix ? a.prefix[b] : 0;
    return s;
}
// how many keys, from the first on, token i of the sequence sees
__device__ __forceinline__ int visible_keys(const AttendArgs &a, const AttendSequence &s, int i) {
    if (!a.causal) return s.keys;
    return min(s.keys, max(s.length - s.count + (i + 1), max(s.prefix, 0)));
}


constexpr float LOG2E = 1.4426950408889634f;
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// cap tanh(u / cap) through one exponential: exact to 1e-7 of the cap, which is what a score's exponential sees
__device__ __forceinline__ float capped(float u, float cap, float two_log2e_over_cap) { return cap - __fdividef(2.f * cap, 1.f + ex2(u * two_log2e_over_cap)); }
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
__device__ __forceinline__ int64_t warp_sum(int64_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}


// Parts of a row's result, in the order of the keys: D sums, the maximum that their exponentials refer to (of the scores as powers of two) and the sum of these.
// A warp: adds up `count` parts, part i's sums at sums(i), its maximum and sum at maximum(i) and total(i); lane x returns the sums of the channels x, x + 32, ..
template <int D, typename Sums, typename Maximum, typename Total>
__device__ __forceinline__ void merge_parts(int count, Sums sums, Maximum maximum, Total total, float (&acc)[D / 32], float &m, float &l) {
    const int lane = threadIdx.x & 31;
    m = -INFINITY;
    for (int i = lane; i < count; i += 32) m = fmaxf(m, __ldcg(maximum(i)));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float base = m == -INFINITY ? 0.f : m;
    l = 0.f;
#pragma unroll
    for (int x = 0; x < D / 32; ++x) acc[x] = 0.f;
    for (int i0 = 0; i0 < count; i0 += 32) {
        float w = 0.f, t = 0.f;
        if (i0 + lane < count) {
            w = ex2(__ldcg(maximum(i0 + lane)) - base);
            t = __ldcg(total(i0 + lane));
        }
        const int here = min(32, count - i0);
#pragma unroll 4
        for (int i = 0; i < here; ++i) {
            const float f = __shfl_sync(0xffffffffu, w, i);
            l = fmaf(__shfl_sync(0xffffffffu, t, i), f, l);
            const float *const from = sums(i0 + i) + lane;
#pragma unroll
            for (int x = 0; x < D / 32; ++x) acc[x] = fmaf(__ldcg(from + x * 32), f, acc[x]);
        }
    }
}
template <int D>
__device__ __forceinline__ void write_row(uint16_t *to, const float (&acc)[D / 32], float l, int bf16) {
    const float f = l == 0.f ? 0.f : __fdividef(1.f, l);
#pragma unroll
    for (int x = 0; x < D / 32; ++x) to[x * 32 + (threadIdx.x & 31)] = (uint16_t)float_to_half_bits(l == 0.f && acc[x] == acc[x] ? 0.f : acc[x] * f, bf16);
}

// ---- sequences of many rows, by tiles (g2d_attend_tc.cu) ----
// Units: for each sequence, each pair of tiles of rows (later rows see more keys), each kv head, the blocks of keys that the last of its rows sees.
constexpr int TA_GRID = 148, TA_ROWS = 256, TA_KEYS = 128;
__device__ __forceinline__ int tile_pairs(const AttendArgs &a, const AttendSequence &s) {
    const int rows = s.count * a.group;  // of no more than tokens x heads
    return rows >= a.rows_from && rows < a.rows_to ? (int)(((unsigned)rows + TA_ROWS - 1) / TA_ROWS) : 0;
}
__device__ __forceinline__ int tile_blocks(const AttendArgs &a, const AttendSequence &s, int pair) {
    const unsigned last = min((unsigned)(s.count * a.group), (unsigned)(pair + 1) * TA_ROWS) - 1u;
    return max((int)(((unsigned)visible_keys(a, s, (int)(last / (unsigned)a.group)) + TA_KEYS - 1) / TA_KEYS), 1);
}
constexpr int FEW_SEQUENCES = 32;  // up to here the lanes of a warp share a sequence's pairs, beyond each has sequences of its own
__device__ __forceinline__ int64_t tile_units(const AttendArgs &a, int b) {  // a thread
    if (b >= a.c.batch) return 0;
    const AttendSequence s = attend_sequence(a, b);
    int64_t sum = 0;
    for (int p = 0, n = tile_pairs(a, s); p < n; ++p) sum += tile_blocks(a, s, p);
    return sum * a.c.kv_heads;
}
__device__ __forceinline__ int64_t warp_tile_units(const AttendArgs &a, const AttendSequence &s) {  // a warp
    int64_t sum = 0;
    for (int p = threadIdx.x & 31, n = tile_pairs(a, s); p < n; p += 32) sum += tile_blocks(a, s, p);
    return warp_sum(sum) * a.c.kv_heads;
}
// All threads of a CTA of WARPS warps: the units of all sequences
template <int WARPS>
__device__ __forceinline__ int64_t all_tile_units(const AttendArgs &a, long long (&totals)[WARPS]) {
    int64_t mine = 0;
    if (a.c.batch < FEW_SEQUENCES) {
        for (int b = threadIdx.x >> 5; b < a.c.batch; b += WARPS) mine += warp_tile_units(a, attend_sequence(a, b));
    } else {
        for (int b = threadIdx.x; b < a.c.batch; b += 32 * WARPS) mine += tile_units(a, b);
        mine = warp_sum(mine);
    }
    if ((threadIdx.x & 31) == 0) totals[threadIdx.x >> 5] = mine;
    __syncthreads();
    int64_t all = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) all += totals[w];
    return all;
}
// A warp: which of the 32 counts of its lanes the unit `at` of the list that begins at `base` falls into (32: none); `base` becomes where that count begins, or the end
__device__ __forceinline__ int lane_of_unit(int64_t count, int64_t at, int64_t &base) {
    const int lane = threadIdx.x & 31;
    int64_t sum = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
    }
    const unsigned past = __ballot_sync(0xffffffffu, base + sum > at);
    const int found = past ? __ffs(past) - 1 : 32;
    if (found > 0) base += __shfl_sync(0xffffffffu, sum, found - 1);
    return found;
}
struct TileCursor {
    int64_t u, end;
    int b, pair, pairs, head, block, blocks;
    AttendSequence s;
    __device__ __forceinline__ void open(const AttendArgs &a) {  // sequence b, or the next one that has units
        for (;; ++b) {
            if (b >= a.c.batch) {  // not reached while u < end
                end = u;
                return;
            }
            s = attend_sequence(a, b);
            pairs = tile_pairs(a, s);
            if (pairs > 0) break;
        }
        pair = head = block = 0;
        blocks = tile_blocks(a, s, 0);
    }
    // A warp: unit `at` of the list, which has more
    __device__ __forceinline__ void find(const AttendArgs &a, int64_t at) {
        const int lane = threadIdx.x & 31;
        int64_t base = 0;
        u = at;
        b = 0;
        if (a.c.batch < FEW_SEQUENCES) {
            for (; b < a.c.batch; ++b) {
                const int64_t here = warp_tile_units(a, attend_sequence(a, b));
                if (base + here > at) break;
                base += here;
            }
        } else {
            for (; b < a.c.batch; b += 32) {
                const int k = lane_of_unit(tile_units(a, b + lane), at, base);
                if (k < 32) {
                    b += k;
                    break;
                }
            }
        }
        open(a);
        for (int p0 = 0; p0 < pairs; p0 += 32) {
            const int k = lane_of_unit(p0 + lane < pairs ? (int64_t)tile_blocks(a, s, p0 + lane) * a.c.kv_heads : 0, at, base);
            if (k < 32) {
                pair = p0 + k;
                break;
            }
        }
        blocks = tile_blocks(a, s, pair);
        head = (int)((at - base) / blocks);
        block = (int)((at - base) % blocks);
    }
    __device__ __forceinline__ int run() const { return (int)min((int64_t)(blocks - block), end - u); }  // blocks of the item in this share
    __device__ __forceinline__ void next(const AttendArgs &a) {                                           // the item behind this run
        u += run();
        if (u >= end) return;
        block = 0;
        if (++head < a.c.kv_heads) return;
        head = 0;
        if (++pair < pairs) {
            blocks = tile_blocks(a, s, pair);
            return;
        }
        ++b;
        open(a);
    }
};
// Partial results: for each of a slot's 256 rows, head_dim sums, the maximum and the sum of the exponentials
template <int D>
__device__ __forceinline__ float *tile_slot(const AttendArgs &a, int64_t slot) {
    return a.partial + slot * (TA_ROWS * (D + 2));
}
size_t attend_tiles_bytes(int head_dim);
int launch_attend_tiles(const AttendArgs &a, cudaStream_t st);

}  // namespace g2d
