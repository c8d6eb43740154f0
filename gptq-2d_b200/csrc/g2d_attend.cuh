// Shared by the attention kernels over the packed cache.
#pragma once
#include "g2d_cache.cuh"
#include "g2d_tc.cuh"

namespace g2d {

int cache_view(const g2d_cache_desc *d, CacheView *c);

// ---- attention: what its kernels share ----
// An item that begins in a share and does not end in it: what is to be added up, and for which rows.  Each share's kernel writes one; count 0: none, -1: the units could not be counted.
struct AttendJoin {
    int count, row0, rows, first, head;  // parts; the first row and how many the sequence has, its first token, kv head
    int reserved[3];
};
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
    int even;                // rows: not 0: every item counts as so many units, and shares have whole items
    int rows_from, rows_to;  // the kernel's sequences: those with rows_from <= queries x group < rows_to
    float *partial;
    AttendJoin *joins;  // one per share
    int clear;          // rows of no sequence become zeros
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


// Where a row's biases are counted from.  A constant added to all of a row's scores changes no result, so that it need not be the query's position: from the key with the largest bias on, the keys
// that count have small ones, whose rounding does not show (slopes of -0.5, 2e5 keys, from the query's position on: off by seven times the bound of a result).
__device__ __forceinline__ int bias_origin(float slope, int limit) { return slope > 0.f ? limit - 1 : 0; }

constexpr float LOG2E = 1.4426950408889634f;
// What a score is taken times, so that its exponential is one to base 2: where it is capped, before that (a cap below 1e-20 is as good as none left)
template <bool MODS>
__device__ __forceinline__ float score_unit(const AttendArgs &a) {
    return MODS && a.softcap > 0.f ? fminf(2.f * LOG2E / a.softcap, 1e20f) : LOG2E;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// two halves, NaN in the place of one that is not finite
__device__ __forceinline__ uint32_t nan_unless_finite(uint32_t halves) {
    const __half2 h = *reinterpret_cast<const __half2 *>(&halves), r = __hfma2(h, __float2half2_rn(0.f), h);
    return *reinterpret_cast<const uint32_t *>(&r);
}
// cap tanh(u / cap) through one exponential, from x = 2 log2(e) u / cap: good to 1e-7 of the cap, which is what a score's exponential sees of a cap up to CAP_NEAR.  Larger caps: tanh's
// series where |u / cap| < 1/4 (relative error 1e-8), so that a cap far above the scores leaves them what they are.
constexpr float CAP_NEAR = 64.f;
__device__ __forceinline__ float capped(float x, float cap, bool near) {
    if (!near) {
        const float y = x * 0.34657359f, z = y * y;  // ln(2) / 2
        if (fabsf(y) < 0.25f) return cap * (y * fmaf(fmaf(fmaf(fmaf(62.f / 2835.f, z, -17.f / 315.f), z, 2.f / 15.f), z, -1.f / 3.f), z, 1.f));
    }
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + ex2(x)));
    return fmaf(-2.f * cap, r, cap);
}
// ---- the list of units, and its shares ----
// Units are counted in 32 bits (the entry point refuses what could have more).  Share i of `count` has the units from begin(i) on.
struct AttendShares {
    unsigned count, each, more;  // the first `more` shares have each + 1
    __device__ __forceinline__ AttendShares(unsigned units, unsigned most) : count(min(units, most)), each(count ? units / count : 0u), more(count ? units - each * count : 0u) {}
    __device__ __forceinline__ unsigned begin(unsigned i) const { return i * each + min(i, more); }
    __device__ __forceinline__ unsigned of(unsigned u) const { return u < more * (each + 1) ? u / (each + 1) : more + (u - more * (each + 1)) / each; }
};
__device__ __forceinline__ unsigned warp_add(unsigned v) { return __reduce_add_sync(0xffffffffu, v); }
// A sequence has fewer than 2^31 units, and all have, as long as no token belongs to two.  Offsets that lie over one another may make more of them: sums stop at UNITS_END.
constexpr unsigned UNITS_END = 0x80000000u;
__device__ __forceinline__ unsigned units_add(unsigned a, unsigned b) { return min(a + b, UNITS_END); }  // of two up to UNITS_END, one of them below it
__device__ __forceinline__ unsigned warp_units(unsigned v) {
    if (warp_add(v >> 6) > UNITS_END >> 6) return UNITS_END;  // else the sum is below 2^31 + 2^11
    return min(warp_add(v), UNITS_END);
}
// All threads of a CTA of WARPS warps: the units of all sequences, units(b) of one, and this lane's first one (of sequence `lane`).  Few sequences: every warp by itself.
template <int WARPS, typename Units>
__device__ __forceinline__ unsigned count_units(int batch, Units units, unsigned (&totals)[WARPS], unsigned &mine) {
    const int lane = threadIdx.x & 31;
    mine = units(lane);
    if (batch <= 32) return warp_units(mine);
    unsigned sum = 0u;
    for (int b = threadIdx.x; b < batch; b += 32 * WARPS) sum = units_add(sum, units(b));
    sum = warp_units(sum);
    if (lane == 0) totals[threadIdx.x >> 5] = sum;
    __syncthreads();
    bool past = false;
    unsigned all = 0u;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        past |= totals[w] == UNITS_END;
        all = units_add(all, totals[w] & (UNITS_END - 1u));
    }
    return past ? UNITS_END : all;
}
// A warp: which of its lanes' counts the unit `at` falls into, the first of them beginning at `base` (32: none); `base` becomes where that count begins, or the end
__device__ __forceinline__ int lane_of_unit(unsigned count, unsigned at, unsigned &base) {
    const int lane = threadIdx.x & 31;
    unsigned sum = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
    }
    const unsigned past = __ballot_sync(0xffffffffu, base + sum > at);
    const int found = past ? __ffs(past) - 1 : 32;
    if (found > 0) base += __shfl_sync(0xffffffffu, sum, found - 1);
    return found;
}
// A warp: the sequence that unit `at` belongs to, and where its units begin; `mine` as count_units has left it
template <typename Units>
__device__ __forceinline__ int sequence_of_unit(int batch, Units units, unsigned mine, unsigned at, unsigned &base) {
    base = 0u;
    for (int b0 = 0; b0 < batch; b0 += 32) {
        const int k = lane_of_unit(b0 == 0 ? mine : units(b0 + (int)(threadIdx.x & 31)), at, base);
        if (k < 32) return b0 + k;
    }
    return batch;
}

// Parts of a row's result, in the order of the keys: D sums, the reference of their exponentials (a power of two) and the sum of these.
// A warp: adds up `count` parts; the row's sums of part i are at row(i), its reference and its sum of exponentials `reference` and `total` floats behind.  Lane x gets the
// sums of the channels x, x + 32, ..
template <int D, typename Row>
__device__ __forceinline__ void merge_parts(int count, Row row, int reference, int total, float (&acc)[D / 32], float &m, float &l) {
    constexpr int TOGETHER = 8;  // parts whose loads travel together, the first ones' with the references
    const int lane = threadIdx.x & 31;
    float mine = -INFINITY, t = 0.f, v[TOGETHER][D / 32];
    const auto fetch = [&](int from) {
#pragma unroll
        for (int k = 0; k < TOGETHER; ++k)
#pragma unroll
            for (int x = 0; x < D / 32; ++x) v[k][x] = from + k < count ? __ldcg(row(from + k) + x * 32 + lane) : 0.f;
    };
    if (lane < count) {
        mine = __ldcg(row(lane) + reference);
        t = __ldcg(row(lane) + total);
    }
    fetch(0);
    m = mine;
    for (int i = lane + 32; i < count; i += 32) m = fmaxf(m, __ldcg(row(i) + reference));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float base = m == -INFINITY ? 0.f : m;
    l = 0.f;
#pragma unroll
    for (int x = 0; x < D / 32; ++x) acc[x] = 0.f;
    float w = 0.f;
#pragma unroll 1
    for (int i = 0; i < count; i += TOGETHER) {
        if (i > 0) fetch(i);
        if (i % 32 == 0) {
            if (i > 0) {
                mine = -INFINITY;
                t = 0.f;
                if (i + lane < count) {
                    mine = __ldcg(row(i + lane) + reference);
                    t = __ldcg(row(i + lane) + total);
                }
            }
            w = ex2(mine - base);
        }
#pragma unroll
        for (int k = 0; k < TOGETHER; ++k) {
            const float f = __shfl_sync(0xffffffffu, w, (i + k) & 31), tk = __shfl_sync(0xffffffffu, t, (i + k) & 31);
            if (i + k < count) {
                l = fmaf(tk, f, l);
#pragma unroll
                for (int x = 0; x < D / 32; ++x) acc[x] = fmaf(v[k][x], f, acc[x]);
            }
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
__device__ __forceinline__ unsigned tile_units(const AttendArgs &a, int b) {  // a thread
    if (b >= a.c.batch) return 0u;
    const AttendSequence s = attend_sequence(a, b);
    unsigned sum = 0u;
    for (int p = 0, n = tile_pairs(a, s); p < n; ++p) sum += tile_blocks(a, s, p);
    return sum * a.c.kv_heads;
}
// The units of sequence `lane`, or of sequence b, by a whole warp: up to 32 sequences, whose pairs of tiles the lanes share
__device__ __forceinline__ unsigned tile_units_of_few(const AttendArgs &a) {
    const int lane = threadIdx.x & 31;
    unsigned mine = 0u;
    for (int b = 0; b < a.c.batch; ++b) {
        const AttendSequence s = attend_sequence(a, b);
        unsigned sum = 0u;
        for (int p = lane, n = tile_pairs(a, s); p < n; p += 32) sum += tile_blocks(a, s, p);
        sum = warp_add(sum) * a.c.kv_heads;
        if (b == lane) mine = sum;
    }
    return mine;
}
template <int WARPS>
__device__ __forceinline__ unsigned count_tile_units(const AttendArgs &a, unsigned (&totals)[WARPS], unsigned &mine) {
    if (a.c.batch <= 8) {
        mine = tile_units_of_few(a);
        return warp_units(mine);
    }
    return count_units<WARPS>(a.c.batch, [&](int b) { return tile_units(a, b); }, totals, mine);
}
struct TileCursor {
    unsigned u, end;
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
    __device__ __forceinline__ void find(const AttendArgs &a, unsigned mine, unsigned at) {
        const int lane = threadIdx.x & 31;
        unsigned base;
        u = at;
        b = sequence_of_unit(a.c.batch, [&](int i) { return tile_units(a, i); }, mine, at, base);
        open(a);
        for (int p0 = 0; p0 < pairs; p0 += 32) {
            const int k = lane_of_unit(p0 + lane < pairs ? (unsigned)tile_blocks(a, s, p0 + lane) * a.c.kv_heads : 0u, at, base);
            if (k < 32) {
                pair = p0 + k;
                break;
            }
        }
        blocks = tile_blocks(a, s, pair);
        head = (int)((at - base) / blocks);
        block = (int)((at - base) % blocks);
    }
    __device__ __forceinline__ int run() const { return (int)min((unsigned)(blocks - block), end - u); }  // blocks of the item in this share
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
int launch_attend_tiles(const AttendArgs &a, bool behind, cudaStream_t st);

// A launch; `behind`: as a programmatic dependent launch behind the one before on the stream
template <typename Args>
inline int launch_attention(void (*kernel)(Args), unsigned grid, int threads, size_t smem, bool behind, const Args &args, cudaStream_t st) {
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(grid);
    config.blockDim = dim3((unsigned)threads);
    config.dynamicSmemBytes = smem;
    config.stream = st;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute;
    config.numAttrs = behind ? 1 : 0;
    return cudaLaunchKernelEx(&config, kernel, args) == cudaSuccess ? check_launch() : G2D_ERR_CUDA;
}

}  // namespace g2d
