// Attention of few query rows per sequence over the packed cache: one token per sequence, or a few drafted ones.
//
//   o_r = sum_j softmax_j(u_rj) v_j,   u_rj = scale q_r . k_j  (capped: cap tanh(u / cap); biased: + slope_h (j - p_r)),   j < limit_r,
//
// with k_j = s_j (c_j - 8), v_j likewise, codes c in 0 .. 15, and zeros where no j is left.  The rows of one kv head are all (token, head of its group).
//
// Work.  A unit is a block of 64 keys of one item (sequence, kv head, eight or sixteen rows).  The units of all items, one after the other, are dealt
// out evenly to the CTAs, and a CTA's to its warps, however long each sequence is: lengths are known on the device only.  A warp goes through its units with a
// running maximum and sum per row and keeps its results in registers; an item that lies within one warp's share is written at once, the others leave
// partial results (at most two per warp), which the CTA adds up in the order of the keys; what of an item lies in several CTAs (at most two parts
// per CTA) attend_join_kernel adds up.
//
// Mathematics.  Codes go to the tensor cores as they are: the bits of c in the lowest (or next) four bits of an fp16 number are c 2^-24 (or c 2^-20), exactly,
// so four codes cost two ANDs and a shift.  The scores are S^T = K Q^T with keys as the rows of A (m16n8k16), the channels of k in the order in which a word of
// codes holds them; Q in fp16 under a power of two per row (bf16 queries lose nothing: 8 bits, and what lies 2^-38 below the row's largest), and the
// products start from -8 sum(q).  The results are O^T = V^T P^T, two keys' words interleaved by a byte permutation, P^T from S^T by
// a transposing matrix move, P s_j in fp16 under a power of two of the block's largest scale: rounded once, to 11 bits, and -8 sum(P s) is formed by
// the same products from the rounded values.  Every block's product starts anew and is added to the results in registers in fp32: the tensor cores truncate, and
// over a long sequence the part -8 sum would leave its truncation behind.
//
// Bound: HBM (head_dim + 4 bytes per key and head), behind it the instructions per key.
#include "g2d_attend.cuh"

namespace g2d {

constexpr int ATTEND_GRID = 148;
// Warps per CTA (a CTA per SM) and stages per warp.  The work of a block is a chain of dependent steps, so warps count for more than stages.
template <int D, int NT>
struct AttendShape {
    static constexpr int WARPS = NT == 1 ? 12 : 8, THREADS = 32 * WARPS, STAGES = NT == 1 ? (D == 128 ? 2 : 4) : 3;
};
constexpr int ATTEND_MOST_WARPS = 12;

template <int D>
struct AttendStage {
    uint8_t k[CACHE_BLOCK * D / 2], v[CACHE_BLOCK * D / 2];
    __half ks[CACHE_BLOCK], vs[CACHE_BLOCK];
};
// A warp's part of an item that it has not the whole of
struct AttendPart {
    int b, item, first, last, blocks;  // blocks first .. last - 1 of `blocks`; last 0: no part
    AttendSequence s;
};
template <int D, int NT>
struct AttendShared {
    using S = AttendShape<D, NT>;
    AttendStage<D> stage[S::WARPS][S::STAGES];
    uint64_t full[S::WARPS][S::STAGES];
    long long totals[S::WARPS];
    AttendPart parts[2 * S::WARPS];
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

// Units of sequence b: of each kv head and each `rows_per_item` rows, its blocks of keys (one at least: rows without keys get their zeros)
__device__ __forceinline__ int64_t attend_units(const AttendArgs &a, const AttendSequence &s, int rows_per_item, int &blocks, int &items) {
    const int64_t rows = (int64_t)s.count * a.group;
    blocks = max((s.keys + CACHE_BLOCK - 1) / CACHE_BLOCK, 1);
    items = rows >= a.rows_from && rows < a.rows_to ? a.c.kv_heads * (int)((rows + rows_per_item - 1) / rows_per_item) : 0;
    return (int64_t)items * blocks;
}
__device__ __forceinline__ int64_t attend_units(const AttendArgs &a, int b, int rows_per_item) {
    int blocks, items;
    return b < a.c.batch ? attend_units(a, attend_sequence(a, b), rows_per_item, blocks, items) : 0;
}
// All threads of a CTA of WARPS warps: the units of all sequences
template <int WARPS>
__device__ __forceinline__ int64_t all_units(const AttendArgs &a, int rows_per_item, long long (&totals)[WARPS]) {
    int64_t mine = 0;
    for (int b = threadIdx.x; b < a.c.batch; b += 32 * WARPS) mine += attend_units(a, b, rows_per_item);
    mine = warp_sum(mine);
    if ((threadIdx.x & 31) == 0) totals[threadIdx.x >> 5] = mine;
    __syncthreads();
    int64_t all = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) all += totals[w];
    return all;
}
// A warp: the sequence that unit u belongs to, and the units before it
__device__ __forceinline__ int sequence_of_unit(const AttendArgs &a, int rows_per_item, int64_t u, int64_t &before) {
    const int lane = threadIdx.x & 31;
    int64_t base = 0;
    for (int b0 = 0; b0 < a.c.batch; b0 += 32) {
        int64_t sum = attend_units(a, b0 + lane, rows_per_item);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t up = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += up;
        }
        const unsigned past = __ballot_sync(0xffffffffu, base + sum > u);
        if (past) {
            const int at = __ffs(past) - 1;
            const int64_t upto = __shfl_sync(0xffffffffu, sum, at > 0 ? at - 1 : 0);
            before = base + (at > 0 ? upto : 0);
            return b0 + at;
        }
        base += __shfl_sync(0xffffffffu, sum, 31);
    }
    before = base;
    return a.c.batch;
}

// A place in the list of units
struct AttendCursor {
    int64_t u, end;
    int b, item, block, blocks, items;
    AttendSequence s;
    __device__ __forceinline__ void open(const AttendArgs &a, int rows_per_item) {  // sequence b, or the next one that has units
        for (;; ++b) {
            if (b >= a.c.batch) {  // not reached while u < end
                end = u;
                return;
            }
            s = attend_sequence(a, b);
            if (attend_units(a, s, rows_per_item, blocks, items) > 0) return;
        }
    }
    __device__ __forceinline__ void step(const AttendArgs &a, int rows_per_item) {
        if (++u >= end) return;
        if (++block < blocks) return;
        block = 0;
        if (++item < items) return;
        item = 0;
        ++b;
        open(a, rows_per_item);
    }
};

// Partial results: for each of a slot's rows, head_dim sums, the maximum and the sum of the exponentials.  Two slots per CTA, behind them two per warp.
template <int D, int ROWS>
__device__ __forceinline__ float *attend_slot(const AttendArgs &a, int64_t slot) {
    return a.partial + slot * (ROWS * (D + 2));
}
constexpr int WARP_SLOTS = 2 * ATTEND_GRID;

template <int D, int NT, bool MODS>
__global__ void __launch_bounds__(AttendShape<D, NT>::THREADS, 1) attend_rows_kernel(const AttendArgs a) {
    constexpr int ATTEND_WARPS = AttendShape<D, NT>::WARPS, ATTEND_STAGES = AttendShape<D, NT>::STAGES;
    constexpr int ROWS = 8 * NT, KSTEPS = D / 16, MTILES = D / 16, WORDS = D / 32, CODE_BYTES = D / 2;
    extern __shared__ __align__(128) unsigned char attend_smem_raw[];
    AttendShared<D, NT> &sh = *reinterpret_cast<AttendShared<D, NT> *>(attend_smem_raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const CacheView &c = a.c;
    if (lane == 0) {
        for (int s = 0; s < ATTEND_STAGES; ++s) mbar_init(&sh.full[warp][s], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    let_the_next_launch_start();
    if (lane < 2) sh.parts[2 * warp + lane].last = 0;
    const int64_t units = all_units<ATTEND_WARPS>(a, ROWS, sh.totals);  // its barrier is that of the initialisation as well
    const int64_t shares = min(units, (int64_t)gridDim.x), share = blockIdx.x;
    AttendCursor cur;
    cur.u = cur.end = 0;
    if (share < shares) {
        const int64_t u0 = share * units / shares, n = (share + 1) * units / shares - u0;
        cur.u = u0 + warp * n / ATTEND_WARPS;
        cur.end = u0 + (warp + 1) * n / ATTEND_WARPS;
    }
    if (cur.u < cur.end) {
        int64_t before;
        cur.b = sequence_of_unit(a, ROWS, cur.u, before);
        cur.open(a, ROWS);
        cur.item = (int)((cur.u - before) / cur.blocks);
        cur.block = (int)((cur.u - before) % cur.blocks);
    }

    // ---- loads: a block's keys lie in one page or in several; lane x brings piece x / 4 of codes or scales, of keys or values ----
    const int piece_shift = min(c.page_shift, 6), piece_keys = 1 << piece_shift, pieces = CACHE_BLOCK >> piece_shift;
    AttendCursor ahead = cur;
    auto page_of = [&](const AttendCursor &at) {  // the page of this lane's piece, or -1
        const int key = at.block * CACHE_BLOCK + (lane >> 2) * piece_keys;
        if (at.u >= at.end || lane >= 4 * pieces || key >= at.s.keys) return -1;
        const int page = c.table[at.b * c.table_stride + (key >> c.page_shift)];
        return page < c.pages ? page : -1;
    };
    int next_page = page_of(ahead);
    unsigned present[ATTEND_STAGES];  // which pieces of a stage were loaded: four bits each
#pragma unroll
    for (int s = 0; s < ATTEND_STAGES; ++s) present[s] = 0u;
    auto issue = [&](int stage, unsigned &here) {
        AttendStage<D> &st = sh.stage[warp][stage];
        uint64_t *bar = &sh.full[warp][stage];
        here = __ballot_sync(0xffffffffu, next_page >= 0);
        const int whole = __popc(here & 0x11111111u);
        if (lane == 0) mbar_expect_tx(bar, (uint32_t)(whole * piece_keys * (2 * CODE_BYTES + 4)));
        __syncwarp();
        if (next_page >= 0) {
            const int place = (ahead.block * CACHE_BLOCK + (lane >> 2) * piece_keys) & (c.page_size - 1), head = ahead.item % c.kv_heads, to = (lane >> 2) * piece_keys;
            const int64_t row = (((int64_t)next_page * c.kv_heads + head) << c.page_shift) + place;
            const int what = lane & 3;
            if (what == 0) bulk_load(st.k + to * CODE_BYTES, c.k_codes + row * CODE_BYTES, piece_keys * CODE_BYTES, bar);
            else if (what == 1) bulk_load(st.v + to * CODE_BYTES, c.v_codes + row * CODE_BYTES, piece_keys * CODE_BYTES, bar);
            else if (what == 2) bulk_load(st.ks + to, c.k_scale + row, piece_keys * 2, bar);
            else bulk_load(st.vs + to, c.v_scale + row, piece_keys * 2, bar);
        }
        ahead.step(a, ROWS);
        next_page = page_of(ahead);
    };
#pragma unroll
    for (int s = 0; s < ATTEND_STAGES; ++s)
        if (ahead.u < ahead.end) issue(s, present[s]);

    const int pi_g = (g & 4) | ((g & 1) << 1) | ((g >> 1) & 1);  // row g of S^T is key pi_g: lanes with neighbouring t then read V from both halves of the banks
    int stage = 0, phase = 0;
    bool sound = true;
    while (cur.u < cur.end) {
        // ---- a run of blocks of one item ----
        const int head = cur.item % c.kv_heads, row0 = cur.item / c.kv_heads * ROWS, rows = cur.s.count * a.group;
        const int first_block = cur.block, last_block = (int)min((int64_t)cur.blocks, (int64_t)cur.block + (cur.end - cur.u));
        const AttendSequence seq = cur.s;
        uint32_t qf[NT][KSTEPS][2];
        float factor[NT][2], start[NT][2], slope[NT][2];
        int limit[NT][2], place[NT][2], least = 0x7fffffff;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int r = row0 + 8 * j + g;
            const bool real = r < rows;
            const int token = real ? r / a.group : 0, h = head * a.group + (real ? r % a.group : 0);
            uint4 raw[WORDS];
            const uint16_t *const q = (const uint16_t *)a.q + (int64_t)(seq.first + token) * a.q_token_stride + (int64_t)h * a.q_head_stride + t * (D / 4);
#pragma unroll
            for (int w = 0; w < WORDS; ++w) raw[w] = real ? reinterpret_cast<const uint4 *>(q)[w] : make_uint4(0u, 0u, 0u, 0u);
            float x[WORDS * 8];
            unsigned largest = 0u;
#pragma unroll
            for (int w = 0; w < WORDS; ++w) {
                const uint32_t word[4] = {raw[w].x, raw[w].y, raw[w].z, raw[w].w};
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[8 * w + e] = half_bits_to_float((word[e >> 1] >> (16 * (e & 1))) & 0xffffu, c.bf16);
                    largest = max(largest, __float_as_uint(x[8 * w + e]) & 0x7fffffffu);
                }
            }
            largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
            largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
            const int e2 = range_exponent(__uint_as_float(largest));
            const float down = power_of_two(-e2);
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < WORDS; ++w) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[8 * w + e] *= down;
                    sum += x[8 * w + e];  // as fp16 below: what that loses of a value lies 2^-38 below the largest
                }
                const float s16 = 0.0625f;
                qf[j][2 * w][0] = pack_halves(x[8 * w], x[8 * w + 4], 0);
                qf[j][2 * w][1] = pack_halves(x[8 * w + 2], x[8 * w + 6], 0);
                qf[j][2 * w + 1][0] = pack_halves(x[8 * w + 1] * s16, x[8 * w + 5] * s16, 0);
                qf[j][2 * w + 1][1] = pack_halves(x[8 * w + 3] * s16, x[8 * w + 7] * s16, 0);
            }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            const float my_factor = 16777216.f * a.scale * (MODS ? 1.f : LOG2E) * power_of_two(e2), my_start = -8.f / 16777216.f * sum;
            const int my_limit = real ? visible_keys(a, seq, token) : seq.keys;
            const float my_slope = MODS && a.slopes ? a.slopes[h] : 0.f;
            const int my_place = seq.length - seq.count + token;
#pragma unroll
            for (int x2 = 0; x2 < 2; ++x2) {
                const int from = (2 * t + x2) * 4;
                factor[j][x2] = __shfl_sync(0xffffffffu, my_factor, from);
                start[j][x2] = __shfl_sync(0xffffffffu, my_start, from);
                limit[j][x2] = __shfl_sync(0xffffffffu, my_limit, from);
                if (MODS) {
                    slope[j][x2] = __shfl_sync(0xffffffffu, my_slope, from);
                    place[j][x2] = __shfl_sync(0xffffffffu, my_place, from);
                }
                least = min(least, limit[j][x2]);
            }
        }
        least = __reduce_min_sync(0xffffffffu, least);
        float m[NT][2], l[NT][2], o[MTILES][NT][4];
        int unit = 0;  // the scales' power of two, as the exponent bits of a float
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            m[j][0] = m[j][1] = -INFINITY;
            l[j][0] = l[j][1] = 0.f;
#pragma unroll
            for (int e = 0; e < MTILES; ++e) o[e][j][0] = o[e][j][1] = o[e][j][2] = o[e][j][3] = 0.f;
        }
        for (int block = first_block; block < last_block; ++block) {
            const AttendStage<D> &st = sh.stage[warp][stage];
            unsigned here = 0u;
#pragma unroll
            for (int s = 0; s < ATTEND_STAGES; ++s)
                if (s == stage) here = present[s];
            if (sound && !mbar_wait(&sh.full[warp][stage], phase, 20, a.wait_cycles)) sound = false;
            sound = __all_sync(0xffffffffu, sound);
            const int key0 = block * CACHE_BLOCK;
            const bool masked = key0 + CACHE_BLOCK > least || (here & 0x11111111u) != (0x11111111u >> (32 - 4 * pieces));
            // ---- scores ----
            float s[4][NT][4];
            uint32_t lo[4][WORDS], hi[4][WORDS];
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) {
                const uint8_t *const at = st.k + (mt * 16 + pi_g) * CODE_BYTES + t * (D / 8);
                if constexpr (WORDS == 4) {
                    const uint4 x = *reinterpret_cast<const uint4 *>(at), y = *reinterpret_cast<const uint4 *>(at + 8 * CODE_BYTES);
                    lo[mt][0] = x.x; lo[mt][1] = x.y; lo[mt][2] = x.z; lo[mt][3] = x.w;
                    hi[mt][0] = y.x; hi[mt][1] = y.y; hi[mt][2] = y.z; hi[mt][3] = y.w;
                } else {
                    const uint2 x = *reinterpret_cast<const uint2 *>(at), y = *reinterpret_cast<const uint2 *>(at + 8 * CODE_BYTES);
                    lo[mt][0] = x.x; lo[mt][1] = x.y;
                    hi[mt][0] = y.x; hi[mt][1] = y.y;
                }
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    s[mt][j][0] = s[mt][j][2] = start[j][0];
                    s[mt][j][1] = s[mt][j][3] = start[j][1];
                }
            }
#pragma unroll
            for (int w = 0; w < WORDS; ++w) {  // four chains of products side by side
#pragma unroll
                for (int mt = 0; mt < 4; ++mt)
#pragma unroll
                    for (int j = 0; j < NT; ++j)
                        mma_f16(s[mt][j], lo[mt][w] & 0x000f000fu, hi[mt][w] & 0x000f000fu, (lo[mt][w] >> 8) & 0x000f000fu, (hi[mt][w] >> 8) & 0x000f000fu, qf[j][2 * w][0], qf[j][2 * w][1]);
#pragma unroll
                for (int mt = 0; mt < 4; ++mt)
#pragma unroll
                    for (int j = 0; j < NT; ++j)
                        mma_f16(s[mt][j], lo[mt][w] & 0x00f000f0u, hi[mt][w] & 0x00f000f0u, (lo[mt][w] >> 8) & 0x00f000f0u, (hi[mt][w] >> 8) & 0x00f000f0u, qf[j][2 * w + 1][0],
                                qf[j][2 * w + 1][1]);
            }
            // ---- scales, masks, maximum ----
            float vs[8], top[NT][2];
            unsigned largest = 0u;
#pragma unroll
            for (int j = 0; j < NT; ++j) top[j][0] = top[j][1] = -INFINITY;
            unsigned hidden[NT][2];  // bit 2 mt + half: masked keys
#pragma unroll
            for (int j = 0; j < NT; ++j) hidden[j][0] = hidden[j][1] = 0u;
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int key = mt * 16 + half * 8 + pi_g;
                    const float ks = __half2float(st.ks[key]);
                    float sv = __half2float(st.vs[key]);
                    const bool gone = masked && (key0 + key >= seq.keys || !((here >> (4 * (key >> piece_shift))) & 1u));
                    if (gone) sv = 0.f;  // what lies there may be anything
                    vs[2 * mt + half] = sv;
                    const unsigned size = __float_as_uint(sv) & 0x7fffffffu;
                    largest = max(largest, size < 0x7f800000u ? size : 0u);  // one that is not finite may be masked for some rows: it sets no unit
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
#pragma unroll
                        for (int x2 = 0; x2 < 2; ++x2) {
                            float u = s[mt][j][2 * half + x2] * factor[j][x2] * ks;
                            if (MODS) {
                                if (a.softcap > 0.f) u = capped(u, a.softcap, 2.f * LOG2E / a.softcap);
                                u = fmaf(slope[j][x2], (float)(key0 + key - place[j][x2]), u) * LOG2E;
                            }
                            if (gone || (masked && key0 + key >= limit[j][x2])) {
                                u = -INFINITY;
                                hidden[j][x2] |= 1u << (2 * mt + half);
                            }
                            s[mt][j][2 * half + x2] = u;
                            top[j][x2] = fmaxf(top[j][x2], u);
                        }
                    }
                }
            }
            largest = __reduce_max_sync(0xffffffffu, largest);
            const int new_unit = max(unit, (int)(largest >> 23));
            const float grown = unit == 0 ? 1.f : power_of_two(max(unit - new_unit, -126));  // nothing to scale yet
            unit = new_unit;
            const float vnorm = power_of_two(min(13 - (unit - 127), 127));
            float keep[NT][2];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
#pragma unroll
                for (int x2 = 0; x2 < 2; ++x2) {
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1) top[j][x2] = fmaxf(top[j][x2], __shfl_xor_sync(0xffffffffu, top[j][x2], off));
                    const float now = fmaxf(m[j][x2], top[j][x2]);
                    const float base = now == -INFINITY ? 0.f : now;
                    keep[j][x2] = ex2(m[j][x2] - base);
                    m[j][x2] = now;
                    l[j][x2] *= keep[j][x2];
                    top[j][x2] = base;
                    keep[j][x2] *= grown;
                }
            }
            // ---- exponentials and their products with the scales, transposed ----
            uint32_t pf[4][NT][2];
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) {
#pragma unroll
                for (int j = 0; j < NT; ++j) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const float p0 = ex2(s[mt][j][2 * half] - top[j][0]), p1 = ex2(s[mt][j][2 * half + 1] - top[j][1]);
                        l[j][0] += p0;
                        l[j][1] += p1;
                        const float w = vs[2 * mt + half] * vnorm;
                        float w0 = p0 * w, w1 = p1 * w;
                        if (masked) {  // a masked key counts for nothing, whatever its scale
                            if ((hidden[j][0] >> (2 * mt + half)) & 1u) w0 = 0.f;
                            if ((hidden[j][1] >> (2 * mt + half)) & 1u) w1 = 0.f;
                        }
                        pf[mt][j][half] = transposed(pack_halves(w0, w1, 0));
                    }
                }
            }
            // ---- results: sixteen keys at a time ----
            float acc[MTILES][NT][4];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                float less[4] = {0.f, 0.f, 0.f, 0.f};  // -8 2^-24 sum of the products, in every row
#pragma unroll
                for (int mt = 0; mt < 4; ++mt) mma_f16(less, 0x80088008u, 0x80088008u, 0x80088008u, 0x80088008u, pf[mt][j][0], pf[mt][j][1]);
#pragma unroll
                for (int e = 0; e < MTILES; ++e) {
                    const float f = e & 1 ? 16.f : 1.f;  // odd places of a word are sixteen times as large
                    acc[e][j][0] = acc[e][j][2] = f * less[0];
                    acc[e][j][1] = acc[e][j][3] = f * less[1];
                }
            }
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) {
                // rows 2t, 2t + 1 (and 8 more) of S^T are the keys t' and t' + 2, t' = 2 (t / 2) ... in the order of pi
                const int k0 = mt * 16 + ((2 * t) & 4) + (t & 1), k1 = k0 + 2;
                uint32_t lo[2][2], hi[2][2];  // [pair of keys][word]: nibbles 0..3 and 4..7 of both keys
#pragma unroll
                for (int pair = 0; pair < 2; ++pair) {
                    if constexpr (D == 128) {
                        const uint2 x = *reinterpret_cast<const uint2 *>(st.v + (k0 + 8 * pair) * CODE_BYTES + g * 8), y = *reinterpret_cast<const uint2 *>(st.v + (k1 + 8 * pair) * CODE_BYTES + g * 8);
                        lo[pair][0] = __byte_perm(x.x, y.x, 0x5410);
                        hi[pair][0] = __byte_perm(x.x, y.x, 0x7632);
                        lo[pair][1] = __byte_perm(x.y, y.y, 0x5410);
                        hi[pair][1] = __byte_perm(x.y, y.y, 0x7632);
                    } else {
                        const uint32_t x = *reinterpret_cast<const uint32_t *>(st.v + (k0 + 8 * pair) * CODE_BYTES + g * 4), y = *reinterpret_cast<const uint32_t *>(st.v + (k1 + 8 * pair) * CODE_BYTES + g * 4);
                        lo[pair][0] = __byte_perm(x, y, 0x5410);
                        lo[pair][1] = __byte_perm(x, y, 0x7632);
                    }
                }
#pragma unroll
                for (int e = 0; e < MTILES; ++e) {
                    const int nibble = e & 3;
                    uint32_t f[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {  // a0, a1: word 0 and 1 of the first pair; a2, a3: of the second
                        const uint32_t word = e < 4 ? lo[x >> 1][x & 1] : hi[x >> 1][x & 1];
                        f[x] = (nibble & 2 ? word >> 8 : word) & (nibble & 1 ? 0x00f000f0u : 0x000f000fu);
                    }
#pragma unroll
                    for (int j = 0; j < NT; ++j) mma_f16(acc[e][j], f[0], f[1], f[2], f[3], pf[mt][j][0], pf[mt][j][1]);
                }
            }
#pragma unroll
            for (int e = 0; e < MTILES; ++e)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int x = 0; x < 4; ++x) o[e][j][x] = fmaf(o[e][j][x], keep[j][x & 1], acc[e][j][x]);
            __syncwarp();  // all lanes have read the stage
            if (sound && ahead.u < ahead.end) {
                unsigned loaded;
                issue(stage, loaded);
#pragma unroll
                for (int s2 = 0; s2 < ATTEND_STAGES; ++s2)
                    if (s2 == stage) present[s2] = loaded;
            }
            if (++stage == ATTEND_STAGES) stage = 0, phase ^= 1;
        }
        // ---- this warp's part of the item ----
        const bool whole = first_block == 0 && last_block == cur.blocks;
        const int part = 2 * warp + (first_block == 0 ? 1 : 0);
        float *const slot = attend_slot<D, ROWS>(a, WARP_SLOTS + 2 * ATTEND_WARPS * share + part);
        if (!whole && lane == 0) sh.parts[part] = AttendPart{cur.b, cur.item, first_block, last_block, cur.blocks, seq};
        const float back = power_of_two(max(24 - 13 + (unit - 127), -126));
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int x2 = 0; x2 < 2; ++x2) {
                const int r = row0 + 8 * j + 2 * t + x2;
                float sum = l[j][x2];
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
                if (r >= rows) continue;
                float f = back;
                if (whole) f = sum == 0.f ? 0.f : __fdividef(f, sum);
                if (!sound) f = NAN;
                float value[D / 8];  // D / 8 neighbouring channels, from g * D / 8 on
#pragma unroll
                for (int e = 0; e < D / 8; ++e) {
                    constexpr int HALF = D / 16;
                    const float x = e < HALF ? o[e][j][x2] : o[e - HALF][j][2 + x2];
                    value[e] = x * (e & 1 ? 0.0625f * f : f);
                }
                if (whole && sum == 0.f && sound) {
#pragma unroll
                    for (int e = 0; e < D / 8; ++e) value[e] = 0.f;
                }
                if (whole) {
                    const int token = r / a.group, h = head * a.group + r % a.group;
                    uint4 *const to = reinterpret_cast<uint4 *>((uint16_t *)a.out + ((int64_t)(seq.first + token) * a.heads + h) * D + g * (D / 8));
#pragma unroll
                    for (int w = 0; w < D / 64; ++w)
                        to[w] = make_uint4(pack_halves(value[8 * w], value[8 * w + 1], c.bf16), pack_halves(value[8 * w + 2], value[8 * w + 3], c.bf16),
                                           pack_halves(value[8 * w + 4], value[8 * w + 5], c.bf16), pack_halves(value[8 * w + 6], value[8 * w + 7], c.bf16));
                } else {
                    const int i = r - row0;
                    float4 *const to = reinterpret_cast<float4 *>(slot + i * D + g * (D / 8));
#pragma unroll
                    for (int w = 0; w < D / 32; ++w) to[w] = make_float4(value[4 * w], value[4 * w + 1], value[4 * w + 2], value[4 * w + 3]);
                    if (g == 0) {
                        slot[ROWS * D + i] = m[j][x2];
                        slot[ROWS * D + ROWS + i] = sum;
                    }
                }
            }
        }
        // on to the next run
        for (int k = last_block - first_block; k > 0; --k) cur.step(a, ROWS);
    }
    if (!sound && lane == 0) {
        let_it_land();  // loads under way must not outlive the shared memory
        if (a.status) atomicExch(a.status, -1);
    }
    // ---- the warps' parts of an item, in the order of the keys: parts that stand together in the list ----
    __syncthreads();
    const auto next_part = [&](int p) {
        while (p < 2 * ATTEND_WARPS && sh.parts[p].last == 0) ++p;
        return p;
    };
    for (int p0 = next_part(0); p0 < 2 * ATTEND_WARPS;) {
        const AttendPart &begin = sh.parts[p0];
        unsigned mask = 1u << p0;
        int p1 = p0, behind = next_part(p0 + 1);
        while (behind < 2 * ATTEND_WARPS && sh.parts[behind].b == begin.b && sh.parts[behind].item == begin.item) {
            p1 = behind;
            mask |= 1u << behind;
            behind = next_part(behind + 1);
        }
        const int count = __popc(mask), first = begin.first, last = sh.parts[p1].last;
        const bool whole = first == 0 && last == begin.blocks;
        const int head = begin.item % c.kv_heads, row0 = begin.item / c.kv_heads * ROWS, rows = begin.s.count * a.group;
        const auto slot_of = [&](int i) {  // the i-th bit of the mask: parts stand close together, so that this is short
            unsigned left = mask;
            for (int k = 0; k < i; ++k) left &= left - 1;
            return attend_slot<D, ROWS>(a, WARP_SLOTS + 2 * ATTEND_WARPS * share + __ffs(left) - 1);
        };
        for (int i = warp; i < ROWS && row0 + i < rows; i += ATTEND_WARPS) {
            float acc[D / 32], m, l;
            merge_parts<D>(count, [&](int k) { return slot_of(k) + i * D; }, [&](int k) { return slot_of(k) + ROWS * D + i; }, [&](int k) { return slot_of(k) + ROWS * D + ROWS + i; }, acc, m, l);
            if (whole) {
                const int token = (row0 + i) / a.group, h = head * a.group + (row0 + i) % a.group;
                write_row<D>((uint16_t *)a.out + ((int64_t)(begin.s.first + token) * a.heads + h) * D, acc, l, c.bf16);
            } else {
                float *const slot = attend_slot<D, ROWS>(a, 2 * share + (first == 0 ? 1 : 0));
#pragma unroll
                for (int x = 0; x < D / 32; ++x) slot[i * D + x * 32 + lane] = acc[x];
                if (lane == 0) {
                    slot[ROWS * D + i] = m;
                    slot[ROWS * D + ROWS + i] = l;
                }
            }
        }
        p0 = behind;
    }
    after_the_launch_before();  // of the tiles' kernel: what follows waits for this one alone
}

// Adds up what items that lie in several CTAs' shares left, in the order of the keys.  A CTA per share and (tiles) 32 rows or (rows) all rows of an item: the one whose
// share an item begins in and does not end in.
constexpr int JOIN_THREADS = 256, TILE_JOINS = TA_ROWS / 32;
struct JoinArgs {
    AttendArgs tiles, rows;
    int tile_ctas;  // the first so many are the tiles'
};
template <int D, int NT>
__global__ void __launch_bounds__(JOIN_THREADS) attend_join_kernel(const JoinArgs j) {
    constexpr int ROWS = 8 * NT, WARPS = JOIN_THREADS / 32;
    __shared__ long long totals[WARPS];
    const int warp = threadIdx.x >> 5;
    if ((int)blockIdx.x < j.tile_ctas) {
        const AttendArgs &a = j.tiles;
        const int64_t units = all_tile_units<WARPS>(a, totals), shares = min(units, (int64_t)TA_GRID), share = blockIdx.x / TILE_JOINS;
        TileCursor cur;
        int64_t u0 = 0, u1 = 0, end = 0;
        if (share + 1 < shares) {
            end = (share + 1) * units / shares;
            cur.find(a, end - 1);
            u0 = end - 1 - cur.block;
            u1 = u0 + cur.blocks;
        }
        after_the_launch_before();  // by every CTA: what follows on the stream must not start before the results are there
        if (u1 <= end || u0 < share * units / shares) return;
        const int count = (int)((u1 * shares - 1) / units - share) + 1;  // the share of unit u1 - 1 is the last one that begins at or before it
        const auto slot_of = [&](int k) { return tile_slot<D>(a, 2 * (share + k) + (k == 0 ? 1 : 0)); };
        for (int i = blockIdx.x % TILE_JOINS * 32 + warp, n = 0; n < 32 / WARPS; ++n, i += WARPS) {
            const int r = cur.pair * TA_ROWS + i;
            if (r >= cur.s.count * a.group) break;
            float acc[D / 32], m, l;
            merge_parts<D>(count, [&](int k) { return slot_of(k) + i * D; }, [&](int k) { return slot_of(k) + TA_ROWS * D + i; }, [&](int k) { return slot_of(k) + TA_ROWS * D + TA_ROWS + i; }, acc, m, l);
            write_row<D>((uint16_t *)a.out + ((int64_t)(cur.s.first + r / a.group) * a.heads + cur.head * a.group + r % a.group) * D, acc, l, a.c.bf16);
        }
    } else {
        const AttendArgs &a = j.rows;
        const int64_t units = all_units<WARPS>(a, ROWS, totals), shares = min(units, (int64_t)ATTEND_GRID), share = blockIdx.x - j.tile_ctas;
        AttendCursor cur;
        int64_t u0 = 0, u1 = 0, end = 0;
        if (share + 1 < shares) {
            int64_t before;
            end = (share + 1) * units / shares;
            cur.u = end - 1;
            cur.end = end;
            cur.b = sequence_of_unit(a, ROWS, end - 1, before);
            cur.open(a, ROWS);
            cur.item = (int)((end - 1 - before) / cur.blocks);
            u0 = before + (int64_t)cur.item * cur.blocks;
            u1 = u0 + cur.blocks;
        }
        after_the_launch_before();
        if (u1 <= end || u0 < share * units / shares) return;
        const int count = (int)((u1 * shares - 1) / units - share) + 1;
        const auto slot_of = [&](int k) { return attend_slot<D, ROWS>(a, 2 * (share + k) + (k == 0 ? 1 : 0)); };
        for (int i = warp; i < ROWS; i += WARPS) {
            const int r = cur.item / a.c.kv_heads * ROWS + i;
            if (r >= cur.s.count * a.group) break;
            float acc[D / 32], m, l;
            merge_parts<D>(count, [&](int k) { return slot_of(k) + i * D; }, [&](int k) { return slot_of(k) + ROWS * D + i; }, [&](int k) { return slot_of(k) + ROWS * D + ROWS + i; }, acc, m, l);
            write_row<D>((uint16_t *)a.out + ((int64_t)(cur.s.first + r / a.group) * a.heads + cur.item % a.c.kv_heads * a.group + r % a.group) * D, acc, l, a.c.bf16);
        }
    }
}

// A launch on the stream behind the one before, as a programmatic dependent launch
template <typename Args>
static int launch_behind(void (*kernel)(Args), unsigned grid, int threads, size_t smem, const Args &args, cudaStream_t st) {
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(grid);
    config.blockDim = dim3((unsigned)threads);
    config.dynamicSmemBytes = smem;
    config.stream = st;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, args) == cudaSuccess ? check_launch() : G2D_ERR_CUDA;
}

// rows and tiles: either or both; both launches share the sequences out between them
template <int D, int NT, bool MODS>
static int launch_rows(const AttendArgs &a, bool behind_tiles, cudaStream_t st) {
    static PerDeviceOnce configured;
    constexpr size_t smem = sizeof(AttendShared<D, NT>);
    if (configured.run([&] { return cudaFuncSetAttribute(attend_rows_kernel<D, NT, MODS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) == cudaSuccess; }) != G2D_OK)
        return G2D_ERR_CUDA;
    if (behind_tiles) return launch_behind(attend_rows_kernel<D, NT, MODS>, ATTEND_GRID, AttendShape<D, NT>::THREADS, smem, a, st);
    attend_rows_kernel<D, NT, MODS><<<ATTEND_GRID, AttendShape<D, NT>::THREADS, smem, st>>>(a);
    return check_launch();
}
template <int D, int NT>
static int launch_attend(const AttendArgs &rows, const AttendArgs &tiles, bool few, bool many, cudaStream_t st) {
    int launched = G2D_OK;
    if (many) launched = launch_attend_tiles(tiles, st);
    if (launched == G2D_OK && few) launched = rows.softcap > 0.f || rows.slopes ? launch_rows<D, NT, true>(rows, many, st) : launch_rows<D, NT, false>(rows, many, st);
    if (launched != G2D_OK) return launched;
    const JoinArgs j{tiles, rows, many ? TA_GRID * TILE_JOINS : 0};
    return launch_behind(attend_join_kernel<D, NT>, (unsigned)(j.tile_ctas + (few ? ATTEND_GRID : 0)), JOIN_THREADS, 0, j, st);
}

// From here on a sequence's rows go by tiles; both sides of the line: see the figures in g2d_attend_tc.cu.
constexpr int TILE_ROWS_FROM = 33;

struct AttendSpace {
    size_t tiles, all;  // the warps' partial results first
};
static AttendSpace attend_space(int head_dim) {
    AttendSpace s;
    s.tiles = ((size_t)ATTEND_GRID * (ATTEND_MOST_WARPS + 1) * 2 * 16 * (head_dim + 2) * sizeof(float) + 255) & ~(size_t)255;
    s.all = s.tiles + attend_tiles_bytes(head_dim);
    return s;
}

}  // namespace g2d

using namespace g2d;

extern "C" int g2d_attend_workspace_bytes(const g2d_attend_desc *desc, size_t *bytes) {
    CacheView c;
    if (!desc || !bytes) return G2D_ERR_BAD_ARGUMENT;
    const int status = cache_view(&desc->cache, &c);
    if (status != G2D_OK) return status;
    *bytes = attend_space(c.head_dim).all;
    return G2D_OK;
}

extern "C" int g2d_cache_attend(const g2d_attend_desc *d, void *stream) {
    AttendArgs a;
    if (!d) return G2D_ERR_BAD_ARGUMENT;
    const int status = cache_view(&d->cache, &a.c);
    if (status != G2D_OK) return status;
    if (d->heads < 1 || d->heads % a.c.kv_heads != 0 || !(d->softcap >= 0.f)) return G2D_ERR_BAD_ARGUMENT;
    if (a.c.tokens == 0 || a.c.batch == 0) return G2D_OK;
    if ((int64_t)a.c.tokens * d->heads > 0x7fffffff) return G2D_ERR_TOO_LARGE;
    if (!d->q || !d->out || (((uintptr_t)d->q | (uintptr_t)d->out) & 15) != 0 || ((d->q_token_stride | d->q_head_stride) & 7) != 0) return G2D_ERR_BAD_ARGUMENT;
    if (!d->workspace || d->workspace_bytes < attend_space(a.c.head_dim).all || ((uintptr_t)d->workspace & 255) != 0) return G2D_ERR_WORKSPACE;
    a.q = d->q;
    a.out = d->out;
    a.q_token_stride = d->q_token_stride;
    a.q_head_stride = d->q_head_stride;
    a.heads = d->heads;
    a.group = d->heads / a.c.kv_heads;
    a.causal = d->causal != 0;
    a.scale = d->scale;
    a.softcap = d->softcap;
    a.slopes = d->slopes;
    a.prefix = d->prefix;
    a.status = d->status;
    a.wait_cycles = WAIT_CYCLES;
    cudaStream_t st = (cudaStream_t)stream;
    // How many rows a sequence has is known here only where all have the same; else the kernels share the sequences out between them.
    const int64_t rows = a.c.offsets ? -1 : (int64_t)(a.c.tokens / a.c.batch) * a.group;
    const bool many = rows < 0 ? (int64_t)a.c.tokens * a.group >= TILE_ROWS_FROM : rows >= TILE_ROWS_FROM, few = rows < TILE_ROWS_FROM;
    AttendArgs t = a;
    t.rows_from = TILE_ROWS_FROM;
    t.rows_to = 0x7fffffff;
    t.partial = (float *)((char *)d->workspace + attend_space(a.c.head_dim).tiles);
    a.rows_from = 1;
    a.rows_to = TILE_ROWS_FROM;
    a.partial = (float *)d->workspace;
    const bool narrow = a.group <= 8 && (rows < 0 || rows <= 8);
    if (a.c.head_dim == 128) return narrow ? launch_attend<128, 1>(a, t, few, many, st) : launch_attend<128, 2>(a, t, few, many, st);
    return narrow ? launch_attend<64, 1>(a, t, few, many, st) : launch_attend<64, 2>(a, t, few, many, st);
}
