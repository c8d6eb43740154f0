// Attention of few query rows per sequence over the packed cache: one token per sequence, or a few drafted ones.
//
//   o_r = sum_j softmax_j(u_rj) v_j,   u_rj = scale q_r . k_j  (capped: cap tanh(u / cap); biased: + slope_h (j - p_r)),   j < limit_r,
//
// with k_j = s_j (c_j - 8), v_j likewise, codes c in 0 .. 15, and zeros where no j is left.  The rows of one kv head are all (token, head of its group).
//
// Work.  A unit is a block of 64 keys of one item (sequence, kv head, eight or sixteen rows).  The units of all items, one after the other, are dealt
// out evenly to the CTAs, and a CTA's to its warps, however long each sequence is: lengths are known on the device only (`even`: whole items to each CTA, where tables are short).  A warp goes through its units with a
// running maximum and sum per row and keeps its results in registers; an item that lies within one warp's share is written at once, the others leave
// partial results (at most two per warp), which the CTA adds up in the order of the keys; what of an item lies in several CTAs (at most two parts
// per CTA) attend_join_kernel adds up.
//
// Mathematics.  Codes go to the tensor cores as they are: the bits of c in the lowest (or next) four bits of an fp16 number are c 2^-24 (or c 2^-20), exactly,
// so four codes cost two ANDs and a shift.  The scores are S^T = K Q^T with keys as the rows of A (m16n8k16), the channels of k in the order in which a word of
// codes holds them; Q in fp16 under a power of two per row (bf16 queries lose nothing: 8 bits, and what lies 2^-38 below the row's largest), and the
// products start from -8 sum(q).  The results are O^T = V^T P^T, two keys' words interleaved by a byte permutation, P^T from S^T by
// a transposing matrix move, P s_j in fp16 under a power of two of the run's largest scale so far (it goes into the exponent, and into the sum of the exponentials alike):
// rounded once, to 11 bits, and -8 sum(P s) is formed by the same products from the rounded values.  Every block's product starts anew and is added to the results in
// registers in fp32: the tensor cores truncate, and over a long sequence the part -8 sum would leave its truncation behind.
// Row g of the tiles of S^T stands for the keys 8 g .. 8 g + 7 of the block, one per tile and half: a lane's scales are one load then.
//
// Bound: HBM (head_dim + 4 bytes per key and head), behind it the products (16 cycles each for a quarter of an SM: 68 for a block of 64 keys and eight rows) and the instructions per key, and
// for short calls the start (counting units, the first pages and codes: about 6 us) and the joins.  64 heads on 8, 128 channels: 131072 keys of one sequence 41 us (3.4 TB/s), 48
// sequences of up to 8191 62 us; 16 sequences of 2000 keys, four queries of 32 heads, capped and biased, 31 us; one of 137 keys 7.2 us.
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
    unsigned totals[S::WARPS];
    AttendPart parts[2 * S::WARPS];
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, const float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ uint32_t transposed(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
// Codes are read once per step: they leave the L2 before what every step reads again (lengths, tables, the kernels' own instructions)
__device__ __forceinline__ uint64_t read_once() {
    uint64_t policy;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    return policy;
}
__device__ __forceinline__ void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar, uint64_t policy) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)), "l"(policy)
                 : "memory");
}

// Units of sequence b: of each kv head and each `rows_per_item` rows, its blocks of keys (one at least: rows without keys get their zeros)
template <int ROWS>
__device__ __forceinline__ unsigned attend_units(const AttendArgs &a, const AttendSequence &s, int &blocks, int &items) {
    const unsigned rows = (unsigned)(s.count * a.group);  // of no more than tokens x heads
    blocks = a.even ? a.even : max((int)(((unsigned)s.keys + CACHE_BLOCK - 1) / CACHE_BLOCK), 1);
    items = rows >= (unsigned)a.rows_from && rows < (unsigned)a.rows_to ? a.c.kv_heads * (int)((rows + ROWS - 1) / ROWS) : 0;
    return (unsigned)items * blocks;
}
template <int ROWS>
__device__ __forceinline__ unsigned attend_units(const AttendArgs &a, int b) {
    int blocks, items;
    return b < a.c.batch ? attend_units<ROWS>(a, attend_sequence(a, b), blocks, items) : 0u;
}

// A place in the list of units
struct AttendCursor {
    int u, end;  // units of the warp's share
    int b, item, block, blocks, items;
    AttendSequence s;
    template <int ROWS>
    __device__ __forceinline__ void open(const AttendArgs &a) {  // sequence b, or the next one that has units
        for (;; ++b) {
            if (b >= a.c.batch) {  // not reached while u < end
                end = u;
                return;
            }
            s = attend_sequence(a, b);
            if (attend_units<ROWS>(a, s, blocks, items) > 0) return;
        }
    }
    template <int ROWS>
    __device__ __forceinline__ void step(const AttendArgs &a) {
        if (++u >= end) return;
        if (++block < blocks) return;
        block = 0;
        if (++item < items) return;
        item = 0;
        ++b;
        open<ROWS>(a);
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
    const auto units_of = [&](int b) { return attend_units<ROWS>(a, b); };
    unsigned mine_units;
    const unsigned grain = max(a.even, 1);  // units that stay together
    const unsigned units = count_units<ATTEND_WARPS>(c.batch, units_of, sh.totals, mine_units);
    if (threadIdx.x == 0) a.joins[blockIdx.x] = AttendJoin{units < UNITS_END ? 0 : -1};
    const AttendShares shares((units < UNITS_END ? units : 0u) / grain, gridDim.x);
    const unsigned share = blockIdx.x;
    AttendCursor cur;
    cur.u = cur.end = 0;
    if (share < shares.count) {
        // of n units the first warps have one each, where there are not enough for all: a warp between two others of an item has a part of it
        const unsigned u0 = shares.begin(share) * grain, n = shares.begin(share + 1) * grain - u0, active = min(n, (unsigned)ATTEND_WARPS);
        if ((unsigned)warp < active) {
            const unsigned mine = u0 + warp * n / active;
            cur.end = (int)(u0 + (warp + 1) * n / active - mine);
            unsigned before;
            cur.b = sequence_of_unit(c.batch, units_of, mine_units, mine, before);
            cur.template open<ROWS>(a);
            cur.item = (int)((mine - before) / cur.blocks);
            cur.block = (int)((mine - before) % cur.blocks);
        }
    }

    // ---- loads: a block's keys lie in one page or in several; lane x brings piece x / 4 of codes or scales, of keys or values ----
    const int piece_shift = min(c.page_shift, 6), piece_keys = 1 << piece_shift, pieces = CACHE_BLOCK >> piece_shift;
    AttendCursor ahead = cur;
    const int what = lane & 3, to = (lane >> 2) * piece_keys;  // this lane's copies: codes of keys, of values, scales of keys, of values, of the keys from `to` on
    const uint32_t key_bytes = what < 2 ? CODE_BYTES : 2;
    const uint8_t *const source = what == 0 ? c.k_codes : what == 1 ? c.v_codes : what == 2 ? (const uint8_t *)c.k_scale : (const uint8_t *)c.v_scale;
    const uint32_t target = (uint32_t)(what == 0 ? offsetof(AttendStage<D>, k) : what == 1 ? offsetof(AttendStage<D>, v) : what == 2 ? offsetof(AttendStage<D>, ks) : offsetof(AttendStage<D>, vs)) + to * key_bytes;
    auto page_of = [&](const AttendCursor &at) {  // what the table says of this lane's piece, or -1
        const int key = at.block * CACHE_BLOCK + to;
        if (at.u >= at.end || lane >= 4 * pieces || key >= at.s.keys) return -1;
        return c.table[at.b * c.table_stride + (key >> c.page_shift)];
    };
    const uint64_t policy = read_once();
    unsigned present[ATTEND_STAGES];  // which pieces of a stage were loaded: four bits each
    auto issue = [&](int stage, unsigned &here, int page, int item, int block) {
        uint64_t *const bar = &sh.full[warp][stage];
        const bool there = page >= 0 && page < c.pages;
        here = __ballot_sync(0xffffffffu, there);
        if (lane == 0) mbar_expect_tx(bar, (uint32_t)(__popc(here & 0x11111111u) * piece_keys * (2 * CODE_BYTES + 4)));
        __syncwarp();
        if (there) {
            const int64_t row = (((int64_t)page * c.kv_heads + item % c.kv_heads) << c.page_shift) + ((block * CACHE_BLOCK + to) & (c.page_size - 1));
            bulk_load(reinterpret_cast<unsigned char *>(&sh.stage[warp][stage]) + target, source + row * key_bytes, piece_keys * key_bytes, bar, policy);
        }
    };
    {
        // the first blocks' pages are asked for together
        int page[ATTEND_STAGES], item[ATTEND_STAGES], block[ATTEND_STAGES];
#pragma unroll
        for (int s = 0; s < ATTEND_STAGES; ++s) {
            page[s] = page_of(ahead);
            item[s] = ahead.u < ahead.end ? ahead.item : -1;
            block[s] = ahead.block;
            if (item[s] >= 0) ahead.template step<ROWS>(a);
        }
#pragma unroll
        for (int s = 0; s < ATTEND_STAGES; ++s) {
            present[s] = 0u;
            if (item[s] >= 0) issue(s, present[s], page[s], item[s], block[s]);
        }
    }
    int next_page = page_of(ahead);

    int stage = 0, phase = 0;
    bool sound = true;
    while (cur.u < cur.end) {
        // ---- a run of blocks of one item ----
        const int head = cur.item % c.kv_heads, row0 = cur.item / c.kv_heads * ROWS, rows = cur.s.count * a.group;
        const int first_block = cur.block, last_block = min(cur.blocks, cur.block + (cur.end - cur.u));
        const AttendSequence seq = cur.s;
        const float cap = a.softcap * LOG2E;
        const bool near = a.softcap <= CAP_NEAR;
        uint32_t qf[NT][KSTEPS][2];
        uint64_t factor[NT];
        float start[NT][2], slope[NT][2];
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
            const float down = power_of_two(-e2) * (a.scale < 0.f ? -1.f : 1.f);  // the scale's sign goes into the queries: the order of a row's products is that of its scores
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
            const float my_factor = fmaxf(16777216.f * fabsf(a.scale) * score_unit<MODS>(a) * power_of_two(e2), 1e-38f),  // above zero: minus infinity stays what it is
                        my_start = -8.f / 16777216.f * sum;
            const int my_limit = real ? visible_keys(a, seq, token) : seq.keys;
            const float my_slope = MODS && a.slopes ? a.slopes[h] * LOG2E : 0.f;
            const int my_place = bias_origin(my_slope, my_limit);
            float two_factors[2];
#pragma unroll
            for (int x2 = 0; x2 < 2; ++x2) {
                const int from = (2 * t + x2) * 4;
                two_factors[x2] = __shfl_sync(0xffffffffu, my_factor, from);
                start[j][x2] = __shfl_sync(0xffffffffu, my_start, from);
                limit[j][x2] = __shfl_sync(0xffffffffu, my_limit, from);
                if (MODS) {
                    slope[j][x2] = __shfl_sync(0xffffffffu, my_slope, from);
                    place[j][x2] = __shfl_sync(0xffffffffu, my_place, from);
                }
                least = min(least, limit[j][x2]);
            }
            factor[j] = pack2(two_factors[0], two_factors[1]);
        }
        least = __reduce_min_sync(0xffffffffu, least);
        // per row: the largest score so far in units of its factor, the reference of the exponentials (as a power of two), their sum; `unit`: the scales' power of two, as exponent bits
        float m[NT][2], refer[NT][2];
        uint64_t l[NT], o[MTILES][NT][2];
        int unit = 0, lift = 0;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            m[j][0] = m[j][1] = -INFINITY;
            refer[j][0] = refer[j][1] = -INFINITY;
            l[j] = 0ull;
#pragma unroll
            for (int e = 0; e < MTILES; ++e) o[e][j][0] = o[e][j][1] = 0ull;
        }
        // MASKED: some row does not see all 64 keys of the block, or some are not there
        const auto take = [&](auto masked, const AttendStage<D> &st, int key0, unsigned here) {
            constexpr bool MASKED = decltype(masked)::value;
            // ---- scores ----
            float s[4][NT][4];
            {
                uint32_t lo[4][WORDS], hi[4][WORDS];
#pragma unroll
                for (int mt = 0; mt < 4; ++mt) {
                    const uint8_t *const at = st.k + (8 * g + 2 * mt) * CODE_BYTES + t * (D / 8);
                    if constexpr (WORDS == 4) {
                        const uint4 x = *reinterpret_cast<const uint4 *>(at), y = *reinterpret_cast<const uint4 *>(at + CODE_BYTES);
                        lo[mt][0] = x.x; lo[mt][1] = x.y; lo[mt][2] = x.z; lo[mt][3] = x.w;
                        hi[mt][0] = y.x; hi[mt][1] = y.y; hi[mt][2] = y.z; hi[mt][3] = y.w;
                    } else {
                        const uint2 x = *reinterpret_cast<const uint2 *>(at), y = *reinterpret_cast<const uint2 *>(at + CODE_BYTES);
                        lo[mt][0] = x.x; lo[mt][1] = x.y;
                        hi[mt][0] = y.x; hi[mt][1] = y.y;
                    }
                }
#pragma unroll
                for (int w = 0; w < WORDS; ++w) {  // four chains of products side by side
#pragma unroll
                    for (int mt = 0; mt < 4; ++mt)
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            const uint32_t a0 = lo[mt][w] & 0x000f000fu, a1 = hi[mt][w] & 0x000f000fu, a2 = (lo[mt][w] >> 8) & 0x000f000fu, a3 = (hi[mt][w] >> 8) & 0x000f000fu;
                            if (w == 0) mma_f16(s[mt][j], a0, a1, a2, a3, qf[j][0][0], qf[j][0][1], {start[j][0], start[j][1], start[j][0], start[j][1]});
                            else mma_f16(s[mt][j], a0, a1, a2, a3, qf[j][2 * w][0], qf[j][2 * w][1]);
                        }
#pragma unroll
                    for (int mt = 0; mt < 4; ++mt)
#pragma unroll
                        for (int j = 0; j < NT; ++j)
                            mma_f16(s[mt][j], lo[mt][w] & 0x00f000f0u, hi[mt][w] & 0x00f000f0u, (lo[mt][w] >> 8) & 0x00f000f0u, (hi[mt][w] >> 8) & 0x00f000f0u, qf[j][2 * w + 1][0],
                                    qf[j][2 * w + 1][1]);
                }
            }
            // ---- scales: of the keys 8 g .. 8 g + 7, key 2 mt + half for the rows of tile mt ----
            const uint4 kraw = *reinterpret_cast<const uint4 *>(st.ks + 8 * g), vraw = *reinterpret_cast<const uint4 *>(st.vs + 8 * g);
            // a scale that is not finite makes its key's scores NaN: for an infinite one, zeros in its codes leave what -8 sum(q) and the products lose to rounding, times infinity
            uint32_t kw[4] = {kraw.x, kraw.y, kraw.z, kraw.w};
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) kw[mt] = nan_unless_finite(kw[mt]);
            uint32_t vw[4] = {vraw.x, vraw.y, vraw.z, vraw.w};
            unsigned gone = 0u;  // MASKED: keys that are not there
            if constexpr (MASKED) {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (key0 + 8 * g + k >= seq.keys || !((here >> (4 * ((8 * g + k) >> piece_shift))) & 1u)) gone |= 1u << k;
#pragma unroll
                for (int mt = 0; mt < 4; ++mt) {  // what lies there may be anything
                    if ((gone >> (2 * mt)) & 1u) vw[mt] &= 0xffff0000u;
                    if ((gone >> (2 * mt + 1)) & 1u) vw[mt] &= 0x0000ffffu;
                }
            }
            unsigned largest = 0u;  // of the values' scales, as the bits of a half; one that is not finite may be masked for some rows: it sets no unit
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) {
                const unsigned x = vw[mt] & 0x7fffu, y = (vw[mt] >> 16) & 0x7fffu;
                largest = max(largest, max(x < 0x7c00u ? x : 0u, y < 0x7c00u ? y : 0u));
            }
            largest = __reduce_max_sync(0xffffffffu, largest);
            const int new_unit = max(unit, (int)(__float_as_uint(__half2float(__ushort_as_half((unsigned short)largest))) >> 23));
            const int new_lift = new_unit == 0 ? 0 : 13 - (new_unit - 127);  // brings the largest scale to 2^13 .. 2^14; of halves: from -2 to 37
            const float grown = power_of_two(new_lift - lift);
            unit = new_unit;
            lift = new_lift;
            // ---- scores in units of the factors, and their maximum ----
            float top[NT][2];
#pragma unroll
            for (int j = 0; j < NT; ++j) top[j][0] = top[j][1] = -INFINITY;
            unsigned hidden[NT][2];  // MASKED: bit k: key 8 g + k is not for this row
            float away[NT][2];       // MODS: the distance of key 8 g
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int x2 = 0; x2 < 2; ++x2) {
                    if (MODS) away[j][x2] = (float)(key0 + 8 * g - place[j][x2]);
                    if (MASKED) hidden[j][x2] = gone | (0xffu << min(max(limit[j][x2] - key0 - 8 * g, 0), 8));
                }
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) {
                const float2 ks = __half22float2(*reinterpret_cast<const __half2 *>(&kw[mt]));
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint64_t k2 = half ? pack2(ks.y, ks.y) : pack2(ks.x, ks.x);
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        float &u0 = s[mt][j][2 * half], &u1 = s[mt][j][2 * half + 1];
                        unpack2(mul2(pack2(u0, u1), k2), u0, u1);
                        if constexpr (MODS) {  // in units of log2 from here on
                            unpack2(mul2(pack2(u0, u1), factor[j]), u0, u1);
                            if (a.softcap > 0.f) u0 = capped(u0, cap, near), u1 = capped(u1, cap, near);
                            u0 = fmaf(slope[j][0], away[j][0] + (float)(2 * mt + half), u0);
                            u1 = fmaf(slope[j][1], away[j][1] + (float)(2 * mt + half), u1);
                        }
                        if constexpr (MASKED) {
                            if ((hidden[j][0] >> (2 * mt + half)) & 1u) u0 = -INFINITY;
                            if ((hidden[j][1] >> (2 * mt + half)) & 1u) u1 = -INFINITY;
                        }
                        top[j][0] = fmaxf(top[j][0], u0);
                        top[j][1] = fmaxf(top[j][1], u1);
                    }
                }
            }
            uint64_t keep[NT], less[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                float f[2] = {1.f, 1.f}, k[2], r[2];
                if constexpr (!MODS) unpack2(factor[j], f[0], f[1]);
#pragma unroll
                for (int x2 = 0; x2 < 2; ++x2) {
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1) top[j][x2] = fmaxf(top[j][x2], __shfl_xor_sync(0xffffffffu, top[j][x2], off));
                    const float old = m[j][x2];
                    m[j][x2] = fmaxf(old, top[j][x2]);
                    const float now = m[j][x2] == -INFINITY ? 0.f : m[j][x2] * f[x2];
                    k[x2] = old == -INFINITY ? grown : ex2(old * f[x2] - now) * grown;
                    r[x2] = now - (float)lift;
                    refer[j][x2] = m[j][x2] == -INFINITY ? -INFINITY : r[x2];
                }
                keep[j] = pack2(k[0], k[1]);
                less[j] = pack2(-r[0], -r[1]);
                l[j] = mul2(l[j], keep[j]);
            }
            // ---- exponentials and their products with the scales, transposed ----
            uint32_t pf[4][NT][2];
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) {
                const float2 vs = __half22float2(*reinterpret_cast<const __half2 *>(&vw[mt]));
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint64_t v2 = half ? pack2(vs.y, vs.y) : pack2(vs.x, vs.x);
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        const uint64_t u = pack2(s[mt][j][2 * half], s[mt][j][2 * half + 1]);
                        float e0, e1, w0, w1;
                        unpack2(MODS ? add2(u, less[j]) : fma2(u, factor[j], less[j]), e0, e1);
                        const uint64_t p = pack2(ex2(e0), ex2(e1));
                        l[j] = add2(l[j], p);
                        unpack2(mul2(p, v2), w0, w1);
                        if constexpr (MASKED) {  // a masked key counts for nothing, whatever its scale
                            if ((hidden[j][0] >> (2 * mt + half)) & 1u) w0 = 0.f;
                            if ((hidden[j][1] >> (2 * mt + half)) & 1u) w1 = 0.f;
                        }
                        pf[mt][j][half] = transposed(pack_halves(w0, w1, 0));
                    }
                }
            }
            // ---- results: sixteen keys at a time, from -8 2^-24 times the sum of the products (sixteen times as much at odd places of a word) ----
            float base[NT][2][4];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                float b[4];
                mma_f16(b, 0x80088008u, 0x80088008u, 0x80088008u, 0x80088008u, pf[0][j][0], pf[0][j][1], {0.f, 0.f, 0.f, 0.f});
#pragma unroll
                for (int mt = 1; mt < 4; ++mt) mma_f16(b, 0x80088008u, 0x80088008u, 0x80088008u, 0x80088008u, pf[mt][j][0], pf[mt][j][1]);
#pragma unroll
                for (int x = 0; x < 4; ++x) base[j][0][x] = b[x & 1], base[j][1][x] = 16.f * b[x & 1];
            }
            // (sixteen rows: half of the channels after the other, as registers are short)
            constexpr int PASSES = NT == 2 && D == 128 ? 2 : 1, HERE = MTILES / PASSES;
#pragma unroll
            for (int pass = 0; pass < PASSES; ++pass) {
                float acc[HERE][NT][4];
#pragma unroll
                for (int mt = 0; mt < 4; ++mt) {
                    const int k0 = 16 * t + 2 * mt;  // rows 2 t and 2 t + 1 of tile mt: the keys k0 and k0 + 8, and the ones behind them
                    uint32_t lo[2][2], hi[2][2];     // [pair of keys][word]: nibbles 0..3 and 4..7 of both keys
#pragma unroll
                    for (int pair = 0; pair < 2; ++pair) {
                        if constexpr (D == 128) {
                            const uint2 x = *reinterpret_cast<const uint2 *>(st.v + (k0 + pair) * CODE_BYTES + g * 8), y = *reinterpret_cast<const uint2 *>(st.v + (k0 + pair + 8) * CODE_BYTES + g * 8);
                            lo[pair][0] = __byte_perm(x.x, y.x, 0x5410);
                            hi[pair][0] = __byte_perm(x.x, y.x, 0x7632);
                            lo[pair][1] = __byte_perm(x.y, y.y, 0x5410);
                            hi[pair][1] = __byte_perm(x.y, y.y, 0x7632);
                        } else {
                            const uint32_t x = *reinterpret_cast<const uint32_t *>(st.v + (k0 + pair) * CODE_BYTES + g * 4), y = *reinterpret_cast<const uint32_t *>(st.v + (k0 + pair + 8) * CODE_BYTES + g * 4);
                            lo[pair][0] = __byte_perm(x, y, 0x5410);
                            lo[pair][1] = __byte_perm(x, y, 0x7632);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < HERE; ++i) {
                        const int e = pass * HERE + i, nibble = e & 3;
                        uint32_t f[4];
#pragma unroll
                        for (int x = 0; x < 4; ++x) {  // a0, a1: word 0 and 1 of the first pair; a2, a3: of the second
                            const uint32_t word = e < 4 ? lo[x >> 1][x & 1] : hi[x >> 1][x & 1];
                            f[x] = (nibble & 2 ? word >> 8 : word) & (nibble & 1 ? 0x00f000f0u : 0x000f000fu);
                        }
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            if (mt == 0) mma_f16(acc[i][j], f[0], f[1], f[2], f[3], pf[mt][j][0], pf[mt][j][1], base[j][e & 1]);
                            else mma_f16(acc[i][j], f[0], f[1], f[2], f[3], pf[mt][j][0], pf[mt][j][1]);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < HERE; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int x = 0; x < 2; ++x) o[pass * HERE + i][j][x] = fma2(o[pass * HERE + i][j][x], keep[j], pack2(acc[i][j][2 * x], acc[i][j][2 * x + 1]));
            }
        };
        for (int block = first_block; block < last_block; ++block) {
            unsigned here = 0u;
#pragma unroll
            for (int s = 0; s < ATTEND_STAGES; ++s)
                if (s == stage) here = present[s];
            if (sound && !mbar_wait(&sh.full[warp][stage], phase, 20, a.wait_cycles)) sound = false;
            sound = __all_sync(0xffffffffu, sound);
            const int key0 = block * CACHE_BLOCK;
            const bool masked = key0 + CACHE_BLOCK > least || (here & 0x11111111u) != (0x11111111u >> (32 - 4 * pieces));
            // capped or biased: one path, as the second would not stay in the instruction caches beside it (16 sequences of 2000 keys, four queries: 46.8 us with two, 41.8 with one)
            if (MODS || masked) take(std::true_type(), sh.stage[warp][stage], key0, here);
            else take(std::false_type(), sh.stage[warp][stage], key0, here);
            __syncwarp();  // all lanes have read the stage
            if (sound && ahead.u < ahead.end) {
                unsigned loaded;
                issue(stage, loaded, next_page, ahead.item, ahead.block);
                ahead.template step<ROWS>(a);
                next_page = page_of(ahead);
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
        constexpr float BACK = 16777216.f;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            float sums[2];
            unpack2(l[j], sums[0], sums[1]);
#pragma unroll
            for (int x2 = 0; x2 < 2; ++x2) {
                const int r = row0 + 8 * j + 2 * t + x2;
                float sum = sums[x2];
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
                if (r >= rows) continue;
                float f = BACK;
                if (whole) f = sum == 0.f ? 0.f : __fdividef(BACK, sum);
                if (!sound) f = NAN;
                float value[D / 8];  // D / 8 neighbouring channels, from g * D / 8 on
#pragma unroll
                for (int e = 0; e < D / 8; ++e) {
                    constexpr int HALF = D / 16;
                    float x0, x1;
                    unpack2(e < HALF ? o[e < HALF ? e : 0][j][0] : o[e < HALF ? 0 : e - HALF][j][1], x0, x1);
                    value[e] = (x2 ? x1 : x0) * (e & 1 ? 0.0625f * f : f);
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
                        slot[ROWS * D + i] = refer[j][x2];
                        slot[ROWS * D + ROWS + i] = sum;
                    }
                }
            }
        }
        // on to the next run
        cur.u += last_block - first_block - 1;
        cur.block = last_block - 1;
        cur.template step<ROWS>(a);
    }
    if (!sound && lane == 0) {
        let_it_land();  // loads under way must not outlive the shared memory
        if (a.status) atomicExch(a.status, -1);
    }
    // ---- the warps' parts of an item, in the order of the keys: parts that stand together in the list ----
    __syncthreads();
    // a lane per part: which are there, and which begin an item
    const AttendPart &at_lane = sh.parts[min(lane, 2 * ATTEND_WARPS - 1)];
    const unsigned there = __ballot_sync(0xffffffffu, lane < 2 * ATTEND_WARPS && at_lane.last != 0);
    const int before = max(31 - __clz((int)(there & ((1u << lane) - 1u))), 0), b_here = at_lane.b, item_here = at_lane.item;
    const int b_before = __shfl_sync(0xffffffffu, b_here, before), item_before = __shfl_sync(0xffffffffu, item_here, before);
    const bool begins = (there >> lane & 1u) && (!(there & ((1u << lane) - 1u)) || b_before != b_here || item_before != item_here);
    for (unsigned left = __ballot_sync(0xffffffffu, begins); left; left &= left - 1) {
        const int p0 = __ffs(left) - 1, end = left & (left - 1) ? __ffs(left & (left - 1)) - 1 : 32;
        const unsigned group = there & ((end < 32 ? 1u << end : 0u) - (1u << p0));
        const int count = __popc(group), p1 = 31 - __clz((int)group);
        const AttendPart &begin = sh.parts[p0];
        const int first = begin.first, last = sh.parts[p1].last;
        const bool whole = first == 0 && last == begin.blocks;
        const int head = begin.item % c.kv_heads, row0 = begin.item / c.kv_heads * ROWS, rows = begin.s.count * a.group;
        if (threadIdx.x == 0 && first == 0 && !whole) {  // it goes on in the next share
            const unsigned behind = shares.begin(share + 1) - last + begin.blocks;
            a.joins[share] = AttendJoin{(int)(shares.of(behind - 1) - share) + 1, row0, rows, begin.s.first, head, {}};
        }
        // the parts of an item but its first are the first ones of the warps that follow
        const float *const from = attend_slot<D, ROWS>(a, WARP_SLOTS + 2 * ATTEND_WARPS * (int64_t)share + p0), *const next = attend_slot<D, ROWS>(a, WARP_SLOTS + 2 * ATTEND_WARPS * (int64_t)share + (p0 & ~1));
        for (int i = warp; i < ROWS && row0 + i < rows; i += ATTEND_WARPS) {
            float acc[D / 32], m, l;
            const auto row = [&](int k) { return (k == 0 ? from : next + k * (2 * ROWS * (D + 2))) + i * D; };
            merge_parts<D>(count, row, ROWS * D + i - i * D, ROWS * D + ROWS + i - i * D, acc, m, l);
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
    }
    after_the_launch_before();  // of the tiles' kernel, where that is the first: what follows waits for this one alone
}

// Adds up what items that lie in several CTAs' shares left, in the order of the keys.  A CTA per share and (tiles) 32 rows or (rows) all rows of an item: the one whose
// share an item begins in and does not end in, as that share's kernel has noted.
constexpr int JOIN_THREADS = 256, TILE_JOINS = TA_ROWS / 32;
struct JoinArgs {
    AttendArgs tiles, rows;
    int tile_ctas;  // the first so many are the tiles'
};
template <int D, int NT>
__global__ void __launch_bounds__(JOIN_THREADS) attend_join_kernel(const JoinArgs j) {
    constexpr int ROWS = 8 * NT, WARPS = JOIN_THREADS / 32;
    const int warp = threadIdx.x >> 5;
    const bool of_tiles = (int)blockIdx.x < j.tile_ctas;
    const AttendArgs &a = of_tiles ? j.tiles : j.rows;
    if (a.clear) {
        const int row = a.heads * D / 8;  // of 16 bytes
        for (int64_t token = blockIdx.x * JOIN_THREADS + threadIdx.x; token < a.c.tokens; token += gridDim.x * JOIN_THREADS) {
            int first, count;
            if (sequence_of(a.c, (int)token, first, count) >= 0) continue;
            for (int i = 0; i < row; ++i) reinterpret_cast<uint4 *>(a.out)[token * row + i] = make_uint4(0u, 0u, 0u, 0u);
        }
    }
    after_the_launch_before();  // by every CTA: what follows on the stream must not start before the results are there
    const int share = of_tiles ? blockIdx.x / TILE_JOINS : blockIdx.x - j.tile_ctas;
    const AttendJoin join = a.joins[share];
    if (join.count == 0) return;
    if (join.count < 0) {  // of every share of the kernel, so that all of its CTAs are here: nothing has been computed
        const int64_t pieces = (int64_t)a.c.tokens * a.heads * (D / 8), ctas = of_tiles ? j.tile_ctas : gridDim.x - j.tile_ctas;
        const int cta = of_tiles ? blockIdx.x : blockIdx.x - j.tile_ctas;
        for (int64_t i = cta * JOIN_THREADS + threadIdx.x; i < pieces; i += ctas * JOIN_THREADS) reinterpret_cast<uint4 *>(a.out)[i] = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);  // NaN in either type
        if (cta == 0 && threadIdx.x == 0 && a.status) atomicExch(a.status, -1);
        return;
    }
    const int rows = of_tiles ? TA_ROWS : ROWS, i0 = of_tiles ? blockIdx.x % TILE_JOINS * 32 : 0, i1 = min(of_tiles ? i0 + 32 : ROWS, join.rows - join.row0);
    const int64_t slot = rows * (D + 2);
    const float *const from = a.partial + (2 * share + 1) * slot, *const next = a.partial + 2 * share * slot;
    for (int i = i0 + warp; i < i1; i += WARPS) {
        float acc[D / 32], m, l;
        const auto row = [&](int k) { return (k == 0 ? from : next + k * (2 * slot)) + i * D; };
        merge_parts<D>(join.count, row, rows * D + i - i * D, rows * D + rows + i - i * D, acc, m, l);
        const int r = join.row0 + i;
        write_row<D>((uint16_t *)a.out + ((int64_t)(join.first + r / a.group) * a.heads + join.head * a.group + r % a.group) * D, acc, l, a.c.bf16);
    }
}

// rows and tiles: either or both; both launches share the sequences out between them
template <int D, int NT, bool MODS>
static int launch_rows(const AttendArgs &a, bool behind, cudaStream_t st) {
    static PerDeviceOnce configured;
    constexpr size_t smem = sizeof(AttendShared<D, NT>);
    if (configured.run([&] { return cudaFuncSetAttribute(attend_rows_kernel<D, NT, MODS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) == cudaSuccess; }) != G2D_OK)
        return G2D_ERR_CUDA;
    return launch_attention(attend_rows_kernel<D, NT, MODS>, ATTEND_GRID, AttendShape<D, NT>::THREADS, smem, behind, a, st);
}
template <int D, int NT>
static int launch_attend(const AttendArgs &rows, const AttendArgs &tiles, bool few, bool many, bool rows_first, cudaStream_t st) {
    const auto launch_few = [&](bool behind) -> int {
        if (!few) return G2D_OK;
        return rows.softcap > 0.f || rows.slopes ? launch_rows<D, NT, true>(rows, behind, st) : launch_rows<D, NT, false>(rows, behind, st);
    };
    int launched = rows_first ? launch_few(false) : G2D_OK;
    if (launched == G2D_OK && many) launched = launch_attend_tiles(tiles, rows_first && few, st);
    if (launched == G2D_OK && !rows_first) launched = launch_few(many);
    if (launched != G2D_OK) return launched;
    if (rows.even) return G2D_OK;  // no item lies in two shares
    const JoinArgs j{tiles, rows, many ? TA_GRID * TILE_JOINS : 0};
    return launch_attention(attend_join_kernel<D, NT>, (unsigned)(j.tile_ctas + (few ? ATTEND_GRID : 0)), JOIN_THREADS, 0, true, j, st);
}

// From how many rows of a kv head on a sequence goes by tiles.  Tiles cost more to begin with, so few items (sequences and kv heads) cross the line later.
// 32 heads on 8, head_dim 128: 1 sequence of 4096 keys, 64 rows: 27.3 us by rows, 35.3 by tiles; 8 of 2000, 64 rows: 47.1, 54.5, 128 rows: 74.5, 59.3;
// 32 of 1000, 32 rows: 62.0, 67.4, 48 rows: 86.8, 69.2
static int tile_rows_from(const CacheView &c) { return (int64_t)c.batch * c.kv_heads <= 64 ? 65 : 33; }

struct AttendSpace {
    size_t tiles, joins, all;  // the warps' partial results first
};
static AttendSpace attend_space(int head_dim) {
    AttendSpace s;
    s.tiles = ((size_t)ATTEND_GRID * (ATTEND_MOST_WARPS + 1) * 2 * 16 * (head_dim + 2) * sizeof(float) + 255) & ~(size_t)255;
    s.joins = (s.tiles + attend_tiles_bytes(head_dim) + 255) & ~(size_t)255;
    s.all = s.joins + (TA_GRID + ATTEND_GRID) * sizeof(AttendJoin);
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
    if (d->heads < 1 || d->heads % a.c.kv_heads != 0 || !(d->softcap >= 0.f) || d->reserved != 0) return G2D_ERR_BAD_ARGUMENT;
    if (a.c.tokens == 0 || a.c.batch == 0) return G2D_OK;
    if ((int64_t)a.c.tokens * d->heads > 0x7fffffff) return G2D_ERR_TOO_LARGE;
    {  // units of 64 keys and eight rows: counted in 32 bits
        const int64_t capacity = (int64_t)a.c.table_width << a.c.page_shift, blocks = ceil_div(capacity < 0x7fffffff ? capacity : 0x7fffffff, (int64_t)CACHE_BLOCK) + 1;
        if (blocks * ((int64_t)a.c.tokens * d->heads / 8 + 2 * (int64_t)a.c.kv_heads * a.c.batch) > 0x7fffffff) return G2D_ERR_TOO_LARGE;
    }
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
    a.slopes = d->slopes;
    a.prefix = d->prefix;
    a.softcap = d->softcap > 1e30f ? 0.f : d->softcap;  // so far above any score that there is none
    a.clear = d->clear != 0 && a.c.offsets;
    a.status = d->status;
    a.wait_cycles = WAIT_CYCLES;
    cudaStream_t st = (cudaStream_t)stream;
    // How many rows a sequence has is known here only where all have the same; else the kernels share the sequences out between them.
    const int64_t rows = a.c.offsets ? -1 : (int64_t)(a.c.tokens / a.c.batch) * a.group;
    const int line = tile_rows_from(a.c);
    const bool many = rows < 0 ? (int64_t)a.c.tokens * a.group >= line : rows >= line, few = rows < line;
    AttendArgs t = a;
    t.rows_from = line;
    t.rows_to = 0x7fffffff;
    const AttendSpace space = attend_space(a.c.head_dim);
    t.partial = (float *)((char *)d->workspace + space.tiles);
    t.joins = (AttendJoin *)((char *)d->workspace + space.joins);
    a.joins = t.joins + TA_GRID;
    t.even = 0;
    a.rows_from = 1;
    a.rows_to = line;
    a.partial = (float *)d->workspace;
    const bool narrow = a.group <= 8 && (rows < 0 ? ceil_div((int64_t)a.c.tokens * a.group, (int64_t)a.c.batch) : rows) <= 8;
    // Short tables, the same number of queries everywhere: items whole in their shares, a CTA's warps some blocks each, and no join; longer ones where there are about as many items as CTAs.  Time cut
    // evenly over time whole, 32 heads on 8, 128 channels, one and four queries, capped or not, all lengths alike or random, by the number of items: up to 300 and 500 keys 0.98 .. 1.37
    // (8 .. 144 items), 0.94 .. 1.43 (152 .. 296), 0.89 .. 1.37 (384, 512); 1000 keys 1.01 .. 1.50 (96 .. 144), 0.89 .. 1.24 (152 .. 176), 1.02 .. 1.53 (200 .. 296); 2000 keys 1.06 .. 1.38 (96 .. 144),
    // 0.80 .. 1.04, 0.89 in the mean (152 .. 176: a second round that few CTAs have), 0.93 .. 1.35 (200 .. 296).  Fewer and more, 2000 keys: 64 items 0.84, one sequence 0.70, 512 0.89.
    const int64_t most_keys = (int64_t)a.c.table_width << a.c.page_shift, items = rows < 0 ? 0 : (int64_t)a.c.batch * a.c.kv_heads * ceil_div(rows, (int64_t)(narrow ? 8 : 16));
    const bool rounds_filled = items >= 96 && items <= 2 * ATTEND_GRID && (items <= ATTEND_GRID || items >= 200 || most_keys <= 1024);
    const bool whole = !many && !a.c.offsets && (most_keys <= 512 || (most_keys <= 2048 && rounds_filled));
    a.even = !whole ? 0 : most_keys > CACHE_BLOCK ? (int)ceil_div(most_keys, (int64_t)CACHE_BLOCK) : 1;
    // Of two kernels one has most of the work, as a rule: the one for the sequences' mean.  The other finds its part, or that it has none, while that one's last CTAs work
    const bool rows_first = (int64_t)a.c.tokens * a.group < (int64_t)line * a.c.batch;
    if (a.c.head_dim == 128) return narrow ? launch_attend<128, 1>(a, t, few, many, rows_first, st) : launch_attend<128, 2>(a, t, few, many, rows_first, st);
    return narrow ? launch_attend<64, 1>(a, t, few, many, rows_first, st) : launch_attend<64, 2>(a, t, few, many, rows_first, st);
}
