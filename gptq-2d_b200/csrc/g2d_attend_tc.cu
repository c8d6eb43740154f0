// Attention of many query rows per sequence over the packed cache, on tcgen05: prompts, and what is added to them.  The formulas are those of g2d_attend.cu.
//
// An item is 256 rows (token, head of the group) of one kv head: two tiles of 128 rows that share every block of 128 keys.  A unit is one block of one item; the units
// of all items, one after the other, are dealt out evenly to the CTAs, whatever the lengths; an item that lies in one CTA's share is written at once, the others
// leave partial results (two per CTA at most) that attend_join_kernel adds up in the order of the keys.
//
// A CTA: four warps turn codes of keys into an operand, code - 8 in the type of the queries, exactly, keys as rows; four others codes of values, code - 8 in fp16, channels as
// rows (two keys' words interleaved by a byte permutation).  One thread issues the products S = Q K^T and O += P V, S in tensor memory (128 columns a tile), P as fp16 over
// S, O beside them.  Sixteen warps, two threads per row with 64 keys each, read S, multiply it by the keys' scales, take maximum and exponentials, and write P = exponential
// times the value's scale, rounded once to fp16 under the power of two of the largest scale so far.  Four such warps per scheduler keep the exponentials' unit busy (with eight warps, a
// thread per row, a block took 7200 cycles, half of them waits).
//
// The maximum that the exponentials refer to moves only when a row's scores exceed it by 2^8 (or the scales' power of two grows): then O is read and scaled in tensor memory.
//
// Bound: the exponentials (16 per cycle and SM: 2048 cycles for the 256 x 128 of a block, as long as its four products at 128 channels) and the instructions and exchanges around them: a
// unit takes about 6700 cycles at 128 channels, where P lies over S and the products wait for it, and 7800 at 64 (168 and 32 units a CTA), so that the exponentials are a third of it at most: the issue slots are
// 53 and 57 % used, the tensor cores 32 and 16 %; S is read twice, and two warps exchange their maxima before the first exponential.  32 heads on 8: 4096 queries on 8192 keys, 128 channels, bf16, 607 us
// (679 TFLOP/s, 0.40 of what the library's products reach); five prompts of up to 1500 on up to 2500 keys, 64 channels, under a prefix, 158 us.  A quarter of the exponentials by a
// polynomial made both slower (665, 164 us: the instructions are the scarcer), the second tile half a block behind the first made no difference.
#include "g2d_attend.cuh"

namespace g2d {

constexpr int TA_THREADS = 896, TA_SCALES = 4, TA_ROW_WARPS = 16;
constexpr int TA_PANEL = 128 * 128;  // bytes of 128 rows of 64 16-bit values
constexpr float TA_SLACK = 8.f;      // how far scores may exceed the maximum that the exponentials refer to, as a power of two
constexpr int TA_UNIT = 6;           // the largest scale is brought to 2^6 .. 2^7: times 2^8, still a number of fp16

template <int D>
struct TileShared {
    static constexpr int Q = 0, Q_TILE = 128 * D * 2, K = 2 * Q_TILE, K_STAGE = 128 * D * 2, V = K + 2 * K_STAGE, V_STAGE = 128 * D * 2, SCALES = V + 2 * V_STAGE;
    static constexpr int SCALE_STAGE = 3 * TA_KEYS * 4;  // ks, vs as floats; where the unit grows behind some rows' limits the exponent of the largest value's scale up to each key
    static constexpr size_t BYTES = SCALES + TA_SCALES * SCALE_STAGE + 1024;
    // Columns of tensor memory.  At 64 channels P has its own, and the scores of the next block are formed as soon as those of this one have been read; at 128 it lies over
    // them, and they have to wait for the products with the values.
    static constexpr bool OWN_P = D == 64;
    static constexpr uint32_t O_AT = 2 * TA_KEYS, P_AT = OWN_P ? O_AT + 2 * D : 0, P_TILE = OWN_P ? TA_KEYS / 2 : TA_KEYS, P_HALF = OWN_P ? TA_KEYS / 4 : TA_KEYS / 2;
};
// Blocks of an item in a CTA's share: written by one warp, read by the others' roles
constexpr int TA_RUNS = 4;
struct TileRun {
    AttendSequence s;
    int b, pair, head, first, n, blocks;  // n 0: there are no more
};
struct TileBarriers {
    uint64_t run_full[TA_RUNS], run_empty[TA_RUNS], q_full, q_empty, o_empty[2], k_full[2], k_empty[2], v_full[2], v_empty[2], scale_full[TA_SCALES], scale_empty[TA_SCALES], s_full[2], s_free[2], p_full[2], o_full[2], tops_full, halves[2][4], drained;
    unsigned present[TA_SCALES][4];  // which keys of a block there are
    int unit[TA_SCALES];             // exponent bits of the largest scale so far
    int tops[2][4];                  // [block's parity][warp]
    TileRun runs[TA_RUNS];
    float tops2[2][2][2][128];       // [block's parity][tile][half of the keys][row]: the halves' maxima
    float sums2[2][2][2][128];       // [item's parity][tile][half][row]: and the sums of their exponentials
    unsigned totals[TA_THREADS / 32];
    uint32_t tmem;
    int failed;
};

__device__ __forceinline__ void mma_from_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tmem_store_32(uint32_t at, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, "
        "%29, %30, %31, %32};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]),
        "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
        "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void store_16s(uint32_t at, uint32_t x, uint32_t y, uint32_t z, uint32_t w) { asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x), "r"(y), "r"(z), "r"(w) : "memory"); }
__device__ __forceinline__ void tmem_store_16(uint32_t at, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                 "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}
__device__ __forceinline__ uint32_t halves_add(uint32_t u, uint32_t v, bool bf16) {
    uint32_t r;
    if (bf16) asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(u), "r"(v));
    else asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(u), "r"(v));
    return r;
}

// A warp, the one of that number: the largest of its lanes' values up to each lane, and of the warps before
__device__ __forceinline__ int largest_up_to(int v, const int *tops, int number) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) v = max(v, __shfl_up_sync(0xffffffffu, v, o));  // of its own below lane o
    for (int w = 0; w < number; ++w) v = max(v, tops[w]);
    return v;
}

struct TileJob {
    CUtensorMap q;  // [tokens][heads][head_dim] in boxes of 64 channels x a group's heads x 128 / group tokens: 128 rows of a tile
    int by_tma;     // 0 where a group does not divide 128
    AttendArgs a;
};
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
                 : "memory");
}

template <int D, bool BF16, bool MODS>
__global__ void __launch_bounds__(TA_THREADS, 1) attend_tiles_kernel(const __grid_constant__ TileJob job) {
    const AttendArgs &a = job.a;
    using M = TileShared<D>;
    extern __shared__ unsigned char tiles_smem[];
    __shared__ __align__(8) TileBarriers bar;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = (smem_u32(tiles_smem) + 1023u) & ~1023u;
    unsigned char *const at_base = tiles_smem + (base - smem_u32(tiles_smem));
    const CacheView &c = a.c;
    const auto wait = [&](uint64_t *b, uint32_t parity, unsigned nap) {
        if (mbar_wait(b, parity, nap, a.wait_cycles)) return true;
        bar.failed = 1;
        return false;
    };
    if (threadIdx.x == 0) {
        for (int s = 0; s < TA_RUNS; ++s) {
            mbar_init(&bar.run_full[s], 1);
            mbar_init(&bar.run_empty[s], 1 + 2 + 4 + 4 + TA_ROW_WARPS);  // the issuing thread, the warps that bring queries, both teams of coders, the rows' warps
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&bar.o_empty[s], TA_ROW_WARPS / 2);
            mbar_init(&bar.k_full[s], 4);
            mbar_init(&bar.k_empty[s], 1);
            mbar_init(&bar.v_full[s], 4);
            mbar_init(&bar.v_empty[s], 1);
            mbar_init(&bar.s_full[s], 1);
            mbar_init(&bar.s_free[s], TA_ROW_WARPS / 2);
            mbar_init(&bar.p_full[s], TA_ROW_WARPS / 2);
            mbar_init(&bar.o_full[s], 1);
            for (int q = 0; q < 4; ++q) mbar_init(&bar.halves[s][q], 2);
        }
        for (int s = 0; s < TA_SCALES; ++s) {
            mbar_init(&bar.scale_full[s], 4);
            mbar_init(&bar.scale_empty[s], TA_ROW_WARPS);
        }
        mbar_init(&bar.q_full, 2);
        mbar_init(&bar.q_empty, 1);
        mbar_init(&bar.tops_full, 4);
        mbar_init(&bar.drained, 1);
        bar.failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    let_the_next_launch_start();
    unsigned mine_units;
    const unsigned units = count_tile_units<TA_THREADS / 32>(a, bar.totals, mine_units);
    if (threadIdx.x == 0) a.joins[blockIdx.x] = AttendJoin{units < UNITS_END ? 0 : -1};
    if (units == 0 || units >= UNITS_END) {  // sequences of few rows only, or more than can be counted
        after_the_launch_before();
        return;
    }
    if (warp == 1) tmem_alloc<false>(&bar.tmem, 512);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = bar.tmem;
    const AttendShares shares(units, gridDim.x);
    const unsigned share = blockIdx.x;
    // the run of that number, for every thread of a role; its entry stays until all roles have let it go
    const auto run_of = [&](uint32_t number, bool &go) -> const TileRun & {
        if (go) go = wait(&bar.run_full[number % TA_RUNS], (number / TA_RUNS) & 1, 0);
        return bar.runs[number % TA_RUNS];
    };
    const auto let_go = [&](uint32_t number) { mbar_arrive(&bar.run_empty[number % TA_RUNS]); };
    const auto second = [&](const TileRun &r) { return (int64_t)r.s.count * a.group - (int64_t)r.pair * TA_ROWS > 128; };  // whether the item has a second tile

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");  // 28 warps of 72 registers in all: 4 x 56 + 8 x 64 + 16 x 80
        if (warp == 0) {
            // ---- the share's runs ----
            TileCursor cur;
            cur.u = cur.end = 0;
            if (share < shares.count) {
                cur.find(a, mine_units, shares.begin(share));
                cur.end = shares.begin(share + 1);
            }
            if (lane == 0) {
                AttendJoin join{};
                for (uint32_t number = 0;; ++number) {
                    if (number >= TA_RUNS && (bar.failed || !wait(&bar.run_empty[number % TA_RUNS], (number / TA_RUNS - 1) & 1, 32))) break;
                    TileRun &r = bar.runs[number % TA_RUNS];
                    r.n = cur.u < cur.end ? cur.run() : 0;
                    if (r.n > 0 && cur.block == 0 && r.n < cur.blocks) {
                        join.count = (int)(shares.of(cur.u + cur.blocks - 1) - share) + 1;
                        join.row0 = cur.pair * TA_ROWS;
                        join.rows = cur.s.count * a.group;
                        join.first = cur.s.first;
                        join.head = cur.head;
                        a.joins[share] = join;
                    }
                    r.s = cur.s;
                    r.b = cur.b;
                    r.pair = cur.pair;
                    r.head = cur.head;
                    r.first = cur.block;
                    r.blocks = cur.blocks;
                    mbar_arrive(&bar.run_full[number % TA_RUNS]);
                    if (cur.u >= cur.end) break;
                    cur.next(a);
                }
            }
        } else if (warp >= 2) {
            // ---- queries: the next item's while the last block of the one before is at its exponentials ----
            constexpr int CHUNKS = D / 8, BATCH = 8;  // of 16 bytes; loads under way
            const int id = threadIdx.x - 64;
            bool go = true;
            uint32_t landed = 0;  // loads issued so far: the last has landed before this CTA ends
            for (uint32_t number = 0;; ++number) {
                const TileRun &run = run_of(number, go);
                if (!__all_sync(0xffffffffu, go) || run.n == 0) break;
                const int row0 = run.pair * TA_ROWS, rows = run.s.count * a.group, local = second(run) ? TA_ROWS : TA_ROWS / 2;
                const int64_t first = run.s.first;
                const int head0 = run.head * a.group;
                __syncwarp();
                if (lane == 0) let_go(number);
                if (number > 0) go = wait(&bar.q_empty, (number - 1) & 1, 32);
                if (!__all_sync(0xffffffffu, go)) break;
                if (job.by_tma) {  // rows past the sequence's last are another's, or zeros: their results go nowhere
                    if (lane == 0 && warp == 2) {
                        mbar_expect_tx(&bar.q_full, (uint32_t)(local * D * 2));
                        for (int t = 0; t < local / 128; ++t)
                            for (int p = 0; p < D / 64; ++p)
                                tma_load_3d(base + M::Q + t * M::Q_TILE + p * TA_PANEL, &job.q, p * 64, head0, (int)(first + (row0 + t * 128) / a.group), &bar.q_full);
                    } else if (lane == 0) {
                        mbar_arrive(&bar.q_full);
                    }
                    landed = number + 1;
                    continue;
                }
                const int chunk = id % CHUNKS;
#pragma unroll 1
                for (int i0 = id / CHUNKS; i0 < local; i0 += BATCH * 64 / CHUNKS) {
                    uint4 v[BATCH];
#pragma unroll
                    for (int k = 0; k < BATCH; ++k) {
                        const int r = row0 + i0 + k * (64 / CHUNKS);
                        v[k] = make_uint4(0u, 0u, 0u, 0u);
                        if (r < rows) {
                            const unsigned token = (unsigned)r / (unsigned)a.group, h = (unsigned)r - token * a.group;
                            v[k] = __ldg(reinterpret_cast<const uint4 *>((const uint16_t *)a.q + (first + token) * a.q_token_stride + (int64_t)(head0 + h) * a.q_head_stride) + chunk);
                        }
                    }
#pragma unroll
                    for (int k = 0; k < BATCH; ++k) {
                        const int i = i0 + k * (64 / CHUNKS);
                        if (i < local) store_16s(base + M::Q + (i >> 7) * M::Q_TILE + (chunk >> 3) * TA_PANEL + (i & 127) * 128 + (((chunk & 7) ^ (i & 7)) << 4), v[k].x, v[k].y, v[k].z, v[k].w);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar.q_full);
            }
            if (landed > 0) mbar_wait(&bar.q_full, (landed - 1) & 1);
        } else if (warp == 1 && elected()) {
            // ---- products ----
            constexpr uint32_t S_DESC = idesc_16(TA_KEYS, BF16 ? 1 : 0), O_DESC = idesc_16(D, 0);
            const uint64_t q0 = umma_desc(base + M::Q), k0 = umma_desc(base + M::K), v0 = umma_desc(base + M::V);
            uint32_t items = 0, pairs = 0, kc = 0, vc = 0, pc0 = 0, pc1 = 0, sc0 = 0, sc1 = 0;
            const auto scores = [&](int tile, int stage) {
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks) {
                    const uint64_t at = (uint64_t)((ks >> 2) * (TA_PANEL >> 4) + (ks & 3) * 2);
                    umma_16(tmem + tile * TA_KEYS, q0 + (uint64_t)(tile * (M::Q_TILE >> 4)) + at, k0 + (uint64_t)(stage * (M::K_STAGE >> 4)) + at, S_DESC, ks > 0);
                }
                umma_commit(&bar.s_full[tile]);
            };
            const auto results = [&](int tile, int stage, bool more) {
#pragma unroll
                for (int ks = 0; ks < TA_KEYS / 16; ++ks)
                    mma_from_tmem(tmem + M::O_AT + tile * D, tmem + M::P_AT + tile * M::P_TILE + (ks >> 2) * M::P_HALF + (ks & 3) * 8, v0 + (uint64_t)(stage * (M::V_STAGE >> 4) + (ks >> 2) * (D * 128 >> 4) + (ks & 3) * 2), O_DESC, more || ks > 0);
            };
            const auto after = [] { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); };
            bool go = true;
            for (;; ++items) {
                const TileRun &run = run_of(items, go);
                if (!go || run.n == 0) break;
                const int n = run.n;
                const bool two = second(run);
                let_go(items);
                go = wait(&bar.q_full, items & 1, 0) && wait(&bar.k_full[kc & 1], (kc >> 1) & 1, 0);
                if (!go) break;
                after();
                scores(0, kc & 1);
                if (two) scores(1, kc & 1);
                if (n == 1) umma_commit(&bar.q_empty);
                umma_commit(&bar.k_empty[kc++ & 1]);
                if constexpr (M::OWN_P) {
                    for (int j = 0; j < n; ++j, ++vc) {
                        const int vs = vc & 1, ks = kc & 1;
                        const bool more = j + 1 < n;
                        if (more) {
                            go = !bar.failed && wait(&bar.s_free[0], sc0 & 1, 0) && wait(&bar.k_full[ks], (kc >> 1) & 1, 0);
                            if (!go) break;
                            after();
                            scores(0, ks);
                        }
                        ++sc0;
                        go = !bar.failed && wait(&bar.v_full[vs], (vc >> 1) & 1, 0) && wait(&bar.p_full[0], pc0++ & 1, 0);
                        if (j == 0 && items > 0) go = go && wait(&bar.o_empty[0], (items - 1) & 1, 0);  // the item before has been read
                        if (!go) break;
                        after();
                        results(0, vs, j > 0);
                        umma_commit(&bar.o_full[0]);
                        if (two) {
                            if (more) {
                                go = wait(&bar.s_free[1], sc1 & 1, 0);
                                if (!go) break;
                                after();
                                scores(1, ks);
                            }
                            ++sc1;
                        }
                        if (more) {
                            if (j + 2 == n) umma_commit(&bar.q_empty);
                            umma_commit(&bar.k_empty[ks]);
                            ++kc;
                        }
                        if (two) {
                            go = wait(&bar.p_full[1], pc1++ & 1, 0);
                            if (j == 0 && pairs > 0) go = go && wait(&bar.o_empty[1], (pairs - 1) & 1, 0);
                            if (!go) break;
                            after();
                            results(1, vs, j > 0);
                            umma_commit(&bar.o_full[1]);
                        }
                        umma_commit(&bar.v_empty[vs]);
                    }
                } else {
                for (int j = 0; j < n; ++j, ++vc) {
                    const int vs = vc & 1, ks = kc & 1;
                    go = !bar.failed && wait(&bar.v_full[vs], (vc >> 1) & 1, 0) && wait(&bar.p_full[0], pc0++ & 1, 0);
                    if (j == 0 && items > 0) go = go && wait(&bar.o_empty[0], (items - 1) & 1, 0);  // the item before has been read
                    if (!go) break;
                    after();
                    results(0, vs, j > 0);
                    if (j + 1 < n) {
                        go = wait(&bar.k_full[ks], (kc >> 1) & 1, 0);
                        if (!go) break;
                        after();
                        scores(0, ks);  // over the P that the products before have read: they are carried out in order
                    } else {
                        umma_commit(&bar.o_full[0]);
                    }
                    if (two) {
                        go = wait(&bar.p_full[1], pc1++ & 1, 0);
                        if (j == 0 && pairs > 0) go = go && wait(&bar.o_empty[1], (pairs - 1) & 1, 0);
                        if (!go) break;
                        after();
                        results(1, vs, j > 0);
                    }
                    umma_commit(&bar.v_empty[vs]);
                    if (j + 1 < n) {
                        if (two) scores(1, ks);
                        if (j + 2 == n) umma_commit(&bar.q_empty);
                        umma_commit(&bar.k_empty[ks]);
                        ++kc;
                    } else if (two) {
                        umma_commit(&bar.o_full[1]);
                    }
                }
                }
                if (two) ++pairs;
            }
            if (bar.failed) {  // what was issued completes, or has its time to, before what it reads and writes is given back
                umma_commit(&bar.drained);
                mbar_wait(&bar.drained, 0);
            } else if (vc > 0) {
                mbar_wait(&bar.v_empty[(vc - 1) & 1], ((vc - 1) >> 1) & 1);
                mbar_wait(&bar.k_empty[(kc - 1) & 1], ((kc - 1) >> 1) & 1);
                mbar_wait(&bar.q_empty, (items - 1) & 1);
            }
        }
        __syncwarp();
    } else if (warp < 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        // ---- operands: four warps for the keys and all scales, four for the values ----
        constexpr int WORDS = D / 8, VW = D / 64;  // words of a key; of a thread's keys in V
        constexpr uint32_t MAGIC = BF16 ? 0x43004300u : 0x64006400u, LESS = BF16 ? 0xc308c308u : 0xe408e408u;
        uint32_t blocks_done = 0, number = 0;
        bool go = true;
        // the block that is on its way: number ahead_j of the run of number ahead
        uint32_t ahead = 0;
        int ahead_n = 0, ahead_j = 0, ahead_keys = 0, ahead_first = 0, ahead_b = 0, ahead_head = 0;
        const auto open_ahead = [&] {
            const TileRun &r = run_of(ahead, go);
            ahead_n = go ? r.n : 0;
            ahead_keys = r.s.keys;
            ahead_first = r.first;
            ahead_b = r.b;
            ahead_head = r.head;
            ahead_j = 0;
        };
        const auto row_of = [&](int at) -> int64_t {  // row of the cache of a key of the block on its way, or -1
            const int position = (ahead_first + ahead_j) * TA_KEYS + at;
            return ahead_n > 0 && position < ahead_keys ? cache_row(c, ahead_b, position, ahead_head) : -1;
        };
        const auto step_ahead = [&] {
            if (ahead_n == 0 || ++ahead_j < ahead_n) return;
            ++ahead;
            open_ahead();
        };
        open_ahead();
        if (warp < 8) {
            const int key = threadIdx.x - 128;
            int unit = 0;
            uint4 kr[WORDS / 4];
            float ks = 0.f, vs = 0.f;
            bool here = false;
            const auto fetch = [&] {
                const int64_t row = row_of(key);
                here = row >= 0;
#pragma unroll
                for (int w = 0; w < WORDS / 4; ++w) kr[w] = here ? __ldg(reinterpret_cast<const uint4 *>(c.k_codes + row * (D / 2)) + w) : make_uint4(0u, 0u, 0u, 0u);
                ks = here ? __half2float(c.k_scale[row]) : 0.f;
                vs = here ? __half2float(c.v_scale[row]) : 0.f;
            };
            fetch();
            for (;; ++number) {
                const TileRun &run = run_of(number, go);
                const int n = run.n;
                if (!__all_sync(0xffffffffu, go) || n == 0) break;
                unit = 0;
                for (int j = 0; j < n; ++j, ++blocks_done) {
                    const int stage = blocks_done & 1, slot = blocks_done % TA_SCALES;
                    if (blocks_done >= 2) go = wait(&bar.k_empty[stage], ((blocks_done >> 1) - 1) & 1, 0);
                    if (blocks_done >= TA_SCALES) go = go && wait(&bar.scale_empty[slot], (blocks_done / TA_SCALES - 1) & 1, 0);
                    go = __all_sync(0xffffffffu, go && !bar.failed);
                    if (!go) break;
                    const uint32_t kt = base + M::K + stage * M::K_STAGE + key * 128;
#pragma unroll
                    for (int w = 0; w < WORDS; ++w) {
                        const uint4 &r = kr[w >> 2];
                        const uint32_t x = (w & 3) == 0 ? r.x : (w & 3) == 1 ? r.y : (w & 3) == 2 ? r.z : r.w, x4 = x >> 4;
                        store_16s(kt + (w >> 3) * TA_PANEL + (((w & 7) ^ (key & 7)) << 4), halves_add((__byte_perm(x, x4, 0x4400) & 0x000f000fu) | MAGIC, LESS, BF16),
                                  halves_add((__byte_perm(x, x4, 0x5511) & 0x000f000fu) | MAGIC, LESS, BF16), halves_add((__byte_perm(x, x4, 0x6622) & 0x000f000fu) | MAGIC, LESS, BF16),
                                  halves_add((__byte_perm(x, x4, 0x7733) & 0x000f000fu) | MAGIC, LESS, BF16));
                    }
                    // the largest scale so far (one that is not finite sets no unit), and the values' scales in its power of two
                    const unsigned bits = __float_as_uint(vs) & 0x7fffffffu, size = bits < 0x7f800000u ? bits : 0u;
                    const unsigned top = __reduce_max_sync(0xffffffffu, size), got = __ballot_sync(0xffffffffu, here);
                    if (lane == 0) {
                        bar.tops[stage][warp - 4] = (int)(top >> 23);
                        mbar_arrive(&bar.tops_full);
                    }
                    go = __all_sync(0xffffffffu, wait(&bar.tops_full, blocks_done & 1, 0));  // of all four warps
                    if (!go) break;
                    const int old_unit = unit;
                    unit = max(max(unit, max(bar.tops[stage][0], bar.tops[stage][1])), max(bar.tops[stage][2], bar.tops[stage][3]));
                    float *const sc = reinterpret_cast<float *>(at_base + M::SCALES + slot * M::SCALE_STAGE) + key;
                    sc[0] = fmaf(ks, 0.f, ks) * (a.scale * score_unit<MODS>(a));  // NaN for a scale that is not finite, whatever the codes
                    sc[TA_KEYS] = vs * power_of_two(min(TA_UNIT - (unit - 127), 127));
                    if (unit != old_unit && (run.first + j + 1) * TA_KEYS > visible_keys(a, run.s, run.pair * TA_ROWS / a.group))  // the item's first row, which sees least, not the whole block
                        sc[2 * TA_KEYS] = __int_as_float(largest_up_to((int)(size >> 23), bar.tops[stage], warp - 4));
                    if (lane == 0) bar.present[slot][warp - 4] = got;
                    if (threadIdx.x == 128) bar.unit[slot] = unit;
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(&bar.scale_full[slot]);
                        mbar_arrive(&bar.k_full[stage]);
                    }
                    step_ahead();
                    fetch();
                }
                // the run's entry is needed no more: the block on its way belongs to the next one
                if (!go) break;
                __syncwarp();
                if (lane == 0) let_go(number);
            }
        } else {
            const int octet = (lane & 7) + 8 * (warp & 1), word = ((lane >> 3) + 4 * ((warp - 8) >> 1)) * VW;  // eight keys, VW words of each
            uint32_t vr[8][VW];
            const auto fetch = [&] {
                const int64_t row = row_of(octet * 8);  // eight keys of one page: those past the last key lie in it, too, and count for nothing
                const uint8_t *const from = c.v_codes + row * (D / 2) + word * 4;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    if constexpr (VW == 2) {
                        const uint2 v = row >= 0 ? __ldg(reinterpret_cast<const uint2 *>(from + k * (D / 2))) : make_uint2(0u, 0u);
                        vr[k][0] = v.x;
                        vr[k][1] = v.y;
                    } else {
                        vr[k][0] = row >= 0 ? __ldg(reinterpret_cast<const uint32_t *>(from + k * (D / 2))) : 0u;
                    }
                }
            };
            fetch();
            for (;; ++number) {
                const int n = run_of(number, go).n;
                if (!__all_sync(0xffffffffu, go) || n == 0) break;
                for (int j = 0; j < n; ++j, ++blocks_done) {
                    const int stage = blocks_done & 1;
                    if (blocks_done >= 2) go = wait(&bar.v_empty[stage], ((blocks_done >> 1) - 1) & 1, 0);
                    go = __all_sync(0xffffffffu, go && !bar.failed);
                    if (!go) break;
                    const uint32_t vt = base + M::V + stage * M::V_STAGE + (octet >> 3) * (D * 128);
#pragma unroll
                    for (int w = 0; w < VW; ++w) {
                        uint32_t lo[4], hi[4];  // of two keys each: the lower and the upper four codes
#pragma unroll
                        for (int p = 0; p < 4; ++p) {
                            lo[p] = __byte_perm(vr[2 * p][w], vr[2 * p + 1][w], 0x5410);
                            hi[p] = __byte_perm(vr[2 * p][w], vr[2 * p + 1][w], 0x7632);
                        }
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int d = (word + w) * 8 + e;
                            uint32_t v[4];
#pragma unroll
                            for (int p = 0; p < 4; ++p) v[p] = halves_add((((e < 4 ? lo[p] : hi[p]) >> (4 * (e & 3))) & 0x000f000fu) | 0x64006400u, 0xe408e408u, false);
                            store_16s(vt + d * 128 + (((octet & 7) ^ (d & 7)) << 4), v[0], v[1], v[2], v[3]);
                        }
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bar.v_full[stage]);
                    step_ahead();
                    fetch();
                }
                if (!go) break;
                __syncwarp();
                if (lane == 0) let_go(number);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 80;");
        // ---- rows: two threads each, with 64 keys of every block and half of the channels ----
        const int tile = (warp - 12) >> 3, half = ((warp - 12) >> 2) & 1, q = warp & 3, row = q * 32 + lane, local = tile * 128 + row;
        const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16), s_at = lanes + tile * TA_KEYS + half * 64, o_at = lanes + M::O_AT + tile * D + half * (D / 2),
                       p_at = lanes + M::P_AT + tile * M::P_TILE + half * M::P_HALF;
        uint32_t hc = 0;
        bool go = true;
        const auto both = [&] {  // the two warps of 32 rows meet (by a barrier whose wait has its limit)
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.halves[tile][q]);
            if (go && !wait(&bar.halves[tile][q], hc & 1, 0)) go = false;
            ++hc;
        };
        uint32_t sc = 0, tc = 0, oc = 0;  // blocks of the CTA, blocks and items of this tile
        for (uint32_t number = 0;; ++number) {
            const TileRun &run = run_of(number, go);
            if (!__all_sync(0xffffffffu, go) || run.n == 0) break;
            const int n = run.n, first = run.first;
            const bool mine = tile == 0 || second(run), whole = first == 0 && n == run.blocks;
            const int r = run.pair * TA_ROWS + local;
            const bool real = r < run.s.count * a.group;
            const int token = real ? r / a.group : 0, h = run.head * a.group + (real ? r % a.group : 0), limit = real ? visible_keys(a, run.s, token) : 0x7fffffff;
            const int64_t at_token = run.s.first + token;
            __syncwarp();
            if (lane == 0) let_go(number);
            if (!mine) {  // blocks that the other tile has alone
                for (int j = 0; j < n; ++j, ++sc) {
                    go = go && !bar.failed && wait(&bar.scale_full[sc % TA_SCALES], (sc / TA_SCALES) & 1, 32);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bar.scale_empty[sc % TA_SCALES]);
                }
                continue;
            }
            const int least = __reduce_min_sync(0xffffffffu, limit);
            const float slope = MODS && a.slopes ? a.slopes[h] * LOG2E : 0.f, cap = a.softcap * LOG2E;
            const int place = bias_origin(slope, limit);
            float m = -INFINITY;
            uint64_t l = 0ull;
            int unit = 0;
            for (int j = 0; j < n; ++j, ++sc, ++tc) {
                const int slot = sc % TA_SCALES, key0 = (first + j) * TA_KEYS + half * 64;
                go = go && !bar.failed && wait(&bar.s_full[tile], tc & 1, 0) && wait(&bar.scale_full[slot], (sc / TA_SCALES) & 1, 0);
                if (!__all_sync(0xffffffffu, go)) go = false;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const ulonglong2 *const scales = reinterpret_cast<const ulonglong2 *>(at_base + M::SCALES + slot * M::SCALE_STAGE) + half * 16;
                const bool masked = key0 + 64 > least || (bar.present[slot][2 * half] & bar.present[slot][2 * half + 1]) != 0xffffffffu;
                // Two passes over S in tensor memory, so that a thread need not hold a row: the maximum, then the exponentials.  Where scores are masked, capped or biased the
                // first pass writes them back.
                const bool stored = MODS || masked;
                float top = -INFINITY;
#pragma unroll 1
                for (int cb = 0; cb < 2; ++cb) {
                    uint32_t v[32];
                    tmem_load_32(s_at + cb * 32, v);
#pragma unroll
                    for (int x = 0; x < 32; x += 4) {
                        const ulonglong2 k4 = scales[cb * 8 + x / 4];
                        float u[4];
                        unpack2(mul2(pack2(v[x], v[x + 1]), k4.x), u[0], u[1]);
                        unpack2(mul2(pack2(v[x + 2], v[x + 3]), k4.y), u[2], u[3]);
#pragma unroll
                        for (int y = 0; y < 4; ++y) v[x + y] = __float_as_uint(u[y]);
                    }
                    if (MODS) {
                        const float away = (float)(key0 + cb * 32 - place);
                        const bool near = a.softcap <= CAP_NEAR;
                        if (a.softcap > 0.f) {
#pragma unroll
                            for (int x = 0; x < 32; ++x) v[x] = __float_as_uint(capped(__uint_as_float(v[x]), cap, near));
                        }
#pragma unroll
                        for (int x = 0; x < 32; ++x) v[x] = __float_as_uint(fmaf(slope, away + (float)x, __uint_as_float(v[x])));
                    }
                    if (stored) {
                        if (masked) {
                            const int seen = min(max(limit - key0 - cb * 32, 0), 32);
                            const unsigned there = bar.present[slot][2 * half + cb] & (uint32_t)((1ull << seen) - 1ull);
#pragma unroll
                            for (int x = 0; x < 32; ++x)
                                if (!((there >> x) & 1u)) v[x] = 0xff800000u;
                        }
                        tmem_store_32(s_at + cb * 32, v);
                    }
#pragma unroll
                    for (int x = 0; x < 32; x += 2) top = fmaxf(fmaxf(top, __uint_as_float(v[x])), __uint_as_float(v[x + 1]));
                }
                if (stored) tmem_stored();
                bar.tops2[tc & 1][tile][half][row] = top;
                both();
                top = fmaxf(top, bar.tops2[tc & 1][tile][half ^ 1][row]);
                if (M::OWN_P && tc > 0) {  // these scores came before the products of the last block with its values, which read P and add to O
                    go = go && wait(&bar.o_full[tile], (tc - 1) & 1, 0);
                    if (!__all_sync(0xffffffffu, go)) go = false;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                }
                // the maximum that the exponentials refer to, and the unit of the scales
                const int new_unit = bar.unit[slot];
                const bool first_seen = m == -INFINITY, moves = top > m + TA_SLACK || (first_seen && top > -INFINITY) || new_unit != unit;
                if (__any_sync(0xffffffffu, moves)) {
                    float now = moves && top > m ? top : m;
                    // A row sees whole blocks up to its limit, and of the block with its limit the first keys: there its reference is lower by as much as the largest scale that it has seen
                    // lies below the unit, so that scales which the mask hides leave its P as large as they would be.  It sees no block behind that.
                    if (new_unit != unit && (first + j + 1) * TA_KEYS > least) {
                        const int visible = min(limit - (first + j) * TA_KEYS, TA_KEYS);
                        const int seen = visible > 0 ? max(unit, __float_as_int(reinterpret_cast<const float *>(at_base + M::SCALES + slot * M::SCALE_STAGE)[2 * TA_KEYS + visible - 1])) : 0;
                        if (seen > 0) now -= (float)(new_unit - seen);
                    }
                    const float keep = first_seen ? 1.f : ex2(m - now);
                    const float f = unit == 0 ? keep : keep * power_of_two(max(unit - new_unit, -126));
                    l = mul2(l, pack2(keep, keep));
                    m = now;
                    unit = new_unit;
                    if (j > 0) {
#pragma unroll 1
                        for (int cb = 0; cb < D / 64; ++cb) {
                            uint32_t v[32];
                            tmem_load_32(o_at + cb * 32, v);
#pragma unroll
                            for (int x = 0; x < 32; ++x) v[x] = __float_as_uint(__uint_as_float(v[x]) * f);
                            tmem_store_32(o_at + cb * 32, v);
                        }
                    }
                }
                const float refer = m == -INFINITY ? 0.f : m;
                const uint64_t less = pack2(-refer, -refer);
                const auto exponentials = [&](auto is_stored, auto is_masked) {
                    constexpr bool STORED = decltype(is_stored)::value, MASKED = decltype(is_masked)::value;
#pragma unroll 1
                for (int cb = 0; cb < 2; ++cb) {
                    uint32_t v[32], p[16];
                    tmem_load_32(s_at + cb * 32, v);
                    if (M::OWN_P && cb == 1) {  // the scores have been read
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&bar.s_free[tile]);
                    }
#pragma unroll
                    for (int x = 0; x < 32; x += 4) {
                        const ulonglong2 k4 = scales[cb * 8 + x / 4], v4 = scales[TA_KEYS / 4 + cb * 8 + x / 4];
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            const uint64_t score = pack2(v[x + 2 * y], v[x + 2 * y + 1]);
                            float e0, e1, w0, w1;
                            unpack2(STORED ? add2(score, less) : fma2(score, y ? k4.y : k4.x, less), e0, e1);
                            const uint64_t e = pack2(ex2(e0), ex2(e1));
                            l = add2(l, e);
                            unpack2(mul2(e, y ? v4.y : v4.x), w0, w1);
                            if constexpr (MASKED) {  // a masked key counts for nothing, whatever its scale
                                if (v[x + 2 * y] == 0xff800000u) w0 = 0.f;
                                if (v[x + 2 * y + 1] == 0xff800000u) w1 = 0.f;
                            }
                            p[x / 2 + y] = pack_halves(w0, w1, 0);
                        }
                    }
                    tmem_store_16(p_at + cb * 16, p);  // 128 channels: over scores that this thread has read
                }
                };
                if (masked) exponentials(std::true_type(), std::true_type());
                else exponentials(std::bool_constant<MODS>(), std::false_type());
                tmem_stored();
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&bar.p_full[tile]);
                    mbar_arrive(&bar.scale_empty[slot]);
                }
            }
            // ---- this CTA's part of the item ----
            float l0, l1;
            unpack2(l, l0, l1);
            l0 += l1;
            bar.sums2[oc & 1][tile][half][row] = l0;
            both();
            l0 = half ? bar.sums2[oc & 1][tile][0][row] + l0 : l0 + bar.sums2[oc & 1][tile][1][row];
            if (go) go = wait(&bar.o_full[tile], (M::OWN_P ? tc - 1 : oc) & 1, 0);
            ++oc;
            if (!__all_sync(0xffffffffu, go)) go = false;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            float f = power_of_two(max((unit - 127) - TA_UNIT, -126));
            if (whole) f = l0 == 0.f ? 0.f : __fdividef(f, l0);
            if (!go) f = NAN;
            const bool none = whole && l0 == 0.f && go;
            float *const slot = tile_slot<D>(a, 2 * share + (first == 0 ? 1 : 0));
#pragma unroll 1
            for (int cb = 0; cb < D / 64; ++cb) {
                uint32_t v[32];
                tmem_load_32(o_at + cb * 32, v);
                if (!real) continue;
#pragma unroll
                for (int x = 0; x < 32; ++x) v[x] = __float_as_uint(none ? 0.f : __uint_as_float(v[x]) * f);
                if (whole) {
                    uint4 *const to = reinterpret_cast<uint4 *>((uint16_t *)a.out + (at_token * a.heads + h) * D + half * (D / 2) + cb * 32);
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        uint32_t w[4];
#pragma unroll
                        for (int y = 0; y < 4; ++y) w[y] = pack_halves(__uint_as_float(v[8 * x + 2 * y]), __uint_as_float(v[8 * x + 2 * y + 1]), BF16);
                        to[x] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                } else {
                    uint4 *const to = reinterpret_cast<uint4 *>(slot + local * D + half * (D / 2) + cb * 32);
#pragma unroll
                    for (int x = 0; x < 8; ++x) to[x] = make_uint4(v[4 * x], v[4 * x + 1], v[4 * x + 2], v[4 * x + 3]);
                }
            }
            if (real && !whole && half == 0) {
                slot[TA_ROWS * D + local] = m;
                slot[TA_ROWS * D + TA_ROWS + local] = l0;
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.o_empty[tile]);
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    after_the_launch_before();  // of the rows' kernel, where that is the first: what follows waits for this one alone
    if (warp == 1) tmem_free<false>(tmem, 512);
    if (threadIdx.x == 0 && bar.failed && a.status) atomicExch(a.status, -1);
}

size_t attend_tiles_bytes(int head_dim) { return (size_t)TA_GRID * 2 * TA_ROWS * (head_dim + 2) * sizeof(float); }

template <int D, bool BF16, bool MODS>
static int launch_tiles(const AttendArgs &a, bool behind, cudaStream_t st) {
    static PerDeviceOnce configured;
    constexpr size_t smem = TileShared<D>::BYTES;
    if (configured.run([&] { return cudaFuncSetAttribute(attend_tiles_kernel<D, BF16, MODS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) == cudaSuccess; }) != G2D_OK) return G2D_ERR_CUDA;
    TileJob job;
    job.a = a;
    job.by_tma = 0;
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return G2D_ERR_CUDA;
    const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)a.heads, (cuuint64_t)a.c.tokens};
    const cuuint64_t strides[2] = {(cuuint64_t)a.q_head_stride * 2, (cuuint64_t)a.q_token_stride * 2};
    const cuuint32_t elem[3] = {1, 1, 1};
    if (128 % a.group == 0 && a.q_head_stride > 0 && a.q_token_stride > 0) {
        const cuuint32_t box[3] = {64, (cuuint32_t)a.group, (cuuint32_t)(128 / a.group)};
        job.by_tma = fn(&job.q, BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void *>(a.q), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    }
    return launch_attention(attend_tiles_kernel<D, BF16, MODS>, TA_GRID, TA_THREADS, smem, behind, job, st);
}

int launch_attend_tiles(const AttendArgs &a, bool behind, cudaStream_t st) {
    const bool mods = a.softcap > 0.f || a.slopes;
    if (a.c.head_dim == 128) {
        if (a.c.bf16) return mods ? launch_tiles<128, true, true>(a, behind, st) : launch_tiles<128, true, false>(a, behind, st);
        return mods ? launch_tiles<128, false, true>(a, behind, st) : launch_tiles<128, false, false>(a, behind, st);
    }
    if (a.c.bf16) return mods ? launch_tiles<64, true, true>(a, behind, st) : launch_tiles<64, true, false>(a, behind, st);
    return mods ? launch_tiles<64, false, true>(a, behind, st) : launch_tiles<64, false, false>(a, behind, st);
}

}  // namespace g2d
