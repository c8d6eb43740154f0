// y = x W^T for a matrix W held as packed 4-bit codes, many tokens, on tcgen05; low-rank adapters of the tokens' requests beside it.
//
// A tile is 128 rows of W times NT tokens: A is W, so a scale belongs to a lane of tensor memory.  Codes travel as they are: the TMA brings 128 rows x 64 columns
// (4 KB) of them to a slot, whose two warps turn them into 16-bit values in the swizzled layout of an MMA operand (code - 8 exactly, plus 8 + qmin - zero rounded to the type), and
// x comes by TMA beside them.  What is accumulated in tensor memory is a slice of the columns under one scale (512 columns at most: the tensor cores add with truncation);
// warps of their own read each slice while the next is accumulated, and add scale times slice in registers, in fp32.
//
// An adapter is two more slices of k: for every adapter among a tile's tokens A is its rows of `up` (times nothing) and B the tokens' inner values, upper and lower
// parts (see g2d_adapters.cu).  The product has a column for every token of the tile; the reading warps add it, times the token's factor, only where the token has this adapter.
//
// Few tokens may each have an adapter of their own, and two turns for each would be nearly as many as the matrix takes (61 tokens of 24 adapters: 112 turns a tile instead of 64): their outer
// halves are added where the pieces are joined (53 us so, 41 that way).
//
// Whole rounds of tiles are done tile by tile; what is left over is cut into pieces of the same length, chunk after chunk on one line, whose sums meet in a second kernel in the order of the
// columns (8192 x 28672, 2048 tokens, 3.46 rounds: 845 us with a fourth round, 738 with the line).
//
// Bound: 256 x 256 tiles by the products and the power that they draw (8192 x 28672, 2048 tokens, adapters of rank 32: 794 us with all launches, one call after the other, 1218 TFLOP/s, 0.72 of what
// the library's 16-bit products reach at once and 0.86 of what they reach for seconds).  64 tokens: a CTA is through with a chunk every 820 cycles (28672 x 8192, 24 tokens: 83.8 us, 194 chunks an SM), while the
// chunk's products take 128 and its decoding about as much, and eight slots are under way; what they all wait for has not been found (issue slots half used, tensor cores 12 %, HBM 12 %;
// 14333 x 4096, 61 tokens 41 us).
#include "g2d_linear.cuh"
#include "g2d_tc.cuh"

namespace g2d {

constexpr int LT_JOIN_TOKENS = 4;
constexpr int LT_W_BYTES = 128 * 128, LT_CODE_BYTES = 128 * 32, LT_SLICE = 8;

// DUO: a pair of CTAs on 256 rows x NT tokens (cta_group::2), each with its rows of W and half of the tokens' rows of x.
// A slot holds one chunk of 64 columns: x, W as 16-bit values, and the codes of the chunk that its W will be next.
template <int NT, bool DUO>
struct LinearShape {
    static constexpr int X_ROWS = DUO ? NT / 2 : NT, X_BYTES = X_ROWS * KH * 2, SLOT = X_BYTES + LT_W_BYTES;
    static constexpr int SLOTS = NT == 64 ? 8 : 6;
    // Two warps per slot turn codes into values, a thread two rows: everything that they wait for comes in the order of their own turns, and while those of one slot wait,
    // load or fence, those of the others work.
    static constexpr int TEAM = 2, CODERS = TEAM * SLOTS, READERS = NT >= 128 ? 8 : 4;  // warps
    static constexpr int THREADS = 32 * (4 + CODERS + READERS);
    static constexpr int MINE = NT * 4 / READERS;  // columns of a reading warp
    static constexpr int ACCUMULATORS = 512 / NT;
    static constexpr size_t SMEM = (size_t)SLOTS * (SLOT + LT_CODE_BYTES) + 1024;
    // registers of a thread that loads or issues, codes, reads: by warpgroups no more than the launch gives, 80 for each of 768 threads
    static constexpr int ISSUE_REGISTERS = NT == 64 ? 64 : 56, CODE_REGISTERS = NT == 64 ? 64 : 40, READ_REGISTERS = 152;
    static_assert(THREADS == 768 && 4 * ISSUE_REGISTERS + CODERS * CODE_REGISTERS + READERS * READ_REGISTERS <= 24 * 80, "setmaxnreg would wait forever");
};

struct LinearTcJob {
    CUtensorMap x, inner, codes, up;
    LinearArgs a;
    LinearTcPlan p;
    int group_chunks;
    const int *plan;  // per tile of tokens: how many adapters, and which
    float *partial;   // [piece][shared tile][token][row]
};

// A CTA's (DUO: a pair's) work.  `p.whole` rounds of whole tiles first; what tiles are left lie on one line, chunk after chunk, and are cut into `p.ctas` pieces of the same length.
struct LinearItem {
    int row0, token0, token_tile, c0, c1;
    int piece;   // which of its tile
    int shared;  // number of the tile among those that are cut, -1: a whole one
};
// the CTA's part of the line, of fewer than 2^31 chunks (8 TB of codes): worked out once
struct LinePart {
    int first, last, tile, begins, piece;  // the tile in which the part begins, where that tile begins, and which of its pieces this is
};
__host__ __device__ __forceinline__ int64_t line_owner(const LinearTcPlan &p, int64_t at) { return ((at + 1) * p.ctas - 1) / p.line; }  // which CTA has a chunk
__device__ __forceinline__ LinePart line_part(const LinearTcPlan &p, int64_t cta) {
    LinePart part{};
    if (p.shared == 0 || cta >= p.ctas) return part;
    part.first = (int)(cta * p.line / p.ctas);
    part.last = (int)((cta + 1) * p.line / p.ctas);
    part.tile = part.first / p.chunks;
    part.begins = part.tile * p.chunks;
    part.piece = (int)(cta - line_owner(p, part.begins));
    return part;
}
template <int NT, bool DUO>
__device__ __forceinline__ bool linear_item(const LinearTcPlan &p, const LinePart &part, int rank, int number, LinearItem &it) {
    const int cta = (int)blockIdx.x / (DUO ? 2 : 1), ctas = (int)gridDim.x / (DUO ? 2 : 1);
    int tile = number * ctas + cta;
    it.c0 = 0;
    it.c1 = p.chunks;
    it.piece = 0;
    it.shared = -1;
    if (number >= p.whole) {
        const int along = number - p.whole, begins = part.begins + along * p.chunks;
        if (max(begins, part.first) >= part.last) return false;
        it.c0 = max(part.first - begins, 0);
        it.c1 = min(p.chunks, part.last - begins);
        it.piece = along == 0 ? part.piece : 0;
        it.shared = part.tile + along;
        tile = p.whole * ctas + it.shared;
    }
    it.token_tile = tile / p.row_tiles;
    it.row0 = (tile - it.token_tile * p.row_tiles) * (DUO ? 256 : 128) + rank * 128;
    it.token0 = it.token_tile * NT;
    return true;
}
// whether a slice ends with chunk ch
__device__ __forceinline__ bool slice_ends(const LinearTcJob &job, int ch, int last) {
    const int in_group = ch % job.group_chunks;
    return ch == last || in_group == job.group_chunks - 1 || in_group % LT_SLICE == LT_SLICE - 1;
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void tma_load_3d_duo(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
                 : "memory");
}

template <bool BF16>
__device__ __forceinline__ uint32_t add2(uint32_t u, uint32_t v) {
    if (BF16) {
        const __nv_bfloat162 r = __hadd2(*reinterpret_cast<__nv_bfloat162 *>(&u), *reinterpret_cast<__nv_bfloat162 *>(&v));
        return *reinterpret_cast<const uint32_t *>(&r);
    }
    const __half2 r = __hadd2(*reinterpret_cast<__half2 *>(&u), *reinterpret_cast<__half2 *>(&v));
    return *reinterpret_cast<const uint32_t *>(&r);
}
// The eight codes of a word, in order, as pairs: the bits of a code under the exponent of 1024 (fp16) or 128 (bf16), plus `add`: -1024 or -128, the origin of
// the codes and the zero point
template <bool BF16>
__device__ __forceinline__ uint4 decoded(uint32_t w, uint32_t add) {
    constexpr uint32_t MAGIC = BF16 ? 0x43004300u : 0x64006400u;
    const uint32_t w4 = w >> 4;
    uint4 r;
    r.x = add2<BF16>((__byte_perm(w, w4, 0x4400) & 0x000f000fu) | MAGIC, add);
    r.y = add2<BF16>((__byte_perm(w, w4, 0x5511) & 0x000f000fu) | MAGIC, add);
    r.z = add2<BF16>((__byte_perm(w, w4, 0x6622) & 0x000f000fu) | MAGIC, add);
    r.w = add2<BF16>((__byte_perm(w, w4, 0x7733) & 0x000f000fu) | MAGIC, add);
    return r;
}
__device__ __forceinline__ uint32_t word_of(const uint4 &v, int w) { return (w & 3) == 0 ? v.x : (w & 3) == 1 ? v.y : (w & 3) == 2 ? v.z : v.w; }
__device__ __forceinline__ void store_16(uint32_t at, const uint4 &v) { asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory"); }
__device__ __forceinline__ uint4 load_16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}

// The W that a CTA's coders have written is read by products that the other CTA, the leader, issues.  Arriving at the leader's barrier with .release takes a thread two thousand cycles (one
// that does nothing else: 8192 x 28672, 2048 tokens, adapters of rank 32 1787 us, two 1079).  So the coders arrive at a barrier of their own CTA, and one thread,
// which acquires that, lets a bulk copy tell the leader: of 16 bytes of that W, to be counted at the leader's barrier.  The copy is carried out behind what its thread has
// acquired, its end is a release for the cluster, and the thread need not wait for it (794 us; 775 with a relaxed arrival, which
// orders nothing; 14336 x 4096, 512 tokens 117, 116, and 125 where each coding warp sends a copy of its own).
__device__ __forceinline__ void tell_leader(uint4 *to, uint32_t from, uint64_t *bar) {
    uint32_t there;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(there) : "r"(smem_u32(to)));
    asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], 16, [%2];" ::"r"(there), "r"(from), "r"(leaders(bar)) : "memory");
}
// The warps that have read an accumulator have written nothing, and their loads have ended: their message to the leader need order nothing (4096 x 4096, 1024 tokens, groups of
// 64: 113 us with .release, 80 us, one scale a row 51 and 49; 8192 x 28672, 2048 tokens 789 and 752).
__device__ __forceinline__ void arrive_relaxed(uint32_t bar) { asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }

template <int NT, bool DUO>
struct LinearBarriers {
    using S = LinearShape<NT, DUO>;
    uint4 told[S::SLOTS];  // what the other CTA's copies leave
    // full: x has landed (or the rows of an adapter) and W is written, in both CTAs: the leader's; coded: W is written, in the other CTA; empty: the products have read the slot
    uint64_t full[S::SLOTS], coded[S::SLOTS], empty[S::SLOTS], code_full[S::SLOTS], code_empty[S::SLOTS], acc_full[S::ACCUMULATORS], acc_empty[S::ACCUMULATORS], drained;
    LinePart part;
    uint32_t tmem;
    int failed;
};

template <bool BF16, int NT, bool DUO>
__global__ void __launch_bounds__(LinearShape<NT, DUO>::THREADS, 1) linear_tc_kernel(const __grid_constant__ LinearTcJob job) {
    using S = LinearShape<NT, DUO>;
    constexpr int CTAS = DUO ? 2 : 1, ACC = S::ACCUMULATORS, SLOTS = S::SLOTS;
    extern __shared__ unsigned char linear_tc_smem[];
    __shared__ __align__(16) LinearBarriers<NT, DUO> bar;
    const LinearArgs &a = job.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = DUO ? (int)cluster_rank() : 0;
    const uint32_t base = (smem_u32(linear_tc_smem) + 1023u) & ~1023u, codes_base = base + SLOTS * S::SLOT;
    const auto wait = [&](uint64_t *b, uint32_t parity, unsigned nap) {
        if (DUO ? mbar_wait_cluster(b, parity, nap, a.wait_cycles) : mbar_wait(b, parity, nap, a.wait_cycles)) return true;
        bar.failed = 1;
        return false;
    };
    if (threadIdx.x == 0) {
        for (int s = 0; s < SLOTS; ++s) {
            mbar_init(&bar.full[s], 1 + S::TEAM);
            mbar_init(&bar.coded[s], S::TEAM);
            mbar_init(&bar.empty[s], 1);
            mbar_init(&bar.code_full[s], 1);
            mbar_init(&bar.code_empty[s], S::TEAM);
        }
        for (int s = 0; s < ACC; ++s) {
            mbar_init(&bar.acc_full[s], 1);
            mbar_init(&bar.acc_empty[s], CTAS * S::READERS);
        }
        mbar_init(&bar.drained, 1);
        bar.part = line_part(job.p, blockIdx.x / CTAS);
        bar.failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc<DUO>(&bar.tmem, 512);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (DUO) {
        __syncwarp();
        cluster_sync();
    }
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = bar.tmem;
    let_the_next_launch_start();
    // how many adapters an item has to add: those of its tile, by the first piece.  The launch before writes them.
    const auto adapters_in = [&](const LinearItem &it) {
        if (job.p.later || a.rank == 0 || it.piece != 0) return 0;
        after_the_launch_before();
        return job.plan[(int64_t)it.token_tile * (NT + 1)];
    };
    const auto adapter_at = [&](const LinearItem &it, int j) { return job.plan[(int64_t)it.token_tile * (NT + 1) + 1 + j]; };
    const auto item = [&](int number, LinearItem &it) { return linear_item<NT, DUO>(job.p, bar.part, rank, number, it); };
    const int first_coder = 4, first_reader = 4 + S::CODERS;

    // Every role counts the turns of the slots over all items of the CTA: a chunk of columns is a turn, and an adapter two (its inner values' upper and lower parts).
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::ISSUE_REGISTERS));
        if (warp == 0 && lane == 0) {  // x
            LinearItem it;
            int slot = 0;
            uint32_t parity = 1, turns = 0;
            const auto begin = [&](uint32_t bytes, uint32_t more) {  // the next slot is free and expects so many bytes in each CTA, and more of the other one's copy
                if (bar.failed || (turns >= SLOTS && !wait(&bar.empty[slot], parity, 32))) return false;
                // DUO: both CTAs' bytes count at the leader's barrier (they may do so before it expects them: the phase waits for its arrival)
                if (rank == 0) mbar_expect_tx(&bar.full[slot], CTAS * bytes + more);
                return true;
            };
            const auto bring = [&](const CUtensorMap *map, int column, int row) {
                if (DUO) tma_load_2d_duo(base + slot * S::SLOT, map, column, row, leaders(&bar.full[slot]));
                else tma_load_2d(base + slot * S::SLOT, map, column, row, &bar.full[slot]);
            };
            const auto next = [&] {
                ++turns;
                if (++slot == SLOTS) slot = 0, parity ^= 1;
            };
            bool go = true;
            for (int i = 0; go && item(i, it); ++i) {
                const int token = it.token0 + rank * S::X_ROWS;
                for (int ch = it.c0; go && ch < it.c1; ++ch) {
                    go = begin(S::X_BYTES, DUO ? 16 : 0);
                    if (!go) break;
                    bring(&job.x, ch * KH, token);
                    next();
                }
                const int extra = go ? 2 * adapters_in(it) : 0;
                for (int e = 0; go && e < extra; ++e) {
                    go = begin(S::X_BYTES + LT_W_BYTES, 0);
                    if (!go) break;
                    bring(&job.inner, (e & 1) * RANK_MAX, token);
                    const uint32_t to = base + slot * S::SLOT + S::X_BYTES;
                    if (DUO) tma_load_3d_duo(to, &job.up, 0, it.row0, adapter_at(it, e >> 1), leaders(&bar.full[slot]));
                    else tma_load_3d(to, &job.up, 0, it.row0, adapter_at(it, e >> 1), &bar.full[slot]);
                    next();
                }
            }
            // What was loaded has landed, and the leader's commits have arrived here, before this CTA ends: the last turn of every slot is awaited to its end.  After a
            // time-out the loads have their time to land.
            if (!bar.failed) {
                for (uint32_t k = turns > SLOTS ? turns - SLOTS : 0; k < turns; ++k) wait(&bar.empty[k % SLOTS], (k / SLOTS) & 1, 32);
            } else if (rank == 0) {
                let_it_land();
            }
        } else if (warp == 2 && lane == 0) {  // codes
            LinearItem it;
            int slot = 0;
            uint32_t used = 0, parity = 0;  // slots whose codes were loaded before; each slot's parity
            bool go = true;
            for (int i = 0; go && item(i, it); ++i) {
                for (int ch = it.c0; ch < it.c1; ++ch) {
                    const uint32_t bit = 1u << slot;
                    if (bar.failed || ((used & bit) && !wait(&bar.code_empty[slot], (parity >> slot) & 1, 32))) { go = false; break; }
                    if (used & bit) parity ^= bit;
                    used |= bit;
                    mbar_expect_tx(&bar.code_full[slot], LT_CODE_BYTES);
                    tma_load_2d(codes_base + slot * LT_CODE_BYTES, &job.codes, ch * (KH / 2), it.row0, &bar.code_full[slot]);
                    if (++slot == SLOTS) slot = 0;
                }
                if (go) slot = (slot + 2 * adapters_in(it)) % SLOTS;
            }
            // every load is awaited by the coders before they end; after a time-out they have their time to land
            if (bar.failed) let_it_land();
        } else if (warp == 1 && rank == 0 && elected()) {  // products
            // One thread issues them all: what it does per product (128 cycles for a pair of CTAs, 32 for narrow tiles) is kept short
            constexpr uint32_t DESC = idesc_16(NT, BF16 ? 1 : 0, DUO ? 2 * MT : MT);
            const uint64_t ws = umma_desc(base + S::X_BYTES), xs = umma_desc(base);
            LinearItem it;
            int slot = 0, slice = 0;
            uint32_t parity = 0;
            const auto ready = [&] {
                if (!wait(&bar.full[slot], parity, 0)) return false;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                return true;
            };
            const auto open = [&] {
                if (slice < ACC) return true;
                if (!wait(&bar.acc_empty[slice % ACC], (slice / ACC - 1) & 1, 0)) return false;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                return true;
            };
            const auto issue = [&](int ks, uint32_t accumulate) {
                const uint32_t d = tmem + (uint32_t)((slice % ACC) * NT);
                const uint64_t at = (uint64_t)((uint32_t)(slot * S::SLOT) >> 4) + 2 * ks;
                if (DUO) umma_16_duo(d, ws + at, xs + at, DESC, accumulate);
                else umma_16(d, ws + at, xs + at, DESC, accumulate);
            };
            const auto done = [&](bool closes) {
                commit<DUO>(&bar.empty[slot]);
                if (closes) commit<DUO>(&bar.acc_full[slice++ % ACC]);
                if (++slot == SLOTS) slot = 0, parity ^= 1;
            };
            bool go = true;
            for (int i = 0; go && item(i, it); ++i) {
                bool opens = true;
                int in_group = it.c0 % job.group_chunks;
                for (int ch = it.c0; ch < it.c1; ++ch) {
                    go = !bar.failed && ready() && (!opens || open());
                    if (!go) break;
                    issue(0, opens ? 0u : 1u);
#pragma unroll
                    for (int ks = 1; ks < KH / 16; ++ks) issue(ks, 1u);
                    const bool group_ends = in_group == job.group_chunks - 1;
                    opens = group_ends || (in_group & (LT_SLICE - 1)) == LT_SLICE - 1 || ch == it.c1 - 1;  // as slice_ends has it
                    in_group = group_ends ? 0 : in_group + 1;
                    done(opens);
                }
                const int extra = go ? 2 * adapters_in(it) : 0;
                for (int e = 0; e < extra; ++e) {  // the rows of `up` against the upper, then the lower parts of the inner values
                    go = !bar.failed && ready() && ((e & 1) || open());
                    if (!go) break;
                    for (int ks = 0; 16 * ks < a.rank; ++ks) issue(ks, (e & 1) || ks > 0 ? 1u : 0u);
                    done(e & 1);
                }
            }
            if (bar.failed) {  // every product that was issued completes, or has its time to, before what it reads and writes is given back
                commit<DUO>(&bar.drained);
                mbar_wait(&bar.drained, 0);
            } else {
                for (int k = max(slice - ACC, 0); k < slice; ++k) mbar_wait(&bar.acc_full[k % ACC], (k / ACC) & 1);
            }
        } else if (DUO && warp == 1 && rank != 0 && elected()) {  // the other CTA's W, slot after slot (rows of `up` come by the TMA, which counts at the leader's barrier itself)
            LinearItem it;
            int slot = 0;
            uint32_t parity = 0;  // each slot's
            bool go = true;
            for (int i = 0; go && item(i, it); ++i) {
                for (int ch = it.c0; ch < it.c1; ++ch) {
                    go = !bar.failed && wait(&bar.coded[slot], (parity >> slot) & 1, 0);
                    if (!go) break;
                    parity ^= 1u << slot;
                    tell_leader(&bar.told[slot], base + slot * S::SLOT + S::X_BYTES, &bar.full[slot]);
                    if (++slot == SLOTS) slot = 0;
                }
                if (go) slot = (slot + 2 * adapters_in(it)) % SLOTS;
            }
        }
        __syncwarp();
    } else if (warp < first_reader) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::CODE_REGISTERS));
        // ---- operands: the rows `row` and `row` + 64 of the turns of one slot ----
        const int slot = (warp - first_coder) / S::TEAM, row = (warp - first_coder) % S::TEAM * 32 + lane;
        const uint32_t to = base + slot * S::SLOT + S::X_BYTES + row * 128, from = codes_base + slot * LT_CODE_BYTES + row * 32;
        constexpr float ORIGIN = BF16 ? 128.f : 1024.f;
        LinearItem it;
        int first = 0;  // the slot of the item's first turn
        uint32_t turns = 0, coded = 0;
        bool go = true;
        const auto free_slot = [&] {
            if (turns > 0) go = go && wait(&bar.empty[slot], (turns - 1) & 1, 0);
            go = __all_sync(0xffffffffu, go && !bar.failed);
            ++turns;
            return go;
        };
        const auto written = [&] {
            if (lane == 0) mbar_arrive(DUO && rank != 0 ? &bar.coded[slot] : &bar.full[slot]);
        };
        for (int i = 0; go && item(i, it); ++i) {
            const float *const zero0 = a.zero + min((int64_t)it.row0 + row, a.m - 1) * a.zero_row, *const zero1 = a.zero + min((int64_t)it.row0 + row + 64, a.m - 1) * a.zero_row;
            int ch = it.c0 + (slot - first + SLOTS) % SLOTS, group_end = -1, next_group = -1;
            float next0 = 0.f, next1 = 0.f;  // the zero points of the group that this thread meets next, on their way
            uint32_t once0 = 0u, once1 = 0u, shift0 = 0u, shift1 = 0u;
            bool exact = true;
            for (; ch < it.c1; ch += SLOTS) {
                if (ch >= group_end) {  // another group
                    const int group = min(ch, job.p.chunks - 1) / job.group_chunks;
                    group_end = (group + 1) * job.group_chunks;
                    const float by0 = a.qmin - (group == next_group ? next0 : __ldg(zero0 + (int64_t)group * a.zero_group));
                    const float by1 = a.qmin - (group == next_group ? next1 : __ldg(zero1 + (int64_t)group * a.zero_group));
                    const int meets = (ch + (group_end - ch + SLOTS - 1) / SLOTS * SLOTS) / job.group_chunks;
                    next_group = min(meets, (job.p.chunks - 1) / job.group_chunks);
                    next0 = __ldg(zero0 + (int64_t)next_group * a.zero_group);
                    next1 = __ldg(zero1 + (int64_t)next_group * a.zero_group);
                    // one addition where -1024 + qmin - zero is a number of the type (integers up to 2048; bf16: -128, 256), else two, the first exact
                    once0 = float_to_bits(by0 - ORIGIN, BF16);
                    once1 = float_to_bits(by1 - ORIGIN, BF16);
                    exact = __all_sync(0xffffffffu, bits_to_float(once0, BF16) == by0 - ORIGIN && bits_to_float(once1, BF16) == by1 - ORIGIN);
                    once0 = exact ? once0 | (once0 << 16) : (BF16 ? 0xc308c308u : 0xe408e408u);
                    once1 = exact ? once1 | (once1 << 16) : once0;
                    shift0 = float_to_bits(by0 + 8.f, BF16) * 0x10001u;
                    shift1 = float_to_bits(by1 + 8.f, BF16) * 0x10001u;
                }
                if (!wait(&bar.code_full[slot], coded++ & 1, 0)) go = false;
                // rows of 32 bytes under the TMA's 32-byte swizzle: the two halves change places in every second group of four rows
                const uint32_t flip = ((row >> 2) & 1) << 4;
                if (!free_slot()) break;  // for the whole warp
#pragma unroll 1
                for (int part = 0; part < 4; ++part) {  // half a row at a time, in a loop: few registers, and few instructions for so many roles to share the caches with
                    const int r = part >> 1, h = part & 1;
                    const uint32_t at = to + r * (64 * 128), once = r ? once1 : once0, shift = r ? shift1 : shift0;
                    const uint4 raw = load_16(from + r * (64 * 32) + ((h << 4) ^ flip));
                    if (part == 3) {
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&bar.code_empty[slot]);
                    }
                    uint4 v[4];
#pragma unroll
                    for (int w = 0; w < 4; ++w) v[w] = decoded<BF16>(word_of(raw, w), once);
                    if (!exact) {
#pragma unroll
                        for (int w = 0; w < 4; ++w) v[w] = make_uint4(add2<BF16>(v[w].x, shift), add2<BF16>(v[w].y, shift), add2<BF16>(v[w].z, shift), add2<BF16>(v[w].w, shift));
                    }
#pragma unroll
                    for (int w = 0; w < 4; ++w) store_16(at + (((4 * h + w) ^ (row & 7)) << 4), v[w]);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                written();
            }
            if (!go) break;
            const int extra = 2 * adapters_in(it);
            first = (first + it.c1 - it.c0) % SLOTS;
            for (int e = (slot - first + SLOTS) % SLOTS; e < extra; e += SLOTS) {  // rows of `up`, which the TMA brings: the slot is free for them
                if (!free_slot()) break;
                if (rank == 0) written();
            }
            first = (first + extra) % SLOTS;
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::READ_REGISTERS));
        // ---- results: a thread has a row and MINE tokens ----
        constexpr int MINE = S::MINE;
        const int q = warp & 3, t0 = ((warp - first_reader) >> 2) * MINE;
        LinearItem it;
        int slice = 0;
        bool go = true;
        for (int i = 0; item(i, it); ++i) {
            const int64_t row = (int64_t)it.row0 + q * 32 + lane;
            const float *const scale = a.scale + min(row, a.m - 1) * a.scale_row;
            float total[MINE];
#pragma unroll
            for (int x = 0; x < MINE; ++x) total[x] = 0.f;
            const auto arrived = [&] {
                const bool ok = go && wait(&bar.acc_full[slice % ACC], (slice / ACC) & 1, 0);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                go = __all_sync(0xffffffffu, ok && !bar.failed);
                return go;
            };
            const auto leave = [&] {
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    if (DUO) arrive_relaxed(leaders(&bar.acc_empty[slice % ACC]));
                    else mbar_arrive(&bar.acc_empty[slice % ACC]);
                }
                ++slice;
            };
            const uint32_t from = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)t0;
            const auto factor_of = [&](int ch) { return __ldg(scale + (int64_t)(min(ch, job.p.chunks - 1) / job.group_chunks) * a.scale_group); };
            float factor = factor_of(it.c0);
            for (int ch = it.c0; go && ch < it.c1; ++ch) {
                if (!slice_ends(job, ch, it.c1 - 1)) continue;
                const float next_factor = factor_of(ch + 1);  // under way while the slice is awaited and read
                if (!arrived()) break;
#pragma unroll
                for (int cb = 0; cb < MINE / 16; ++cb) {
                    uint32_t v[16];
                    tmem_load_16(from + (uint32_t)((slice % ACC) * NT + cb * 16), v);
#pragma unroll
                    for (int x = 0; x < 16; ++x) total[cb * 16 + x] = fmaf(__uint_as_float(v[x]), factor, total[cb * 16 + x]);
                }
                leave();
                factor = next_factor;
            }
            const int extra = go ? adapters_in(it) : 0;
            if (extra > 0) {
                // every 32 tokens' adapters and factors, a token per lane: loaded once per tile, whatever the number of adapters
                int ids[MINE / 32];
                float factors[MINE / 32];
#pragma unroll
                for (int cb = 0; cb < MINE / 32; ++cb) {
                    const int token = it.token0 + t0 + cb * 32 + lane;
                    ids[cb] = adapter_of(a, token);
                    factors[cb] = ids[cb] >= 0 ? a.factor[token] : 0.f;
                }
                int id = adapter_at(it, 0);
                for (int e = 0; go && e < extra; ++e) {
                    const int next_id = e + 1 < extra ? adapter_at(it, e + 1) : 0;
                    if (!arrived()) break;
#pragma unroll
                    for (int cb = 0; cb < MINE / 16; ++cb) {
                        const unsigned takes = __ballot_sync(0xffffffffu, ids[cb / 2] == id) >> (cb % 2 * 16) & 0xffffu;
                        if (takes == 0u) continue;
                        uint32_t v[16];
                        tmem_load_16(from + (uint32_t)((slice % ACC) * NT + cb * 16), v);
#pragma unroll
                        for (int x = 0; x < 16; ++x) {  // a token of another adapter keeps its sum, whatever this one's rows hold
                            const float f = __shfl_sync(0xffffffffu, factors[cb / 2], cb % 2 * 16 + x);
                            if ((takes >> x) & 1u) total[cb * 16 + x] = fmaf(__uint_as_float(v[x]), f, total[cb * 16 + x]);
                        }
                    }
                    leave();
                    id = next_id;
                }
            }
            if (!go) {
#pragma unroll
                for (int x = 0; x < MINE; ++x) total[x] = NAN;
            }
            if (row < a.m) {
                const int count = min(MINE, a.tokens - it.token0 - t0);
                if (it.shared >= 0) {
                    constexpr int ROWS = DUO ? 256 : 128;
                    float *to = job.partial + (((int64_t)it.piece * job.p.shared + it.shared) * NT + t0) * ROWS + rank * 128 + q * 32 + lane;
#pragma unroll
                    for (int x = 0; x < MINE; ++x)
                        if (x < count) to[x * ROWS] = total[x];
                } else {
                    uint16_t *to = (uint16_t *)a.out + (int64_t)(it.token0 + t0) * a.out_stride + row;
#pragma unroll
                    for (int x = 0; x < MINE; ++x)
                        if (x < count) to[x * a.out_stride] = (uint16_t)float_to_bits(total[x], BF16);
                }
            }
        }
    }
    if (a.rank) after_the_launch_before();  // by every CTA: what follows on the stream must not start before the launch before has ended
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (DUO) {
        // neither CTA leaves while the other's MMAs may read its shared memory or arrive at its barriers
        if (threadIdx.x == 0 && bar.failed) let_it_land();
        __syncwarp();
        cluster_sync();
    }
    if (warp == 1) tmem_free<DUO>(tmem, 512);
    if (threadIdx.x == 0 && bar.failed && a.status) atomicExch(a.status, -1);
}

// The tiles that were cut: sums of their pieces, in their order, and (`later`) the outer halves of the adapters.  A thread has a row and LT_JOIN_TOKENS tokens.
template <bool STAGED>
__global__ void __launch_bounds__(128) linear_join_kernel(const LinearArgs a, const LinearTcPlan p, const float *__restrict__ partial, int grid_ctas) {
    __shared__ float4 inner[LT_JOIN_TOKENS][RANK_MAX / 4];
    __shared__ uint4 up_rows[STAGED ? 128 * (RANK_MAX / 8 + 1) : 1];
    const int rows = p.duo ? 256 : 128, parts = rows / 128;
    const int64_t shared = blockIdx.x / parts, tile = (int64_t)p.whole * grid_ctas + shared;
    const int in_tile = blockIdx.y * LT_JOIN_TOKENS;
    const int64_t token0 = tile / p.row_tiles * p.tile + in_tile, row_in_tile = blockIdx.x % parts * 128 + threadIdx.x, row = tile % p.row_tiles * rows + row_in_tile;
    const int pieces = (int)(line_owner(p, (shared + 1) * p.chunks - 1) - line_owner(p, shared * p.chunks)) + 1;
    const bool outer = p.later;
    int id[LT_JOIN_TOKENS];
#pragma unroll
    for (int e = 0; e < LT_JOIN_TOKENS; ++e) id[e] = outer ? adapter_of(a, (int)token0 + e) : -1;
    after_the_launch_before();
    if (outer) {
        for (int e = threadIdx.x; e < LT_JOIN_TOKENS * RANK_MAX; e += 128) {
            const int64_t token = token0 + e / RANK_MAX;
            const uint16_t *const h = a.inner + token * INNER_LD + e % RANK_MAX;
            if (token < a.tokens) reinterpret_cast<float *>(inner)[e] = bits_to_float(h[0], a.bf16) + bits_to_float(h[RANK_MAX], a.bf16);
        }
        __syncthreads();
    }
    const int count = (int)min((int64_t)LT_JOIN_TOKENS, a.tokens - token0);
    // The CTA's rows of a token's `up` are one piece of memory: they come as that, through shared memory, the next token's under way while one's are used.  (32 tokens, 40 adapters of rank 64,
    // 4096 rows: 14 us; each thread its own row, 16 bytes after the others: 78, as the first-level cache is small beside the products' shared memory.)  Rows of 16 bytes are read
    // as well as they lie (61 tokens, rank 8, 14333 rows, the whole call: 41.0 us, through shared memory 43.7).
    const int words = a.rank / 8, pitch = words | 1, per_row = words > 0 ? (65535 + words) / words : 0;  // x / words = x per_row >> 16 for x up to 1024
    uint4 next[RANK_MAX / 8];
    const auto fetch = [&](int e) {
        if (e >= count || id[e] < 0) return;
        const int64_t first = row - threadIdx.x;
        const uint4 *const up = reinterpret_cast<const uint4 *>((const uint16_t *)a.up + ((int64_t)id[e] * a.m + first) * a.rank);
        const int there = (int)min((int64_t)128, a.m - first) * words;
#pragma unroll
        for (int i = 0; i < RANK_MAX / 8; ++i)
            if (i < words && i * 128 + (int)threadIdx.x < there) next[i] = __ldg(up + i * 128 + threadIdx.x);
    };
    if (STAGED) fetch(0);
    float sum[LT_JOIN_TOKENS];
#pragma unroll
    for (int e = 0; e < LT_JOIN_TOKENS; ++e) sum[e] = 0.f;
    if (row < a.m) {
        const float *from = partial + (shared * p.tile + in_tile) * rows + row_in_tile;
#pragma unroll 2
        for (int k = 0; k < pieces; ++k, from += p.shared * p.tile * rows) {
#pragma unroll
            for (int e = 0; e < LT_JOIN_TOKENS; ++e)
                if (e < count) sum[e] += from[e * rows];
        }
    }
#pragma unroll
    for (int e = 0; e < LT_JOIN_TOKENS; ++e) {
        if (e >= count) break;
        if (STAGED && id[e] >= 0) {
            __syncthreads();  // the rows before have been read
#pragma unroll
            for (int i = 0; i < RANK_MAX / 8; ++i) {
                const int x = i * 128 + (int)threadIdx.x, r = x * per_row >> 16;
                if (i < words) up_rows[r * pitch + x - r * words] = next[i];
            }
            __syncthreads();
        }
        if (STAGED && e + 1 < LT_JOIN_TOKENS) fetch(e + 1);
        if (id[e] >= 0 && row < a.m) {
            const uint4 *const up = reinterpret_cast<const uint4 *>((const uint16_t *)a.up + ((int64_t)id[e] * a.m + row) * a.rank);
            float more = 0.f;
            for (int r = 0; r < words; ++r) {
                const uint4 v = STAGED ? up_rows[threadIdx.x * pitch + r] : __ldg(up + r);
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                const float4 h[2] = {inner[e][2 * r], inner[e][2 * r + 1]};
                const float hh[8] = {h[0].x, h[0].y, h[0].z, h[0].w, h[1].x, h[1].y, h[1].z, h[1].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    more = fmaf(bits_to_float(w[i] & 0xffffu, a.bf16), hh[2 * i], more);
                    more = fmaf(bits_to_float(w[i] >> 16, a.bf16), hh[2 * i + 1], more);
                }
            }
            sum[e] = fmaf(more, a.factor[token0 + e], sum[e]);
        }
        if (row < a.m) ((uint16_t *)a.out)[(token0 + e) * a.out_stride + row] = (uint16_t)float_to_bits(sum[e], a.bf16);
    }
}

static bool make_map_codes(CUtensorMap *map, const uint8_t *codes, int64_t rows, int64_t bytes, int64_t pitch) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)bytes, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)pitch};
    const cuuint32_t box[2] = {32, 128};
    const cuuint32_t elem[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t *>(codes), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_32B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// rows of `up`: boxes of 128 rows of one adapter, the rank padded to 64 with zeros
static bool make_map_up(CUtensorMap *map, const LinearArgs &a) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)a.rank, (cuuint64_t)a.m, (cuuint64_t)a.adapters};
    const cuuint64_t strides[2] = {(cuuint64_t)a.rank * 2, (cuuint64_t)a.rank * 2 * (cuuint64_t)a.m};
    const cuuint32_t box[3] = {KH, 128, 1};
    const cuuint32_t elem[3] = {1, 1, 1};
    return fn(map, a.bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void *>(a.up), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Adapters' outer halves at the join: up to LINEAR_FEW tokens always; up to 256 where so many adapters may be among a tile's tokens that two turns for each are many, and a rank is short enough for
// the join's fp32 sums.  14336 x 4096, 128 tokens: 32 adapters of rank 8 62.5 us at the join, 73.9 as turns, 100 of rank 16 76.4, 89.2; 8 of rank 64 86.9, 61.5, 4 of rank 16 60.0, 48.9; 512 tokens, 100
// of rank 16 159.6, 158.3.  256 tokens: 32 of rank 8 70.0, 80.0, of rank 16 92.4, 82.2; 4096 x 4096 41.1, 56.3
// and 47.4, 56.2.
constexpr int64_t LATER_TOKENS = 256, LATER_ADAPTERS = 24;
constexpr int LATER_RANK = 16;
LinearTcPlan linear_tc_plan(int64_t m, int64_t n, int64_t tokens, int rank, int64_t adapters) {
    LinearTcPlan p;
    p.tile = tokens <= LINEAR_FEW ? LINEAR_FEW : 128;
    p.duo = 0;
    int64_t rows = ceil_div(m, (int64_t)128), columns = ceil_div(tokens, (int64_t)p.tile);
    // 256 x 256 by pairs of CTAs, four times the work of a 128 x 128 tile in little more than its time, unless a pair's share is too short for what each tile costs besides.  2048 x 2048, 256 tokens
    // (3.5 chunks a pair) 14.6 us by 128 x 128, 16.1 by pairs; 512 tokens (7) 19.4, 17.9; 4096 x 4096, 256 tokens (14) 25.6, 23.5; 8192 x 8192, 512 tokens 110.6, 70.3.  Up to 128 tokens half of
    // such a tile would be empty: 8192 x 8192, 100 tokens 36.3, 37.5, in groups of 128 45.7, 51.6.
    const int64_t pairs = ceil_div(m, (int64_t)256) * ceil_div(tokens, (int64_t)256);
    if (tokens > 128 && pairs * ceil_div(n, (int64_t)KH) >= 74 * 6) {
        p.tile = 256;
        p.duo = 1;
        rows = ceil_div(m, (int64_t)256);
        columns = ceil_div(tokens, (int64_t)256);
    }
    p.row_tiles = (int)rows;
    p.token_tiles = (int)columns;
    p.chunks = (int)ceil_div(n, (int64_t)KH);
    const int64_t tiles = rows * columns, at_once = p.duo ? 74 : 148;
    p.later = rank > 0 && (tokens <= LINEAR_FEW || (tokens <= LATER_TOKENS && adapters >= LATER_ADAPTERS && rank <= LATER_RANK));
    p.whole = p.later ? 0 : (int)(tiles / at_once);
    p.shared = tiles - p.whole * at_once;
    p.line = p.shared * p.chunks;
    p.ctas = p.line / 8 < at_once ? (p.line / 8 > 0 ? p.line / 8 : 1) : at_once;  // pieces of eight chunks at least
    p.pieces = 0;
    if (p.shared > 0) {
        p.pieces = ceil_div((int64_t)p.chunks - 1, p.line / p.ctas) + 1;
        if (p.pieces > p.ctas) p.pieces = p.ctas;
    }
    p.partial_bytes = (size_t)p.pieces * p.shared * p.tile * (p.duo ? 256 : 128) * sizeof(float);
    return p;
}

template <bool BF16, int NT, bool DUO>
static int launch_tc(const LinearArgs &a, const LinearTcPlan &p, const int *plan, float *partial, cudaStream_t st) {
    using S = LinearShape<NT, DUO>;
    static PerDeviceOnce configured;
    if (configured.run([&] { return cudaFuncSetAttribute(linear_tc_kernel<BF16, NT, DUO>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::SMEM) == cudaSuccess; }) != G2D_OK) return G2D_ERR_CUDA;
    LinearTcJob job;
    job.a = a;
    job.p = p;
    job.group_chunks = a.group >= a.n ? p.chunks : (int)(a.group / KH);
    job.plan = plan;
    job.partial = partial;
    if (!make_map_16(&job.x, a.x, a.tokens, a.n, S::X_ROWS, BF16, a.x_stride) || !make_map_codes(&job.codes, a.codes, a.m, a.n / 2, a.row_bytes)) return G2D_ERR_CUDA;
    if (a.rank > 0 && (!make_map_16(&job.inner, a.inner, a.tokens, INNER_LD, S::X_ROWS, BF16) || !make_map_up(&job.up, a))) return G2D_ERR_CUDA;
    if (a.rank == 0) job.inner = job.up = job.x;
    const int64_t ctas = p.whole > 0 ? (DUO ? 74 : 148) : p.ctas;
    const int launched = launch_dependent(linear_tc_kernel<BF16, NT, DUO>, dim3((unsigned)(DUO ? 2 * ctas : ctas)), S::THREADS, S::SMEM, DUO ? 2 : 1, a.rank > 0, st, job);
    if (launched != G2D_OK || p.shared == 0) return launched;
    const auto join = p.later && a.rank > 8 ? linear_join_kernel<true> : linear_join_kernel<false>;
    return launch_dependent(join, dim3((unsigned)p.shared * (DUO ? 2 : 1), NT / LT_JOIN_TOKENS), 128, 0, 1, true, st, a, p, partial, (int)ctas);
}

int launch_linear_tc(const LinearArgs &a, const LinearTcPlan &p, const int *plan, float *partial, cudaStream_t st) {
    if (p.tile == 64) return a.bf16 ? launch_tc<true, 64, false>(a, p, plan, partial, st) : launch_tc<false, 64, false>(a, p, plan, partial, st);
    if (p.tile == 128) return a.bf16 ? launch_tc<true, 128, false>(a, p, plan, partial, st) : launch_tc<false, 128, false>(a, p, plan, partial, st);
    return a.bf16 ? launch_tc<true, 256, true>(a, p, plan, partial, st) : launch_tc<false, 256, true>(a, p, plan, partial, st);
}

}  // namespace g2d
