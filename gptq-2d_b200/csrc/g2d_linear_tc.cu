// y = x W^T for a matrix W held as packed 4-bit codes, many tokens, on tcgen05; low-rank adapters of the tokens' requests beside it.
//
// A tile is 128 rows of W times NT tokens: A is W, so a scale belongs to a lane of tensor memory.  Codes travel as they are: the TMA brings 128 rows x 256 columns
// (16 KB) of them, four or eight warps turn 64 columns at a time into 16-bit values in the swizzled layout of an MMA operand (code - 8 exactly, plus 8 + qmin - zero rounded to the type), and
// x comes by TMA beside them.  What is accumulated in tensor memory is a slice of the columns under one scale (512 columns at most: the tensor cores add with truncation);
// warps of their own read each slice while the next is accumulated, and add scale times slice in registers, in fp32.
//
// An adapter is two more slices of k: for every adapter among a tile's tokens A is its rows of `up` (times nothing) and B the tokens' inner values, upper and lower
// parts (see g2d_adapters.cu).  The product has a column for every token of the tile; the reading warps add it, times the token's factor, only where the token has this adapter.
//
// Few tiles: the columns are split over several CTAs, whose sums meet in a second kernel, in a fixed order.
#include "g2d_linear.cuh"
#include "g2d_tc.cuh"

namespace g2d {

constexpr int LT_CODE_BYTES = 128 * 128, LT_W_BYTES = 128 * 128, LT_SUB = 2, LT_CODE_CHUNKS = 4, LT_SLICE = 8;

// DUO: a pair of CTAs on 256 rows x NT tokens (cta_group::2), each with its rows of W and half of the tokens' rows of x
template <int NT, bool DUO>
struct LinearShape {
    static constexpr int X_ROWS = DUO ? NT / 2 : NT, X_BYTES = X_ROWS * KH * 2, STAGE = LT_SUB * (X_BYTES + LT_W_BYTES);  // two chunks of 64 columns
    static constexpr int CODE_STAGES = 2, STAGES = NT == 64 ? 4 : 3;
    static constexpr int CODERS = 4, READERS = NT >= 128 ? 8 : 4;  // warps; the coders of a team take a stage together, a row per thread
    static constexpr int TEAMS = NT == 64 ? 4 : 2;                  // that take the stages in turn: one waits and fences while another works
    static constexpr int THREADS = 32 * (4 + TEAMS * CODERS + READERS);
    // registers of a thread that loads or issues, codes, reads: by warpgroups no more than the launch gives (96 or, of 768 threads, 80 each)
    static constexpr int ISSUE_REGISTERS = NT == 64 ? 40 : 48, CODE_REGISTERS = NT == 64 ? 72 : 64, READ_REGISTERS = 152;
    static_assert(4 * ISSUE_REGISTERS + TEAMS * CODERS * CODE_REGISTERS + READERS * READ_REGISTERS <= THREADS / 32 * (NT == 64 ? 80 : 96), "setmaxnreg would wait forever");
    static constexpr int MINE = NT * 4 / READERS;                               // columns of a reading warp
    static constexpr int ACCUMULATORS = 512 / NT;
    static constexpr size_t SMEM = (size_t)STAGES * STAGE + CODE_STAGES * LT_CODE_BYTES + 1024;
};

struct LinearTcJob {
    CUtensorMap x, inner, codes, up;
    LinearArgs a;
    int row_tiles, token_tiles, splits, chunks, group_chunks;  // chunks: an even number of them
    const int *plan;  // per tile of tokens: how many adapters, and which
    float *partial;   // [splits][tokens][m], where splits > 1
};

struct LinearItem {
    int row0, token0, token_tile, split, c0, c1;
};
template <int NT, bool DUO>
__device__ __forceinline__ bool linear_item(const LinearTcJob &job, int rank, int number, LinearItem &it) {
    const int64_t at = (blockIdx.x + (int64_t)number * gridDim.x) / (DUO ? 2 : 1);
    if (at >= (int64_t)job.row_tiles * job.token_tiles * job.splits) return false;
    it.split = (int)(at % job.splits);
    const int64_t tile = at / job.splits;
    it.token_tile = (int)(tile / job.row_tiles);
    it.row0 = (int)(tile % job.row_tiles) * (DUO ? 256 : 128) + rank * 128;
    it.token0 = it.token_tile * NT;
    const int quads = (job.chunks + LT_CODE_CHUNKS - 1) / LT_CODE_CHUNKS;  // splits begin where codes' stages do
    it.c0 = (int)((int64_t)it.split * quads / job.splits) * LT_CODE_CHUNKS;
    it.c1 = min((int)((int64_t)(it.split + 1) * quads / job.splits) * LT_CODE_CHUNKS, job.chunks);
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

// One thread of the warp, all of whose threads are here.  The compiler knows that a branch on this leaves one thread, and keeps what a product's instruction takes
// from uniform registers there; behind a comparison of lane numbers it does not.
__device__ __forceinline__ bool elected() {
    uint32_t one;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(one));
    return one != 0;
}

__device__ __forceinline__ void arrive_relaxed(uint32_t bar) { asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }

template <int NT, bool DUO>
struct LinearBarriers {
    using S = LinearShape<NT, DUO>;
    uint64_t x_full[S::STAGES], w_here[S::STAGES], w_full[S::STAGES], empty[S::STAGES], code_full[S::CODE_STAGES], code_empty[S::CODE_STAGES], acc_full[S::ACCUMULATORS], acc_empty[S::ACCUMULATORS], drained;
    uint32_t tmem;
    int failed;
};

template <bool BF16, int NT, bool DUO>
__global__ void __launch_bounds__(LinearShape<NT, DUO>::THREADS, 1) linear_tc_kernel(const __grid_constant__ LinearTcJob job) {
    using S = LinearShape<NT, DUO>;
    constexpr int CTAS = DUO ? 2 : 1, ACC = S::ACCUMULATORS;
    extern __shared__ unsigned char linear_tc_smem[];
    __shared__ __align__(8) LinearBarriers<NT, DUO> bar;
    const LinearArgs &a = job.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = DUO ? (int)cluster_rank() : 0;
    const uint32_t base = (smem_u32(linear_tc_smem) + 1023u) & ~1023u, codes_base = base + S::STAGES * S::STAGE;
    const auto wait = [&](uint64_t *b, uint32_t parity, unsigned nap) {
        if (mbar_wait(b, parity, nap, a.wait_cycles)) return true;
        bar.failed = 1;
        return false;
    };
    const auto arrive = [&](uint64_t *b) {  // at the leader's barrier
        if (DUO) mbar_arrive_at(leaders(b));
        else mbar_arrive(b);
    };
    if (threadIdx.x == 0) {
        for (int s = 0; s < S::STAGES; ++s) {
            mbar_init(&bar.x_full[s], 1);
            mbar_init(&bar.w_here[s], S::CODERS);
            mbar_init(&bar.w_full[s], CTAS);
            mbar_init(&bar.empty[s], 1);
        }
        for (int s = 0; s < S::CODE_STAGES; ++s) {
            mbar_init(&bar.code_full[s], 1);
            mbar_init(&bar.code_empty[s], S::TEAMS * S::CODERS);
        }
        for (int s = 0; s < ACC; ++s) {
            mbar_init(&bar.acc_full[s], 1);
            mbar_init(&bar.acc_empty[s], CTAS * S::READERS);
        }
        mbar_init(&bar.drained, 1);
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
    // how many adapters an item has to add: those of its tile, by the first split.  The launch before writes them.
    const auto adapters_in = [&](const LinearItem &it) {
        if (a.rank == 0 || it.split != 0) return 0;
        after_the_launch_before();
        return job.plan[(int64_t)it.token_tile * (NT + 1)];
    };
    const auto adapter_at = [&](const LinearItem &it, int j) { return job.plan[(int64_t)it.token_tile * (NT + 1) + 1 + j]; };
    const auto item = [&](int number, LinearItem &it) { return linear_item<NT, DUO>(job, rank, number, it); };
    const int first_coder = 4, first_reader = 4 + S::TEAMS * S::CODERS;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::ISSUE_REGISTERS));
        if (warp == 0 && lane == 0) {  // x
            LinearItem it;
            int c = 0;
            const auto begin = [&](uint32_t bytes) {  // the next stage is free and expects so many bytes in each CTA
                const int stage = c % S::STAGES, round = c / S::STAGES;
                if (bar.failed || (round > 0 && !wait(&bar.empty[stage], (round - 1) & 1, 32))) return false;
                // DUO: both CTAs' bytes count at the leader's barrier (they may do so before it expects them: the phase waits for its arrival)
                if (rank == 0) mbar_expect_tx(&bar.x_full[stage], CTAS * bytes);
                return true;
            };
            const auto bring = [&](uint32_t at, const CUtensorMap *map, int column, int row) {
                uint64_t *const full = &bar.x_full[c % S::STAGES];
                const uint32_t to = base + (c % S::STAGES) * S::STAGE + at;
                if (DUO) tma_load_2d_duo(to, map, column, row, leaders(full));
                else tma_load_2d(to, map, column, row, full);
            };
            bool go = true;
            for (int i = 0; go && item(i, it); ++i) {
                const int token = it.token0 + rank * S::X_ROWS;
                for (int ch = it.c0; go && ch < it.c1; ch += LT_SUB) {
                    go = begin(LT_SUB * S::X_BYTES);
                    if (!go) break;
                    for (int s = 0; s < LT_SUB; ++s) bring(s * S::X_BYTES, &job.x, (ch + s) * KH, token);
                    ++c;
                }
                const int extra = go ? adapters_in(it) : 0;
                for (int e = 0; go && e < extra; ++e) {
                    go = begin(LT_SUB * S::X_BYTES + LT_W_BYTES);
                    if (!go) break;
                    for (int s = 0; s < LT_SUB; ++s) bring(s * S::X_BYTES, &job.inner, s * RANK_MAX, token);
                    uint64_t *const full = &bar.x_full[c % S::STAGES];
                    const uint32_t to = base + (c % S::STAGES) * S::STAGE + LT_SUB * S::X_BYTES;
                    if (DUO) tma_load_3d_duo(to, &job.up, 0, it.row0, adapter_at(it, e), leaders(full));
                    else tma_load_3d(to, &job.up, 0, it.row0, adapter_at(it, e), full);
                    ++c;
                }
            }
            // landed, or had their time to, before the memory is given back
            if (rank == 0)
                for (int k = max(c - S::STAGES, 0); k < c; ++k) mbar_wait(&bar.x_full[k % S::STAGES], (k / S::STAGES) & 1);
            if (DUO && !bar.failed) {  // the leader's commits arrive here as well: none may be under way when this CTA ends
                for (int k = max(c - S::STAGES, 0); k < c; ++k) wait(&bar.empty[k % S::STAGES], (k / S::STAGES) & 1, 32);
            }
        } else if (warp == 2 && lane == 0) {  // codes
            LinearItem it;
            int c = 0;
            bool go = true;
            for (int i = 0; go && item(i, it); ++i) {
                for (int ch = it.c0; ch < it.c1; ch += LT_CODE_CHUNKS, ++c) {
                    const int stage = c % S::CODE_STAGES, round = c / S::CODE_STAGES;
                    if (bar.failed || (round > 0 && !wait(&bar.code_empty[stage], (round - 1) & 1, 32))) { go = false; break; }
                    mbar_expect_tx(&bar.code_full[stage], LT_CODE_BYTES);
                    tma_load_2d(codes_base + stage * LT_CODE_BYTES, &job.codes, ch * (KH / 2), it.row0, &bar.code_full[stage]);
                }
            }
            for (int k = max(c - S::CODE_STAGES, 0); k < c; ++k) mbar_wait(&bar.code_full[k % S::CODE_STAGES], (k / S::CODE_STAGES) & 1);
        } else if (DUO && warp == 3 && lane == 0) {
            // The coders arrive at this CTA's barrier; this thread passes it on to the leader's.  What they wrote stays in this CTA's shared memory and is read by this
            // SM's tensor core alone: they have brought it there by their proxy fence before they arrive, so that the message itself need order nothing (with
            // .release it takes a thousand cycles of this chain: 8192 x 28672, 2048 tokens, 940 and 885 us).
            LinearItem it;
            int c = 0;
            bool go = true;
            for (int i = 0; go && item(i, it); ++i) {
                const int stages = (it.c1 - it.c0 + LT_SUB - 1) / LT_SUB + adapters_in(it);
                for (int k = 0; go && k < stages; ++k, ++c) {
                    go = !bar.failed && wait(&bar.w_here[c % S::STAGES], (c / S::STAGES) & 1, 20);
                    if (go) arrive_relaxed(leaders(&bar.w_full[c % S::STAGES]));
                }
            }
        } else if (warp == 1 && rank == 0 && elected()) {  // products
            // One thread issues them all: what it does per product (128 cycles for a pair of CTAs, 32 for narrow tiles) is kept short
            constexpr uint32_t DESC = idesc_16(NT, BF16 ? 1 : 0, DUO ? 2 * MT : MT);
            const uint64_t ws = umma_desc(base + LT_SUB * S::X_BYTES), xs = umma_desc(base);
            LinearItem it;
            int stage = 0, slice = 0;
            uint32_t parity = 0;
            const auto ready = [&] {
                if (bar.failed || !wait(DUO ? &bar.w_full[stage] : &bar.w_here[stage], parity, 20) || !wait(&bar.x_full[stage], parity, 20)) return false;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                return true;
            };
            const auto open = [&] {
                if (slice < ACC) return true;
                if (!wait(&bar.acc_empty[slice % ACC], (slice / ACC - 1) & 1, 20)) return false;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                return true;
            };
            const auto issue = [&](uint64_t w, uint64_t x, uint32_t accumulate) {
                const uint32_t d = tmem + (uint32_t)((slice % ACC) * NT);
                if (DUO) umma_16_duo(d, w, x, DESC, accumulate);
                else umma_16(d, w, x, DESC, accumulate);
            };
            const auto done = [&] {
                commit<DUO>(&bar.empty[stage]);
                if (++stage == S::STAGES) stage = 0, parity ^= 1;
            };
            bool go = true;
            for (int i = 0; go && item(i, it); ++i) {
                bool opens = true;
                int in_group = it.c0 % job.group_chunks;
                for (int ch = it.c0; go && ch < it.c1; ch += LT_SUB) {
                    go = ready();
                    const uint64_t w0 = ws + (uint64_t)((uint32_t)(stage * S::STAGE) >> 4), x0 = xs + (uint64_t)((uint32_t)(stage * S::STAGE) >> 4);
#pragma unroll
                    for (int s = 0; s < LT_SUB; ++s) {
                        if (opens) go = go && open();
                        if (!go) break;
                        const uint64_t w = w0 + (uint64_t)(s * (LT_W_BYTES >> 4)), x = x0 + (uint64_t)(s * (S::X_BYTES >> 4));
                        issue(w, x, opens ? 0u : 1u);
#pragma unroll
                        for (int ks = 1; ks < KH / 16; ++ks) issue(w + 2 * ks, x + 2 * ks, 1u);
                        const bool group_ends = in_group == job.group_chunks - 1;
                        opens = group_ends || (in_group & (LT_SLICE - 1)) == LT_SLICE - 1 || ch + s == it.c1 - 1;  // as slice_ends has it
                        in_group = group_ends ? 0 : in_group + 1;
                        if (opens) commit<DUO>(&bar.acc_full[slice++ % ACC]);
                    }
                    done();
                }
                const int extra = go ? adapters_in(it) : 0;
                for (int e = 0; go && e < extra; ++e) {  // the rows of `up` against both parts of the inner values
                    go = ready() && open();
                    if (!go) break;
                    const uint64_t w0 = ws + (uint64_t)((uint32_t)(stage * S::STAGE) >> 4), x0 = xs + (uint64_t)((uint32_t)(stage * S::STAGE) >> 4);
                    for (int ks = 0; 16 * ks < a.rank; ++ks) {
                        issue(w0 + 2 * ks, x0 + 2 * ks, ks > 0);
                        issue(w0 + 2 * ks, x0 + (S::X_BYTES >> 4) + 2 * ks, 1u);
                    }
                    commit<DUO>(&bar.acc_full[slice++ % ACC]);
                    done();
                }
            }
            if (bar.failed) {  // every product that was issued completes, or has its time to, before what it reads and writes is given back
                commit<DUO>(&bar.drained);
                mbar_wait(&bar.drained, 0);
            } else {
                for (int k = max(slice - ACC, 0); k < slice; ++k) mbar_wait(&bar.acc_full[k % ACC], (k / ACC) & 1);
            }
        }
        __syncwarp();
    } else if (warp < first_reader) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::CODE_REGISTERS));
        // ---- operands: a thread has a row and, with four warps, both chunks of a stage, else one ----
        const int team = (warp - first_coder) / S::CODERS, id = threadIdx.x - 32 * (first_coder + team * S::CODERS), row = id;
        LinearItem it;
        int stage = 0, turn = 0, code_stage = 0;
        uint32_t parity = 1, code_parity = 0;  // of the stage's last release (the first time round there is none to wait for)
        bool go = true, again = false;
        const auto released = [&] { return !again || wait(&bar.empty[stage], parity, 20); };
        const auto free_stage = [&] {
            go = go && released();
            go = __all_sync(0xffffffffu, go && !bar.failed);
            return go;
        };
        const auto advance = [&](bool mine) {
            // Where a team does not come back to the same stages, it awaits the other turns' releases too (they come before its own): a wait that left out a
            // phase could take the one before for it.
            if (!mine && S::STAGES % S::TEAMS != 0) go = go && released();
            if (++stage == S::STAGES) stage = 0, parity ^= 1, again = true;
            if (++turn == S::TEAMS) turn = 0;
        };
        constexpr float ORIGIN = BF16 ? 128.f : 1024.f;
        for (int i = 0; go && item(i, it); ++i) {
            const float *const zero = a.zero + min((int64_t)it.row0 + row, a.m - 1) * a.zero_row;
            const int groups = (job.chunks - 1) / job.group_chunks + 1;
            // the zero point of the next group that this thread meets is on its way
            int group_end = -1;
            const auto zero_of = [&](int g) { return __ldg(zero + (int64_t)min(g, groups - 1) * a.zero_group); };
            float next_zero = 0.f;
            int next_group = -2;
            uint32_t once = 0u, shift = 0u;
            bool exact = true;
            for (int ch = it.c0; ch < it.c1; ch += LT_SUB) {
                const int quarter = ch % LT_CODE_CHUNKS;
                // by all teams, theirs or not, as for the releases
                if (quarter == 0 && !wait(&bar.code_full[code_stage], code_parity, 20)) go = false;
                if (turn == team) {
                    const uint32_t from = codes_base + code_stage * LT_CODE_BYTES + row * 128;
                    uint4 raw[2 * LT_SUB];
#pragma unroll
                    for (int w = 0; w < 2 * LT_SUB; ++w) raw[w] = load_16(from + (((quarter * 2 + w) ^ (row & 7)) << 4));
                    if (!free_stage()) break;  // for the whole warp
#pragma unroll
                    for (int s = 0; s < LT_SUB; ++s) {
                        if (ch + s >= group_end) {  // another group
                            const int group = (ch + s) / job.group_chunks;
                            group_end = (group + 1) * job.group_chunks;
                            const float by = a.qmin - (group == next_group ? next_zero : zero_of(group));
                            next_group = (group_end > ch + LT_SUB - 1 ? max(group_end, ch + LT_SUB * S::TEAMS) : group_end) / job.group_chunks;
                            next_zero = zero_of(next_group);
                            // one addition where -1024 + qmin - zero is a number of the type (integers up to 2048; bf16: -128, 256), else two, the first exact
                            const uint32_t whole = float_to_bits(by - ORIGIN, BF16), apart = float_to_bits(by + 8.f, BF16);
                            exact = __all_sync(0xffffffffu, bits_to_float(whole, BF16) == by - ORIGIN);
                            once = exact ? whole | (whole << 16) : (BF16 ? 0xc308c308u : 0xe408e408u);
                            shift = apart | (apart << 16);
                        }
                        const uint32_t to = base + stage * S::STAGE + LT_SUB * S::X_BYTES + s * LT_W_BYTES + row * 128;
                        if (exact) {
#pragma unroll
                            for (int w = 0; w < 8; ++w) store_16(to + ((w ^ (row & 7)) << 4), decoded<BF16>(word_of(raw[2 * s + (w >> 2)], w), once));
                        } else {
#pragma unroll
                            for (int w = 0; w < 8; ++w) {
                                const uint4 v = decoded<BF16>(word_of(raw[2 * s + (w >> 2)], w), once);
                                store_16(to + ((w ^ (row & 7)) << 4), make_uint4(add2<BF16>(v.x, shift), add2<BF16>(v.y, shift), add2<BF16>(v.z, shift), add2<BF16>(v.w, shift)));
                            }
                        }
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bar.w_here[stage]);
                }
                advance(turn == team);
                if (quarter + LT_SUB >= LT_CODE_CHUNKS || ch + LT_SUB >= it.c1) {
                    if (lane == 0) mbar_arrive(&bar.code_empty[code_stage]);  // behind the warp's barrier: all lanes have read
                    if (++code_stage == S::CODE_STAGES) code_stage = 0, code_parity ^= 1;
                }
            }
            const int extra = go ? adapters_in(it) : 0;
            for (int e = 0; go && e < extra; ++e) {  // rows of `up`, which the TMA brings: the stage is free for them
                if (turn == team) {
                    if (!free_stage()) break;
                    if (lane == 0) mbar_arrive(&bar.w_here[stage]);
                }
                advance(turn == team);
            }
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
                const bool ok = go && wait(&bar.acc_full[slice % ACC], (slice / ACC) & 1, 20);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                go = __all_sync(0xffffffffu, ok && !bar.failed);
                return go;
            };
            const auto leave = [&] {
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) arrive(&bar.acc_empty[slice % ACC]);
                ++slice;
            };
            const uint32_t from = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)t0;
            const auto factor_of = [&](int ch) { return __ldg(scale + (int64_t)(min(ch, job.chunks - 1) / job.group_chunks) * a.scale_group); };
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
            for (int e = 0; go && e < extra; ++e) {
                const int id = adapter_at(it, e);
                if (!arrived()) break;
#pragma unroll
                for (int cb = 0; cb < MINE / 16; ++cb) {
                    const int token = it.token0 + t0 + cb * 16 + (lane & 15);
                    const bool has = adapter_of(a, token) == id;
                    const float f = has ? a.factor[token] : 0.f;
                    const unsigned takes = __ballot_sync(0xffffffffu, has);
                    if (takes == 0u) continue;
                    uint32_t v[16];
                    tmem_load_16(from + (uint32_t)((slice % ACC) * NT + cb * 16), v);
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        const float fx = __shfl_sync(0xffffffffu, f, x);
                        if ((takes >> x) & 1u) total[cb * 16 + x] = fmaf(__uint_as_float(v[x]), fx, total[cb * 16 + x]);
                    }
                }
                leave();
            }
            if (!go) {
#pragma unroll
                for (int x = 0; x < MINE; ++x) total[x] = NAN;
            }
            if (row < a.m) {
                const int count = min(MINE, a.tokens - it.token0 - t0);
                if (job.splits > 1) {
                    float *to = job.partial + ((int64_t)it.split * a.tokens + it.token0 + t0) * a.m + row;
#pragma unroll
                    for (int x = 0; x < MINE; ++x)
                        if (x < count) to[x * a.m] = total[x];
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

// sums of the splits
__global__ void __launch_bounds__(256) linear_join_kernel(const LinearArgs a, const float *__restrict__ partial, int splits) {
    const int64_t count = (int64_t)a.tokens * a.m;
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < count; e += (int64_t)gridDim.x * 256) {
        float sum = partial[e];
        for (int s = 1; s < splits; ++s) sum += partial[s * count + e];
        ((uint16_t *)a.out)[e / a.m * a.out_stride + e % a.m] = (uint16_t)float_to_bits(sum, a.bf16);
    }
}

static bool make_map_codes(CUtensorMap *map, const uint8_t *codes, int64_t rows, int64_t bytes, int64_t pitch) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)bytes, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)pitch};
    const cuuint32_t box[2] = {128, 128};
    const cuuint32_t elem[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t *>(codes), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
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

LinearTcPlan linear_tc_plan(int64_t m, int64_t n, int64_t tokens) {
    LinearTcPlan p;
    p.tile = tokens <= 64 ? 64 : 128;
    p.duo = 0;
    int64_t rows = ceil_div(m, (int64_t)128), columns = ceil_div(tokens, (int64_t)p.tile);
    // 256 x 256 by pairs of CTAs where they fill the GPU as well: four times the work of a 128 x 128 tile in 1.6 times its time
    const int64_t pairs = ceil_div(m, (int64_t)256) * ceil_div(tokens, (int64_t)256);
    if (p.tile == 128 && 8 * ceil_div(pairs, (int64_t)74) <= 5 * ceil_div(rows * columns, (int64_t)148)) {
        p.tile = 256;
        p.duo = 1;
        rows = ceil_div(m, (int64_t)256);
        columns = ceil_div(tokens, (int64_t)256);
    }
    p.row_tiles = (int)rows;
    p.token_tiles = (int)columns;
    const int64_t tiles = rows * columns, quads = ceil_div(n, (int64_t)(KH * LT_CODE_CHUNKS));
    int64_t splits = (p.duo ? 74 : 148) / tiles;
    if (splits > quads / 2) splits = quads / 2;
    p.splits = splits < 1 ? 1 : (int)splits;
    return p;
}

template <bool BF16, int NT, bool DUO>
static int launch_tc(const LinearArgs &a, const LinearTcPlan &p, const int *plan, float *partial, cudaStream_t st) {
    using S = LinearShape<NT, DUO>;
    static PerDeviceOnce configured;
    if (configured.run([&] { return cudaFuncSetAttribute(linear_tc_kernel<BF16, NT, DUO>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::SMEM) == cudaSuccess; }) != G2D_OK) return G2D_ERR_CUDA;
    LinearTcJob job;
    job.a = a;
    job.row_tiles = p.row_tiles;
    job.token_tiles = p.token_tiles;
    job.splits = p.splits;
    job.chunks = (int)ceil_div(a.n, (int64_t)(LT_SUB * KH)) * LT_SUB;
    job.group_chunks = a.group >= a.n ? job.chunks : (int)(a.group / KH);
    job.plan = plan;
    job.partial = partial;
    if (!make_map_16(&job.x, a.x, a.tokens, a.n, S::X_ROWS, BF16, a.x_stride) || !make_map_codes(&job.codes, a.codes, a.m, a.n / 2, a.row_bytes)) return G2D_ERR_CUDA;
    if (a.rank > 0 && (!make_map_16(&job.inner, a.inner, a.tokens, INNER_LD, S::X_ROWS, BF16) || !make_map_up(&job.up, a))) return G2D_ERR_CUDA;
    if (a.rank == 0) job.inner = job.up = job.x;
    const int64_t items = (int64_t)p.row_tiles * p.token_tiles * p.splits;
    const unsigned grid = DUO ? 2 * (unsigned)(items < 74 ? items : 74) : (unsigned)(items < 148 ? items : 148);
    const int launched = launch_dependent(linear_tc_kernel<BF16, NT, DUO>, dim3(grid), S::THREADS, S::SMEM, DUO ? 2 : 1, a.rank > 0, st, job);
    if (launched != G2D_OK || p.splits == 1) return launched;
    const int64_t blocks = ceil_div((int64_t)a.tokens * a.m, (int64_t)256);
    linear_join_kernel<<<(unsigned)(blocks < 148 * 8 ? blocks : 148 * 8), 256, 0, st>>>(a, partial, p.splits);
    return check_launch();
}

int launch_linear_tc(const LinearArgs &a, const LinearTcPlan &p, const int *plan, float *partial, cudaStream_t st) {
    if (p.tile == 64) return a.bf16 ? launch_tc<true, 64, false>(a, p, plan, partial, st) : launch_tc<false, 64, false>(a, p, plan, partial, st);
    if (p.tile == 128) return a.bf16 ? launch_tc<true, 128, false>(a, p, plan, partial, st) : launch_tc<false, 128, false>(a, p, plan, partial, st);
    return a.bf16 ? launch_tc<true, 256, true>(a, p, plan, partial, st) : launch_tc<false, 256, true>(a, p, plan, partial, st);
}

}  // namespace g2d
