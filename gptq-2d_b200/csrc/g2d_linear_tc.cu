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

constexpr int LT_THREADS = 512, LT_CODE_BYTES = 128 * 128, LT_W_BYTES = 128 * 128, LT_SUB = 2, LT_CODE_CHUNKS = 4, LT_SLICE = 8;

// DUO: a pair of CTAs on 256 rows x NT tokens (cta_group::2), each with its rows of W and half of the tokens' rows of x
template <int NT, bool DUO>
struct LinearShape {
    static constexpr int X_ROWS = DUO ? NT / 2 : NT, X_BYTES = X_ROWS * KH * 2, STAGE = LT_SUB * (X_BYTES + LT_W_BYTES);  // two chunks of 64 columns
    static constexpr int CODE_STAGES = 2, STAGES = NT == 64 ? 4 : 3;
    static constexpr int CODERS = NT >= 128 ? 4 : 8, READERS = NT >= 128 ? 8 : 4;  // warps
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
// The eight codes of a word, in order, as pairs of code - 8: the bits of a code under the exponent of 1024 (fp16) or 128 (bf16), and that minus 1032 or 136
template <bool BF16>
__device__ __forceinline__ uint4 decoded(uint32_t w) {
    constexpr uint32_t MAGIC = BF16 ? 0x43004300u : 0x64006400u, LESS = BF16 ? 0xc308c308u : 0xe408e408u;
    const uint32_t w4 = w >> 4;
    uint4 r;
    r.x = add2<BF16>((__byte_perm(w, w4, 0x4400) & 0x000f000fu) | MAGIC, LESS);
    r.y = add2<BF16>((__byte_perm(w, w4, 0x5511) & 0x000f000fu) | MAGIC, LESS);
    r.z = add2<BF16>((__byte_perm(w, w4, 0x6622) & 0x000f000fu) | MAGIC, LESS);
    r.w = add2<BF16>((__byte_perm(w, w4, 0x7733) & 0x000f000fu) | MAGIC, LESS);
    return r;
}
__device__ __forceinline__ void store_16(uint32_t at, const uint4 &v) { asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory"); }
__device__ __forceinline__ uint4 load_16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}

template <int NT, bool DUO>
struct LinearBarriers {
    using S = LinearShape<NT, DUO>;
    uint64_t x_full[S::STAGES], w_full[S::STAGES], empty[S::STAGES], code_full[S::CODE_STAGES], code_empty[S::CODE_STAGES], acc_full[S::ACCUMULATORS], acc_empty[S::ACCUMULATORS], drained;
    uint32_t tmem;
    int failed;
};

template <bool BF16, int NT, bool DUO>
__global__ void __launch_bounds__(LT_THREADS, 1) linear_tc_kernel(const __grid_constant__ LinearTcJob job) {
    using S = LinearShape<NT, DUO>;
    constexpr int CTAS = DUO ? 2 : 1, ACC = S::ACCUMULATORS;
    constexpr bool HEAVY = S::MINE > 64;  // the readers need more than 128 registers
    extern __shared__ unsigned char linear_tc_smem[];
    __shared__ __align__(8) LinearBarriers<NT, DUO> bar;
    const LinearArgs &a = job.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = DUO ? (int)cluster_rank() : 0;
    const uint32_t base = (smem_u32(linear_tc_smem) + 1023u) & ~1023u, codes_base = base + S::STAGES * S::STAGE;
    const auto await = [](uint64_t *b, uint32_t parity, unsigned nap, long long cycles) { return DUO ? mbar_wait_cluster(b, parity, nap, cycles) : mbar_wait(b, parity, nap, cycles); };
    const auto wait = [&](uint64_t *b, uint32_t parity, unsigned nap) {
        if (await(b, parity, nap, a.wait_cycles)) return true;
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
            mbar_init(&bar.w_full[s], CTAS * S::CODERS);
            mbar_init(&bar.empty[s], 1);
        }
        for (int s = 0; s < S::CODE_STAGES; ++s) {
            mbar_init(&bar.code_full[s], 1);
            mbar_init(&bar.code_empty[s], S::CODERS);
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
    const int first_coder = 4, first_reader = 4 + S::CODERS;

    if (warp < 4) {
        if (HEAVY) asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
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
                for (int k = max(c - S::STAGES, 0); k < c; ++k) await(&bar.x_full[k % S::STAGES], (k / S::STAGES) & 1, 32, WAIT_CYCLES);
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
        } else if (warp == 1 && lane == 0 && rank == 0) {  // products
            constexpr uint32_t DESC = idesc_16(NT, BF16 ? 1 : 0, DUO ? 2 * MT : MT);
            LinearItem it;
            int c = 0, slice = 0;
            const auto ready = [&] {
                const int stage = c % S::STAGES, round = c / S::STAGES;
                if (bar.failed || !wait(&bar.w_full[stage], round & 1, 20) || !wait(&bar.x_full[stage], round & 1, 20)) return false;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                return true;
            };
            const auto product = [&](int w, int x, bool opens, bool closes, int steps) {  // chunks w and x of the stage
                const int buf = slice % ACC;
                if (opens && slice >= ACC) {
                    if (!wait(&bar.acc_empty[buf], (slice / ACC - 1) & 1, 20)) return false;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                }
                const uint32_t d = tmem + (uint32_t)(buf * NT), at = base + (c % S::STAGES) * S::STAGE, xs = at + x * S::X_BYTES, ws = at + LT_SUB * S::X_BYTES + w * LT_W_BYTES;
                for (int ks = 0; ks < steps; ++ks) mma<DUO>(d, ws + ks * 32, xs + ks * 32, DESC, (opens && ks == 0) ? 0u : 1u);
                if (closes) {
                    commit<DUO>(&bar.acc_full[buf]);
                    ++slice;
                }
                return true;
            };
            bool go = true;
            for (int i = 0; go && item(i, it); ++i) {
                bool opens = true;
                for (int ch = it.c0; go && ch < it.c1; ch += LT_SUB) {
                    go = ready();
                    for (int s = 0; go && s < LT_SUB; ++s) {
                        const bool closes = slice_ends(job, ch + s, it.c1 - 1);
                        go = product(s, s, opens, closes, KH / 16);
                        opens = closes;
                    }
                    commit<DUO>(&bar.empty[c++ % S::STAGES]);
                }
                const int extra = go ? adapters_in(it) : 0;
                for (int e = 0; go && e < extra; ++e) {
                    go = ready() && product(0, 0, true, false, (a.rank + 15) / 16) && product(0, 1, false, true, (a.rank + 15) / 16);
                    commit<DUO>(&bar.empty[c++ % S::STAGES]);
                }
            }
            if (bar.failed) {  // every product that was issued completes, or has its time to, before what it reads and writes is given back
                commit<DUO>(&bar.drained);
                await(&bar.drained, 0, 32, WAIT_CYCLES);
            } else {
                for (int k = max(slice - ACC, 0); k < slice; ++k) await(&bar.acc_full[k % ACC], (k / ACC) & 1, 32, WAIT_CYCLES);
            }
        }
        __syncwarp();
    } else if (warp < first_reader) {
        if (HEAVY) asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
        // ---- operands: a thread has a row and, with four warps, both chunks of a stage, else one ----
        constexpr int EACH = LT_SUB * 4 / S::CODERS;  // chunks
        const int id = threadIdx.x - 32 * first_coder, row = id & 127, first = (id >> 7) * EACH;
        LinearItem it;
        int c = 0, cc = 0;
        bool go = true;
        const auto free_stage = [&] {
            const int stage = c % S::STAGES, round = c / S::STAGES;
            if (round > 0) go = go && wait(&bar.empty[stage], (round - 1) & 1, 20);
            go = __all_sync(0xffffffffu, go && !bar.failed);
            return go;
        };
        for (int i = 0; go && item(i, it); ++i) {
            const float *const zero = a.zero + min((int64_t)it.row0 + row, a.m - 1) * a.zero_row;
            const auto shift_of = [&](int ch) { return 8.f + a.qmin - __ldg(zero + (int64_t)(min(ch, job.chunks - 1) / job.group_chunks) * a.zero_group); };
            float next_shift = shift_of(it.c0 + first);
            int group_end = -1;  // first chunk past the group whose shift is at hand
            uint32_t shift = 0u;
            bool shifted = false;
            for (int ch = it.c0; ch < it.c1; ch += LT_SUB, ++c) {
                const int code_stage = cc % S::CODE_STAGES;
                if (ch % LT_CODE_CHUNKS == 0) go = wait(&bar.code_full[code_stage], (cc / S::CODE_STAGES) & 1, 20);
                uint4 raw[EACH][2];
                const uint32_t from = codes_base + code_stage * LT_CODE_BYTES + row * 128;
#pragma unroll
                for (int s = 0; s < EACH; ++s)
#pragma unroll
                    for (int w = 0; w < 2; ++w) raw[s][w] = load_16(from + ((((ch % LT_CODE_CHUNKS + first + s) * 2 + w) ^ (row & 7)) << 4));
                if (!free_stage()) break;
                const uint32_t to = base + (c % S::STAGES) * S::STAGE + LT_SUB * S::X_BYTES + row * 128;
#pragma unroll
                for (int s = 0; s < EACH; ++s) {
                    if (ch + first + s >= group_end) {
                        const uint32_t bits = float_to_bits(next_shift, BF16);
                        shift = bits | (bits << 16);
                        shifted = __any_sync(0xffffffffu, next_shift != 0.f);
                        group_end = ((ch + first + s) / job.group_chunks + 1) * job.group_chunks;
                        next_shift = shift_of(S::CODERS == 8 && job.group_chunks == 1 ? group_end + 1 : group_end);  // one of two chunks: every other group
                    }
#pragma unroll
                    for (int w = 0; w < 8; ++w) {
                        const uint4 &r = raw[s][w >> 2];
                        uint4 v = decoded<BF16>((w & 3) == 0 ? r.x : (w & 3) == 1 ? r.y : (w & 3) == 2 ? r.z : r.w);
                        if (shifted) v = make_uint4(add2<BF16>(v.x, shift), add2<BF16>(v.y, shift), add2<BF16>(v.z, shift), add2<BF16>(v.w, shift));
                        store_16(to + (first + s) * LT_W_BYTES + ((w ^ (row & 7)) << 4), v);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) arrive(&bar.w_full[c % S::STAGES]);
                if (ch % LT_CODE_CHUNKS + LT_SUB >= LT_CODE_CHUNKS || ch + LT_SUB >= it.c1) {
                    if (lane == 0) mbar_arrive(&bar.code_empty[code_stage]);  // behind the warp's barrier: all lanes have read
                    ++cc;
                }
            }
            const int extra = go ? adapters_in(it) : 0;
            for (int e = 0; go && e < extra; ++e, ++c) {  // rows of `up`, which the TMA brings: the stage is free for them
                if (!free_stage()) break;
                if (lane == 0) arrive(&bar.w_full[c % S::STAGES]);
            }
        }
    } else {
        if (HEAVY) asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
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
            for (int ch = it.c0; go && ch < it.c1; ++ch) {
                if (!slice_ends(job, ch, it.c1 - 1)) continue;
                const float factor = factor_of(ch);
                if (!arrived()) break;
#pragma unroll
                for (int cb = 0; cb < MINE / 16; ++cb) {
                    uint32_t v[16];
                    tmem_load_16(from + (uint32_t)((slice % ACC) * NT + cb * 16), v);
#pragma unroll
                    for (int x = 0; x < 16; ++x) total[cb * 16 + x] = fmaf(__uint_as_float(v[x]), factor, total[cb * 16 + x]);
                }
                leave();
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
    const int launched = launch_dependent(linear_tc_kernel<BF16, NT, DUO>, dim3(grid), LT_THREADS, S::SMEM, DUO ? 2 : 1, a.rank > 0, st, job);
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
