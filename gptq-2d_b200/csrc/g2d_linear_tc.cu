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

constexpr int LT_THREADS = 512, LT_CODE_BYTES = 128 * 128, LT_W_BYTES = 128 * 128, LT_CODE_CHUNKS = 4, LT_SLICE = 8;

template <int NT>
struct LinearShape {
    static constexpr int X_BYTES = NT * KH * 2, STAGE = X_BYTES + LT_W_BYTES;
    static constexpr int CODE_STAGES = NT == 256 ? 2 : 3, STAGES = NT == 256 ? 4 : NT == 128 ? 5 : 7;
    static constexpr int CODERS = NT >= 128 ? 4 : 8, READERS = NT >= 128 ? 8 : 4;  // warps
    static constexpr int MINE = NT * 4 / READERS;                               // columns of a reading warp
    static constexpr size_t SMEM = (size_t)STAGES * STAGE + CODE_STAGES * LT_CODE_BYTES + 1024;
};

struct LinearTcJob {
    CUtensorMap x, inner, codes;
    LinearArgs a;
    int row_tiles, token_tiles, splits, chunks, group_chunks;
    const int *plan;  // per tile of tokens: how many adapters, and which
    float *partial;   // [splits][tokens][m], where splits > 1
};

struct LinearItem {
    int row0, token0, token_tile, split, c0, c1;
};
__device__ __forceinline__ bool linear_item(const LinearTcJob &job, int nt, int number, LinearItem &it) {
    const int64_t at = blockIdx.x + (int64_t)number * gridDim.x;
    if (at >= (int64_t)job.row_tiles * job.token_tiles * job.splits) return false;
    it.split = (int)(at % job.splits);
    const int64_t tile = at / job.splits;
    it.token_tile = (int)(tile / job.row_tiles);
    it.row0 = (int)(tile % job.row_tiles) * 128;
    it.token0 = it.token_tile * nt;
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

template <int NT>
struct LinearBarriers {
    using S = LinearShape<NT>;
    uint64_t x_full[S::STAGES], w_full[S::STAGES], empty[S::STAGES], code_full[S::CODE_STAGES], code_empty[S::CODE_STAGES], acc_full[2], acc_empty[2], drained;
    uint32_t tmem;
    int failed;
};

template <bool BF16, int NT>
__global__ void __launch_bounds__(LT_THREADS, 1) linear_tc_kernel(const __grid_constant__ LinearTcJob job) {
    using S = LinearShape<NT>;
    extern __shared__ unsigned char linear_tc_smem[];
    __shared__ __align__(8) LinearBarriers<NT> bar;
    const LinearArgs &a = job.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = (smem_u32(linear_tc_smem) + 1023u) & ~1023u, codes_base = base + S::STAGES * S::STAGE;
    constexpr uint32_t COLS = 2 * NT;
    const auto wait = [&](uint64_t *b, uint32_t parity, unsigned nap) {
        if (mbar_wait(b, parity, nap, a.wait_cycles)) return true;
        bar.failed = 1;
        return false;
    };
    if (threadIdx.x == 0) {
        for (int s = 0; s < S::STAGES; ++s) {
            mbar_init(&bar.x_full[s], 1);
            mbar_init(&bar.w_full[s], S::CODERS);
            mbar_init(&bar.empty[s], 1);
        }
        for (int s = 0; s < S::CODE_STAGES; ++s) {
            mbar_init(&bar.code_full[s], 1);
            mbar_init(&bar.code_empty[s], S::CODERS);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&bar.acc_full[s], 1);
            mbar_init(&bar.acc_empty[s], S::READERS);
        }
        mbar_init(&bar.drained, 1);
        bar.failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc<false>(&bar.tmem, COLS);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = bar.tmem;
    // how many adapters an item has to add: those of its tile, by the first split.  The launch before writes them.
    const auto adapters_in = [&](const LinearItem &it) {
        if (a.rank == 0 || it.split != 0) return 0;
        after_the_launch_before();
        return job.plan[(int64_t)it.token_tile * (NT + 1)];
    };
    const auto adapter_at = [&](const LinearItem &it, int j) { return job.plan[(int64_t)it.token_tile * (NT + 1) + 1 + j]; };
    const int first_coder = 4, first_reader = 4 + S::CODERS;

    if (warp < 4) {
        if (NT == 256) asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        if (warp == 0 && lane == 0) {  // x
            LinearItem it;
            int c = 0;
            const auto bring = [&](const CUtensorMap *map, int column, int token) {
                const int stage = c % S::STAGES, round = c / S::STAGES;
                if (bar.failed || (round > 0 && !wait(&bar.empty[stage], (round - 1) & 1, 32))) return false;
                mbar_expect_tx(&bar.x_full[stage], S::X_BYTES);
                tma_load_2d(base + stage * S::STAGE, map, column, token, &bar.x_full[stage]);
                ++c;
                return true;
            };
            bool go = true;
            for (int i = 0; go && linear_item(job, NT, i, it); ++i) {
                for (int ch = it.c0; go && ch < it.c1; ++ch) go = bring(&job.x, ch * KH, it.token0);
                const int extra = go ? 2 * adapters_in(it) : 0;
                for (int e = 0; go && e < extra; ++e) go = bring(&job.inner, (e & 1) * RANK_MAX, it.token0);
            }
            for (int k = max(c - S::STAGES, 0); k < c; ++k) mbar_wait(&bar.x_full[k % S::STAGES], (k / S::STAGES) & 1);  // landed before the memory is given back
        } else if (warp == 2 && lane == 0) {  // codes
            LinearItem it;
            int c = 0;
            bool go = true;
            for (int i = 0; go && linear_item(job, NT, i, it); ++i) {
                for (int ch = it.c0; ch < it.c1; ch += LT_CODE_CHUNKS, ++c) {
                    const int stage = c % S::CODE_STAGES, round = c / S::CODE_STAGES;
                    if (bar.failed || (round > 0 && !wait(&bar.code_empty[stage], (round - 1) & 1, 32))) { go = false; break; }
                    mbar_expect_tx(&bar.code_full[stage], LT_CODE_BYTES);
                    tma_load_2d(codes_base + stage * LT_CODE_BYTES, &job.codes, ch * (KH / 2), it.row0, &bar.code_full[stage]);
                }
            }
            for (int k = max(c - S::CODE_STAGES, 0); k < c; ++k) mbar_wait(&bar.code_full[k % S::CODE_STAGES], (k / S::CODE_STAGES) & 1);
        } else if (warp == 1 && lane == 0) {  // products
            constexpr uint32_t DESC = idesc_16(NT, BF16 ? 1 : 0);
            LinearItem it;
            int c = 0, slice = 0;
            const auto product = [&](bool opens, bool closes, int steps) {
                const int stage = c % S::STAGES, round = c / S::STAGES, buf = slice & 1;
                if (bar.failed || (opens && slice >= 2 && !wait(&bar.acc_empty[buf], ((slice >> 1) - 1) & 1, 20))) return false;
                if (!wait(&bar.w_full[stage], round & 1, 20) || !wait(&bar.x_full[stage], round & 1, 20)) return false;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t d = tmem + (uint32_t)(buf * NT), x = base + stage * S::STAGE, w = x + S::X_BYTES;
                for (int ks = 0; ks < steps; ++ks) umma_16(d, umma_desc(w + ks * 32), umma_desc(x + ks * 32), DESC, (opens && ks == 0) ? 0u : 1u);
                umma_commit(&bar.empty[stage]);
                if (closes) {
                    umma_commit(&bar.acc_full[buf]);
                    ++slice;
                }
                ++c;
                return true;
            };
            bool go = true;
            for (int i = 0; go && linear_item(job, NT, i, it); ++i) {
                bool opens = true;
                for (int ch = it.c0; go && ch < it.c1; ++ch) {
                    const bool closes = slice_ends(job, ch, it.c1 - 1);
                    go = product(opens, closes, KH / 16);
                    opens = closes;
                }
                const int extra = go ? adapters_in(it) : 0;
                for (int e = 0; go && e < 2 * extra; ++e) go = product(!(e & 1), e & 1, (a.rank + 15) / 16);
            }
            if (bar.failed) {  // every product that was issued completes, or has its time to, before what it reads and writes is given back
                umma_commit(&bar.drained);
                mbar_wait(&bar.drained, 0);
            } else if (slice > 0) {
                mbar_wait(&bar.acc_full[(slice - 1) & 1], ((slice - 1) >> 1) & 1);
            }
        }
        __syncwarp();
    } else if (warp < first_reader) {
        if (NT == 256) asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
        // ---- operands: a thread has a row and, with eight warps, half of its columns ----
        constexpr int PARTS = S::CODERS / 4, WORDS = 8 / PARTS;
        const int id = threadIdx.x - 32 * first_coder, row = id & 127, part = id >> 7;
        LinearItem it;
        int c = 0, cc = 0;
        bool go = true;
        const auto ready = [&](int stage) {  // all of the warp's values are written
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.w_full[stage]);
        };
        for (int i = 0; go && linear_item(job, NT, i, it); ++i) {
            const float *const zero = a.zero + min((int64_t)it.row0 + row, a.m - 1) * a.zero_row;
            const auto shift_of = [&](int ch) { return 8.f + a.qmin - __ldg(zero + (int64_t)(min(ch, job.chunks - 1) / job.group_chunks) * a.zero_group); };
            float next_shift = shift_of(it.c0);
            uint32_t shift = 0u;
            bool shifted = false;
            for (int ch = it.c0; ch < it.c1; ++ch, ++c) {
                if (ch == it.c0 || ch % job.group_chunks == 0) {
                    const uint32_t bits = float_to_bits(next_shift, BF16);
                    shift = bits | (bits << 16);
                    shifted = __any_sync(0xffffffffu, next_shift != 0.f);
                    next_shift = shift_of((ch / job.group_chunks + 1) * job.group_chunks);
                }
                const int stage = c % S::STAGES, round = c / S::STAGES, code_stage = cc % S::CODE_STAGES;
                if (ch % LT_CODE_CHUNKS == 0) go = wait(&bar.code_full[code_stage], (cc / S::CODE_STAGES) & 1, 20);
                uint4 raw[WORDS / 4];
                const uint32_t from = codes_base + code_stage * LT_CODE_BYTES + row * 128;
#pragma unroll
                for (int w = 0; w < WORDS / 4; ++w) raw[w] = load_16(from + ((((ch % LT_CODE_CHUNKS) * 2 + part * (WORDS / 4) + w) ^ (row & 7)) << 4));
                if (round > 0) go = go && wait(&bar.empty[stage], (round - 1) & 1, 20);
                go = __all_sync(0xffffffffu, go && !bar.failed);
                if (!go) break;
                const uint32_t to = base + stage * S::STAGE + S::X_BYTES + row * 128;
#pragma unroll
                for (int w = 0; w < WORDS; ++w) {
                    const uint32_t word = (w & 3) == 0 ? raw[w / 4].x : (w & 3) == 1 ? raw[w / 4].y : (w & 3) == 2 ? raw[w / 4].z : raw[w / 4].w;
                    uint4 v = decoded<BF16>(word);
                    if (shifted) v = make_uint4(add2<BF16>(v.x, shift), add2<BF16>(v.y, shift), add2<BF16>(v.z, shift), add2<BF16>(v.w, shift));
                    store_16(to + (((part * WORDS + w) ^ (row & 7)) << 4), v);
                }
                ready(stage);
                if (ch % LT_CODE_CHUNKS == LT_CODE_CHUNKS - 1 || ch == it.c1 - 1) {
                    if (lane == 0) mbar_arrive(&bar.code_empty[code_stage]);  // behind the warp's barrier: all lanes have read
                    ++cc;
                }
            }
            const int extra = go ? adapters_in(it) : 0;
            for (int e = 0; go && e < 2 * extra; ++e, ++c) {  // rows of `up`, twice: against the upper and the lower parts of the inner values
                const int stage = c % S::STAGES, round = c / S::STAGES;
                const uint4 *const up = reinterpret_cast<const uint4 *>((const uint16_t *)a.up + ((int64_t)adapter_at(it, e >> 1) * a.m + it.row0 + row) * a.rank);
                uint4 v[WORDS];
#pragma unroll
                for (int w = 0; w < WORDS; ++w) {
                    const int at = part * WORDS + w;
                    v[w] = 8 * at < a.rank && it.row0 + row < a.m ? __ldg(up + at) : make_uint4(0u, 0u, 0u, 0u);
                }
                if (round > 0) go = wait(&bar.empty[stage], (round - 1) & 1, 20);
                go = __all_sync(0xffffffffu, go && !bar.failed);
                if (!go) break;
                const uint32_t to = base + stage * S::STAGE + S::X_BYTES + row * 128;
#pragma unroll
                for (int w = 0; w < WORDS; ++w) store_16(to + (((part * WORDS + w) ^ (row & 7)) << 4), v[w]);
                ready(stage);
            }
        }
    } else {
        if (NT == 256) asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
        // ---- results: a thread has a row and MINE tokens ----
        constexpr int MINE = S::MINE;
        const int q = warp & 3, t0 = ((warp - first_reader) >> 2) * MINE;
        LinearItem it;
        int slice = 0;
        bool go = true;
        for (int i = 0; linear_item(job, NT, i, it); ++i) {
            const int64_t row = (int64_t)it.row0 + q * 32 + lane;
            const float *const scale = a.scale + min(row, a.m - 1) * a.scale_row;
            float total[MINE];
#pragma unroll
            for (int x = 0; x < MINE; ++x) total[x] = 0.f;
            const auto arrived = [&] {
                const bool ok = go && wait(&bar.acc_full[slice & 1], (slice >> 1) & 1, 64);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                go = __all_sync(0xffffffffu, ok && !bar.failed);
                return go;
            };
            const auto leave = [&] {
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar.acc_empty[slice & 1]);
                ++slice;
            };
            const uint32_t from = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)t0;
            for (int ch = it.c0; go && ch < it.c1; ++ch) {
                if (!slice_ends(job, ch, it.c1 - 1)) continue;
                const float factor = __ldg(scale + (int64_t)(ch / job.group_chunks) * a.scale_group);
                if (!arrived()) break;
#pragma unroll
                for (int cb = 0; cb < MINE / 16; ++cb) {
                    uint32_t v[16];
                    tmem_load_16(from + (uint32_t)((slice & 1) * NT + cb * 16), v);
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
                    tmem_load_16(from + (uint32_t)((slice & 1) * NT + cb * 16), v);
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
    if (warp == 1) tmem_free<false>(tmem, COLS);
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

LinearTcPlan linear_tc_plan(int64_t m, int64_t n, int64_t tokens) {
    LinearTcPlan p;
    p.tile = tokens <= 64 ? 64 : tokens <= 128 ? 128 : 256;
    p.row_tiles = (int)ceil_div(m, (int64_t)128);
    p.token_tiles = (int)ceil_div(tokens, (int64_t)p.tile);
    const int64_t tiles = (int64_t)p.row_tiles * p.token_tiles, quads = ceil_div(n, (int64_t)(KH * LT_CODE_CHUNKS));
    int64_t splits = 148 / tiles;
    if (splits > quads / 2) splits = quads / 2;
    p.splits = splits < 1 ? 1 : (int)splits;
    return p;
}

template <bool BF16, int NT>
static int launch_tc(const LinearArgs &a, const LinearTcPlan &p, const int *plan, float *partial, cudaStream_t st) {
    static PerDeviceOnce configured;
    constexpr size_t smem = LinearShape<NT>::SMEM;
    if (configured.run([&] { return cudaFuncSetAttribute(linear_tc_kernel<BF16, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) == cudaSuccess; }) != G2D_OK) return G2D_ERR_CUDA;
    LinearTcJob job;
    job.a = a;
    job.row_tiles = p.row_tiles;
    job.token_tiles = p.token_tiles;
    job.splits = p.splits;
    job.chunks = (int)ceil_div(a.n, (int64_t)KH);
    job.group_chunks = a.group >= a.n ? job.chunks : (int)(a.group / KH);
    job.plan = plan;
    job.partial = partial;
    if (!make_map_16(&job.x, a.x, a.tokens, a.n, NT, BF16, a.x_stride) || !make_map_codes(&job.codes, a.codes, a.m, a.n / 2, a.row_bytes)) return G2D_ERR_CUDA;
    if (a.rank > 0 && !make_map_16(&job.inner, a.inner, a.tokens, INNER_LD, NT, BF16)) return G2D_ERR_CUDA;
    if (a.rank == 0) job.inner = job.x;
    const int64_t items = (int64_t)p.row_tiles * p.token_tiles * p.splits;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3((unsigned)(items < 148 ? items : 148));
    config.blockDim = dim3(LT_THREADS);
    config.dynamicSmemBytes = smem;
    config.stream = st;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute;
    config.numAttrs = a.rank > 0 ? 1 : 0;
    if (cudaLaunchKernelEx(&config, linear_tc_kernel<BF16, NT>, job) != cudaSuccess) return G2D_ERR_CUDA;
    if (check_launch() != G2D_OK) return G2D_ERR_CUDA;
    if (p.splits == 1) return G2D_OK;
    const int64_t blocks = ceil_div((int64_t)a.tokens * a.m, (int64_t)256);
    linear_join_kernel<<<(unsigned)(blocks < 148 * 8 ? blocks : 148 * 8), 256, 0, st>>>(a, partial, p.splits);
    return check_launch();
}

int launch_linear_tc(const LinearArgs &a, const LinearTcPlan &p, const int *plan, float *partial, cudaStream_t st) {
    if (p.tile == 64) return a.bf16 ? launch_tc<true, 64>(a, p, plan, partial, st) : launch_tc<false, 64>(a, p, plan, partial, st);
    if (p.tile == 128) return a.bf16 ? launch_tc<true, 128>(a, p, plan, partial, st) : launch_tc<false, 128>(a, p, plan, partial, st);
    return a.bf16 ? launch_tc<true, 256>(a, p, plan, partial, st) : launch_tc<false, 256>(a, p, plan, partial, st);
}

}  // namespace g2d
