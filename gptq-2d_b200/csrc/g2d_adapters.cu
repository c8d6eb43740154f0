// The inner halves of low-rank adapters: h_t = down[i_t] x_t for every token t and its adapter i_t.
//
// The outer halves, up[i_t] h_t, are added inside the product with the packed codes, or where its pieces are joined, while its sums are still in fp32; for the tensor cores h travels as a pair of
// 16-bit values hi + lo in the type of the activations under a power of two per token (22 bits for fp16, 16 for bf16: nothing that a 16-bit result
// shows), the power and the adapter's scaling as one factor per token.
//
// A cluster of eight CTAs shares the n columns; its sums meet through distributed shared memory in a fixed order.
//   * Up to 64 tokens (inner_rows_kernel): a cluster per token.  Each token may have an adapter of its own, so the work is reading 2 rank n bytes per
//     token, by warps that take one or more rows of `down` each.
//   * More (inner_block_kernel): a cluster per 32 tokens and adapter among them, on the tensor cores (m16n8k16).  Tokens of a prompt stand together, so a
//     block has one or two adapters and `down` is read once per 32 tokens (from the L2).  The order of k in a product is free as long as both operands agree: a lane
//     reads 16 bytes of its row of x and of its row of `down` and uses them as the fragments of two products.
// Bound: HBM (x once, each adapter in use once) and, for few tokens, the latency of one launch, which the product's own loads of codes hide: it is
// launched as a dependent launch and waits only before it adds the adapters.
#include "g2d_linear.cuh"
#include "g2d_tc.cuh"

namespace g2d {

constexpr int INNER_SPLIT = 8, INNER_THREADS = 256, INNER_BLOCK = 32;

// 64 threads (two warps) of a token: thread r brings its sum; writes the inner row and the factor.  `shared`: two floats of the two warps.
__device__ __forceinline__ void write_inner(const LinearArgs &a, int token, int id, int r, float h, float *shared) {
    unsigned largest = __float_as_uint(h) & 0x7fffffffu;
    largest = __reduce_max_sync(0xffffffffu, largest);
    if ((threadIdx.x & 31) == 0) shared[(threadIdx.x >> 5) & 1] = __uint_as_float(largest);
    asm volatile("bar.sync %0, 64;" ::"r"(1 + (int)(threadIdx.x >> 6)) : "memory");
    const float top = __uint_as_float(max(__float_as_uint(shared[0]), __float_as_uint(shared[1])));
    const int e = top > 0.f && top < INFINITY ? min(range_exponent(top) + 14, 126) : 0;  // the largest in [1, 2), or in [1, 4) at the end of the range
    const float scaled = h * power_of_two(-e);
    const uint32_t hi = float_to_bits(scaled, a.bf16), lo = float_to_bits(scaled - bits_to_float(hi, a.bf16), a.bf16);
    a.inner[(int64_t)token * INNER_LD + r] = (uint16_t)hi;
    a.inner[(int64_t)token * INNER_LD + RANK_MAX + r] = (uint16_t)(top < INFINITY ? lo : 0u);
    if (r == 0) a.factor[token] = id < 0 ? 0.f : power_of_two(e) * (a.scaling ? a.scaling[id] : 1.f);
}

__device__ __forceinline__ float dot8(const uint4 &p, const uint4 &q, int bf16, float sum) {
    const uint32_t u[4] = {p.x, p.y, p.z, p.w}, v[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        sum = fmaf(bits_to_float(u[e] & 0xffffu, bf16), bits_to_float(v[e] & 0xffffu, bf16), sum);
        sum = fmaf(bits_to_float(u[e] >> 16, bf16), bits_to_float(v[e] >> 16, bf16), sum);
    }
    return sum;
}

// All threads of a CTA: the adapters of the `tile` <= INNER_THREADS tokens from token0 on, in the order in which they appear
__device__ void write_plan(const LinearArgs &a, int *plan, int tile, int token0) {
    __shared__ int ids[INNER_THREADS], counts[INNER_THREADS / 32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int id = (int)threadIdx.x < tile ? adapter_of(a, token0 + threadIdx.x) : -1;
    ids[threadIdx.x] = id;
    __syncthreads();
    bool first = id >= 0;
    for (int k = 0; k < (int)threadIdx.x && first; ++k) first = ids[k] != id;
    const unsigned found = __ballot_sync(0xffffffffu, first);
    if (lane == 0) counts[warp] = __popc(found);
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < INNER_THREADS / 32; ++w) {
        if (w < warp) before += counts[w];
        all += counts[w];
    }
    if (first) plan[1 + before + __popc(found & ((1u << lane) - 1u))] = id;
    if (threadIdx.x == 0) plan[0] = all;
}

__global__ void __launch_bounds__(INNER_THREADS) inner_rows_kernel(const LinearArgs a) {
    __shared__ float part[RANK_MAX], tops[2];
    let_the_next_launch_start();
    const int token = blockIdx.x / INNER_SPLIT, rank = (int)cluster_rank(), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int id = adapter_of(a, token);
    const int64_t chunks = a.n / 8, c0 = rank * chunks / INNER_SPLIT, c1 = (rank + 1) * chunks / INNER_SPLIT;  // eight columns each
    if (threadIdx.x < RANK_MAX) part[threadIdx.x] = 0.f;
    __syncthreads();
    if (id >= 0) {
        const uint4 *const x = reinterpret_cast<const uint4 *>((const uint16_t *)a.x + token * a.x_stride);
        for (int r = warp; r < a.rank; r += INNER_THREADS / 32) {
            const uint4 *const d = reinterpret_cast<const uint4 *>((const uint16_t *)a.down + ((int64_t)id * a.rank + r) * a.n);
            float sum = 0.f;
#pragma unroll 4
            for (int64_t c = c0 + lane; c < c1; c += 32) sum = dot8(d[c], x[c], a.bf16, sum);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane == 0) part[r] = sum;
        }
    }
    __syncthreads();
    cluster_sync();
    if (rank == 0 && threadIdx.x < RANK_MAX) {
        float h = 0.f;
        for (int k = 0; k < INNER_SPLIT; ++k) h += peer_float(&part[threadIdx.x], k);
        write_inner(a, token, id, threadIdx.x, h, tops);
    }
    __syncwarp();
    cluster_sync();  // the others' shared memory is read until here
}

template <bool BF16>
__device__ __forceinline__ void mma_16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// TILES: of eight inner values each
template <bool BF16, int TILES>
__global__ void __launch_bounds__(INNER_THREADS, TILES == 8 ? 1 : 2) inner_block_kernel(const LinearArgs a, int *plan, int tile) {
    constexpr int WARPS = INNER_THREADS / 32;
    __shared__ float part[WARPS / 2][INNER_BLOCK][RANK_MAX + 2];  // two warps at a time
    __shared__ int ids[INNER_BLOCK];
    __shared__ unsigned firsts;
    __shared__ float tops[4][2];
    let_the_next_launch_start();
    const int block = blockIdx.x / INNER_SPLIT, rank = (int)cluster_rank(), warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int token0 = block * INNER_BLOCK;
    if (plan && rank == INNER_SPLIT - 1 && blockIdx.y == 0 && token0 % tile == 0) write_plan(a, plan + (int64_t)(token0 / tile) * (tile + 1), tile, token0);
    if (warp == 0) {  // the block's adapters: each by its first token
        const int id = adapter_of(a, token0 + lane);
        ids[lane] = id;
        const unsigned same = __match_any_sync(0xffffffffu, id);
        const unsigned first = __ballot_sync(0xffffffffu, __ffs(same) - 1 == lane);
        if (lane == 0) firsts = first;
    }
    __syncthreads();
    const int64_t steps = ceil_div(a.n, (int64_t)32), s0 = rank * steps / INNER_SPLIT, s1 = (rank + 1) * steps / INNER_SPLIT;  // 32 columns each; n is a multiple of 32
    int number = 0;  // of the adapter among the block's
    for (unsigned left = firsts; left; left &= left - 1) {
        if (number++ % gridDim.y != blockIdx.y) continue;  // the same for the whole cluster
        const int id = ids[__ffs(left) - 1];
        float acc[2][TILES][4];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < TILES; ++j) acc[i][j][0] = acc[i][j][1] = acc[i][j][2] = acc[i][j][3] = 0.f;
        if (id >= 0) {
            const uint16_t *const d = (const uint16_t *)a.down + (int64_t)id * a.rank * a.n;
            const uint16_t *const x = (const uint16_t *)a.x + 8 * t;
            // a step's loads are under way while the one before is multiplied
            uint4 xr[4], br[TILES];
            const auto fetch = [&](int64_t s, uint4 (&xv)[4], uint4 (&bv)[TILES]) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int token = token0 + 8 * i + g;
                    xv[i] = s < s1 && token < a.tokens ? __ldg(reinterpret_cast<const uint4 *>(x + token * a.x_stride + s * 32)) : make_uint4(0u, 0u, 0u, 0u);
                }
#pragma unroll
                for (int j = 0; j < TILES; ++j)
                    bv[j] = s < s1 && 8 * j < a.rank ? __ldg(reinterpret_cast<const uint4 *>(d + (int64_t)(8 * j + g) * a.n + s * 32 + 8 * t)) : make_uint4(0u, 0u, 0u, 0u);
            };
            fetch(s0 + warp, xr, br);
            for (int64_t s = s0 + warp; s < s1; s += WARPS) {
                uint4 xn[4], bn[TILES];
                fetch(s + WARPS, xn, bn);
#pragma unroll
                for (int j = 0; j < TILES; ++j) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        mma_16<BF16>(acc[i][j], xr[2 * i].x, xr[2 * i + 1].x, xr[2 * i].y, xr[2 * i + 1].y, br[j].x, br[j].y);
                        mma_16<BF16>(acc[i][j], xr[2 * i].z, xr[2 * i + 1].z, xr[2 * i].w, xr[2 * i + 1].w, br[j].z, br[j].w);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) xr[i] = xn[i];
#pragma unroll
                for (int j = 0; j < TILES; ++j) br[j] = bn[j];
            }
        }
        // the warps' sums, in order: the upper four into shared memory, the lower four add theirs
        for (int half = 1; half >= 0; --half) {
            if (warp / (WARPS / 2) == half) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < TILES; ++j)
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            float &to = part[warp % (WARPS / 2)][16 * i + 8 * (x >> 1) + g][8 * j + 2 * t + (x & 1)];
                            to = half ? acc[i][j][x] : to + acc[i][j][x];
                        }
            }
            __syncthreads();
        }
        for (int e = threadIdx.x; e < INNER_BLOCK * RANK_MAX; e += INNER_THREADS) {
            if (e % RANK_MAX >= 8 * TILES) {
                part[0][e / RANK_MAX][e % RANK_MAX] = 0.f;
                continue;
            }
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS / 2; ++w) sum += part[w][e / RANK_MAX][e % RANK_MAX];
            part[0][e / RANK_MAX][e % RANK_MAX] = sum;
        }
        cluster_sync();
        {  // four of the tokens are this CTA's to write
            const int local = rank * (INNER_BLOCK / INNER_SPLIT) + (int)(threadIdx.x >> 6), r = threadIdx.x & 63;
            float h = 0.f;
            for (int k = 0; k < INNER_SPLIT; ++k) h += peer_float(&part[0][local][r], k);
            // by all 64 threads of a token or none
            if (ids[local] == id && token0 + local < a.tokens) write_inner(a, token0 + local, id, r, h, tops[threadIdx.x >> 6]);
        }
        __syncwarp();
        cluster_sync();  // before the next adapter's sums overwrite these
    }
}

int launch_inner(const LinearArgs &a, int *plan, int tile, cudaStream_t st) {
    // Whole calls, 4096 x 4096, 64 tokens of 40 adapters of rank 64: 38.7 us by tokens, 63.1 by blocks; of 32 of rank 16: 25.2, 45.3; of one or four alike (23.6, 23.3; 34.8, 33.7).  Beyond, a
    // prompt's tokens stand together: 2048 of 8 adapters of rank 32 over 28672 columns 53 us by blocks, and one adapter would be read 2048 times by tokens.
    if (a.tokens <= LINEAR_FEW) return launch_dependent(inner_rows_kernel, dim3((unsigned)a.tokens * INNER_SPLIT), INNER_THREADS, 0, INNER_SPLIT, false, st, a);
    const unsigned blocks = (unsigned)ceil_div((int64_t)a.tokens, (int64_t)INNER_BLOCK);
    // several CTAs share a block's adapters only while blocks are few (256 x 28672, 4096 tokens of 32 adapters of rank 64: 270 us with four always, 252)
    const int64_t room = 2 * 148 / ((int64_t)blocks * INNER_SPLIT), most = a.adapters < 4 ? a.adapters + 1 : 4;
    const dim3 grid(blocks * INNER_SPLIT, (unsigned)(room < 1 ? 1 : room < most ? room : most));
    const auto launch = [&](auto kernel) { return launch_dependent(kernel, grid, INNER_THREADS, 0, INNER_SPLIT, false, st, a, plan, tile); };
    if (a.rank <= 16) return a.bf16 ? launch(inner_block_kernel<true, 2>) : launch(inner_block_kernel<false, 2>);
    if (a.rank <= 32) return a.bf16 ? launch(inner_block_kernel<true, 4>) : launch(inner_block_kernel<false, 4>);
    return a.bf16 ? launch(inner_block_kernel<true, 8>) : launch(inner_block_kernel<false, 8>);
}

}  // namespace g2d
