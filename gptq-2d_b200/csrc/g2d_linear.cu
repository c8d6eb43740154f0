// y = x W^T for a matrix W held as packed 4-bit codes, few tokens:  y[t, o] = sum_g s[o, g] sum_{k in g} (c[o, k] + qmin - z[o, g]) x[t, k]  (+ adapters).
//
// The rows of W are the rows of A of m16n8k16 products, the tokens its columns.  A code goes to the tensor cores as it lies in its word: the bits of c in the lowest
// (or next) four bits of a 16-bit float are c (or 16 c) times the smallest subnormal, exactly, so eight codes cost a shift and four ANDs; the products
// with the 16 c go to sums of their own.  fp16 activations are taken as they are; bf16 ones times 2^56, for codes of c 2^-133, or, where
// a token's largest lies outside 2^-12 .. 2^64, times a power of two of the token's own: x is brought once more
// then (8192 x 8192, 16 tokens: 20.2 us, then 28.2; looking for such tokens costs 2 %).
// What the codes' origin and zero point add is (qmin - z) sum x, from sums of x over each group that the CTA forms while it brings x to shared memory.
// A lane reads 16 bytes of codes (32 columns) of two rows, four times ahead; x lies in shared memory in the order in which such
// words hold their columns, so a fragment of it is one 16-byte load.  With groups of an odd number of 64 columns a lane reads 8 bytes at a time.
//
// A CTA has 128 rows, each of its eight warps 16; a cluster of CTAs splits the columns, and sums meet through shared memory in a fixed order.  (64 rows and the
// columns halved between warps: 1024 x 4096, 1 token 5.5 us where this takes 5.2; 8192 x 8192, 16 tokens 28.6, 20.2.)
// Bound: HBM (half a byte per weight) and, from about 12 tokens on, the rate of these products (16 cycles each for a quarter of an SM); for small matrices the latency of one chain
// of loads.  Without adapters 8192 x 8192 takes 16.0 us with 1 token (2.1 TB/s) and 20.2 with 16; 28672 x 4096 25.8 (2.3 TB/s); 1024 x 4096, 1 token, an adapter of rank 16 6.8.
#include "g2d_linear.cuh"
#include "g2d_tc.cuh"

namespace g2d {

constexpr int ROWS_WARPS = 8, ROWS_THREADS = 32 * ROWS_WARPS;

// bf16: the power of two that brings a token's largest activation (its bits) to 2^100 .. 2^101, so that 2^93 below it nothing is lost to the codes' 2^-133
__device__ __forceinline__ int token_exponent(unsigned top) { return top == 0u || top >= 0x7f80u ? 56 : 227 - (int)(top >> 7); }  // -27 .. 227
__device__ __forceinline__ bool token_is_far(unsigned top) { return top != 0u && (top < 0x3980u || (top >= 0x5f80u && top < 0x7f80u)); }  // outside 2^-12 .. 2^64, and finite
__device__ __forceinline__ uint32_t bf16_pair_times(uint32_t pair, uint32_t factors) {
    const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162 *>(&pair), *reinterpret_cast<const __nv_bfloat162 *>(&factors));
    return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t bf16_pair_of_powers(int e) { return (uint32_t)(e + 127) * 0x00800080u; }  // of 2^e twice

template <bool BF16>
__device__ __forceinline__ void mma_codes(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// KB: columns of a block, 128 or 64; NT: tiles of eight tokens
template <bool BF16, int NT, int KB>
__global__ void __launch_bounds__(ROWS_THREADS, 2) linear_rows_kernel(const LinearArgs a) {
    constexpr int WORDS = KB / 32, ROWS = 16 * ROWS_WARPS, TOKENS = 8 * NT, CHUNKS = KB / 8, AHEAD = 4;
    extern __shared__ __align__(16) unsigned char linear_smem_raw[];
    __shared__ unsigned tops[TOKENS];  // bf16: the bits of each token's largest magnitude in this CTA's columns
    const int splits = (int)gridDim.x, rank = (int)blockIdx.x;  // a cluster has all CTAs along x
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int64_t row0 = (int64_t)blockIdx.y * ROWS;
    const int token0 = blockIdx.z * TOKENS;
    const int64_t blocks = ceil_div(a.n, (int64_t)KB), b_first = rank * blocks / splits, b_last = (rank + 1) * blocks / splits;
    const int mine = (int)(b_last - b_first), most = (int)ceil_div(blocks, (int64_t)splits);  // the same layout in every CTA of the cluster
    uint4 *const xs = reinterpret_cast<uint4 *>(linear_smem_raw);            // [block][word][tile of tokens][lane]
    float *const sums = reinterpret_cast<float *>(xs + (int64_t)most * WORDS * NT * 32);  // [block][token]
    float *const part = sums + most * TOKENS;                                // [token][row]

    // the first codes are on their way while x is brought
    uint32_t code[AHEAD][2][WORDS];
    const int64_t row_lo = row0 + warp * 16 + g, row_hi = row_lo + 8;
    const auto fetch = [&](int slot, int block) {
        const int64_t k = (b_first + block) * KB + t * (KB / 4);
        const bool inside = block < mine && k < a.n;  // n is a multiple of 32: a lane's columns are all inside or, 64 of 128 (or 32 of 64), checked by word
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t row = h ? row_hi : row_lo;
            const uint8_t *const p = a.codes + row * a.row_bytes + (k >> 1);
#pragma unroll
            for (int w = 0; w < WORDS; ++w) code[slot][h][w] = 0u;
            if (inside && row < a.m) {
                if constexpr (WORDS == 4) {
                    const uint4 v = __ldg(reinterpret_cast<const uint4 *>(p));
                    code[slot][h][0] = v.x; code[slot][h][1] = v.y; code[slot][h][2] = v.z; code[slot][h][3] = v.w;
                } else {
                    const uint2 v = __ldg(reinterpret_cast<const uint2 *>(p));
                    code[slot][h][0] = v.x; code[slot][h][1] = v.y;
                }
            }
        }
    };
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) fetch(s, s);

    // ---- x: a thread takes eight columns of a token; the CHUNKS threads of a block and token stand together and add up its sum ----
    constexpr int TOGETHER = 4;  // loads of a thread on their way at once
    const auto piece = [&](int e, int &chunk, int &token, int &block) -> uint4 {  // number e of the share's pieces of eight columns
        chunk = e % CHUNKS;
        token = e / CHUNKS % TOKENS;
        block = e / (CHUNKS * TOKENS);
        const int64_t k = (b_first + block) * KB + 8 * chunk;
        return block < mine && k < a.n && token0 + token < a.tokens ? __ldg(reinterpret_cast<const uint4 *>((const uint16_t *)a.x + (int64_t)(token0 + token) * a.x_stride + k)) : make_uint4(0u, 0u, 0u, 0u);
    };
    const int all = mine * TOKENS * CHUNKS;
    float largest = 0.f;  // bf16: what shows that a token may be outside the range of the common power; its exact largest is looked at only then
    bool small = false;
    const auto bring = [&](auto own_powers) {
        constexpr bool OWN = decltype(own_powers)::value;
        for (int e0 = threadIdx.x; e0 - (int)threadIdx.x < all; e0 += TOGETHER * ROWS_THREADS) {
            uint4 v[TOGETHER];
            int chunk, token, block;
#pragma unroll
            for (int q = 0; q < TOGETHER; ++q) v[q] = piece(e0 + q * ROWS_THREADS, chunk, token, block);
#pragma unroll
            for (int q = 0; q < TOGETHER; ++q) {
                const int e = e0 + q * ROWS_THREADS;
                if (e - (int)threadIdx.x >= all) break;
                chunk = e % CHUNKS;
                token = e / CHUNKS % TOKENS;
                block = e / (CHUNKS * TOKENS);
                float sum = 0.f;
                uint32_t u[4] = {v[q].x, v[q].y, v[q].z, v[q].w};
                if (OWN) {
                    const int power = token_exponent(tops[token]), half = power >> 1;
#pragma unroll
                    for (int i = 0; i < 4; ++i) u[i] = bf16_pair_times(bf16_pair_times(u[i], bf16_pair_of_powers(half)), bf16_pair_of_powers(power - half));
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x0 = bits_to_float(u[i] & 0xffffu, BF16), x1 = bits_to_float(u[i] >> 16, BF16);
                    sum += x0 + x1;
                    if (BF16 && !OWN) {
                        largest = fmaxf(fmaxf(largest, fabsf(x0)), fabsf(x1));
                        u[i] = bf16_pair_times(u[i], bf16_pair_of_powers(56));
                    }
                }
#pragma unroll
                for (int o = 1; o < CHUNKS; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                if (block < mine) {
                    // columns (0, 4), (2, 6), (1, 5), (3, 7): two codes of a word that lie sixteen bits apart
                    const uint4 f = make_uint4(__byte_perm(u[0], u[2], 0x5410), __byte_perm(u[1], u[3], 0x5410), __byte_perm(u[0], u[2], 0x7632), __byte_perm(u[1], u[3], 0x7632));
                    const int w = chunk % WORDS, lane_of = (token & 7) * 4 + chunk / WORDS;
                    xs[((block * WORDS + w) * NT + (token >> 3)) * 32 + lane_of] = f;
                    if (BF16 && !OWN) small |= fabsf(sum) < 9.3e-10f && (u[0] | u[1] | u[2] | u[3]) != 0u;  // 2^-30: where a block's sum is not below that, its largest is not below 2^-37; zeros are no matter
                    if (chunk == 0) sums[block * TOKENS + token] = OWN ? sum * 1.3877787807814457e-17f : sum;  // 2^-56: in the units of the common power's products
                }
            }
        }
    };
    bring(std::false_type());
    bool own = false;  // bf16: every token under a power of two of its own
    if (!BF16) {
        __syncthreads();
    } else if (__syncthreads_or(small || largest >= 18446744073709551616.f)) {  // 2^64
        if (threadIdx.x < TOKENS) tops[threadIdx.x] = 0u;
        __syncthreads();
        for (int e = threadIdx.x; e < all; e += ROWS_THREADS) {
            int chunk, token, block;
            const uint4 v = piece(e, chunk, token, block);
            const uint32_t pair = __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
            atomicMax(&tops[token], max(pair & 0xffffu, pair >> 16));
        }
        __syncthreads();
        for (int i = 0; i < TOKENS; ++i) own |= token_is_far(tops[i]);
        if (own) bring(std::true_type());
        __syncthreads();
    }

    // ---- products ----
    constexpr float BACK = BF16 ? 151115727451828646838272.f : 16777216.f;  // 2^(133 - 56) = 2^77, or 2^24
    const int per_group = (int)(a.group / KB);  // blocks of a group (one scale per row: all)
    float total[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j) total[j][0] = total[j][1] = total[j][2] = total[j][3] = 0.f;
    const bool single = a.group >= a.n;
    const float *const scale_lo = a.scale + min(row_lo, a.m - 1) * a.scale_row, *const scale_hi = a.scale + min(row_hi, a.m - 1) * a.scale_row;
    const float *const zero_lo = a.zero + min(row_lo, a.m - 1) * a.zero_row, *const zero_hi = a.zero + min(row_hi, a.m - 1) * a.zero_row;
    int block = 0;
    while (block < mine) {
        // a run of blocks under one scale
        const int64_t group = single ? 0 : (b_first + block) / per_group;
        const int end = single ? mine : (int)min((int64_t)mine, (group + 1) * per_group - b_first);
        const float s_lo = __ldg(scale_lo + group * a.scale_group), s_hi = __ldg(scale_hi + group * a.scale_group);
        const float o_lo = a.qmin - __ldg(zero_lo + group * a.zero_group), o_hi = a.qmin - __ldg(zero_hi + group * a.zero_group);
        float low[NT][4], high[NT][4], xsum[NT][2];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            low[j][0] = low[j][1] = low[j][2] = low[j][3] = high[j][0] = high[j][1] = high[j][2] = high[j][3] = xsum[j][0] = xsum[j][1] = 0.f;
        }
        while (block < end) {
#pragma unroll
            for (int s = 0; s < AHEAD; ++s) {
                // the slots go round with the blocks of the whole share, not of the run
                if ((block & (AHEAD - 1)) != s || block >= end) continue;
                const uint4 *const xb = xs + (int64_t)block * WORDS * NT * 32 + lane;
                uint32_t lo[WORDS], hi[WORDS];
#pragma unroll
                for (int w = 0; w < WORDS; ++w) lo[w] = code[s][0][w], hi[w] = code[s][1][w];
                fetch(s, block + AHEAD);
#pragma unroll
                for (int w = 0; w < WORDS; ++w) {
                    const uint32_t lo8 = lo[w] >> 8, hi8 = hi[w] >> 8;
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        const uint4 f = xb[(w * NT + j) * 32];
                        mma_codes<BF16>(low[j], lo[w] & 0x000f000fu, hi[w] & 0x000f000fu, lo8 & 0x000f000fu, hi8 & 0x000f000fu, f.x, f.y);
                        mma_codes<BF16>(high[j], lo[w] & 0x00f000f0u, hi[w] & 0x00f000f0u, lo8 & 0x00f000f0u, hi8 & 0x00f000f0u, f.z, f.w);
                    }
                }
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const float2 v = *reinterpret_cast<const float2 *>(sums + block * TOKENS + 8 * j + 2 * t);
                    xsum[j][0] += v.x;
                    xsum[j][1] += v.y;
                }
                ++block;
            }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const float products = fmaf(high[j][x], 0.0625f, low[j][x]) * BACK;
                total[j][x] = fmaf(x < 2 ? s_lo : s_hi, fmaf(x < 2 ? o_lo : o_hi, xsum[j][x & 1], products), total[j][x]);
            }
        }
    }
    if (BF16 && own) {  // from units of the token's power over the common one
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int power = token_exponent(tops[8 * j + 2 * t + (x & 1)]) - 56, half = power >> 1;
                total[j][x] = total[j][x] * power_of_two(-half) * power_of_two(half - power);
            }
    }
    // ---- sums of the cluster ----
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) part[(8 * j + 2 * t + (x & 1)) * ROWS + warp * 16 + 8 * (x >> 1) + g] = total[j][x];
    bool sound = true;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) sound &= fabsf(total[j][x]) < INFINITY;
    if (__syncthreads_or(!sound)) {
        // An infinite activation: codes and their origin, added up apart, would leave NaN of it.  Such activations alone decide a token's results: a thread adds up their products with the
        // weights, for a row and every second token, from the blocks whose sums of x show that they have some (8192 x 8192, 16 tokens, one infinity: 30 us instead of 20).
        const int row_here = threadIdx.x % ROWS;
        const int64_t row = min(row0 + row_here, a.m - 1);
        for (int token = threadIdx.x / ROWS; token < min(TOKENS, a.tokens - token0); token += ROWS_THREADS / ROWS) {
            float sum = 0.f;
            for (int block = 0; block < mine && sum == sum; ++block) {
                if (fabsf(sums[block * TOKENS + token]) < INFINITY) continue;
                const int64_t k0 = (b_first + block) * KB;
#pragma unroll 4
                for (int chunk = 0; chunk < CHUNKS; ++chunk) {
                    const uint4 v = k0 + 8 * chunk < a.n ? __ldg(reinterpret_cast<const uint4 *>((const uint16_t *)a.x + (token0 + token) * a.x_stride + k0) + chunk) : make_uint4(0u, 0u, 0u, 0u);
                    const uint32_t word[4] = {v.x, v.y, v.z, v.w};
                    unsigned odd = 0u;  // which of the eight are not finite
#pragma unroll
                    for (int i = 0; i < 8; ++i) odd |= fabsf(bits_to_float((word[i >> 1] >> (16 * (i & 1))) & 0xffffu, BF16)) < INFINITY ? 0u : 1u << i;
                    for (; odd && sum == sum; odd &= odd - 1u) {  // a NaN stays
                        const int64_t k = k0 + 8 * chunk + __ffs(odd) - 1, group = k / a.group;
                        const float x = bits_to_float(__ldg((const uint16_t *)a.x + (token0 + token) * a.x_stride + k), BF16), origin = a.qmin - __ldg(a.zero + row * a.zero_row + group * a.zero_group);
                        const uint32_t code = (__ldg(a.codes + row * a.row_bytes + (k >> 1)) >> (4 * (k & 1))) & 15u;
                        sum += ((float)code + origin) * __ldg(a.scale + row * a.scale_row + group * a.scale_group) * x;
                    }
                }
            }
            if (!(fabsf(sum) < INFINITY)) part[token * ROWS + row_here] = sum;
        }
        __syncthreads();
    }
    if (splits > 1) cluster_sync();
    if (a.rank) after_the_launch_before();
    // results: the cluster's CTAs share them, each a part of the rows and tokens; consecutive threads have consecutive rows
    const int results = min(TOKENS, a.tokens - token0) * ROWS;
    for (int e = rank * ROWS_THREADS + threadIdx.x; e < results; e += splits * ROWS_THREADS) {
        const int token = token0 + e / ROWS;
        const int64_t row = row0 + e % ROWS;
        float sum = 0.f;
        if (splits > 1) {
            for (int k = 0; k < splits; ++k) sum += peer_float(part + e, k);
        } else {
            sum = part[e];
        }
        if (row >= a.m) continue;
        const int id = adapter_of(a, token);
        if (id >= 0) {
            const uint4 *const up = reinterpret_cast<const uint4 *>((const uint16_t *)a.up + ((int64_t)id * a.m + row) * a.rank);
            const uint16_t *const inner = a.inner + (int64_t)token * INNER_LD;
            float more = 0.f;
            for (int r = 0; r < a.rank; r += 8) {
                const uint4 u = __ldg(up + r / 8), hi = *reinterpret_cast<const uint4 *>(inner + r), lo = *reinterpret_cast<const uint4 *>(inner + RANK_MAX + r);
                const uint32_t uu[4] = {u.x, u.y, u.z, u.w}, hh[4] = {hi.x, hi.y, hi.z, hi.w}, ll[4] = {lo.x, lo.y, lo.z, lo.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    more = fmaf(bits_to_float(uu[i] & 0xffffu, BF16), bits_to_float(hh[i] & 0xffffu, BF16) + bits_to_float(ll[i] & 0xffffu, BF16), more);
                    more = fmaf(bits_to_float(uu[i] >> 16, BF16), bits_to_float(hh[i] >> 16, BF16) + bits_to_float(ll[i] >> 16, BF16), more);
                }
            }
            sum = fmaf(more, a.factor[token], sum);
        }
        ((uint16_t *)a.out)[token * a.out_stride + row] = (uint16_t)float_to_bits(sum, BF16);
    }
    if (splits > 1) {
        __syncwarp();
        cluster_sync();  // the others' shared memory is read until here
    }
}

template <bool BF16, int NT, int KB>
static int launch_rows_kernel(const LinearArgs &a, cudaStream_t st) {
    static PerDeviceOnce configured;
    constexpr int ROWS = 16 * ROWS_WARPS, TOKENS = 8 * NT;
    constexpr size_t MOST = 200 * 1024;
    const int64_t blocks = ceil_div(a.n, (int64_t)KB), rows = ceil_div(a.m, (int64_t)ROWS), tiles = ceil_div((int64_t)a.tokens, (int64_t)TOKENS);
    const auto bytes = [&](int64_t splits) {
        const int64_t most = ceil_div(blocks, splits);
        return (size_t)(most * (KB * TOKENS * 2 + TOKENS * 4) + TOKENS * ROWS * 4);
    };
    // as many parts of the columns as two CTAs per SM take at once, of four blocks per warp at least; more where x would not fit
    int splits = 1;
    while (splits < 8 && ((rows * tiles * splits * 2 <= 2 * 148 && blocks >= 2 * splits * 4) || bytes(splits) > 96 * 1024)) splits *= 2;
    if (bytes(splits) > MOST) return G2D_ERR_TOO_LARGE;
    if (rows > 65535 || tiles > 65535) return G2D_ERR_TOO_LARGE;
    if (configured.run([&] { return cudaFuncSetAttribute(linear_rows_kernel<BF16, NT, KB>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)MOST) == cudaSuccess; }) != G2D_OK)
        return G2D_ERR_CUDA;
    return launch_dependent(linear_rows_kernel<BF16, NT, KB>, dim3((unsigned)splits, (unsigned)rows, (unsigned)tiles), ROWS_THREADS, bytes(splits), splits, a.rank > 0, st, a);
}

template <bool BF16, int NT>
static int launch_rows_tokens(const LinearArgs &a, cudaStream_t st) {
    const bool odd = a.group < a.n && a.group % 128 != 0;
    return odd ? launch_rows_kernel<BF16, NT, 64>(a, st) : launch_rows_kernel<BF16, NT, 128>(a, st);
}

int launch_linear_rows(const LinearArgs &a, cudaStream_t st) {
    if (a.tokens <= 8) return a.bf16 ? launch_rows_tokens<true, 1>(a, st) : launch_rows_tokens<false, 1>(a, st);
    return a.bf16 ? launch_rows_tokens<true, 2>(a, st) : launch_rows_tokens<false, 2>(a, st);
}

}  // namespace g2d

using namespace g2d;

// Up to here the tokens are columns of m16n8k16 products.  28672 x 8192, no adapters: 16 tokens 68.3 us, by tiles 83.9; 24 tokens 117 (two tiles of 16), by tiles 83.8; 4096 x 4096: 16 tokens 8.7,
// by tiles 16.5; 24 tokens 14.5, by tiles 16.8.
constexpr int64_t ROWS_TOKENS = 16;
// ... where x fits the shared memory of a cluster, and the rows a grid: else the tiles, which take x as it comes.
static bool linear_many(const g2d_linear_desc *d) { return d->tokens > ROWS_TOKENS || d->n > 32768 || d->m > (int64_t)65535 * 128; }

struct LinearSpace {
    size_t factor, plan, partial, all;  // inner values first
};
static LinearSpace linear_space(const g2d_linear_desc *d) {
    const auto whole = [](size_t bytes) { return (bytes + 255) & ~(size_t)255; };
    LinearSpace s{};
    size_t at = 0;
    const bool many = linear_many(d);
    const LinearTcPlan p = many ? linear_tc_plan(d->m, d->n, d->tokens, d->adapters > 0 ? (int)d->rank : 0, d->adapters) : LinearTcPlan{};
    if (d->rank > 0) {
        s.factor = at += whole((size_t)d->tokens * INNER_LD * 2);
        s.plan = at += whole((size_t)d->tokens * sizeof(float));
        if (d->tokens > LINEAR_FEW) at += whole((size_t)p.token_tiles * (p.tile + 1) * sizeof(int));
    }
    s.partial = at;
    if (many) at += whole(p.partial_bytes);
    s.all = at;
    return s;
}

static int linear_check(const g2d_linear_desc *d) {
    if (!d || (d->half != G2D_FP16 && d->half != G2D_BF16) || d->m < 0 || d->n < 0 || d->tokens < 0 || d->groups < 1 || d->rank < 0 || d->adapters < 0 || d->reserved != 0) return G2D_ERR_BAD_ARGUMENT;
    if (d->bits != 4 || d->n % 32 != 0 || d->row_bytes % 16 != 0 || d->rank % 8 != 0 || d->rank > RANK_MAX) return G2D_ERR_UNSUPPORTED;
    if (d->row_bytes < d->n / 2) return G2D_ERR_BAD_ARGUMENT;
    if (d->groups > 1 && (d->n % d->groups != 0 || d->n / d->groups % 64 != 0)) return G2D_ERR_UNSUPPORTED;
    if (d->m > 0x3fffffff || d->n > 0x3fffffff || d->tokens > 0x3fffffff || d->adapters > 0x7fffffff) return G2D_ERR_TOO_LARGE;
    return G2D_OK;
}

extern "C" int g2d_linear_workspace_bytes(const g2d_linear_desc *desc, size_t *bytes) {
    const int status = linear_check(desc);
    if (status != G2D_OK) return status;
    if (!bytes) return G2D_ERR_BAD_ARGUMENT;
    *bytes = linear_space(desc).all;
    return G2D_OK;
}

extern "C" int g2d_packed_linear(const g2d_linear_desc *d, void *stream) {
    const int status = linear_check(d);
    if (status != G2D_OK) return status;
    if (d->m == 0 || d->tokens == 0) return G2D_OK;
    if (!d->out || ((uintptr_t)d->out & 1) != 0 || d->out_stride < d->m) return G2D_ERR_BAD_ARGUMENT;
    if (d->n == 0) return G2D_ERR_UNSUPPORTED;
    if (!d->x || !d->codes || !d->scale || !d->zero || (((uintptr_t)d->x | (uintptr_t)d->codes) & 15) != 0 || d->x_stride % 8 != 0) return G2D_ERR_BAD_ARGUMENT;
    if (linear_many(d) && d->tokens > 1 && d->x_stride < d->n) return G2D_ERR_BAD_ARGUMENT;  // the tiles' copies take x as rows that stand apart
    if (d->rank > 0 && (!d->down || !d->up || !d->index || (((uintptr_t)d->down | (uintptr_t)d->up) & 15) != 0)) return G2D_ERR_BAD_ARGUMENT;
    const LinearSpace space = linear_space(d);
    if (space.all > 0 && (!d->workspace || d->workspace_bytes < space.all || ((uintptr_t)d->workspace & 255) != 0)) return G2D_ERR_WORKSPACE;
    LinearArgs a;
    a.x = d->x;
    a.codes = d->codes;
    a.scale = d->scale;
    a.zero = d->zero;
    a.out = d->out;
    a.m = d->m;
    a.n = d->n;
    a.row_bytes = d->row_bytes;
    a.x_stride = d->tokens > 1 ? d->x_stride : d->n;  // of one row it says nothing
    a.out_stride = d->out_stride;
    a.scale_row = d->scale_row_stride;
    a.scale_group = d->scale_group_stride;
    a.zero_row = d->zero_row_stride;
    a.zero_group = d->zero_group_stride;
    a.group = d->n / d->groups;
    a.tokens = (int)d->tokens;
    a.bf16 = d->half == G2D_BF16;
    a.qmin = (float)d->qmin;
    a.down = d->down;
    a.up = d->up;
    a.scaling = d->scaling;
    a.index = d->index;
    a.adapters = d->adapters;
    a.rank = d->adapters > 0 ? d->rank : 0;
    a.inner = (uint16_t *)d->workspace;
    a.factor = d->rank > 0 ? (float *)((char *)d->workspace + space.factor) : nullptr;
    a.status = d->status;
    a.wait_cycles = WAIT_CYCLES;
    cudaStream_t st = (cudaStream_t)stream;
    const bool many = linear_many(d);
    const LinearTcPlan p = many ? linear_tc_plan(a.m, a.n, a.tokens, a.rank, a.adapters) : LinearTcPlan{};
    int *const plan = a.tokens > LINEAR_FEW && a.rank > 0 ? (int *)((char *)d->workspace + space.plan) : nullptr;
    if (a.rank > 0) {
        const int launched = launch_inner(a, plan, p.tile, st);
        if (launched != G2D_OK) return launched;
    }
    return many ? launch_linear_tc(a, p, plan, (float *)((char *)d->workspace + space.partial), st) : launch_linear_rows(a, st);
}
