// Shared by the kernels of the product with packed codes and its low-rank adapters.
#pragma once
#include "g2d_common.cuh"

namespace g2d {

constexpr int RANK_MAX = 64;
constexpr int LINEAR_FEW = 64;  // up to so many tokens each has its adapter for itself: no plan
constexpr int INNER_LD = 2 * RANK_MAX;  // an inner row: 64 upper parts, 64 lower parts

struct LinearArgs {
    const void *x;         // [tokens, n], rows of x_stride
    const uint8_t *codes;  // [m, row_bytes], two codes a byte, the lower half first
    const float *scale, *zero;
    void *out;  // [tokens, m], rows of out_stride
    int64_t m, n, row_bytes, x_stride, out_stride;
    int64_t scale_row, scale_group, zero_row, zero_group;
    int64_t group;  // columns under one scale; n for one scale per row
    int tokens, bf16;
    float qmin;
    // adapters: down [adapters, rank, n], up [adapters, m, rank], scaling [adapters] or null, index [tokens]; rank 0: none
    const void *down, *up;
    const float *scaling;
    const int32_t *index;
    int64_t adapters;
    int rank;
    // the inner values h = down x of every token, times 2^-e of its own, as pairs of 16-bit values hi + lo; factor: 2^e scaling, 0 for a token without an adapter
    uint16_t *inner;  // [tokens, INNER_LD]
    float *factor;    // [tokens]
    int *status;
    long long wait_cycles;
};

// A token's adapter, or -1
__device__ __forceinline__ int adapter_of(const LinearArgs &a, int token) {
    if (a.rank == 0 || token >= a.tokens) return -1;
    const int id = a.index[token];
    return id >= 0 && id < a.adapters ? id : -1;
}
__device__ __forceinline__ float bits_to_float(uint32_t bits, int bf16) { return bf16 ? __uint_as_float(bits << 16) : __half2float(__ushort_as_half((unsigned short)bits)); }
__device__ __forceinline__ uint32_t float_to_bits(float v, int bf16) { return bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v)); }

// Many tokens: tiles of 128 rows (duo: 256, by two CTAs) x `tile` tokens, in chunks of 64 columns.  Whole rounds of whole tiles, then `shared` tiles on one line
// of chunks, cut into `ctas` pieces; a tile has at most `pieces` of them.
struct LinearTcPlan {
    int tile, duo, row_tiles, token_tiles, chunks, whole;
    int later;  // the adapters' outer halves are added where the pieces are joined, and every tile is cut
    int64_t shared, line, ctas, pieces;
    size_t partial_bytes;
};
LinearTcPlan linear_tc_plan(int64_t m, int64_t n, int64_t tokens, int rank, int64_t adapters);

// Inner values and factors of all tokens; where they are more than LINEAR_FEW, also the adapters of each tile of `tile` tokens: plan[i * (tile + 1)] of them, their numbers behind it
int launch_inner(const LinearArgs &a, int *plan, int tile, cudaStream_t st);
int launch_linear_rows(const LinearArgs &a, cudaStream_t st);  // few tokens
int launch_linear_tc(const LinearArgs &a, const LinearTcPlan &p, const int *plan, float *partial, cudaStream_t st);

template <typename... Params, typename... Args>
inline int launch_dependent(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, int cluster, bool dependent, cudaStream_t st, const Args &...args) {
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = dim3((unsigned)threads);
    config.dynamicSmemBytes = smem;
    config.stream = st;
    cudaLaunchAttribute attributes[2]{};
    unsigned count = 0;
    if (cluster > 1) {
        attributes[count].id = cudaLaunchAttributeClusterDimension;
        attributes[count].val.clusterDim.x = (unsigned)cluster;
        attributes[count].val.clusterDim.y = attributes[count].val.clusterDim.z = 1;
        ++count;
    }
    if (dependent) {
        attributes[count].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attributes[count].val.programmaticStreamSerializationAllowed = 1;
        ++count;
    }
    config.attrs = attributes;
    config.numAttrs = count;
    return cudaLaunchKernelEx(&config, kernel, Params(args)...) == cudaSuccess ? check_launch() : G2D_ERR_CUDA;
}

// shared memory of another CTA of the cluster
__device__ __forceinline__ float peer_float(const float *mine, uint32_t rank) {
    uint32_t at;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(mine)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}

}  // namespace g2d
