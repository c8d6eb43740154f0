// Shared by the attention kernels over the packed cache.
#pragma once
#include "g2d_cache.cuh"
#include "g2d_tc.cuh"

namespace g2d {

int cache_view(const g2d_cache_desc *d, CacheView *c);

// ---- attention: what its kernels share ----
struct AttendArgs {
    CacheView c;
    const void *q;
    void *out;  // [tokens, heads, head_dim]
    int64_t q_token_stride, q_head_stride;
    int heads, group;
    int causal;
    float scale;             // of the scores
    float softcap;           // 0: none
    const float *slopes;     // per head, or null
    const int32_t *prefix;   // per sequence, or null
    int rows_from, rows_to;  // the kernel's sequences: those with rows_from <= queries x group < rows_to
    float *partial;
    int *status;
    long long wait_cycles;
};
struct AttendSequence {
    int first, count, length, keys, prefix;
};
__device__ __forceinline__ AttendSequence attend_sequence(const AttendArgs &a, int b) {
    AttendSequence s;
    tokens_of(a.c, b, s.first, s.count);
    s.length = a.c.lengths[b];
    s.keys = keys_of(a.c, s.length);
    s.prefix = a.prefix ? a.prefix[b] : 0;
    return s;
}
// how many keys, from the first on, token i of the sequence sees
__device__ __forceinline__ int visible_keys(const AttendArgs &a, const AttendSequence &s, int i) {
    if (!a.causal) return s.keys;
    const int64_t p = (int64_t)s.length - s.count + i;
    return (int)min((int64_t)s.keys, max(p + 1, max((int64_t)s.prefix, (int64_t)0)));
}


constexpr float LOG2E = 1.4426950408889634f;
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// cap tanh(u / cap) through one exponential: exact to 1e-7 of the cap, which is what a score's exponential sees
__device__ __forceinline__ float capped(float u, float cap, float two_log2e_over_cap) { return cap - __fdividef(2.f * cap, 1.f + ex2(u * two_log2e_over_cap)); }
__device__ __forceinline__ int64_t warp_sum(int64_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Sequences of many rows, by tiles (g2d_attend_tc.cu)
size_t attend_tiles_bytes(int head_dim);
int launch_attend_tiles(const AttendArgs &a, cudaStream_t st);

}  // namespace g2d
