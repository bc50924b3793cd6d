// topk.cu - the k largest logits of every row in falling order (cngpt_cuda_topk).
#include "common.cuh"
#include "kernels.h"
#include "rank.cuh"

namespace cg {
namespace {

#define LAUNCH_CHECK() do { ++g_launch_count; CG_CUDA(cudaGetLastError()); } while (0)

constexpr int NT = 512;

__device__ int block_count(int v, int *sh) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    int s = 0;
    for (int w = 0; w < NT / 32; ++w) s += sh[w];
    return s;
}

// Block per row. A token's rank is the number of 64-bit keys (logit key, index
// inverted) above its own; the k-th largest such key is found by bisection, the
// k tokens at or above it are collected and ordered by counting.
__global__ void __launch_bounds__(NT)
topk_kernel(const float *__restrict__ logits, long ldl, int V, int k, float *__restrict__ values,
            int *__restrict__ indices) {
    __shared__ int sh[NT / 32];
    __shared__ unsigned long long cand[TOPK_MAX];
    __shared__ int n;
    const float *x = logits + (long)blockIdx.x * ldl;
    auto key = [&](int i) { return ((unsigned long long)rank_key(x[i]) << 32) | (0xFFFFFFFFu - (uint32_t)i); };
    unsigned long long lo = 0, hi = ~0ull;
    while (lo < hi) {
        const unsigned long long mid = lo + (hi - lo) / 2;
        int c = 0;
        for (int i = threadIdx.x; i < V; i += NT) c += key(i) > mid;
        if (block_count(c, sh) < k) hi = mid;
        else lo = mid + 1;
    }
    if (threadIdx.x == 0) n = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < V; i += NT)
        if (key(i) >= lo) cand[atomicAdd(&n, 1)] = key(i);
    __syncthreads();
    for (int c = threadIdx.x; c < k; c += NT) {
        int r = 0;
        for (int j = 0; j < k; ++j) r += cand[j] > cand[c];
        values[(long)blockIdx.x * k + r] = rank_value((uint32_t)(cand[c] >> 32));
        indices[(long)blockIdx.x * k + r] = (int)(0xFFFFFFFFu - (uint32_t)cand[c]);
    }
}

}  // namespace

int topk_rows(const float *logits, long ldl, int rows, int V, int k, float *values, int *indices, cudaStream_t s) {
    if (rows <= 0) return OK;
    topk_kernel<<<rows, NT, 0, s>>>(logits, ldl, V, k, values, indices);
    LAUNCH_CHECK();
    return OK;
}

}  // namespace cg
