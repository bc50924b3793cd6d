// distill.cu - loss and gradient of a student's logits against a teacher's
// list of top logits and hard targets (cngpt_cuda_distill).
#include <cmath>

#include "common.cuh"
#include "kernels.h"

namespace cg {
namespace {

#define LAUNCH_CHECK() do { ++g_launch_count; CG_CUDA(cudaGetLastError()); } while (0)

constexpr int NT = 512;

template <bool MAX>
__device__ float block_reduce(float v, float *sh) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float w = __shfl_xor_sync(0xffffffffu, v, o);
        v = MAX ? fmaxf(v, w) : v + w;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh[0];
    for (int w = 1; w < NT / 32; ++w) v = MAX ? fmaxf(v, sh[w]) : v + sh[w];
    return v;
}

// Block per row: the row's maximum, the two softmax sums, the list's softmax,
// then the gradient. In place the row is read for the last time before any of
// it is written, except by the thread that rewrites the element itself.
__global__ void __launch_bounds__(NT)
distill_kernel(const float *logits, long ldl, int V, const float *__restrict__ tv, const int *__restrict__ ti, int k,
               const int *__restrict__ targets, float tau, float alpha, float scale, float *__restrict__ row_loss,
               float *dlogits, long ldd) {
    __shared__ float sh[NT / 32];
    __shared__ float sp[TOPK_MAX], sx[TOPK_MAX];
    __shared__ int si[TOPK_MAX];
    const long row = blockIdx.x;
    const float *x = logits + row * ldl;
    const float it = 1.0f / tau;
    // the list: values / tau where the entry counts, else -inf
    float lm = -INFINITY;
    for (int j = threadIdx.x; j < k; j += NT) {
        const int i = ti[row * k + j];
        const float v = tv[row * k + j];
        const bool ok = i >= 0 && i < V && v > -INFINITY;
        si[j] = ok ? i : -1;
        sp[j] = ok ? v : -INFINITY;
        sx[j] = ok ? x[i] : 0.0f;
        lm = fmaxf(lm, sp[j]);
    }
    lm = block_reduce<true>(lm, sh);
    float m = -INFINITY;
    bool nan = false;
    for (int i = threadIdx.x; i < V; i += NT) {
        m = fmaxf(m, x[i]);
        nan |= x[i] != x[i];
    }
    m = block_reduce<true>(m, sh);
    nan = block_reduce<true>(nan ? 1.0f : 0.0f, sh) > 0.0f;
    const int tgt = targets ? targets[row] : -1;
    const bool live = m > -INFINITY || nan;
    const bool soft = live && lm > -INFINITY, hard = live && tgt >= 0 && tgt < V;
    float st = 0.0f, s1 = 0.0f;
    for (int i = threadIdx.x; i < V; i += NT) {
        const float d = x[i] - m;
        st += expf(d * it);
        s1 += expf(d);
    }
    st = block_reduce<false>(st, sh);
    s1 = block_reduce<false>(s1, sh);
    float lz = 0.0f;
    for (int j = threadIdx.x; j < k; j += NT) lz += sp[j] > -INFINITY ? expf((sp[j] - lm) * it) : 0.0f;
    lz = block_reduce<false>(lz, sh);
    const float llz = logf(lz), lst = logf(st);
    float loss = 0.0f;
    if (soft)
        for (int j = threadIdx.x; j < k; j += NT) {
            const float z = (sp[j] - lm) * it;
            const float p = sp[j] > -INFINITY ? expf(z) / lz : 0.0f;
            if (p > 0.0f) loss += p * ((z - llz) - ((sx[j] - m) * it - lst));
            sp[j] = p;
        }
    loss = block_reduce<false>(loss, sh) * (alpha * tau * tau);
    if (hard) loss += (1.0f - alpha) * (logf(s1) - (x[tgt] - m));
    if (threadIdx.x == 0) row_loss[row] = loss;
    if (!dlogits) return;
    __syncthreads();
    float *d = dlogits + row * ldd;
    const float ct = soft ? scale * alpha * tau / st : 0.0f, c1 = hard ? scale * (1.0f - alpha) / s1 : 0.0f;
    for (int i = threadIdx.x; i < V; i += NT) {
        const float e = x[i] - m;
        float g = 0.0f;
        if (ct != 0.0f) g += ct * expf(e * it);
        if (c1 != 0.0f) g += c1 * expf(e);
        if (hard && i == tgt) g -= scale * (1.0f - alpha);
        d[i] = g;
    }
    __syncthreads();
    if (soft)
        for (int j = threadIdx.x; j < k; j += NT) {
            // the first entry of a token takes off the sum over all its entries
            if (si[j] < 0) continue;
            bool first = true;
            float p = 0.0f;
            for (int l = 0; l < k; ++l)
                if (si[l] == si[j]) {
                    first &= l >= j;
                    p += sp[l];
                }
            if (first) d[si[j]] -= scale * alpha * tau * p;
        }
}

// 1024 threads each sum a fixed strided subset, then a fixed-shape tree.
__global__ void __launch_bounds__(1024)
loss_sum_kernel(const float *__restrict__ row_loss, int rows, float scale, float *__restrict__ loss) {
    __shared__ float sh[1024];
    float acc = 0.0f;
    for (int r = threadIdx.x; r < rows; r += 1024) acc += row_loss[r];
    sh[threadIdx.x] = acc;
    __syncthreads();
    for (int w = 512; w > 0; w >>= 1) {
        if ((int)threadIdx.x < w) sh[threadIdx.x] += sh[threadIdx.x + w];
        __syncthreads();
    }
    if (threadIdx.x == 0) *loss = scale * sh[0];
}

}  // namespace

int distill_rows(const float *logits, long ldl, int rows, int V, const float *tv, const int *ti, int k,
                 const int *targets, float tau, float alpha, float scale, float *row_loss, float *dlogits, long ldd,
                 cudaStream_t s) {
    if (rows <= 0) return OK;
    distill_kernel<<<rows, NT, 0, s>>>(logits, ldl, V, tv, ti, k, targets, tau, alpha, scale, row_loss, dlogits, ldd);
    LAUNCH_CHECK();
    return OK;
}

int distill_loss_sum(const float *row_loss, int rows, float scale, float *loss, cudaStream_t s) {
    loss_sum_kernel<<<1, 1024, 0, s>>>(row_loss, rows, scale, loss);
    LAUNCH_CHECK();
    return OK;
}

}  // namespace cg
