// sample.cu - one token per row of logits from given uniform numbers, with
// temperature, top-k, top-p and min-p of every row (cngpt_cuda_sample).
#include <cmath>

#include "common.cuh"
#include "kernels.h"
#include "rank.cuh"

namespace cg {
namespace {

#define LAUNCH_CHECK() do { ++g_launch_count; CG_CUDA(cudaGetLastError()); } while (0)

constexpr int NT = 1024;

// Sum over the block in a fixed order, the same value in every thread.
template <class T>
__device__ T block_sum(T v, T *sh) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    T s = 0;
    for (int w = 0; w < NT / 32; ++w) s += sh[w];
    return s;
}

struct Row {
    const float *x;
    int V;
    float mx;
    double t;
    uint32_t key;  // tokens with a higher key stay, and at this key those up to index `cut`
    int cut;
    __device__ bool keeps(int i, uint32_t k) const { return k > key || (k == key && i <= cut); }
    __device__ double weight(int i) const {
        const float l = x[i];
        if (isinf(mx)) return l == mx ? 1.0 : 0.0;
        return exp(((double)l - (double)mx) / t);
    }
};

// The threshold that keeps the kept tokens above `key`, and the first `m` (in
// index order) at it.
__device__ int nth_at_key(const Row &r, uint32_t key, int m, int *shi) {
    int lo = 0, hi = r.V - 1;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        int c = 0;
        for (int i = threadIdx.x; i <= mid; i += NT) {
            const uint32_t k = rank_key(r.x[i]);
            c += k == key && r.keeps(i, k);
        }
        if (block_sum(c, shi) >= m) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

__global__ void __launch_bounds__(NT)
sample_kernel(SampleRows a) {
    __shared__ double shd[NT / 32];
    __shared__ int shi[NT / 32];
    __shared__ unsigned long long best;
    __shared__ double part[NT];
    const long row = blockIdx.x;
    Row r;
    const int V = a.V;
    const long at = a.step ? (long)*a.step * a.rows + row : row;
    auto put = [&](int tok, float lp) {
        a.tokens[at] = tok;
        if (a.next) a.next[row] = max(tok, 0);
        if (a.logprob) a.logprob[row] = lp;
    };
    r.x = a.logits + row * a.ldl;
    r.V = V;
    const float T = a.temperature ? a.temperature[row] : 1.0f;
    r.t = (double)T;
    if (threadIdx.x == 0) best = 0;
    __syncthreads();
    unsigned long long b = 0;
    for (int i = threadIdx.x; i < V; i += NT)
        b = max(b, ((unsigned long long)rank_key(r.x[i]) << 32) | (0xFFFFFFFFu - (uint32_t)i));
    atomicMax(&best, b);
    __syncthreads();
    const uint32_t bk = (uint32_t)(best >> 32);
    const int bi = (int)(0xFFFFFFFFu - (uint32_t)best);
    float p = a.top_p ? a.top_p[row] : 1.0f;
    if (bk <= RANK_NEG_INF || !(T > 0.0f) || p <= 0.0f) {
        if (threadIdx.x == 0) {
            if (bk <= RANK_NEG_INF) put(-1, -INFINITY);
            else put(bi, 0.0f);
        }
        return;
    }
    r.mx = rank_value(bk);
    r.key = RANK_NEG_INF;
    r.cut = -1;
    const int k = a.top_k ? a.top_k[row] : 0;
    if (k > 0 && k < V) {
        // the lowest key that fewer than k keys exceed: the k-th largest
        uint32_t lo = RANK_NEG_INF, hi = 0xFFFFFFFFu;
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2;
            int c = 0;
            for (int i = threadIdx.x; i < V; i += NT) c += rank_key(r.x[i]) > mid;
            if (block_sum(c, shi) < k) hi = mid;
            else lo = mid + 1;
        }
        if (lo > RANK_NEG_INF) {
            int c = 0;
            for (int i = threadIdx.x; i < V; i += NT) c += rank_key(r.x[i]) > lo;
            c = block_sum(c, shi);
            r.key = lo - 1;  // all at `lo` while their order is looked at
            const int cut = nth_at_key(r, lo, k - c, shi);
            r.key = lo;
            r.cut = cut;
        }
    }
    auto mass = [&](uint32_t above) {
        double s = 0.0;
        for (int i = threadIdx.x; i < V; i += NT) {
            const uint32_t kk = rank_key(r.x[i]);
            if (kk > above && r.keeps(i, kk)) s += r.weight(i);
        }
        return block_sum(s, shd);
    };
    if (p < 1.0f) {
        const double want = (double)p * mass(RANK_NEG_INF);
        uint32_t lo = r.key, hi = 0xFFFFFFFFu;
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (mass(mid) < want) hi = mid;
            else lo = mid + 1;
        }
        if (lo > RANK_NEG_INF) {
            const double above = mass(lo);
            const double w = isinf(r.mx) ? 1.0 : exp(((double)rank_value(lo) - (double)r.mx) / r.t);
            const double m = w > 0.0 ? ceil((want - above) / w) : (double)V;
            if (m < (double)V) {
                const int cut = nth_at_key(r, lo, max(1, (int)m), shi);
                r.cut = r.key == lo ? min(r.cut, cut) : cut;
                r.key = lo;
            }
        }
    }
    const float mp = a.min_p ? a.min_p[row] : 0.0f;
    const double floor_w = mp > 0.0f ? (double)fminf(1.0f, mp) : 0.0;  // NaN: off
    auto drawn = [&](int i) {
        const uint32_t kk = rank_key(r.x[i]);
        if (!r.keeps(i, kk)) return 0.0;
        const double w = r.weight(i);
        return w < floor_w ? 0.0 : w;
    };
    // index order: every thread sums its own stretch, the crossing stretch is walked
    const int n = (V + NT - 1) / NT, i0 = min(V, (int)threadIdx.x * n), i1 = min(V, i0 + n);
    double s = 0.0;
    for (int i = i0; i < i1; ++i) s += drawn(i);
    part[threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.x != 0) return;
    double total = 0.0;
    for (int t = 0; t < NT; ++t) total += part[t];
    const double target = (double)a.u[at] * total;
    double c = 0.0;
    int tok = bi;
    double wt = 1.0;
    for (int t = 0; t < NT; ++t) {
        if (part[t] <= 0.0) continue;
        const bool here = c + part[t] > target;
        double c2 = c;
        bool hit = false;
        for (int i = t * n; i < min(V, t * n + n); ++i) {
            const double w = drawn(i);
            if (w <= 0.0) continue;
            c2 += w;
            tok = i;
            wt = w;
            if (here && c2 > target) {
                hit = true;
                break;
            }
        }
        if (hit) break;
        c += part[t];
    }
    put(tok, (float)log(wt / total));
}

}  // namespace

int sample_rows(const SampleRows &a, cudaStream_t s) {
    if (a.rows <= 0) return OK;
    sample_kernel<<<a.rows, NT, 0, s>>>(a);
    LAUNCH_CHECK();
    return OK;
}

}  // namespace cg
