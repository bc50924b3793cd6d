// prefix_attention.cu - decode attention of sequences that share a prefix
// (cngpt_cuda_prefix_attention).
#include <cmath>

#include "common.cuh"
#include "kernels.h"

namespace cg {
namespace {

#define LAUNCH_CHECK() do { ++g_launch_count; CG_CUDA(cudaGetLastError()); } while (0)

// One warp per (sequence, head), keys in order, the softmax's running maximum
// and sum in registers; lane l holds dimensions l, l + 32, ...
__global__ void __launch_bounds__(128)
prefix_attn_kernel(PrefixAttn a) {
    const long w = ((long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    if (w >= (long)a.B * a.H) return;
    const long b = w / a.H;
    const int h = (int)(w % a.H), hk = h / (a.H / a.Hk);
    float q[8], o[8] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int d = lane + 32 * i;
        q[i] = d < a.hs ? a.q[b * a.ldq + (long)h * a.hs + d] * a.scale : 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    const int S = a.S > 0 ? min(max(a.suffix_len[b], 0), a.S) : 0;
    for (long j = 0; j < (long)a.P + S; ++j) {
        const bool pre = j < a.P;
        const long at = (pre ? j * a.ldp : b * a.seq_stride + (j - a.P) * a.lds) + (long)hk * a.hs;
        const float *kr = (pre ? a.pk : a.sk) + at, *vr = (pre ? a.pv : a.sv) + at;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (lane + 32 * i < a.hs) s = fmaf(q[i], kr[lane + 32 * i], s);
        s = warp_sum(s);
        if (s == -INFINITY) continue;
        const float mn = fmaxf(m, s), c = expf(m - mn), p = expf(s - mn);
        l = l * c + p;
        m = mn;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (lane + 32 * i < a.hs) o[i] = fmaf(p, vr[lane + 32 * i], o[i] * c);
    }
    const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int d = lane + 32 * i;
        if (d < a.hs) a.out[b * a.ldo + (long)h * a.hs + d] = o[i] * inv;
    }
}

__global__ void shared_advance_kernel(int *ctr, int *suffix_len, int n) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) suffix_len[i] += 1;
    if (threadIdx.x < 3) ctr[threadIdx.x] += 1;
}

}  // namespace

int shared_advance(int *ctr, int *suffix_len, int n, cudaStream_t s) {
    shared_advance_kernel<<<1, 256, 0, s>>>(ctr, suffix_len, n);
    LAUNCH_CHECK();
    return OK;
}

size_t prefix_attention_ws_bytes(int, int, int, int, int, int) { return 0; }

int prefix_attention(const PrefixAttn &a, void *, cudaStream_t s) {
    if (a.B <= 0) return OK;
    const long warps = (long)a.B * a.H;
    prefix_attn_kernel<<<(unsigned)((warps + 3) / 4), 128, 0, s>>>(a);
    LAUNCH_CHECK();
    return OK;
}

}  // namespace cg
