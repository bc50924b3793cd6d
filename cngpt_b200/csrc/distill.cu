// distill.cu - loss and gradient of a student's logits against a teacher's
// list of top logits and hard targets (cngpt_cuda_distill).
//
// With c = log2(e) / t, a row's softmax at temperature t needs m = max x and
// s_t = sum 2^((x - m) c); loss and gradient then are
//   sum p (log p - (x - m) / tau + log s_tau)  and  a 2^((x - m) c) / s_t - ...,
// the list's and the target's entries apart. Reading a row once and writing its
// gradient once is all that has to move (8 bytes a logit, 4 without gradient),
// so a cluster of blocks keeps the row in its shared memory between the pass
// that forms m and the sums and the pass that writes.
#include <algorithm>
#include <cmath>

#include <cooperative_groups.h>

#include "common.cuh"
#include "kernels.h"

namespace cg {
namespace {

namespace coop = cooperative_groups;

#define LAUNCH_CHECK() do { ++g_launch_count; CG_CUDA(cudaGetLastError()); } while (0)

constexpr int NT = 256;
constexpr int QUADS = 4;                // 16-byte loads of a thread in flight
constexpr int MAX_PARTS = 8;
constexpr int SLICE_BYTES = 52 * 1024;  // of a row in a block's shared memory: four blocks an SM
constexpr int SLICE_MAX = 200 * 1024;   // where eight blocks need more than that: one block an SM
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Maximum and the sums at both temperatures of a part of a row. A part of -inf
// alone has m = -inf and sums of 0; NaN stays in the sums.
struct Stats {
    float m, st, s1;
};

__device__ __forceinline__ float ref_of(float m) { return m == -INFINITY ? 0.0f : m; }

__device__ __forceinline__ Stats merge(const Stats &a, const Stats &b, float ct) {
    Stats r;
    r.m = fmaxf(a.m, b.m);
    const float ref = ref_of(r.m), da = a.m - ref, db = b.m - ref;
    r.st = a.st * ex2(da * ct) + b.st * ex2(db * ct);
    r.s1 = a.s1 * ex2(da * LOG2E) + b.s1 * ex2(db * LOG2E);
    return r;
}

struct DistillArgs {
    const float *logits;
    long ldl;
    int V, stretch;
    const float *tv;
    const int *ti;
    int k;
    const int *targets;
    float tau, alpha, scale;
    float *row_loss;
    float *dlogits;
    long ldd;
};

// Cluster of 1 to 8 blocks per row, a stretch of it each. BOTH: the hard part's
// softmax (temperature 1) is needed beside the list's. CACHE: the stretch stays
// in shared memory for the gradient; without it, it is read again.
template <bool GRAD, bool BOTH, bool CACHE>
__global__ void __launch_bounds__(NT)
distill_kernel(DistillArgs a) {
    extern __shared__ float4 slice4[];  // [cached stretch + 8], then the list: sp, sx, si [k]
    __shared__ Stats sw[NT / 32], sc[MAX_PARTS];
    __shared__ float red[NT / 32];
    __shared__ int twice;
    float *slice = (float *)slice4;
    float *sp = slice + (CACHE ? a.stretch + 8 : 0), *sx = sp + a.k;
    int *si = (int *)(sx + a.k);
    auto cluster = coop::this_cluster();
    const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
    if (parts > 1) cluster.barrier_arrive();  // waited for before the first write to another block
    const long row = blockIdx.x / parts;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int lo = min(a.V, part * a.stretch), hi = min(a.V, lo + a.stretch), n = hi - lo, k = a.k;
    const float *xr = a.logits + row * a.ldl, *x = xr + lo;
    const float ct = LOG2E / a.tau;
    // elements before the first 16-byte boundary, whole groups of four, the rest;
    // element i of the stretch is kept at slice[pad + i], groups at float4s
    const int head = min(n, (int)(((16 - (uintptr_t)x % 16) / 4) % 4)), quads = (n - head) / 4, pad = (4 - head) & 3;
    const float4 *x4 = (const float4 *)(x + head);
    float4 *s4 = (float4 *)(slice + pad + head);

    Stats s{-INFINITY, 0.0f, 0.0f};
    auto add = [&](float v, float ref) {
        const float d = v - ref;
        s.st += ex2(d * ct);
        if (BOTH) s.s1 += ex2(d * LOG2E);
    };
    auto raise = [&](float m) {  // to a maximum over what comes next
        if (m > s.m) {
            const float d = s.m - m;
            s.st *= ex2(d * ct);
            if (BOTH) s.s1 *= ex2(d * LOG2E);
            s.m = m;
        }
        return ref_of(s.m);
    };
    {
        const int i = tid < head ? tid : tid < n - 4 * quads ? tid + 4 * quads : -1;  // the odd ones at both ends
        if (i >= 0) {
            const float v = x[i];
            if (CACHE) slice[pad + i] = v;
            add(v, raise(v));
        }
    }
    for (int q0 = tid; q0 < quads; q0 += QUADS * NT) {
        float4 v[QUADS];
#pragma unroll
        for (int j = 0; j < QUADS; ++j)
            v[j] = q0 + j * NT < quads ? __ldcs(x4 + q0 + j * NT) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        float m = -INFINITY;
#pragma unroll
        for (int j = 0; j < QUADS; ++j) {
            m = fmaxf(m, fmaxf(fmaxf(v[j].x, v[j].y), fmaxf(v[j].z, v[j].w)));
            if (CACHE && q0 + j * NT < quads) s4[q0 + j * NT] = v[j];
        }
        const float ref = raise(m);
#pragma unroll
        for (int j = 0; j < QUADS; ++j) {
            add(v[j].x, ref);
            add(v[j].y, ref);
            add(v[j].z, ref);
            add(v[j].w, ref);
        }
    }
    // the list: its softmax sp and the student's logits sx there, in every block
    float lm = -INFINITY;
    for (int j = tid; j < k; j += NT) {
        const int i = a.ti[row * k + j];
        const float v = a.tv[row * k + j];
        const bool ok = i >= 0 && i < a.V && v > -INFINITY;
        si[j] = ok ? i : -1;
        sp[j] = ok ? v : -INFINITY;
        sx[j] = ok ? xr[i] : 0.0f;
        lm = fmaxf(lm, sp[j]);
    }
    const int tgt = a.targets ? a.targets[row] : -1;
    const bool has_tgt = tgt >= 0 && tgt < a.V;
    const float xt = has_tgt ? xr[tgt] : 0.0f;

    // the row's statistics: lanes, warps, blocks, each in a fixed order
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const Stats b{__shfl_xor_sync(0xffffffffu, s.m, o), __shfl_xor_sync(0xffffffffu, s.st, o),
                      __shfl_xor_sync(0xffffffffu, s.s1, o)};
        // the lower lane's value first, so that both lanes form the same sum
        s = (lane & o) ? merge(b, s, ct) : merge(s, b, ct);
    }
    lm = warp_max(lm);
    if (lane == 0) {
        sw[warp] = s;
        red[warp] = lm;
    }
    __syncthreads();
    s = sw[0];
    lm = red[0];
#pragma unroll
    for (int w = 1; w < NT / 32; ++w) {
        s = merge(s, sw[w], ct);
        lm = fmaxf(lm, red[w]);
    }
    if (parts > 1) {
        cluster.barrier_wait();
        if (tid < parts) *cluster.map_shared_rank(&sc[part], tid) = s;
        cluster.sync();  // also: every block has read what another one will overwrite
        s = sc[0];
        for (int p = 1; p < parts; ++p) s = merge(s, sc[p], ct);
    }
    const float ref = ref_of(s.m);
    const bool live = !(s.m == -INFINITY && s.st == 0.0f);
    const bool soft = live && lm > -INFINITY, hard = live && has_tgt;
    auto sum = [&](float v) {
        v = warp_sum(v);
        __syncthreads();
        if (lane == 0) red[warp] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int w = 1; w < NT / 32; ++w) v += red[w];
        return v;
    };
    if (soft) {
        const float it = 1.0f / a.tau;
        float lz = 0.0f;
        for (int j = tid; j < k; j += NT) lz += sp[j] > -INFINITY ? expf((sp[j] - lm) * it) : 0.0f;
        lz = sum(lz);
        const float llz = logf(lz), lst = logf(s.st);
        float loss = 0.0f;
        for (int j = tid; j < k; j += NT) {
            const float z = (sp[j] - lm) * it;
            const float p = sp[j] > -INFINITY ? expf(z) / lz : 0.0f;
            if (p > 0.0f) loss += p * ((z - llz) - ((sx[j] - ref) * it - lst));
            sp[j] = p;
        }
        if (part == 0) {
            loss = sum(loss) * (a.alpha * a.tau * a.tau);
            if (hard) loss += (1.0f - a.alpha) * (logf(s.s1) - (xt - ref));
            if (tid == 0) a.row_loss[row] = loss;
        }
    } else if (part == 0 && tid == 0) {
        a.row_loss[row] = hard ? (1.0f - a.alpha) * (logf(s.s1) - (xt - ref)) : 0.0f;
    }
    if (!GRAD) return;

    float *dr = a.dlogits + row * a.ldd, *d = dr + lo;
    const float gt = soft ? a.scale * a.alpha * a.tau / s.st : 0.0f;
    const float g1 = BOTH && hard ? a.scale * (1.0f - a.alpha) / s.s1 : 0.0f;
    const float ot = a.scale * a.alpha * a.tau, o1 = a.scale * (1.0f - a.alpha);
    auto grad = [&](float v) {
        const float e = v - ref;
        // a part that is switched off counts as 0 whatever its exponential
        float g = soft ? gt * ex2(e * ct) : 0.0f;
        if (BOTH && hard) g = fmaf(g1, ex2(e * LOG2E), g);
        return g;
    };
    {
        const int i = tid < head ? tid : tid < n - 4 * quads ? tid + 4 * quads : -1;
        if (i >= 0) d[i] = grad(CACHE ? slice[pad + i] : x[i]);
    }
    const bool whole = ((uintptr_t)(d + head) & 15) == 0;  // the groups of x are groups of d too
    for (int q = tid; q < quads; q += NT) {
        float4 v = CACHE ? s4[q] : __ldcs(x4 + q);
        v = make_float4(grad(v.x), grad(v.y), grad(v.z), grad(v.w));
        if (whole) {
            __stcs((float4 *)(d + head) + q, v);
        } else {
            float *p = d + head + 4 * q;
            p[0] = v.x;
            p[1] = v.y;
            p[2] = v.z;
            p[3] = v.w;
        }
    }
    if (!soft && !hard) return;
    // entries of the list and the target in this stretch: written again with
    // their own part taken off, by the first entry of a token for all of its
    if (tid == 0) twice = !CACHE;
    __syncthreads();
    if (soft && CACHE) {
        // the cached stretch has done its service: every entry leaves its number
        // at its token, and one that finds another there has company
        for (int j = tid; j < k; j += NT)
            if (si[j] >= lo && si[j] < hi) slice[pad + si[j] - lo] = __int_as_float(j);
        __syncthreads();
        for (int j = tid; j < k; j += NT)
            if (si[j] >= lo && si[j] < hi && __float_as_int(slice[pad + si[j] - lo]) != j) twice = 1;
        __syncthreads();
    }
    const bool search = twice;
    if (soft)
        for (int j = tid; j < k; j += NT) {
            const int i = si[j];
            if (i < lo || i >= hi) continue;
            float p = sp[j];
            if (search) {
                bool first = true;
                p = 0.0f;
                for (int l = 0; l < k; ++l)
                    if (si[l] == i) {
                        first &= l >= j;
                        p += sp[l];
                    }
                if (!first) continue;
            }
            float g = grad(sx[j]) - ot * p;
            if (hard && i == tgt) g -= o1;
            dr[i] = g;
        }
    if (hard && tgt >= lo && tgt < hi) {
        __shared__ int listed;
        if (tid == 0) listed = 0;
        __syncthreads();
        if (soft)
            for (int j = tid; j < k; j += NT)
                if (si[j] == tgt) listed = 1;
        __syncthreads();
        if (tid == 0 && !listed) dr[tgt] = grad(xt) - o1;
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

template <bool GRAD, bool BOTH, bool CACHE>
int launch(const DistillArgs &a, int rows, int parts, size_t smem, cudaStream_t s) {
    static bool set = false;
    if (!set) {
        CG_CUDA(cudaFuncSetAttribute(distill_kernel<GRAD, BOTH, CACHE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     SLICE_MAX + 12 * TOPK_MAX));
        set = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * parts));
    cfg.blockDim = dim3(NT);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)parts;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    CG_CUDA(cudaLaunchKernelEx(&cfg, distill_kernel<GRAD, BOTH, CACHE>, a));
    ++g_launch_count;
    return OK;
}

}  // namespace

int distill_rows(const float *logits, long ldl, int rows, int V, const float *tv, const int *ti, int k,
                 const int *targets, float tau, float alpha, float scale, float *row_loss, float *dlogits, long ldd,
                 cudaStream_t s) {
    if (rows <= 0) return OK;
    // Blocks of a row: as many as keep four blocks' stretches on an SM, more
    // while there are rows for half the SMs at most. The same with and without
    // gradient, so that the loss is the same to the bit.
    int parts = 1;
    while (parts < MAX_PARTS && ((long)V * 4 > (long)parts * SLICE_BYTES ||
                                 ((long)rows * parts * 2 <= num_sms() && V >= parts * 4096)))
        parts *= 2;
    if ((long)rows * parts > 0x7FFFFFFFL) {
        set_last_error(ERR_ARG, "distill: %d rows are too many", rows);
        return ERR_ARG;
    }
    DistillArgs a{logits, ldl, V, ((V + parts - 1) / parts + 3) / 4 * 4, tv, ti, k, targets, tau, alpha, scale, row_loss,
                  dlogits, ldd};
    const size_t list = (size_t)k * 12, bytes = ((size_t)a.stretch + 8) * sizeof(float);
    const bool both = alpha < 1.0f && targets;
    if (!dlogits)
        return both ? launch<false, true, false>(a, rows, parts, list, s) : launch<false, false, false>(a, rows, parts, list, s);
    if (bytes <= SLICE_MAX)
        return both ? launch<true, true, true>(a, rows, parts, bytes + list, s)
                    : launch<true, false, true>(a, rows, parts, bytes + list, s);
    return both ? launch<true, true, false>(a, rows, parts, list, s) : launch<true, false, false>(a, rows, parts, list, s);
}

int distill_loss_sum(const float *row_loss, int rows, float scale, float *loss, cudaStream_t s) {
    loss_sum_kernel<<<1, 1024, 0, s>>>(row_loss, rows, scale, loss);
    LAUNCH_CHECK();
    return OK;
}

}  // namespace cg
