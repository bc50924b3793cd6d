// distill.cu - loss and gradient of a student's logits against a teacher's
// list of top logits and hard targets (cngpt_cuda_distill).
//
// With c = log2(e) / t and R = max x c, a row's softmax at temperature t needs
// s_t = sum 2^(x c - R): loss and gradient then are
//   sum p (log p - ln2 (x c - R - log2 s_tau))  and  a 2^(x c - R) / s_t - ...,
// the list's and the target's entries apart. R is one rounded number that both
// passes subtract inside one fma, so its rounding cancels. Reading a row once and
// writing its gradient once is all that has to move (8 bytes a logit, 4 without
// gradient), so a cluster of blocks keeps the row in its shared memory between
// the pass that forms the sums and the pass that writes.
//
// The list's dependent loads, its softmax and the second writing of its entries are
// one warp's; eight others look after the stretch and wait for it only at the end
// (with the list's warp among them they waited twice: 0.76 ms where it is 0.675).
//
// On B200, 8192 x 50257 with both softmaxes and the gradient: 0.675 ms (4.9 TB/s, 75 %
// of the copy rate); the loss of 1024 rows alone: 56.6 us (3.6 TB/s). What is left is the
// latency of a row's phases (loads, two block barriers, one cluster barrier), which
// four blocks an SM do not hide; the exponentials take half of the special-function
// units' time. Two to seven more warps took 0.68 to 1.09 ms, shorter stretches 1.06,
// sums of chunks while the next ones arrive 8 % more, clusters that prefetch their
// next row three times as long. Short rows have a warp each: 7000 x 500 18 us.
#include <algorithm>
#include <cmath>

#include <cooperative_groups.h>

#include "common.cuh"
#include "kernels.h"

namespace cg {
namespace {

namespace coop = cooperative_groups;

#define LAUNCH_CHECK() do { ++g_launch_count; CG_CUDA(cudaGetLastError()); } while (0)

constexpr int COPY = 256;  // threads of a stretch, behind the list's warp
constexpr int ROWS = 4;    // of a block whose warps have a row each
constexpr int MAX_PARTS = 8;
constexpr int SLICE_BYTES = 52 * 1024;  // of a row in a block's shared memory: four blocks an SM
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Maximum of a part of a row and its sums at both temperatures, relative to
// R(m). A part of -inf alone has m = -inf and sums of 0; NaN stays in the sums.
struct Stats {
    float m, st, s1;
};

__device__ __forceinline__ float scaled_max(float m, float c) { return m == -INFINITY ? 0.0f : __fmul_rn(m, c); }

// the sums of `s` relative to the maximum m >= s.m; those of a part of -inf alone
// stay what they are (0, or NaN), whatever R(m) is
template <bool BOTH>
__device__ __forceinline__ void raise(Stats &s, float m, float ct) {
    if (s.m > -INFINITY) {
        s.st *= ex2(scaled_max(s.m, ct) - scaled_max(m, ct));
        if (BOTH) s.s1 *= ex2(scaled_max(s.m, LOG2E) - scaled_max(m, LOG2E));
    }
    s.m = m;
}

struct DistillArgs {
    const float *logits;
    long ldl;
    int rows, V, stretch;
    const float *tv;
    const int *ti;
    int k;
    const int *targets;
    float tau, alpha, scale;
    float *row_loss;
    float *dlogits;
    long ldd;
};

// of shared memory: the stretch and the list
__host__ __device__ __forceinline__ size_t row_bytes(int stretch, int k) {
    return (((size_t)stretch + 8) * 4 + (size_t)k * 12 + 15) / 16 * 16;
}

// Cluster of 1 to 8 blocks per row, a stretch of it each. BOTH: the hard part's
// softmax (temperature 1) is needed beside the list's. Warp 0 looks after the
// list; until the first barrier the others read from shared memory only what they
// copied there themselves.
// ALONE: one warp does all of it for a whole row, ROWS of them a block.
template <bool GRAD, bool BOTH, bool ALONE>
__global__ void __launch_bounds__(ALONE ? 32 * ROWS : 32 + COPY)
distill_kernel(DistillArgs a) {
    constexpr int NT = ALONE ? 32 : 32 + COPY, STEP = ALONE ? 32 : COPY;
    extern __shared__ float4 slice4[];  // [stretch + 8], then the list: sp, sx, si [k]
    __shared__ Stats sw_of[ALONE ? ROWS : NT / 32], sc[MAX_PARTS];
    __shared__ int flags[ALONE ? ROWS : 1][3];
    const int own = ALONE ? threadIdx.x >> 5 : 0;  // of the block's rows
    Stats *sw = sw_of + own;
    int &soft_list = flags[own][0], &twice = flags[own][1], &listed = flags[own][2];
    float *slice = (float *)((char *)slice4 + own * row_bytes(a.stretch, a.k)), *sp = slice + a.stretch + 8, *sx = sp + a.k;
    int *si = (int *)(sx + a.k);
    auto cluster = coop::this_cluster();
    const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
    if (parts > 1) cluster.barrier_arrive();  // waited for before the first write to another block
    const long row = ALONE ? (long)blockIdx.x * ROWS + own : blockIdx.x / parts;
    if (ALONE && row >= a.rows) return;
    auto sync = [] {
        if (ALONE) __syncwarp();
        else __syncthreads();
    };
    const int tid = ALONE ? threadIdx.x & 31 : threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int lo = min(a.V, part * a.stretch), hi = min(a.V, lo + a.stretch), n = hi - lo, k = a.k;
    const float *xr = a.logits + row * a.ldl, *x = xr + lo;
    const float ct = LOG2E / a.tau;
    // elements before the first 16-byte boundary, whole groups of four, the rest;
    // element i of the stretch is kept at slice[pad + i], groups at float4s
    const int head = min(n, (int)(((16 - (uintptr_t)x % 16) / 4) % 4)), quads = (n - head) / 4, pad = (4 - head) & 3;
    const int at = ALONE ? tid : tid - 32;  // among the threads of the stretch
    const int odd = at < 0 ? -1 : at < head ? at : at < n - 4 * quads ? at + 4 * quads : -1;  // this thread's of those at both ends
    float4 *s4 = (float4 *)(slice + pad + head);
    for (int q = at; at >= 0 && q < quads; q += STEP)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(s4 + q)), "l"(x + head + 4 * q) : "memory");
    if (odd >= 0)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(slice + pad + odd)), "l"(x + odd) : "memory");
    asm volatile("cp.async.commit_group;" ::: "memory");

    // the list, where it counts, and the student's logits at its tokens
    float lm = -INFINITY;
    const int tgt = a.targets ? a.targets[row] : -1;
    const bool has_tgt = tgt >= 0 && tgt < a.V;
    const float xt = has_tgt ? xr[tgt] : 0.0f;
    if (warp == 0) {
        for (int j = lane; j < k; j += 32) {
            const int i = a.ti[row * k + j];
            const float v = a.tv[row * k + j];
            const bool ok = i >= 0 && i < a.V && v > -INFINITY;
            si[j] = ok ? i : -1;
            sp[j] = ok ? v : -INFINITY;
            sx[j] = ok ? xr[i] : 0.0f;
            lm = fmaxf(lm, sp[j]);
        }
        lm = warp_max(lm);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // statistics of the thread, the warp, the block and the row, in a fixed order
    Stats s{-INFINITY, 0.0f, 0.0f};
    for (int q = at; at >= 0 && q < quads; q += STEP) {
        const float4 v = s4[q];
        s.m = fmaxf(s.m, fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)));
    }
    if (odd >= 0) s.m = fmaxf(s.m, slice[pad + odd]);
    {
        const float m = warp_max(s.m), rt = scaled_max(m, ct), r1 = scaled_max(m, LOG2E);
        auto add = [&](float v) {
            s.st += ex2(fmaf(v, ct, -rt));
            if (BOTH) s.s1 += ex2(fmaf(v, LOG2E, -r1));
        };
#pragma unroll 2
        for (int q = at; at >= 0 && q < quads; q += STEP) {
            const float4 v = s4[q];
            add(v.x);
            add(v.y);
            add(v.z);
            add(v.w);
        }
        if (odd >= 0) add(slice[pad + odd]);
        s.m = m;
        s.st = warp_sum(s.st);
        if (BOTH) s.s1 = warp_sum(s.s1);
    }
    if (lane == 0) sw[warp] = s;
    if (tid == 0) soft_list = lm > -INFINITY;
    sync();
    auto join = [&](const Stats *v, int count) {
        float m = v[0].m;
        for (int w = 1; w < count; ++w) m = fmaxf(m, v[w].m);
        Stats r{m, 0.0f, 0.0f};
        for (int w = 0; w < count; ++w) {
            Stats u = v[w];
            raise<BOTH>(u, m, ct);
            r.st += u.st;
            r.s1 += u.s1;
        }
        return r;
    };
    if (parts > 1) {
        if (warp == 0) s = join(sw, NT / 32);
        cluster.barrier_wait();
        if (tid < parts) *cluster.map_shared_rank(&sc[part], tid) = s;
        cluster.sync();  // also: every block has read what another one will overwrite
        s = join(sc, parts);
    } else {
        s = join(sw, NT / 32);
    }
    const float rt = scaled_max(s.m, ct), r1 = scaled_max(s.m, LOG2E);
    const bool live = !(s.m == -INFINITY && s.st == 0.0f);
    const bool soft = live && soft_list, hard = live && has_tgt;
    if (warp == 0) {
        float loss = 0.0f;
        if (soft) {
            const float it = 1.0f / a.tau;
            float lz = 0.0f;
            for (int j = lane; j < k; j += 32) lz += sp[j] > -INFINITY ? expf((sp[j] - lm) * it) : 0.0f;
            lz = warp_sum(lz);
            const float llz = logf(lz), l2 = log2f(s.st);
            for (int j = lane; j < k; j += 32) {
                const float z = (sp[j] - lm) * it;
                const float p = sp[j] > -INFINITY ? expf(z) / lz : 0.0f;
                if (p > 0.0f) loss += p * ((z - llz) - LN2 * (fmaf(sx[j], ct, -rt) - l2));
                sp[j] = p;
            }
            loss = warp_sum(loss) * (a.alpha * a.tau * a.tau);
        }
        if (hard) loss -= (1.0f - a.alpha) * (LN2 * (fmaf(xt, LOG2E, -r1) - log2f(BOTH ? s.s1 : 1.0f)));
        if (part == 0 && lane == 0) a.row_loss[row] = loss;
    }
    if (!GRAD) return;
    float *dr = a.dlogits + row * a.ldd, *d = dr + lo;
    const float ot = a.scale * a.alpha * a.tau, o1 = a.scale * (1.0f - a.alpha);
    const float gt = soft ? ot / s.st : 0.0f, g1 = BOTH && hard ? o1 / s.s1 : 0.0f;
    const bool none = !soft && !hard;
    auto grad = [&](float v) {
        float g = gt * ex2(fmaf(v, ct, -rt));
        if (BOTH) g = fmaf(g1, ex2(fmaf(v, LOG2E, -r1)), g);
        return none ? 0.0f : g;
    };
    if (odd >= 0) d[odd] = grad(slice[pad + odd]);
    if (((uintptr_t)(d + head) & 15) == 0 && at >= 0) {  // the groups of x are groups of d too
#pragma unroll 2
        for (int q = at; q < quads; q += STEP) {
            const float4 v = s4[q];
            __stcs((float4 *)(d + head) + q, make_float4(grad(v.x), grad(v.y), grad(v.z), grad(v.w)));
        }
    } else if (at >= 0) {  // another alignment: element by element, from the whole block's copies
        for (int i = head + at; i < head + 4 * quads; i += STEP) d[i] = grad(slice[pad + i]);
    }
    if (none) return;
    sync();
    // entries of the list and the target in this stretch: written again with
    // their own part taken off, by the first entry of a token for all of its
    if (warp != 0) return;
    if (lane == 0) {
        twice = 0;
        listed = 0;
    }
    __syncwarp();
    auto mine = [&](int j) { return si[j] >= lo && si[j] < hi; };
    if (soft) {
        // the stretch has done its service: every entry leaves its number at its
        // token, and one that finds another there has company
        for (int j = lane; j < k; j += 32)
            if (mine(j)) slice[pad + si[j] - lo] = __int_as_float(j);
        __syncwarp();
        for (int j = lane; j < k; j += 32)
            if (mine(j)) {
                if (__float_as_int(slice[pad + si[j] - lo]) != j) twice = 1;
                if (si[j] == tgt) listed = 1;
            }
        __syncwarp();
        const bool search = twice;
        for (int j = lane; j < k; j += 32) {
            if (!mine(j)) continue;
            float p = sp[j];
            if (search) {
                bool first = true;
                p = 0.0f;
                for (int l = 0; l < k; ++l)
                    if (si[l] == si[j]) {
                        first &= l >= j;
                        p += sp[l];
                    }
                if (!first) continue;
            }
            float g = grad(sx[j]) - ot * p;
            if (hard && si[j] == tgt) g -= o1;
            dr[si[j]] = g;
        }
        __syncwarp();
    }
    if (hard && tgt >= lo && tgt < hi && lane == 0 && !listed) dr[tgt] = grad(xt) - o1;
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

template <bool GRAD, bool BOTH, bool ALONE>
int launch_as(const DistillArgs &a, int rows, int parts, cudaStream_t s) {
    static bool set_on[MAX_DEVICES];
    bool *set;
    CG_TRY(this_device(set_on, &set));
    if (!*set) {
        CG_CUDA(cudaFuncSetAttribute(distill_kernel<GRAD, BOTH, ALONE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     ALONE ? ROWS * (4096 * 4 + 64 + 12 * TOPK_MAX)
                                           : ROW_MAX_VOCAB / MAX_PARTS * 4 + 64 + 12 * TOPK_MAX));
        *set = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ALONE ? (unsigned)((rows - 1) / ROWS + 1) : (unsigned)(rows * parts));
    cfg.blockDim = dim3(ALONE ? 32 * ROWS : 32 + COPY);
    cfg.dynamicSmemBytes = row_bytes(a.stretch, a.k) * (ALONE ? ROWS : 1);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)parts;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    CG_CUDA(cudaLaunchKernelEx(&cfg, distill_kernel<GRAD, BOTH, ALONE>, a));
    ++g_launch_count;
    return OK;
}

template <bool GRAD, bool BOTH>
int launch(const DistillArgs &a, int rows, int parts, bool alone, cudaStream_t s) {
    return alone ? launch_as<GRAD, BOTH, true>(a, rows, parts, s) : launch_as<GRAD, BOTH, false>(a, rows, parts, s);
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
    // Short rows of which every SM gets some leave a block's warps waiting for one
    // another: a warp each (7000 x 500 with gradient 18 us, 61 by blocks; 7000 x 2600 47
    // us, 80; 600 x 2600 11.8 us, 13.8; 150 x 2600 10.4, 8.5).
    const bool alone = parts == 1 && (V <= 512 || (V <= 4096 && rows >= 2 * num_sms()));
    if ((long)rows * parts > 0x7FFFFFFFL) {
        set_last_error(ERR_ARG, "distill: %d rows are too many", rows);
        return ERR_ARG;
    }
    DistillArgs a{logits, ldl, rows, V, ((V + parts - 1) / parts + 3) / 4 * 4, tv, ti, k, targets, tau, alpha, scale, row_loss,
                  dlogits, ldd};
    if (alpha < 1.0f && targets)
        return dlogits ? launch<true, true>(a, rows, parts, alone, s) : launch<false, true>(a, rows, parts, alone, s);
    return dlogits ? launch<true, false>(a, rows, parts, alone, s) : launch<false, false>(a, rows, parts, alone, s);
}

int distill_loss_sum(const float *row_loss, int rows, float scale, float *loss, cudaStream_t s) {
    loss_sum_kernel<<<1, 1024, 0, s>>>(row_loss, rows, scale, loss);
    LAUNCH_CHECK();
    return OK;
}

}  // namespace cg
