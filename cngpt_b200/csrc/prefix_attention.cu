// prefix_attention.cu - decode attention of sequences that share a prefix
// (cngpt_cuda_prefix_attention).
//
// out = softmax(scale q K^T) V over the prefix's and the sequence's own keys.
// For a set of keys the triple (m, l, o) = (max s, sum 2^(s - m), sum 2^(s - m) v)
// with s = scale log2(e) q.k is enough: triples of disjoint sets join by
// rescaling to the larger m. Three kernels form and join them:
//
//   prefix_part_kernel  all B * (n_head / n_kv_head) queries of a key/value head
//                       against a stretch of the prefix, on the tensor cores:
//                       the prefix is read once for all of them;
//   suffix_part_kernel  a sequence's own queries against a stretch of its own
//                       keys, on the CUDA cores: every key is used by one
//                       sequence only, so its bytes set the time;
//   join_kernel         a query's triples, in the order of the stretches.
//
//
// Few keys take direct_kernel alone. The three are chained by programmatic dependent launch, so the suffix blocks
// fill the SMs that the prefix blocks leave.
//
// On B200: 48 samples x 16 heads of 64 over 16384 shared keys and up to 512 own (36 us
// of bytes): 94 us, of which the prefix takes 76 us at half the tf32 mma.sync rate
// (276 TFLOP/s measured; three products a product), the suffixes partly beside it;
// 16 samples x 12 heads, 768 + 255 keys (4.6 us of bytes): 13.1 us; 12 samples x 24
// heads of 128 over 6, 5003 + 77 keys (5.2 us): 31 us; one sample, 109 keys: 4.0 us
// in one launch (direct_kernel). fp16 products with scaled rows need half the tensor time and gave
// half the error, but took as long: splitting the rows then sets the pace.
#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "kernels.h"

namespace cg {
namespace {

#define LAUNCH_CHECK() do { ++g_launch_count; CG_CUDA(cudaGetLastError()); } while (0)

constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// not volatile: independent products may be interleaved
__device__ __forceinline__ void mma8(float (&d)[4], const uint32_t *a, uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// d = a b: the first product of a sum
__device__ __forceinline__ void mma8_first(float (&d)[4], const uint32_t *a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

// x = hi + lo in two tf32 numbers. Rounded: hi is x to 11 significant bits (half
// away from zero, on the bit pattern), lo the exact rest with half a step added
// before the tensor core cuts it to 11 bits: x to 2^-23. For what is loaded anew
// for every tile (K, V) both are cut, two instructions for four: x to 2^-21,
// 2^-22 on average and towards zero, so a score or an output shrinks by 1e-7.
__device__ __forceinline__ void split_tf32(float x, uint32_t &hi, uint32_t &lo) {
    hi = (__float_as_uint(x) + 0x1000u) & 0xFFFFE000u;
    lo = __float_as_uint(x - __uint_as_float(hi)) + 0x1000u;
}
__device__ __forceinline__ void cut_tf32(float x, uint32_t &hi, uint32_t &lo) {
    hi = __float_as_uint(x) & 0xFFFFE000u;
    lo = __float_as_uint(x - __uint_as_float(hi));
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], const float *p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_u32(p)));
}

__device__ __forceinline__ void cp_async16(float *dst, const float *src, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(float *dst, const float *src, bool ok) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(ok ? 4 : 0) : "memory");
}

struct Parts {  // the triples, [stretch][B * H]
    float *o;     // [pitch] each, pitch = hs rounded up to 4
    float2 *ml;
    int pitch;
    int n_pre, chunk;      // prefix stretches and their keys
    int n_suf, suf_chunk;  // suffix stretches (of the capacity) and their keys
};

// ------------------------------------------------------------------ prefix
constexpr int TK = 64;       // keys of a tile

template <int HSP, int RG>
struct PrefixCfg {
    // key groups: 8 warps up to two row groups, four warps a row group beyond
    static constexpr int KG = RG == 1 ? 8 : 4, WARPS = RG * KG, KW = TK / KG;
    static constexpr bool QREG = RG <= 2 && HSP <= 64;  // fragments of Q in registers, else in shared memory
    static constexpr int QBUF = QREG ? 0 : 16 * RG * HSP * 2;
    static constexpr int LDK = HSP + 4;  // pitches without bank conflicts for ldmatrix rows and
    static constexpr int LDV = HSP + 8;  // for column-wise reads of four rows
    static constexpr int STAGE = TK * (LDK + LDV);
    static constexpr int STAGES = HSP <= 64 ? 3 : HSP <= 128 ? 2 : 1;
    static constexpr int JOIN = KG * 16 * RG * (HSP + 2);
    static constexpr int FLOATS = (STAGES * STAGE > JOIN ? STAGES * STAGE : JOIN) + QBUF;
};

// Block: 16 RG query rows of a key/value head against `chunk` keys. Warp (rg, kg)
// takes rows 16 rg .. 16 rg + 15 and the keys [KW kg, KW kg + KW) of every tile,
// with its own running maximum, so warps meet only where tiles are exchanged.
// Products are split in three (lo*hi + hi*lo + hi*hi). The tensor core truncates
// as it accumulates, so the small products of a score have their own accumulator
// and P V starts a fresh one in every tile, which is added in fp32.
// 48 rows keep 128 registers a thread, so that a suffix block fits beside them.
template <int HSP, int RG, bool SPLIT>
__global__ void __launch_bounds__(RG == 3 ? 512 : PrefixCfg<HSP, RG>::WARPS * 32, 1)
prefix_part_kernel(PrefixAttn a, Parts w, int n_tiles, bool vec) {
    using Cfg = PrefixCfg<HSP, RG>;
    constexpr int KG = Cfg::KG, KW = Cfg::KW, NK = KW / 8, KK = HSP / 8, ND = HSP / 8;
    constexpr int NT = Cfg::WARPS * 32;
    extern __shared__ float sm[];
    pdl_trigger();
    const int split = blockIdx.x % w.n_pre, tile = blockIdx.x / w.n_pre % n_tiles, hk = blockIdx.x / w.n_pre / n_tiles;
    const int G = a.H / a.Hk, R = a.B * G, hs = a.hs;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rg = warp % RG, kg = warp / RG;
    const int k_lo = split * w.chunk, k_hi = min(a.P, k_lo + w.chunk);
    const int tiles = (k_hi - k_lo + TK - 1) / TK;
    const float *kbase = a.pk + (long)hk * hs, *vbase = a.pv + (long)hk * hs;

    auto load = [&](int i) {
        float *dk = sm + (i % Cfg::STAGES) * Cfg::STAGE, *dv = dk + TK * Cfg::LDK;
        const int k0 = k_lo + i * TK;
        if (vec) {
#pragma unroll
            for (int c = 0; c < (TK * (HSP / 4) + NT - 1) / NT; ++c) {
                const int e = c * NT + threadIdx.x, r = e / (HSP / 4), d = e % (HSP / 4) * 4;
                if (TK * (HSP / 4) % NT && r >= TK) break;
                const bool ok = k0 + r < k_hi && d < hs;
                const long at = ok ? (long)(k0 + r) * a.ldp + d : 0;
                cp_async16(dk + r * Cfg::LDK + d, kbase + at, ok);
                cp_async16(dv + r * Cfg::LDV + d, vbase + at, ok);
            }
        } else {
            for (int e = threadIdx.x; e < TK * HSP; e += NT) {
                const int r = e / HSP, d = e % HSP;
                const bool ok = k0 + r < k_hi && d < hs;
                const long at = ok ? (long)(k0 + r) * a.ldp + d : 0;
                cp_async4(dk + r * Cfg::LDK + d, kbase + at, ok);
                cp_async4(dv + r * Cfg::LDV + d, vbase + at, ok);
            }
        }
    };
    constexpr int AHEAD = Cfg::STAGES > 1 ? Cfg::STAGES - 1 : 1;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
        if (i < tiles) load(i);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }

    // the rows' fragments of Q scale log2(e), split
    constexpr int QK = Cfg::QREG ? KK : 1;
    uint32_t qh[QK][4], ql[QK][4];
    uint4 *sq = (uint4 *)(sm + Cfg::FLOATS - Cfg::QBUF) + rg * KK * 64 + lane;  // [KK][hi, lo][32 lanes] of the row group
    {
        const float sc = a.scale * LOG2E;
        const int r0 = tile * 16 * RG + rg * 16 + g, r1 = r0 + 8;
        auto row = [&](int r) { return a.q + (long)(r / G) * a.ldq + (long)(hk * G + r % G) * hs; };
        const float *p0 = row(min(r0, R - 1)), *p1 = row(min(r1, R - 1));
        auto fragment = [&](int k, uint32_t (&h)[4], uint32_t (&l)[4]) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = 8 * k + t + (e >> 1) * 4;
                const bool ok = d < hs && ((e & 1) ? r1 : r0) < R;
                const float v = ok ? ((e & 1) ? p1 : p0)[d] * sc : 0.0f;
                if constexpr (SPLIT) split_tf32(v, h[e], l[e]);
                else h[e] = l[e] = __float_as_uint(v);
            }
        };
        if constexpr (Cfg::QREG) {
#pragma unroll
            for (int k = 0; k < KK; ++k) fragment(k, qh[k], ql[k]);
        } else {
            for (int k = kg; k < KK; k += KG) {  // the first tile's barrier shows them to the group
                fragment(k, qh[0], ql[0]);
                sq[k * 64] = make_uint4(qh[0][0], qh[0][1], qh[0][2], qh[0][3]);
                sq[k * 64 + 32] = make_uint4(ql[0][0], ql[0][1], ql[0][2], ql[0][3]);
            }
        }
    }

    float o[ND][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    for (int i = 0; i < tiles; ++i) {
        if constexpr (Cfg::STAGES > 1) asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD - 1) : "memory");
        else asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();  // tile i is there, and every warp is done with tile i - 1
        if constexpr (Cfg::STAGES > 1) {
            if (i + AHEAD < tiles) load(i + AHEAD);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        const float *sk = sm + (i % Cfg::STAGES) * Cfg::STAGE, *sv = sk + TK * Cfg::LDK;
        const int valid = min(TK, k_hi - k_lo - i * TK);
        if (kg * KW < valid) {
            float s[NK][4], sl[NK][4];
            // accumulator column n of a group of 8 holds key (n >> 1) + 4 (n & 1),
            // so that a thread's two columns are the keys t and t + 4 of the A
            // fragment that the same registers form in P V
            const float *kr = sk + (kg * KW + ((lane & 7) >> 1) + 4 * (lane & 1)) * Cfg::LDK + (lane >> 3) * 4;
#pragma unroll
            for (int k = 0; k < KK; k += 2) {
                uint32_t b[NK][4];
#pragma unroll
                for (int j = 0; j < NK; ++j) ldsm4(b[j], kr + j * 8 * Cfg::LDK + k * 8);
                // the products of one kind over all keys in a row: none waits for the one before
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    uint32_t ah[4], al[4];
                    if constexpr (Cfg::QREG) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            ah[e] = qh[k + u][e];
                            al[e] = ql[k + u][e];
                        }
                    } else {
                        const uint4 x = sq[(k + u) * 64], y = SPLIT ? sq[(k + u) * 64 + 32] : x;
                        ah[0] = x.x, ah[1] = x.y, ah[2] = x.z, ah[3] = x.w;
                        al[0] = y.x, al[1] = y.y, al[2] = y.z, al[3] = y.w;
                    }
                    if constexpr (SPLIT) {
                        uint32_t h[NK][2], l[NK][2];
#pragma unroll
                        for (int j = 0; j < NK; ++j) {
                            cut_tf32(__uint_as_float(b[j][2 * u]), h[j][0], l[j][0]);
                            cut_tf32(__uint_as_float(b[j][2 * u + 1]), h[j][1], l[j][1]);
                        }
#pragma unroll
                        for (int j = 0; j < NK; ++j)
                            k + u ? mma8(sl[j], al, h[j][0], h[j][1]) : mma8_first(sl[j], al, h[j][0], h[j][1]);
#pragma unroll
                        for (int j = 0; j < NK; ++j)
                            k + u ? mma8(s[j], ah, h[j][0], h[j][1]) : mma8_first(s[j], ah, h[j][0], h[j][1]);
#pragma unroll
                        for (int j = 0; j < NK; ++j) mma8(sl[j], ah, l[j][0], l[j][1]);
                    } else {
#pragma unroll
                        for (int j = 0; j < NK; ++j)
                            k + u ? mma8(s[j], ah, b[j][2 * u], b[j][2 * u + 1])
                                  : mma8_first(s[j], ah, b[j][2 * u], b[j][2 * u + 1]);
                    }
                }
            }
            float mx[2] = {m[0], m[1]};
            if (SPLIT)
#pragma unroll
                for (int j = 0; j < NK; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[j][e] += sl[j][e];
            if (valid < TK)  // the last tile
#pragma unroll
                for (int j = 0; j < NK; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (kg * KW + j * 8 + t + (e & 1) * 4 >= valid) s[j][e] = -INFINITY;
#pragma unroll
            for (int j = 0; j < NK; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) mx[e >> 1] = fmaxf(mx[e >> 1], s[j][e]);
            float c[2], ref[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
                ref[r] = mx[r] == -INFINITY ? 0.0f : mx[r];
                c[r] = ex2(m[r] - ref[r]);
                m[r] = mx[r];
                l[r] *= c[r];
            }
            uint32_t ph[NK][4], pl[NK][4];
#pragma unroll
            for (int j = 0; j < NK; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float p = ex2(s[j][e] - ref[e >> 1]);
                    l[e >> 1] += p;
                    const int x = (e >> 1) + 2 * (e & 1);  // C fragment {0,1,2,3} -> A fragment {0,2,1,3}
                    if constexpr (SPLIT) split_tf32(p, ph[j][x], pl[j][x]);
                    else ph[j][x] = __float_as_uint(p);
                }
            const float *vr = sv + (kg * KW + t) * Cfg::LDV + g;
#pragma unroll
            for (int n0 = 0; n0 < ND; n0 += 4) {
                float acc[4][4];  // the tile's own sum, the small products first
#pragma unroll
                for (int j = 0; j < NK; ++j) {
                    float v[4][2];
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        v[n][0] = vr[j * 8 * Cfg::LDV + (n0 + n) * 8];
                        v[n][1] = vr[(j * 8 + 4) * Cfg::LDV + (n0 + n) * 8];
                    }
                    if constexpr (SPLIT) {
                        uint32_t h[4][2], l[4][2];
#pragma unroll
                        for (int n = 0; n < 4; ++n) {
                            cut_tf32(v[n][0], h[n][0], l[n][0]);
                            cut_tf32(v[n][1], h[n][1], l[n][1]);
                        }
#pragma unroll
                        for (int n = 0; n < 4; ++n)
                            j ? mma8(acc[n], pl[j], h[n][0], h[n][1]) : mma8_first(acc[n], pl[j], h[n][0], h[n][1]);
#pragma unroll
                        for (int n = 0; n < 4; ++n) mma8(acc[n], ph[j], l[n][0], l[n][1]);
#pragma unroll
                        for (int n = 0; n < 4; ++n) mma8(acc[n], ph[j], h[n][0], h[n][1]);
                    } else {
#pragma unroll
                        for (int n = 0; n < 4; ++n) {
                            const uint32_t v0 = __float_as_uint(v[n][0]), v1 = __float_as_uint(v[n][1]);
                            j ? mma8(acc[n], ph[j], v0, v1) : mma8_first(acc[n], ph[j], v0, v1);
                        }
                    }
                }
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        o[n0 + n][e] = fmaf(o[n0 + n][e], c[e >> 1], acc[n][e]);
            }
        }
        if constexpr (Cfg::STAGES == 1) {
            __syncthreads();
            if (i + 1 < tiles) load(i + 1);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();

    // join the KG warps of a row group, in their order
    float *so = sm;                                       // [KG][16 RG][HSP]
    float2 *sml = (float2 *)(so + KG * 16 * RG * HSP);    // [KG][16 RG]
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        const int rr = rg * 16 + g + 8 * r;
        if (t == 0) sml[kg * 16 * RG + rr] = make_float2(m[r], l[r]);
#pragma unroll
        for (int n = 0; n < ND; ++n)
            *(float2 *)(so + (kg * 16 * RG + rr) * HSP + n * 8 + 2 * t) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
    }
    __syncthreads();
    const long BH = (long)a.B * a.H;
    for (int e = threadIdx.x; e < 16 * RG * HSP; e += NT) {
        const int rr = e / HSP, d = e % HSP, r = tile * 16 * RG + rr;
        if (r >= R) continue;
        float mm = -INFINITY;
#pragma unroll
        for (int k = 0; k < KG; ++k) mm = fmaxf(mm, sml[k * 16 * RG + rr].x);
        const float ref = mm == -INFINITY ? 0.0f : mm;
        float ll = 0.0f, oo = 0.0f;
#pragma unroll
        for (int k = 0; k < KG; ++k) {
            const float2 p = sml[k * 16 * RG + rr];
            const float f = ex2(p.x - ref);
            ll = fmaf(p.y, f, ll);
            oo = fmaf(so[(k * 16 * RG + rr) * HSP + d], f, oo);
        }
        const long id = split * BH + (long)(r / G) * a.H + hk * G + r % G;
        if (d < hs) w.o[id * w.pitch + d] = oo;
        if (d == 0) w.ml[id] = make_float2(mm, ll);
    }
}

// ------------------------------------------------------------------ suffix
// Block: one sequence, one key/value head, one stretch of CH keys. LPK lanes hold
// one key's row (NF float4 each), so a warp reads 32 / LPK whole rows at a time;
// all K and V rows of the stretch are on their way before the first is used.
constexpr int SWARPS = 4;

template <int LPK, int NF>
struct SuffixCfg {
    static constexpr int KPI = 32 / LPK, ITER = 8 / NF, CH = SWARPS * KPI * ITER;
};

__device__ __forceinline__ float4 row4(const float *p, int d, int hs, bool ok, bool vec) {
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (!ok) return v;
    if (vec) {
        if (d < hs) v = *(const float4 *)(p + d);
    } else {
        if (d < hs) v.x = p[d];
        if (d + 1 < hs) v.y = p[d + 1];
        if (d + 2 < hs) v.z = p[d + 2];
        if (d + 3 < hs) v.w = p[d + 3];
    }
    return v;
}

template <int LPK, int NF>
__global__ void __launch_bounds__(SWARPS * 32, 4)
suffix_part_kernel(PrefixAttn a, Parts w, bool vec) {
    using Cfg = SuffixCfg<LPK, NF>;
    __shared__ float so[SWARPS][LPK * 4 * NF];
    __shared__ float2 sml[SWARPS];
    pdl_trigger();
    const int chunk = blockIdx.x % w.n_suf, hk = blockIdx.x / w.n_suf % a.Hk, b = blockIdx.x / w.n_suf / a.Hk;
    const int len = min(max(a.suffix_len[b], 0), a.S), j0 = chunk * Cfg::CH;
    if (j0 < len) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane / LPK, li = lane % LPK;
        const int G = a.H / a.Hk, hs = a.hs;
        const float *kb = a.sk + b * a.seq_stride + (long)hk * hs, *vb = a.sv + b * a.seq_stride + (long)hk * hs;
        float4 k[Cfg::ITER][NF], v[Cfg::ITER][NF];
#pragma unroll
        for (int i = 0; i < Cfg::ITER; ++i) {
            const int j = j0 + (i * SWARPS + warp) * Cfg::KPI + sub;
#pragma unroll
            for (int f = 0; f < NF; ++f) k[i][f] = row4(kb + (long)j * a.lds, (li + f * LPK) * 4, hs, j < len, vec);
        }
#pragma unroll
        for (int i = 0; i < Cfg::ITER; ++i) {
            const int j = j0 + (i * SWARPS + warp) * Cfg::KPI + sub;
#pragma unroll
            for (int f = 0; f < NF; ++f) v[i][f] = row4(vb + (long)j * a.lds, (li + f * LPK) * 4, hs, j < len, vec);
        }
        const float sc = a.scale * LOG2E;
        for (int gq = 0; gq < G; ++gq) {
            const float *qr = a.q + b * a.ldq + (long)(hk * G + gq) * hs;
            float s[Cfg::ITER] = {}, m = -INFINITY;
#pragma unroll
            for (int f = 0; f < NF; ++f) {
                const float4 q = row4(qr, (li + f * LPK) * 4, hs, true, false);
#pragma unroll
                for (int i = 0; i < Cfg::ITER; ++i)
                    s[i] = fmaf(q.x, k[i][f].x, fmaf(q.y, k[i][f].y, fmaf(q.z, k[i][f].z, fmaf(q.w, k[i][f].w, s[i]))));
            }
#pragma unroll
            for (int i = 0; i < Cfg::ITER; ++i) {
#pragma unroll
                for (int x = LPK / 2; x > 0; x >>= 1) s[i] += __shfl_xor_sync(0xffffffffu, s[i], x);
                const int j = j0 + (i * SWARPS + warp) * Cfg::KPI + sub;
                s[i] = j < len ? s[i] * sc : -INFINITY;
                m = fmaxf(m, s[i]);
            }
#pragma unroll
            for (int x = LPK; x < 32; x <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
            const float ref = m == -INFINITY ? 0.0f : m;
            float l = 0.0f;
            float4 o[NF];
#pragma unroll
            for (int f = 0; f < NF; ++f) o[f] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int i = 0; i < Cfg::ITER; ++i) {
                const float p = ex2(s[i] - ref);
                l += p;
#pragma unroll
                for (int f = 0; f < NF; ++f) {
                    o[f].x = fmaf(p, v[i][f].x, o[f].x);
                    o[f].y = fmaf(p, v[i][f].y, o[f].y);
                    o[f].z = fmaf(p, v[i][f].z, o[f].z);
                    o[f].w = fmaf(p, v[i][f].w, o[f].w);
                }
            }
#pragma unroll
            for (int x = LPK; x < 32; x <<= 1) {
                l += __shfl_xor_sync(0xffffffffu, l, x);
#pragma unroll
                for (int f = 0; f < NF; ++f) {
                    o[f].x += __shfl_xor_sync(0xffffffffu, o[f].x, x);
                    o[f].y += __shfl_xor_sync(0xffffffffu, o[f].y, x);
                    o[f].z += __shfl_xor_sync(0xffffffffu, o[f].z, x);
                    o[f].w += __shfl_xor_sync(0xffffffffu, o[f].w, x);
                }
            }
            if (gq) __syncthreads();  // the head before has been read
            if (lane == 0) sml[warp] = make_float2(m, l);
            if (sub == 0)
#pragma unroll
                for (int f = 0; f < NF; ++f) *(float4 *)&so[warp][(li + f * LPK) * 4] = o[f];
            __syncthreads();
            const long id = (long)(w.n_pre + chunk) * a.B * a.H + (long)b * a.H + hk * G + gq;
            float mm = -INFINITY, ll = 0.0f;
#pragma unroll
            for (int x = 0; x < SWARPS; ++x) mm = fmaxf(mm, sml[x].x);
            const float r2 = mm == -INFINITY ? 0.0f : mm;
            for (int d = threadIdx.x; d < hs; d += SWARPS * 32) {
                float oo = 0.0f;
#pragma unroll
                for (int x = 0; x < SWARPS; ++x) oo = fmaf(so[x][d], ex2(sml[x].x - r2), oo);
                w.o[id * w.pitch + d] = oo;
            }
            if (threadIdx.x == 0) {
#pragma unroll
                for (int x = 0; x < SWARPS; ++x) ll = fmaf(sml[x].y, ex2(sml[x].x - r2), ll);
                w.ml[id] = make_float2(mm, ll);
            }
        }
    }
    pdl_wait();  // the prefix blocks: the kernel that waits for this one waits for them too
}

// ------------------------------------------------------------------ direct
// Few keys: one block does a query's all of them, prefix and suffix, in one launch
// without the workspace; the prefix comes from L2 as often as there are queries.
// The lanes of one key's row keep their own (m, l, o), joined at the end in the order
// of lanes and warps.
constexpr int DWARPS = 16;

template <int LPK, int NF>
__global__ void __launch_bounds__(DWARPS * 32, 1)
direct_kernel(PrefixAttn a, bool vec) {
    constexpr int KPI = 32 / LPK, ITER = 8 / NF;
    __shared__ float so[DWARPS][LPK * 4 * NF];
    __shared__ float2 sml[DWARPS];
    const int h = blockIdx.x % a.H, b = blockIdx.x / a.H, hs = a.hs;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane / LPK, li = lane % LPK;
    const int n = a.P + (a.S > 0 ? min(max(a.suffix_len[b], 0), a.S) : 0);
    const long head = (long)(h / (a.H / a.Hk)) * hs, own = b * a.seq_stride;
    const float sc = a.scale * LOG2E, *qr = a.q + b * a.ldq + (long)h * hs;
    float4 q[NF], o[NF];
#pragma unroll
    for (int f = 0; f < NF; ++f) {
        q[f] = row4(qr, (li + f * LPK) * 4, hs, true, false);
        o[f] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    float m = -INFINITY, l = 0.0f;
    for (int t = warp * KPI * ITER; t < n; t += DWARPS * KPI * ITER) {
        float4 k[ITER][NF], v[ITER][NF];
        float s[ITER] = {};
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int j = t + i * KPI + sub;
            const long at = head + (j < a.P ? (long)j * a.ldp : own + (long)(j - a.P) * a.lds);
            const float *kr = (j < a.P ? a.pk : a.sk) + at, *vr = (j < a.P ? a.pv : a.sv) + at;
#pragma unroll
            for (int f = 0; f < NF; ++f) {
                k[i][f] = row4(kr, (li + f * LPK) * 4, hs, j < n, vec);
                v[i][f] = row4(vr, (li + f * LPK) * 4, hs, j < n, vec);
            }
        }
        float mx = m;
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
#pragma unroll
            for (int f = 0; f < NF; ++f)
                s[i] = fmaf(q[f].x, k[i][f].x, fmaf(q[f].y, k[i][f].y, fmaf(q[f].z, k[i][f].z, fmaf(q[f].w, k[i][f].w, s[i]))));
#pragma unroll
            for (int x = LPK / 2; x > 0; x >>= 1) s[i] += __shfl_xor_sync(0xffffffffu, s[i], x);
            s[i] = t + i * KPI + sub < n ? s[i] * sc : -INFINITY;
            mx = fmaxf(mx, s[i]);
        }
        const float ref = mx == -INFINITY ? 0.0f : mx, c = ex2(m - ref);
        m = mx;
        l *= c;
#pragma unroll
        for (int f = 0; f < NF; ++f) o[f] = make_float4(o[f].x * c, o[f].y * c, o[f].z * c, o[f].w * c);
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const float p = ex2(s[i] - ref);
            l += p;
#pragma unroll
            for (int f = 0; f < NF; ++f)
                o[f] = make_float4(fmaf(p, v[i][f].x, o[f].x), fmaf(p, v[i][f].y, o[f].y), fmaf(p, v[i][f].z, o[f].z),
                                   fmaf(p, v[i][f].w, o[f].w));
        }
    }
    // the warp's, then the block's
    float wm = m;
#pragma unroll
    for (int x = LPK; x < 32; x <<= 1) wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, x));
    const float c = ex2(m - (wm == -INFINITY ? 0.0f : wm));
    l *= c;
#pragma unroll
    for (int f = 0; f < NF; ++f) o[f] = make_float4(o[f].x * c, o[f].y * c, o[f].z * c, o[f].w * c);
#pragma unroll
    for (int x = LPK; x < 32; x <<= 1) {
        l += __shfl_xor_sync(0xffffffffu, l, x);
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            o[f].x += __shfl_xor_sync(0xffffffffu, o[f].x, x);
            o[f].y += __shfl_xor_sync(0xffffffffu, o[f].y, x);
            o[f].z += __shfl_xor_sync(0xffffffffu, o[f].z, x);
            o[f].w += __shfl_xor_sync(0xffffffffu, o[f].w, x);
        }
    }
    if (lane == 0) sml[warp] = make_float2(wm, l);
    if (sub == 0)
#pragma unroll
        for (int f = 0; f < NF; ++f) *(float4 *)&so[warp][(li + f * LPK) * 4] = o[f];
    __syncthreads();
    if ((int)threadIdx.x >= hs) return;
    float mm = -INFINITY, ll = 0.0f, oo = 0.0f;
#pragma unroll
    for (int x = 0; x < DWARPS; ++x) mm = fmaxf(mm, sml[x].x);
    const float ref = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
    for (int x = 0; x < DWARPS; ++x) {
        const float f = ex2(sml[x].x - ref);
        ll = fmaf(sml[x].y, f, ll);
        oo = fmaf(so[x][threadIdx.x], f, oo);
    }
    a.out[b * a.ldo + (long)h * hs + threadIdx.x] = n > 0 ? oo / ll : 0.0f;
}

// -------------------------------------------------------------------- join
constexpr int JT = 128, JBATCH = 4;

// Block: one query. Groups of `lp` threads (four dimensions each) take every JT / lp
// -th stretch, JBATCH of them on their way at a time; the groups' triples are then
// joined in order.
__global__ void __launch_bounds__(JT)
join_kernel(PrefixAttn a, Parts w, int lp) {
    __shared__ float4 so[JT];
    __shared__ float2 sml[JT];
    const long row = blockIdx.x, BH = (long)a.B * a.H;
    const int b = (int)(row / a.H), h = (int)(row % a.H), hs = a.hs;
    const int sub = threadIdx.x / lp, li = threadIdx.x % lp, groups = JT / lp;
    const int len = a.S > 0 ? min(max(a.suffix_len[b], 0), a.S) : 0;
    const int n = w.n_pre + (len > 0 ? (len + w.suf_chunk - 1) / w.suf_chunk : 0);
    const bool on = 4 * li < hs;
    pdl_wait();
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s0 = sub; s0 < n; s0 += JBATCH * groups) {
        float2 p[JBATCH];
        float4 v[JBATCH];
#pragma unroll
        for (int j = 0; j < JBATCH; ++j) {
            const int s = s0 + j * groups;
            p[j] = s < n ? w.ml[s * BH + row] : make_float2(-INFINITY, 0.0f);
            v[j] = s < n && on ? *(const float4 *)(w.o + (s * BH + row) * w.pitch + 4 * li) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        float mx = m;
#pragma unroll
        for (int j = 0; j < JBATCH; ++j) mx = fmaxf(mx, p[j].x);
        const float ref = mx == -INFINITY ? 0.0f : mx, c = ex2(m - ref);
        m = mx;
        l *= c;
        o = make_float4(o.x * c, o.y * c, o.z * c, o.w * c);
#pragma unroll
        for (int j = 0; j < JBATCH; ++j) {
            const float f = ex2(p[j].x - ref);
            l = fmaf(p[j].y, f, l);
            o = make_float4(fmaf(v[j].x, f, o.x), fmaf(v[j].y, f, o.y), fmaf(v[j].z, f, o.z), fmaf(v[j].w, f, o.w));
        }
    }
    so[threadIdx.x] = o;
    if (li == 0) sml[sub] = make_float2(m, l);
    __syncthreads();
    if (sub != 0 || !on) return;
    m = -INFINITY;
    for (int x = 0; x < groups; ++x) m = fmaxf(m, sml[x].x);
    const float ref = m == -INFINITY ? 0.0f : m;
    l = 0.0f;
    o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int x = 0; x < groups; ++x) {
        const float f = ex2(sml[x].x - ref);
        const float4 v = so[x * lp + li];
        l = fmaf(sml[x].y, f, l);
        o = make_float4(fmaf(v.x, f, o.x), fmaf(v.y, f, o.y), fmaf(v.z, f, o.z), fmaf(v.w, f, o.w));
    }
    const float inv = n > 0 ? 1.0f / l : 0.0f, e[4] = {o.x, o.y, o.z, o.w};
    float *out = a.out + b * a.ldo + (long)h * hs + 4 * li;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (4 * li + j < hs) out[j] = n > 0 ? e[j] * inv : 0.0f;
}

__global__ void shared_advance_kernel(int *ctr, int *suffix_len, int n) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) suffix_len[i] += 1;
    if (threadIdx.x < 3) ctr[threadIdx.x] += 1;
}

// ------------------------------------------------------------- the launches
// Rows of 16 that a block takes: up to 64 rows read a tile once. Above 128
// dimensions the tile and the queries of more than 32 rows do not fit.
int row_groups(long R, int hs) {
    if (R <= 16) return 1;
    if (R <= 32 || hs > 128) return 2;
    // 48 rows a block where that takes as few blocks as 64 would
    return (R + 47) / 48 == (R + 63) / 64 ? 3 : 4;
}

// Stretches: the prefix is cut so that its blocks fill the SMs about once (one
// block an SM), but not below one tile; the suffixes into what one block loads
// at once.
Parts plan(int B, int H, int Hk, int hs, int P, int S) {
    Parts w{};
    w.pitch = (hs + 3) / 4 * 4;
    const long R = (long)B * (H / Hk);
    const int rg = row_groups(R, hs);
    if (P > 0) {
        const long n_tiles = (R + 16 * rg - 1) / (16 * rg), tiles = (P + TK - 1) / TK;
        const long want = std::max<long>(1, 148 / std::max<long>(1, Hk * n_tiles));
        const long per = (tiles + std::min(want, tiles) - 1) / std::min(want, tiles);
        w.chunk = (int)(per * TK);
        w.n_pre = (int)((P + (long)w.chunk - 1) / w.chunk);
    }
    w.suf_chunk = hs <= 32 ? SuffixCfg<8, 1>::CH : hs <= 64 ? SuffixCfg<16, 1>::CH
                : hs <= 128 ? SuffixCfg<32, 1>::CH : SuffixCfg<32, 2>::CH;
    w.n_suf = (int)(((long)S + w.suf_chunk - 1) / w.suf_chunk);
    return w;
}

template <class K, class... A>
int launch_pdl(K kernel, long grid, int threads, size_t smem, bool chained, cudaStream_t s, A... args) {
    if (grid > 0x7FFFFFFFL) {
        set_last_error(ERR_ARG, "prefix_attention: %ld blocks are too many", grid);
        return ERR_ARG;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = chained ? 1 : 0;
    CG_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
    ++g_launch_count;
    return OK;
}

template <int HSP, int RG, bool SPLIT>
int launch_prefix(const PrefixAttn &a, const Parts &w, cudaStream_t s) {
    using Cfg = PrefixCfg<HSP, RG>;
    constexpr size_t smem = (size_t)Cfg::FLOATS * sizeof(float);
    static_assert(smem <= 227 * 1024, "shared memory of a block");
    static bool set_on[MAX_DEVICES];
    bool *set;
    CG_TRY(this_device(set_on, &set));
    if (!*set) {
        CG_CUDA(cudaFuncSetAttribute(prefix_part_kernel<HSP, RG, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)smem));
        *set = true;
    }
    const long R = (long)a.B * (a.H / a.Hk), n_tiles = (R + 16 * RG - 1) / (16 * RG);
    const bool vec = a.hs % 4 == 0 && a.ldp % 4 == 0 && ((uintptr_t)a.pk | (uintptr_t)a.pv) % 16 == 0;
    return launch_pdl(prefix_part_kernel<HSP, RG, SPLIT>, (long)w.n_pre * n_tiles * a.Hk, Cfg::WARPS * 32, smem, false, s, a, w,
                      (int)n_tiles, vec);
}

template <int HSP, bool SPLIT>
int dispatch_rows(const PrefixAttn &a, const Parts &w, cudaStream_t s) {
    const int rg = row_groups((long)a.B * (a.H / a.Hk), a.hs);
    if (rg == 1) return launch_prefix<HSP, 1, SPLIT>(a, w, s);
    if constexpr (HSP <= 128) {
        if (rg == 3) return launch_prefix<HSP, 3, SPLIT>(a, w, s);
        if (rg == 4) return launch_prefix<HSP, 4, SPLIT>(a, w, s);
    }
    return launch_prefix<HSP, 2, SPLIT>(a, w, s);
}

template <bool SPLIT>
int dispatch_hs(const PrefixAttn &a, const Parts &w, cudaStream_t s) {
    if (a.hs <= 32) return dispatch_rows<32, SPLIT>(a, w, s);
    if (a.hs <= 64) return dispatch_rows<64, SPLIT>(a, w, s);
    if (a.hs <= 96) return dispatch_rows<96, SPLIT>(a, w, s);
    if (a.hs <= 128) return dispatch_rows<128, SPLIT>(a, w, s);
    return dispatch_rows<256, SPLIT>(a, w, s);
}

}  // namespace

int shared_advance(int *ctr, int *suffix_len, int n, cudaStream_t s) {
    shared_advance_kernel<<<1, 256, 0, s>>>(ctr, suffix_len, n);
    LAUNCH_CHECK();
    return OK;
}

size_t prefix_attention_ws_bytes(int B, int H, int Hk, int hs, int P, int S) {
    const Parts w = plan(B, H, Hk, hs, P, S);
    const size_t rows = (size_t)(w.n_pre + w.n_suf) * B * H;
    return rows * (w.pitch * sizeof(float) + sizeof(float2));
}

int prefix_attention(const PrefixAttn &a, void *ws, cudaStream_t s) {
    if (a.B <= 0) return OK;
    // One launch where that is no longer than three: 109 keys, 12 queries 4.0 us (6.6),
    // 16 x 12 queries 6.9 (8.2), 355 keys 11.0 (11.1); but 528 keys 14.7 (10.7), and
    // 48 x 12 queries, four rounds of blocks, 109 keys 12.7 (12.1).
    if ((long)a.P + a.S <= 384 && (long)a.B * a.H <= 2 * num_sms()) {
        const bool vec = a.hs % 4 == 0 &&
                         (a.P == 0 || (a.ldp % 4 == 0 && ((uintptr_t)a.pk | (uintptr_t)a.pv) % 16 == 0)) &&
                         (a.S == 0 || ((a.lds | a.seq_stride) % 4 == 0 && ((uintptr_t)a.sk | (uintptr_t)a.sv) % 16 == 0));
        auto go = [&](auto kernel) { return launch_pdl(kernel, (long)a.B * a.H, DWARPS * 32, 0, false, s, a, vec); };
        if (a.hs <= 32) return go(direct_kernel<8, 1>);
        if (a.hs <= 64) return go(direct_kernel<16, 1>);
        if (a.hs <= 128) return go(direct_kernel<32, 1>);
        return go(direct_kernel<32, 2>);
    }
    Parts w = plan(a.B, a.H, a.Hk, a.hs, a.P, a.S);
    w.o = (float *)ws;
    const size_t rows = (size_t)(w.n_pre + w.n_suf) * a.B * a.H;
    w.ml = (float2 *)(w.o + rows * w.pitch);
    bool chained = false;
    if (w.n_pre > 0) {
        CG_TRY(precision() == PREC_TF32 ? dispatch_hs<false>(a, w, s) : dispatch_hs<true>(a, w, s));
        chained = true;
    }
    if (w.n_suf > 0) {
        const bool vec = a.hs % 4 == 0 && a.lds % 4 == 0 && a.seq_stride % 4 == 0 &&
                         ((uintptr_t)a.sk | (uintptr_t)a.sv) % 16 == 0;
        const long grid = (long)w.n_suf * a.Hk * a.B;
        auto go = [&](auto kernel) { return launch_pdl(kernel, grid, SWARPS * 32, 0, chained, s, a, w, vec); };
        if (a.hs <= 32) CG_TRY(go(suffix_part_kernel<8, 1>));
        else if (a.hs <= 64) CG_TRY(go(suffix_part_kernel<16, 1>));
        else if (a.hs <= 128) CG_TRY(go(suffix_part_kernel<32, 1>));
        else CG_TRY(go(suffix_part_kernel<32, 2>));
        chained = true;
    }
    int lp = 8;  // threads of a row in the join
    while (4 * lp < a.hs) lp *= 2;
    return launch_pdl(join_kernel, (long)a.B * a.H, JT, 0, chained, s, a, w, lp);
}

}  // namespace cg
