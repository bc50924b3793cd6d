// sample.cu - one token per row of logits from given uniform numbers, with
// temperature, top-k, top-p and min-p of every row (cngpt_cuda_sample).
//
// A token's rank is that of its 64-bit key (ordered bits of the logit, then the
// inverted index), its weight exp((l - max) / T) in fixed point: 2^SH parts of the
// largest weight, SH = 62 - log2(vocabulary), 50 at most, at least one part if it is not zero
// in 64-bit floating point. Sums of such weights are exact whatever their order,
// so atomics and any split of the row give the same token; a weight itself is right
// to 1e-9, in fp32 and integer instructions (in fp64 ones it took twice as long).
//
// A cluster of blocks holds the row in shared memory. Few tokens decide, and they
// are found without ranking the others: a bar from the threads' maxima, which at
// least k tokens (top-k up to 256) or some 300 (top-p) reach, or the bound of min-p.
// With top-p one pass sums all weights and those from the bar on: do these hold top-p
// of the whole, the border is among them. Up to 512 such tokens are ranked and drawn
// from by one block. Otherwise both cuts of the ranking
// (top-k: the first k keys; top-p: the keys before which less than p of the weight
// lies) are thresholds on the key, found alike: a histogram of the counts or
// weights over 1024 bins of the span in question, whose prefix sums give the bin that the
// border falls into; the few hundred keys of that bin are then compared with one
// another. Where a bin holds more than that (runs of equal logits, outliers that
// stretch the bins), it is cut again by the bits of its keys until it does not.
//
// On B200: 1 x 50257 with top-k and top-p 12.8 us, 64 rows with min-p 11 us, 32 rows
// with settings of their own 24 us, 256 rows by top-p alone 93 us (reading them:
// 7.9 us; a histogram of every row 122 us). The last is bound by instruction issue:
// some 60 a logit for its weight, and 15 % of the rows there have a nucleus of
// thousands, whose histograms' atomics (30 cycles a warp) make them twice as long.
#include <algorithm>
#include <cfloat>
#include <cmath>

#include <cooperative_groups.h>

#include "common.cuh"
#include "kernels.h"
#include "rank.cuh"

namespace cg {
namespace {

namespace coop = cooperative_groups;

typedef unsigned long long u64;

constexpr int NT = 256;
constexpr int WARPS = NT / 32;
constexpr int MAX_PARTS = 8;
constexpr int SLICE_BYTES = 52 * 1024;  // of a row in a block's shared memory: three blocks an SM
constexpr int BINS = 4 * NT;
constexpr int TABLE = 256;   // entries of the exponential, for 2^(-j / 256)
constexpr double SHIFT = 0.51;  // the entries are those of j - SHIFT
constexpr int BORDER = 512;  // keys that are compared with one another
constexpr float ALL = NAN;   // as a high end: no logit is at or above it

__device__ __forceinline__ u64 make_key(uint32_t rank, int i) { return ((u64)rank << 32) | (0xFFFFFFFFu - (uint32_t)i); }

// 2^31 2^((SHIFT - j) / TABLE) from the Taylor series of e^x
struct Pow2 {
    uint32_t v[TABLE];
    constexpr Pow2() : v() {
        for (int j = 0; j < TABLE; ++j) {
            const double x = 0.6931471805599453 * (SHIFT - j) / TABLE;
            double term = 1.0, sum = 0.0;
            for (int n = 1; n < 30; ++n) {
                sum += term;
                term *= x / n;
            }
            v[j] = (uint32_t)(sum * 2147483648.0 + 0.5);
        }
    }
};
__device__ const Pow2 pow2_table;

struct Border {  // what a block has of the border's bin
    int count;
    u64 lowest, highest;
};

struct Smem {
    union {
        struct {
            uint32_t lo[BINS], hi[BINS];  // a bin's count, or its weight in two halves
        };
        struct {
            u64 key[BORDER], measure[BORDER];  // the border's keys of all blocks
        };
    };
    uint32_t table[TABLE];
    u64 list[BORDER];  // this block's keys of the border
    Border mine;
    float max_of[MAX_PARTS], min_of[MAX_PARTS];
    u64 total_of[MAX_PARTS], upper_of[MAX_PARTS], sum_of[MAX_PARTS];
    float bar_of[MAX_PARTS];
    int first_of[MAX_PARTS];
    union {
        struct {
            uint32_t fine_lo[NT], fine_hi[NT];
        };
        int index_of[BORDER];
    };
    union {
        short list_of[BORDER];
        int slot[BORDER];
    };
    __align__(16) uint32_t rank_of[BORDER];
    int few;
    u64 warp[WARPS], upper[WARPS];
    float fwarp[3][WARPS];
    float bar;
    __align__(16) float own[NT];
    int bin;
    u64 above, cut;
};

struct Row {
    const float *s;  // the block's stretch in shared memory
    int n, lo, per;  // its length, the index of its first token, tokens of a thread (odd: no bank conflicts)
    float mx, mf;    // the row's largest logit, and the largest finite one up to it
    double m, t, it; // maximum, temperature, 1 / temperature
    float ch, cl;    // TABLE log2(e) / temperature in two parts
    int sh;
    const uint32_t *table;
    float cut_at;    // tokens above this logit stay, and of those at it
    int cut_index;   // the ones up to this index

    __device__ bool keeps(float x, int i) const { return x > cut_at || (x == cut_at && i <= cut_index); }
    // drops what weighs less than min_p: log w >= log min_p as a bound on the logit,
    // rounded up to the next one
    __device__ void least(float min_p) {
        if (!(min_p > 0.0f)) return;
        const double l = log(fmin(1.0, (double)min_p));
        const float bound = l < 0.0 ? __double2float_ru(m + l * t) : mx;
        if (bound > cut_at) {
            cut_at = bound;
            cut_index = 0x7FFFFFFF;
        }
    }
    __device__ void cut(u64 key) {
        const float at = rank_value((uint32_t)(key >> 32));
        const int i = (int)(0xFFFFFFFFu - (uint32_t)key);
        if (!keeps(at, i)) return;  // below an earlier cut
        cut_at = at;
        cut_index = i;
    }
    // log of the weight; -inf for a finite logit beside a maximum of +inf
    __device__ double exponent(float x) const {
        if (x == mx) return 0.0;
        const double d = (double)x - m;
        return isinf(d) ? d : d * it;
    }
    // The weight of a token that stays, in parts, to 1e-9 of itself and rounded up: 2^(-z / 256) with z = (max - x) c in
    // two floats (the difference's rounding error is exact, the product's an fma's).
    // z = k + f - 0.51, 0 < f < 1.02, gives the table's entry for k mod 256 times
    // 2^(-f / 256) = 1 - g as 32-bit fractions, moved down by k / 256; g from the
    // Taylor series (the fourth power, 2e-12, is left out). Adding 1.5 2^23 to a
    // float (2^23 to one above 0) leaves a rounded integer in its low bits.
    __device__ u64 weight(float x) const {
        constexpr double B = 0.6931471805599453 / TABLE, F = 2147483648.0;
        x = fminf(x, FLT_MAX);
        const float d = __fsub_rn(mf, x), xr = __fsub_rn(mf, d), mr = __fadd_rn(d, xr);
        const float dl = __fadd_rn(__fsub_rn(mf, mr), __fsub_rn(xr, x));
        const float p = __fmul_rn(d, ch);
        const float e = fmaf(dl, ch, fmaf(d, cl, fmaf(d, ch, -p)));
        const float kd = __fadd_rn(p, 12582912.0f);
        const uint32_t k = (uint32_t)__float_as_int(kd);  // 0x4B400000 + k
        const float f = __fadd_rn(__fsub_rn(p, __fsub_rn(kd, 12582912.0f)), __fadd_rn(e, (float)SHIFT));
        const float q = fmaf(fmaf((float)(F * B * B * B / 6), f, (float)(-F * B * B / 2)), f, (float)(F * B));
        const uint32_t g = 2 * ((uint32_t)__float_as_int(fmaf(q, f, 8388608.0f)) - 0x4B000000u);
        const u64 w = (u64)table[k & (TABLE - 1)] * (0xFFFFFFFFu - g);  // 2^63 parts of 1
        return (w >> min(63u, k / TABLE - (uint32_t)(0x4B400000 / TABLE - 63 + sh))) + 1;
    }
};

// inclusive sum over the lanes up to this one
__device__ __forceinline__ u64 warp_scan(u64 v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    return v;
}

// the lowest and the highest over the block's threads, to sm.mine
__device__ __forceinline__ void merge_span(u64 low, u64 high, Smem &sm) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        low = min(low, __shfl_xor_sync(0xffffffffu, low, o));
        high = max(high, __shfl_xor_sync(0xffffffffu, high, o));
    }
    if ((threadIdx.x & 31) == 0 && high) {
        atomicMin(&sm.mine.lowest, low);
        atomicMax(&sm.mine.highest, high);
    }
}

// The lowest of sm.key[0, n) before which, in the ranking, the measure (1, or
// sm.measure) and what lies `above` all of them stay below `limit`; above < limit
// <= above + the sum of all. By the block.
__device__ u64 border_cut(int n, u64 lowest, u64 highest, u64 above, u64 limit, bool weigh, Smem &sm) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // 256 bins of the keys' span first, one a thread
    const int fine = max(0, 64 - __clzll((long long)(highest - lowest)) - 8);
    auto fine_of = [&](u64 key) { return (int)((highest - key) >> fine); };
    sm.fine_lo[tid] = sm.fine_hi[tid] = 0;
    if (tid == 0) {
        sm.cut = ~0ull;
        sm.few = 0;
    }
    __syncthreads();
    for (int e = tid; e < n; e += NT) {
        const int f = fine_of(sm.key[e]);
        const u64 w = weigh ? sm.measure[e] : 1;
        const uint32_t l = (uint32_t)w, old = atomicAdd(&sm.fine_lo[f], l);
        const uint32_t h = (uint32_t)(w >> 32) + (old + l < old ? 1u : 0u);
        if (h) atomicAdd(&sm.fine_hi[f], h);
    }
    __syncthreads();
    const u64 mine = ((u64)sm.fine_hi[tid] << 32) + sm.fine_lo[tid], scan = warp_scan(mine, lane);
    if (lane == 31) sm.warp[warp] = scan;
    __syncthreads();
    u64 base = above + scan - mine;
    for (int w = 0; w < warp; ++w) base += sm.warp[w];
    if (base < limit && base + mine >= limit) {
        sm.bin = tid;
        sm.above = base;
    }
    __syncthreads();
    for (int e = tid; e < n; e += NT)
        if (fine_of(sm.key[e]) == sm.bin) sm.list_of[atomicAdd(&sm.few, 1)] = (short)e;
    __syncthreads();
    // each of those few against the others
    u64 cut = ~0ull;
    for (int e = tid; e < sm.few; e += NT) {
        const u64 key = sm.key[sm.list_of[e]];
        u64 b = sm.above;
        for (int j = 0; j < sm.few; ++j) {
            const int o = sm.list_of[j];
            if (sm.key[o] > key) b += weigh ? sm.measure[o] : 1;
        }
        if (b < limit) cut = min(cut, key);
    }
    if (cut != ~0ull) atomicMin(&sm.cut, cut);
    __syncthreads();
    return sm.cut;
}

// every block's list to sm.key, block q's by warp q; lane q knows its length
__device__ void gather(int n, int have, int parts, Smem &sm) {
    auto cluster = coop::this_cluster();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int upto = have;
#pragma unroll
    for (int o = 1; o < MAX_PARTS; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    if (warp < parts) {
        const int m = __shfl_sync(0xffffffffu, have, warp), at = __shfl_sync(0xffffffffu, upto, warp) - m;
        const u64 *other = cluster.map_shared_rank(sm.list, warp);
        for (int i = lane; i < m; i += 32) sm.key[at + i] = other[i];
    }
}

// Raises r's cut to the border of the ranking at which the measure of the tokens
// before (their number, or with WEIGHT their weight) reaches a limit below that of the
// whole. It lies among the tokens from low_end up to but without high_end, and the
// measure of those from high_end on is `above`.
template <bool WEIGHT, class Each>
__device__ void cut_ranking(Row &r, u64 limit, float low_end, float high_end, u64 above, Smem &sm, Each each) {
    auto cluster = coop::this_cluster();
    const int parts = (int)cluster.num_blocks(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    u64 lowest = 0, highest = 0;
    // bins over the span, at most 64 wide (an outlier would stretch them)
    const float from = fminf(high_end, r.mx);
    const float scale = low_end < from ? fminf((float)BINS / fminf(from - low_end, 64.0f), 1e30f) : 0.0f;
    int shift = 0;
    for (int level = 0;; ++level) {
        // bin of a token, the best ones first; -1: not (any more) in question
        auto bin_of = [&](float x, int i) {
            if (level == 0)
                return x >= low_end && !(x >= high_end) && r.keeps(x, i)
                           ? (int)fminf((x == from ? 0.0f : from - x) * scale, (float)(BINS - 1)) : -1;
            const u64 key = make_key(rank_key(x), i);
            return key >= lowest && key <= highest ? (int)((highest - key) >> shift) : -1;
        };
        *((uint4 *)sm.lo + tid) = make_uint4(0, 0, 0, 0);
        *((uint4 *)sm.hi + tid) = make_uint4(0, 0, 0, 0);
        __syncthreads();
        each([&](const float(&x)[4], int i) {
            int b[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = bin_of(x[j], i + j);
            if (max(max(b[0], b[1]), max(b[2], b[3])) < 0) return;
            u64 w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = WEIGHT ? r.weight(x[j]) : 1;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (b[j] < 0) continue;
                const uint32_t l = (uint32_t)w[j], old = atomicAdd(&sm.lo[b[j]], l);
                if (!WEIGHT) continue;
                const uint32_t h = (uint32_t)(w[j] >> 32) + (old + l < old ? 1u : 0u);  // with the carry
                if (h) atomicAdd(&sm.hi[b[j]], h);
            }
        });
        cluster.sync();
        // thread t sums bins 4 t .. 4 t + 3 over the blocks; exclusive scan
        u64 c[4] = {}, s = 0;
        for (int q = 0; q < parts; ++q) {
            const uint4 l = *((const uint4 *)cluster.map_shared_rank(sm.lo, q) + tid);
            c[0] += l.x;
            c[1] += l.y;
            c[2] += l.z;
            c[3] += l.w;
            if (WEIGHT) {
                const uint4 h = *((const uint4 *)cluster.map_shared_rank(sm.hi, q) + tid);
                c[0] += (u64)h.x << 32;
                c[1] += (u64)h.y << 32;
                c[2] += (u64)h.z << 32;
                c[3] += (u64)h.w << 32;
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) s += c[j];
        const u64 inc = warp_scan(s, lane);
        if (lane == 31) sm.warp[warp] = inc;
        __syncthreads();
        u64 before = above + inc - s, total = 0;
        for (int w = 0; w < WARPS; ++w) {
            if (w < warp) before += sm.warp[w];
            total += sm.warp[w];
        }
        if (!WEIGHT && level == 0 && total <= limit) {  // nothing to cut (the same in every block)
            cluster.sync();                             // the bins have been read
            return;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (before < limit && before + c[j] >= limit) {
                sm.bin = 4 * tid + j;
                sm.above = before;
            }
            before += c[j];
        }
        if (tid == 0) sm.mine = {0, ~0ull, 0};
        __syncthreads();
        above = sm.above;
        const int bin = sm.bin;
        u64 low = ~0ull, high = 0;
        each([&](const float(&x)[4], int i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (bin_of(x[j], i + j) != bin) continue;
                const u64 key = make_key(rank_key(x[j]), i + j);
                const int at = atomicAdd(&sm.mine.count, 1);
                if (at < BORDER) sm.list[at] = key;
                low = min(low, key);
                high = max(high, key);
            }
        });
        merge_span(low, high, sm);
        cluster.sync();  // also: the bins have been read
        // every warp: lane q asks block q, then warp q fetches block q's keys
        int have = 0;
        lowest = ~0ull;
        highest = 0;
        if (lane < parts) {
            const Border *b = cluster.map_shared_rank(&sm.mine, lane);
            have = b->count;
            lowest = b->lowest;
            highest = b->highest;
        }
#pragma unroll
        for (int o = 1; o < MAX_PARTS; o <<= 1) {
            lowest = min(lowest, __shfl_xor_sync(0xffffffffu, lowest, o));
            highest = max(highest, __shfl_xor_sync(0xffffffffu, highest, o));
        }
        lowest = __shfl_sync(0xffffffffu, lowest, 0);
        highest = __shfl_sync(0xffffffffu, highest, 0);
        const int n = __reduce_add_sync(0xffffffffu, have);
        if (n <= BORDER) {
            gather(n, have, parts, sm);
            __syncthreads();
            if (WEIGHT)
                for (int e = tid; e < n; e += NT) sm.measure[e] = r.weight(rank_value((uint32_t)(sm.key[e] >> 32)));
            __syncthreads();
            r.cut(border_cut(n, lowest, highest, above, limit, WEIGHT, sm));
            return;
        }
        // 10 bits of the span of the keys that are left
        shift = max(0, 64 - __clzll((long long)(highest - lowest)) - 10);
    }
}

// The draw by one block among sm.key[0, n), which hold the first k of the ranking;
// those stay before which less than `limit` of the weight lies (0: less than the
// part p of theirs).
template <class Put>
__device__ void draw_brief(Row &r, int n, int k, u64 limit, float p, float min_p, float u, Smem &sm, Put put) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int PER = BORDER / NT;
    auto logit = [&](int e) { return rank_value((uint32_t)(sm.list[e] >> 32)); };
    auto index = [&](int e) { return (int)(0xFFFFFFFFu - (uint32_t)sm.list[e]); };
    // The ranking: a key's place is the number of larger logits, those with as many
    // (equal ones) are told apart by their indices.
    for (int e = tid; e < BORDER; e += NT) {
        sm.rank_of[e] = e < n ? (uint32_t)(sm.key[e] >> 32) : 0;
        sm.slot[e] = 0;
    }
    __syncthreads();
    int place[PER] = {};
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int e = tid + j * NT;
        if (e >= n) break;
        const uint32_t mine = sm.rank_of[e];
#pragma unroll 4
        for (int q = 0; q < n; q += 4) {
            const uint4 o = *(const uint4 *)(sm.rank_of + q);
            place[j] += (o.x > mine) + (o.y > mine) + (o.z > mine) + (o.w > mine);
        }
        atomicAdd(&sm.slot[place[j]], 1);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int e = tid + j * NT;
        if (e >= n) break;
        const u64 key = sm.key[e];
        if (sm.slot[place[j]] > 1)
            for (int q = 0; q < n; ++q) place[j] += sm.key[q] > key && sm.key[q] >> 32 == key >> 32;
        sm.list[place[j]] = key;
        const float x = rank_value((uint32_t)(key >> 32));
        sm.measure[place[j]] = r.keeps(x, (int)(0xFFFFFFFFu - (uint32_t)key)) ? r.weight(x) : 0;
    }
    __syncthreads();
    // its running sums, two tokens a thread; those that stay come first
    u64 w[PER], s = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) s += w[j] = PER * tid + j < min(n, k) ? sm.measure[PER * tid + j] : 0;
    u64 before = warp_scan(s, lane), total = 0;
    if (lane == 31) sm.warp[warp] = before;
    __syncthreads();
    before -= s;
    for (int q = 0; q < WARPS; ++q) {
        if (q < warp) before += sm.warp[q];
        total += sm.warp[q];
    }
    if (!limit) limit = p < 1.0f ? max(1ull, (u64)ceil((double)p * (double)total)) : total;
    r.least(min_p);
    bool stay[PER];
    u64 upto[PER];
    int left = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int e = PER * tid + j;
        stay[j] = w[j] && before < limit && r.keeps(logit(e), index(e));
        upto[j] = before += w[j];
        left += __syncthreads_count(stay[j]);
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int e = PER * tid + j;
        if (stay[j]) sm.index_of[e] = index(e);
        if (e == left - 1) sm.above = upto[j];
    }
    __syncthreads();
    total = sm.above;
    const int *at = sm.index_of;
    const u64 *weight = sm.measure;
    const u64 target = u < 1.0f ? min(total - 1, (u64)fmax(0.0, (double)u * (double)total)) : total - 1;
    const double whole = ldexp((double)total, -r.sh);
    if (target == 0 && u > 0.0f) {  // below one part: the weights as they are, see sample_kernel
        if (tid != 0) return;
        double c = 0.0;
        for (int last = -1, more = left;; --more) {
            int e = -1;  // the next one in index order
            for (int j = 0; j < left; ++j)
                if (at[j] > last && (e < 0 || at[j] < at[e])) e = j;
            last = at[e];
            const double y = r.exponent(logit(e));
            c += exp(y);
            if (c > (double)u * whole || more == 1) {
                put(last, (float)(y - log(whole)));
                return;
            }
        }
    }
    if (left <= NT / 2) {  // each against the others
        if (tid >= left) return;
        u64 lower = 0;
#pragma unroll 4
        for (int j = 0; j < left; ++j) lower += at[j] < at[tid] ? weight[j] : 0;
        if (lower <= target && lower + weight[tid] > target)
            put(at[tid], (float)(r.exponent(logit(tid)) - log(whole)));
        return;
    }
    // The first in index order whose sum exceeds the target: with the index as the
    // key's upper half the lowest before which it does not.
    if (tid == 0) sm.mine = {0, ~0ull, 0};
    __syncthreads();
    u64 lowest = ~0ull, highest = 0;
    for (int e = tid; e < left; e += NT) {
        const u64 key = sm.list[e] << 32 | sm.list[e] >> 32;
        sm.key[e] = key;
        lowest = min(lowest, key);
        highest = max(highest, key);
    }
    merge_span(lowest, highest, sm);
    __syncthreads();
    const u64 drawn = border_cut(left, sm.mine.lowest, sm.mine.highest, 0, target + 1, true, sm);
    if (tid == 0) {
        const float v = rank_value((uint32_t)drawn);
        put((int)(0xFFFFFFFFu - (uint32_t)(drawn >> 32)), (float)(r.exponent(v) - log(whole)));
    }
}

__global__ void __launch_bounds__(NT, 3)
sample_kernel(SampleRows a, int stretch, int sh) {
    extern __shared__ float4 slice4[];
    __shared__ __align__(16) Smem sm;
    float *slice = (float *)slice4;
    auto cluster = coop::this_cluster();
    const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
    cluster.barrier_arrive();  // waited for before the first write to another block
    const long row = blockIdx.x / parts, at = a.step ? (long)*a.step * a.rows + row : row;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    Row r;
    r.lo = min(a.V, part * stretch);
    r.n = min(a.V, r.lo + stretch) - r.lo;
    r.per = ((r.n + NT - 1) / NT) | 1;
    r.sh = sh;
    r.table = sm.table;
    const float *x = a.logits + row * a.ldl + r.lo;
    // elements before the first 16-byte boundary, whole groups of four, the rest;
    // element i of the stretch is kept at slice[pad + i], groups at float4s
    const int head = min(r.n, (int)(((16 - (uintptr_t)x % 16) / 4) % 4)), quads = (r.n - head) / 4, pad = (4 - head) & 3;
    const int odd = tid < head ? tid : tid < r.n - 4 * quads ? tid + 4 * quads : -1;
    float4 *s4 = (float4 *)(slice + pad + head);
    for (int q = tid; q < quads; q += NT)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(s4 + q)), "l"(x + head + 4 * q) : "memory");
    if (odd >= 0)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(slice + pad + odd)), "l"(x + odd) : "memory");
    asm volatile("cp.async.commit_group;" ::: "memory");
    float T = a.temperature ? a.temperature[row] : 1.0f;
    if (T > 0.0f) T = fminf(fmaxf(T, 0x1p-100f), 0x1p100f);  // the exponential's range
    const float p = a.top_p ? a.top_p[row] : 1.0f;
    const float min_p = a.min_p ? a.min_p[row] : 0.0f, u = a.u[at];
    const int k = a.top_k ? a.top_k[row] : 0;
    sm.table[tid] = pow2_table.v[tid];
    auto put = [&](int token, float logprob) {
        a.tokens[at] = token;
        if (a.next) a.next[row] = max(token, 0);
        if (a.logprob) a.logprob[row] = logprob;
    };
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    r.s = slice + pad;

    // the row's largest logit and its smallest above -inf
    float mx = -INFINITY, mn = INFINITY;
    auto look = [&](float v) {
        mx = fmaxf(mx, v);
        mn = fminf(mn, v == -INFINITY ? INFINITY : v);
    };
    for (int q = tid; q < quads; q += NT) {
        const float4 v = s4[q];
        look(v.x);
        look(v.y);
        look(v.z);
        look(v.w);
    }
    if (odd >= 0) look(r.s[odd]);
    // a bar for a short top-k: of the threads' maxima the one that ceil(k / blocks)
    // reach, the lowest over the blocks; k tokens reach it
    const bool brief = k > 0 && k <= BORDER / 2 && T > 0.0f && p > 0.0f;
    const float own = mx;  // of this thread
    mx = warp_max(mx);
    mn = -warp_max(-mn);
    // a bar for top-p that some 300 tokens reach: the mean over the row's warps of the
    // one of the lanes' maxima that 256 of the row's (22 of a lone block's warp) reach
    const bool nucleus = !brief && T > 0.0f && p > 0.0f && p < 1.0f;
    float reach = -INFINITY;
    if (nucleus && a.V > BORDER) {
        int rank = 0;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            const float v = __shfl_sync(0xffffffffu, own, j);
            rank += v > own || (v == own && j < lane);
        }
        const int at = 31 - __clz(__ballot_sync(0xffffffffu, rank == min(22, 32 / parts) - 1));
        reach = __shfl_sync(0xffffffffu, own, at);
    }
    if (lane == 0) {
        sm.fwarp[0][warp] = mx;
        sm.fwarp[1][warp] = mn;
        sm.fwarp[2][warp] = reach;
        if (warp == 0) sm.mine = {0, ~0ull, 0};
    }
    sm.own[tid] = own;
    __syncthreads();
    for (int w = 0; w < WARPS; ++w) {
        mx = fmaxf(mx, sm.fwarp[0][w]);
        mn = fminf(mn, sm.fwarp[1][w]);
    }
    if (nucleus) {
        float s = 0.0f;
        int n = 0;
        for (int w = 0; w < WARPS; ++w)
            if (sm.fwarp[2][w] > -INFINITY) {
                s += sm.fwarp[2][w];
                ++n;
            }
        reach = n ? s / n : -INFINITY;
    }
    if (brief) {
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < NT; j += 4) {
            const float4 v = *(const float4 *)(sm.own + j);
            rank += (v.x > own || (v.x == own && j < tid)) + (v.y > own || (v.y == own && j + 1 < tid)) +
                    (v.z > own || (v.z == own && j + 2 < tid)) + (v.w > own || (v.w == own && j + 3 < tid));
        }
        if (rank == (k + parts - 1) / parts - 1) sm.bar = own;  // exactly one thread
        __syncthreads();
    }
    float bar = brief ? sm.bar : reach;
    cluster.barrier_wait();
    if (tid < parts) {
        *cluster.map_shared_rank(&sm.max_of[part], tid) = mx;
        *cluster.map_shared_rank(&sm.min_of[part], tid) = mn;
        *cluster.map_shared_rank(&sm.bar_of[part], tid) = bar;
    }
    cluster.sync();
    for (int q = 0; q < parts; ++q) {
        mx = fmaxf(mx, sm.max_of[q]);
        mn = fminf(mn, sm.min_of[q]);
        bar = fminf(bar, sm.bar_of[q]);
    }
    if (nucleus) {
        float s = 0.0f;
        int n = 0;
        for (int q = 0; q < parts; ++q)
            if (sm.bar_of[q] > -INFINITY) {
                s += sm.bar_of[q];
                ++n;
            }
        bar = n ? s / n : -INFINITY;
    }
    if (mx == -INFINITY) {  // the same in every block, as all that follows
        if (part == 0 && tid == 0) put(-1, -INFINITY);
        return;
    }
    const int i0 = min(r.n, tid * r.per), i1 = min(r.n, i0 + r.per);
    if (!(T > 0.0f) || p <= 0.0f) {  // the first of the ranking
        int first = 0x7FFFFFFF;
        for (int i = i0; i < i1; ++i)
            if (r.s[i] == mx) {
                first = r.lo + i;
                break;
            }
        first = (int)__reduce_min_sync(0xffffffffu, (unsigned)first);
        if (lane == 0) sm.warp[warp] = (u64)first;
        __syncthreads();
        for (int w = 0; w < WARPS; ++w) first = min(first, (int)sm.warp[w]);
        if (tid == 0) *cluster.map_shared_rank(&sm.first_of[part], 0) = first;
        cluster.sync();
        if (part == 0 && tid == 0) {
            for (int q = 0; q < parts; ++q) first = min(first, sm.first_of[q]);
            put(first, 0.0f);
        }
        return;
    }
    r.mx = mx;
    r.m = (double)mx;
    r.t = (double)T;
    r.it = 1.0 / r.t;
    const double factor = TABLE * 1.4426950408889634 * r.it;
    r.ch = (float)factor;
    r.cl = (float)(factor - (double)r.ch);
    r.mf = fminf(mx, FLT_MAX);
    // nothing stays beside +inf, nor what has no weight in 64-bit floating point
    r.cut_at = fminf(__double2float_rd(r.m - 745.0 * r.t), nextafterf(mx, -INFINITY));
    if (mx == INFINITY) r.cut_at = FLT_MAX;
    r.cut_index = -1;
    // the stretch's logits in no order, four at a time (NaN: none), whose weights
    // have no need to wait for one another
    auto each = [&](auto &&f) {
        for (int q = tid - NT; q < quads; q += NT) {
            float v[4] = {NAN, NAN, NAN, NAN};
            if (q >= 0) {
                const float4 w = s4[q];
                v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
                f(v, r.lo + head + 4 * q);
            } else if (odd >= 0) {
                v[0] = r.s[odd];
                f(v, r.lo + odd);
            }
        }
    };
    // the tokens that reach a bar, to the list
    auto collect = [&](float v, int i) {
        const int e = atomicAdd(&sm.mine.count, 1);
        if (e < BORDER) sm.list[e] = make_key(rank_key(v), i);
    };
    // in all blocks, after the next cluster.sync(): their number; and block 0 draws among them
    auto listed = [&](int &have) {
        have = lane < parts ? cluster.map_shared_rank(&sm.mine, lane)->count : 0;
        return __reduce_add_sync(0xffffffffu, have);
    };
    auto draw = [&](int n, int have, int first, u64 limit) {
        if (part == 0) gather(n, have, parts, sm);
        cluster.sync();  // the others' keys have been read
        if (part == 0) draw_brief(r, n, first, limit, p, min_p, u, sm, put);
    };
    if (brief && bar > -INFINITY) {
        // A short top-k: the tokens that reach the bar, some 2 k, decide alone.
        if (own >= bar)
            each([&](const float(&v)[4], int i) {
                if (!(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])) >= bar)) return;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (v[j] >= bar) collect(v[j], i + j);
            });
        cluster.sync();
        int have;
        const int n = listed(have);
        if (n <= BORDER) {
            draw(n, have, k, 0);
            return;
        }
        // too many equal logits: the general way
    }
    if (k > 0 && k < a.V) {
        cut_ranking<false>(r, (u64)k, mn, ALL, 0, sm, each);
        cluster.sync();  // the blocks' lists have been read
    }
    if (tid == 0) sm.mine = {0, ~0ull, 0};
    __syncthreads();
    if (p < 1.0f) {
        // the whole weight, and the tokens that reach the bar with theirs
        u64 s = 0, upper = 0;
        each([&](const float(&v)[4], int i) {
            u64 kept[4];
            bool any = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const u64 w = r.weight(v[e]);
                kept[e] = r.keeps(v[e], i + e) ? w : 0;
                s += kept[e];
                any |= v[e] >= bar;
            }
            if (!any) return;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (v[e] >= bar && kept[e]) {
                    upper += kept[e];
                    collect(v[e], i + e);
                }
        });
        s = warp_scan(s, lane);
        upper = warp_scan(upper, lane);
        if (lane == 31) {
            sm.warp[warp] = s;
            sm.upper[warp] = upper;
        }
        __syncthreads();
        if (tid < 2 * parts) {
            const u64 *of = tid < parts ? sm.warp : sm.upper;
            u64 v = 0;
            for (int w = 0; w < WARPS; ++w) v += of[w];
            *cluster.map_shared_rank(&(tid < parts ? sm.total_of : sm.upper_of)[part], tid % parts) = v;
        }
        cluster.sync();
        u64 whole = 0;
        upper = 0;
        for (int q = 0; q < parts; ++q) {
            whole += sm.total_of[q];
            upper += sm.upper_of[q];
        }
        const u64 limit = max(1ull, (u64)ceil((double)p * (double)whole));
        int have;
        const int n = listed(have);
        if (n <= BORDER && limit < whole && limit <= upper) {
            draw(n, have, n, limit);
            return;
        }
        if (limit < whole) {
            // A wide nucleus. Its border is not below a floor: V tokens under it would weigh
            // less than what lies behind the border; two parts (for the rounding) less than
            // an equal share, and 1e-8 of it for the exponential's error.
            const double share = ldexp((double)(whole - limit) / a.V - 2.0, -sh) * (1.0 - 1e-8);
            const float floor = share > 0.0 ? fminf(mx, __double2float_rd(r.m + r.t * log(share))) : -INFINITY;
            if (limit <= upper)
                cut_ranking<true>(r, limit, fmaxf(bar, mn), ALL, 0, sm, each);
            else
                cut_ranking<true>(r, limit, fmaxf(floor, mn), bar, upper, sm, each);
        }
        r.least(min_p);
    } else if (min_p > 0.0f) {
        r.least(min_p);
        each([&](const float(&v)[4], int i) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (r.keeps(v[e], i + e)) collect(v[e], i + e);
        });
        cluster.sync();
        int have;
        const int n = listed(have);
        if (n <= BORDER) {
            draw(n, have, n, 0);
            return;
        }
    }

    // cumulative weights in index order: threads, warps, blocks
    auto drawn = [&](int i) -> u64 {
        const float v = r.s[i];
        return r.keeps(v, r.lo + i) ? r.weight(v) : 0;
    };
    u64 s = 0;
    for (int i = i0; i < i1; i += 4) {  // four that need not wait for one another
        float v[4];
        bool stay[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] = i + e < i1 ? r.s[i + e] : NAN;
            stay[e] = r.keeps(v[e], r.lo + i + e);
        }
        if (!(stay[0] || stay[1] || stay[2] || stay[3])) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const u64 w = r.weight(v[e]);
            s += stay[e] ? w : 0;
        }
    }
    const u64 inc = warp_scan(s, lane);
    if (lane == 31) sm.warp[warp] = inc;
    __syncthreads();
    u64 before = inc - s, block = 0;
    for (int w = 0; w < WARPS; ++w) {
        if (w < warp) before += sm.warp[w];
        block += sm.warp[w];
    }
    if (tid < parts) *cluster.map_shared_rank(&sm.sum_of[part], tid) = block;
    cluster.sync();
    u64 total = 0;
    for (int q = 0; q < parts; ++q) {
        if (q < part) before += sm.sum_of[q];
        total += sm.sum_of[q];
    }
    // the first token whose cumulative weight exceeds u total: an integer that
    // exceeds floor(u total)
    const u64 target = u < 1.0f ? min(total - 1, (u64)fmax(0.0, (double)u * (double)total)) : total - 1;
    if (target == 0 && u > 0.0f) {
        // A number below one part of the whole: what the parts round up decides, so
        // the weights are summed as they are. No generator of 24 or 32 bits gives
        // such a number, so one thread walks the stretch that holds the border.
        const double tau = ldexp((double)u * (double)total, -sh);
        auto real = [&](int i) { return drawn(i) ? exp(r.exponent(r.s[i])) : 0.0; };
        double d = 0.0;
        for (int i = i0; i < i1; ++i) d += real(i);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
        __syncthreads();
        if (lane == 0) sm.warp[warp] = (u64)__double_as_longlong(d);
        __syncthreads();
        d = 0.0;
        for (int w = 0; w < WARPS; ++w) d += __longlong_as_double((long long)sm.warp[w]);
        cluster.sync();  // sum_of has been read
        if (tid < parts) *cluster.map_shared_rank(&sm.sum_of[part], tid) = (u64)__double_as_longlong(d);
        cluster.sync();
        double base = 0.0;
        int owner = 0;
        for (; owner < parts - 1; ++owner) {
            const double next = base + __longlong_as_double((long long)sm.sum_of[owner]);
            if (next > tau) break;
            base = next;
        }
        if (part != owner || tid != 0) return;
        int token = 0;
        for (int i = 0; i < r.n; ++i) {
            const double w = real(i);
            if (w > 0.0) token = i;
            base += w;
            if (base > tau) break;
        }
        put(r.lo + token, (float)(r.exponent(r.s[token]) - log(ldexp((double)total, -sh))));
        return;
    }
    const bool here = before <= target && before + s > target;
    const uint32_t who = __ballot_sync(0xffffffffu, here);
    if (!who) return;
    const int owner = __ffs(who) - 1, o0 = __shfl_sync(0xffffffffu, i0, owner), o1 = __shfl_sync(0xffffffffu, i1, owner);
    u64 c = __shfl_sync(0xffffffffu, before, owner);
    for (int i = o0; i < o1; i += 32) {
        const u64 w = i + lane < o1 ? drawn(i + lane) : 0;
        const u64 sum = c + warp_scan(w, lane);
        const uint32_t over = __ballot_sync(0xffffffffu, sum > target);
        if (over) {
            if (lane == __ffs(over) - 1) {
                const float v = r.s[i + lane];
                put(r.lo + i + lane, (float)(r.exponent(v) - log(ldexp((double)total, -sh))));
            }
            return;
        }
        c = __shfl_sync(0xffffffffu, sum, 31);
    }
}

}  // namespace

int sample_rows(const SampleRows &a, cudaStream_t s) {
    if (a.rows <= 0) return OK;
    // Blocks of a row: as many as the shared memory for its stretches asks for,
    // more while there are rows for half the SMs at most.
    int parts = 1;
    while (parts < MAX_PARTS && ((long)a.V * 4 > (long)parts * SLICE_BYTES ||
                                 ((long)a.rows * parts <= num_sms() && a.V >= parts * 2048)))
        parts *= 2;
    if ((long)a.rows * parts > 0x7FFFFFFFL) {
        set_last_error(ERR_ARG, "sample: %d rows are too many", a.rows);
        return ERR_ARG;
    }
    const int stretch = ((a.V + parts - 1) / parts + 3) / 4 * 4;
    int sh = 50;
    while ((a.V - 1) >> (62 - sh)) --sh;  // V weights of 2^sh stay below 2^62
    static bool set_on[MAX_DEVICES];
    bool *set;
    CG_TRY(this_device(set_on, &set));
    if (!*set) {
        CG_CUDA(cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (SAMPLE_MAX_VOCAB / MAX_PARTS + 16) * 4));
        *set = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.rows * parts));
    cfg.blockDim = dim3(NT);
    cfg.dynamicSmemBytes = ((size_t)stretch + 8) * sizeof(float);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)parts;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    CG_CUDA(cudaLaunchKernelEx(&cfg, sample_kernel, a, stretch, sh));
    ++g_launch_count;
    return OK;
}

}  // namespace cg
