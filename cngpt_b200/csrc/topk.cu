// topk.cu - the k largest logits of every row in falling order (cngpt_cuda_topk).
//
// One pass over the row. The block keeps the k best of what it has seen as
// 64-bit keys (ordered bits of the logit, then the inverted index, so that the
// lower index wins among equals) and the logit `low` of the worst of them; of
// the next chunk only logits above `low` can matter (an equal one has a higher
// index than all k). In a row of random order the k-th best rises so fast that
// about k (1 + log(chunks)) logits pass after the first chunk; whenever many have
// passed, a selection cuts the candidates back to k. So the time is that of
// reading the logits once as long as k is small.
//
// On B200, 8192 x 50257: k = 8 0.278 ms (5.9 TB/s, 90 % of the copy rate), k = 64
// 0.331 ms (5.0 TB/s), k = 256 0.62 ms, where lists outgrow one warp's registers;
// 7615 x 1261, k = 24, a warp a row: 26 us;
// 37 x 32003, k = 20, cut among clusters: 9.4 us. What passes costs issue slots
// beside the loads. Tried: the row resident in a cluster's shared memory (0.66 ms,
// its latencies are not hidden), a cp.async ring (0.57 ms), 128 threads (the same).
#include <algorithm>

#include <cooperative_groups.h>

#include "common.cuh"
#include "kernels.h"
#include "rank.cuh"

namespace cg {
namespace {

namespace coop = cooperative_groups;

typedef unsigned long long u64;

constexpr int NT = 256;              // threads
constexpr int QUADS = 4;             // 16-byte loads of a thread and chunk
constexpr int CHUNK = NT * QUADS * 4;
constexpr int BINS = 2048;           // radix 2^11
constexpr int TRIGGER = 448;         // candidates below which no selection is worth its time

__device__ __forceinline__ u64 make_key(float x, uint32_t i) { return ((u64)rank_key(x) << 32) | (0xFFFFFFFFu - i); }

struct Smem {
    // hist is also where a selection collects the k it keeps (TOPK_MAX * 8 bytes)
    union {
        uint32_t hist[BINS];
        uint4 hist4[BINS / 4];
        u64 keep[TOPK_MAX];
    };
    uint32_t warp[NT / 32];
    int count;             // candidates in the buffer
    int bin, need, equal;  // of a selection: the bin that holds the k-th, how many of it belong, how many it has
    int kept;
    uint32_t low;          // rank_key of the worst one kept
};

// The same cut for up to SMALL candidates by warp 0 alone, while the others wait
// at the barrier behind it: it bisects the logits' bits with the candidates in
// registers and, among those that equal the k-th, the index's. Some 500
// instructions of one warp take the place of some 5000 of all warps.
constexpr int SMALL = 512;

template <int PER>
__device__ uint32_t select_part(u64 *buf, int n, int k) {
    const int lane = threadIdx.x & 31;
    uint32_t key[PER], top = 0, bottom = 0xFFFFFFFFu;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int i = lane + 32 * j;
        key[j] = i < n ? (uint32_t)(buf[i] >> 32) : 0u;
        top = max(top, key[j]);
        if (i < n) bottom = min(bottom, key[j]);
    }
    uint32_t hi = __reduce_max_sync(0xffffffffu, top), lo = __reduce_min_sync(0xffffffffu, bottom);
    // lo: the highest value that at least k candidates reach
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2 + 1;
        int c = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) c += key[j] >= mid;
        c = __reduce_add_sync(0xffffffffu, c);
        if (c >= k) lo = mid;
        else hi = mid - 1;
        if (c == k) break;  // just these; whether `lo` is one of them does not matter
    }
    int above = 0, equal = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        above += key[j] > lo;
        equal += key[j] == lo && lane + 32 * j < n;
    }
    above = __reduce_add_sync(0xffffffffu, above);
    equal = __reduce_add_sync(0xffffffffu, equal);
    // of the equal ones the k - above with the largest inverted index
    uint32_t bar = 0;
    if (above + equal > k) {
        uint32_t a = 0, b = 0xFFFFFFFFu;
        while (a < b) {
            const uint32_t mid = a + (b - a) / 2 + 1;
            int c = 0;
            for (int j = 0; j < PER; ++j) c += key[j] == lo && lane + 32 * j < n && (uint32_t)buf[lane + 32 * j] >= mid;
            if (__reduce_add_sync(0xffffffffu, c) >= k - above) a = mid;
            else b = mid - 1;
        }
        bar = a;
    }
    // compaction in place: a round's survivors never pass the round's own places
    int at = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int i = lane + 32 * j;
        const u64 c = i < n ? buf[i] : 0;
        const bool keep = i < n && (key[j] > lo || (key[j] == lo && (uint32_t)c >= bar));
        const uint32_t mask = __ballot_sync(0xffffffffu, keep);
        if (keep) buf[at + __popc(mask & ((1u << lane) - 1))] = c;
        at += __popc(mask);
        __syncwarp();
    }
    // between NaN (0) and -inf lies no logit: k numbers, what follows has to exceed -inf
    return lo == 0u ? 0u : max(lo, RANK_NEG_INF);
}

// returns the new `low`
__device__ __forceinline__ uint32_t select_small(u64 *buf, int n, int k) {
    return n <= 128 ? select_part<4>(buf, n, k) : n <= 256 ? select_part<8>(buf, n, k) : select_part<SMALL / 32>(buf, n, k);
}

// Cuts the n > k candidates in buf to the k largest (any order) and sets low.
// Radix from the top: 11, 11 and 10 bits of the logit, then of the index (only
// where equal logits straddle the cut); ends as soon as the bin that holds the
// k-th is needed whole. hist is zero before and after.
__device__ void select_k(u64 *buf, int n, int k, Smem &sm) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (n <= SMALL) {
        if (warp == 0) {
            const uint32_t low = select_small(buf, n, k);
            if (lane == 0) {
                sm.count = k;
                sm.low = low;
            }
        }
        __syncthreads();
        return;
    }
    u64 prefix = 0;
    int need = k, top = 64;
    while (true) {
        const int bits = (top == 42 || top == 10) ? 10 : 11, shift = top - bits;
        for (int i = tid; i < n; i += NT) {
            const u64 key = buf[i];
            if (top == 64 || (key >> top) == prefix) atomicAdd(&sm.hist[(uint32_t)(key >> shift) & ((1u << bits) - 1)], 1u);
        }
        __syncthreads();
        // thread t sums 8 bins from the top; exclusive scan over the threads
        const int hi = BINS - 8 * tid;
        const uint4 q1 = sm.hist4[hi / 4 - 1], q0 = sm.hist4[hi / 4 - 2];
        sm.hist4[hi / 4 - 1] = sm.hist4[hi / 4 - 2] = make_uint4(0, 0, 0, 0);
        const uint32_t c[8] = {q1.w, q1.z, q1.y, q1.x, q0.w, q0.z, q0.y, q0.x};
        uint32_t s = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) s += c[j];
        uint32_t inc = s;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        if (lane == 31) sm.warp[warp] = inc;
        __syncthreads();
        uint32_t before = inc - s;
        for (int w = 0; w < warp; ++w) before += sm.warp[w];
        if (before < (uint32_t)need && before + s >= (uint32_t)need) {
            uint32_t b = before;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (b < (uint32_t)need && b + c[j] >= (uint32_t)need) {
                    sm.bin = hi - 1 - j;
                    sm.need = need - (int)b;
                    sm.equal = (int)c[j];
                }
                b += c[j];
            }
        }
        __syncthreads();
        prefix = (prefix << bits) | (u64)sm.bin;
        need = sm.need;
        top = shift;
        if (sm.equal == need || top == 0) break;  // at the last bit the keys differ
    }
    const u64 cut = prefix << top;
    if (tid == 0) {
        sm.kept = 0;
        sm.low = 0xFFFFFFFFu;
    }
    __syncthreads();
    uint32_t low = 0xFFFFFFFFu;
    for (int i = tid; i < n; i += NT) {
        const u64 key = buf[i];
        if (key >= cut) {
            sm.keep[atomicAdd(&sm.kept, 1)] = key;
            low = min(low, (uint32_t)(key >> 32));
        }
    }
    low = __reduce_min_sync(0xffffffffu, low);
    if (lane == 0) atomicMin(&sm.low, low);
    __syncthreads();
    for (int i = tid; i < k; i += NT) buf[i] = sm.keep[i];
    __syncthreads();
    for (int i = tid; i < 2 * k; i += NT) sm.hist[i] = 0;  // where keep was
    if (tid == 0) sm.count = k;
    __syncthreads();
}

// Cluster of 1 to 8 blocks per row, each with a stretch of it; block 0 then
// joins the stretches' candidates from the others' shared memory.
__global__ void __launch_bounds__(NT, 4)
topk_kernel(const float *__restrict__ logits, long ldl, int V, int k, float *__restrict__ values,
            int *__restrict__ indices, int stretch) {
    extern __shared__ u64 buf[];  // [max(2 k, TRIGGER) + CHUNK + 8]
    __shared__ Smem sm;
    auto cluster = coop::this_cluster();
    const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
    const long row = blockIdx.x / parts;
    const int tid = threadIdx.x, lane = tid & 31;
    const int lo = min(V, part * stretch), hi = min(V, lo + stretch), n = hi - lo;
    const float *x = logits + row * ldl + lo;
    for (int i = tid; i < BINS / 4; i += NT) sm.hist4[i] = make_uint4(0, 0, 0, 0);
    if (tid == 0) sm.count = 0;
    // elements before the first 16-byte boundary, whole groups of four, the rest
    const int head = min(n, (int)(((16 - (uintptr_t)x % 16) / 4) % 4)), quads = (n - head) / 4;
    const float4 *x4 = (const float4 *)(x + head);
    float4 v[QUADS], nx[QUADS];
    const float4 none = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    auto fetch = [&](float4 *dst, int c) {
        const float4 *p = x4 + c * QUADS * NT + tid;
        if ((c + 1) * QUADS * NT <= quads) {
#pragma unroll
            for (int j = 0; j < QUADS; ++j) dst[j] = __ldcs(p + j * NT);
        } else {
#pragma unroll
            for (int j = 0; j < QUADS; ++j) dst[j] = (c * QUADS + j) * NT + tid < quads ? __ldcs(p + j * NT) : none;
        }
    };
    fetch(nx, 0);
    __syncthreads();
    if (tid < head) buf[atomicAdd(&sm.count, 1)] = make_key(x[tid], lo + tid);
    __syncthreads();
    const int chunks = (quads + QUADS * NT - 1) / (QUADS * NT);
    const int trigger = max(2 * k, TRIGGER);
    bool all = true;  // fewer than k kept: every element is a candidate, NaN too
    float low = 0.0f;
    if (k <= NT) {
        // A first bar from the first chunk: each warp's ceil(k / warps)-th largest
        // of its lanes' maxima, the lowest of them. At least k elements of the
        // chunk reach it, so what lies below it cannot count, nor can an equal one
        // of a later chunk. If it is -inf, NaN may count: no bar then.
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < QUADS; ++j) mx = fmaxf(mx, fmaxf(fmaxf(nx[j].x, nx[j].y), fmaxf(nx[j].z, nx[j].w)));
        uint32_t key = rank_key(mx);
#pragma unroll
        for (int size = 2; size <= 32; size <<= 1)  // the lanes' keys in falling order
#pragma unroll
            for (int d = size >> 1; d > 0; d >>= 1) {
                const uint32_t o = __shfl_xor_sync(0xffffffffu, key, d);
                const bool up = ((lane & size) == 0) == ((lane & d) == 0);  // this lane takes the larger
                key = up ? max(key, o) : min(key, o);
            }
        key = __shfl_sync(0xffffffffu, key, (k + NT / 32 - 1) / (NT / 32) - 1);
        if (lane == 0) sm.warp[tid / 32] = key;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NT / 32; ++w) key = min(key, sm.warp[w]);
        if (key > RANK_NEG_INF) {
            all = false;
            low = rank_value(key);
        }
    }
    // takes what `accept`s of a chunk; cuts where more than that might not fit
    auto take = [&](int c, bool any, auto accept) {
        bool full = false;
        if (any) {
            uint32_t pass = 0;
#pragma unroll
            for (int j = 0; j < QUADS; ++j)
                if ((c * QUADS + j) * NT + tid < quads)
                    pass |= ((accept(v[j].x) ? 1u : 0u) | (accept(v[j].y) ? 2u : 0u) | (accept(v[j].z) ? 4u : 0u) |
                             (accept(v[j].w) ? 8u : 0u)) << (4 * j);
            if (pass) {
                int at = atomicAdd(&sm.count, __popc(pass));
                full = at + __popc(pass) >= (all ? k + 1 : trigger);  // the last of the chunk to add sees the whole count
                do {
                    const int b = __ffs(pass) - 1;
                    pass &= pass - 1;
                    const float4 f = b & 8 ? (b & 4 ? v[3] : v[2]) : (b & 4 ? v[1] : v[0]);
                    const float e = b & 2 ? (b & 1 ? f.w : f.z) : (b & 1 ? f.y : f.x);
                    buf[at++] = make_key(e, (uint32_t)(lo + head + 4 * ((c * QUADS + (b >> 2)) * NT + tid) + (b & 3)));
                } while (pass);
            }
        }
        // the buffer holds what may stay uncut and one more chunk
        if (__syncthreads_or(full)) {
            select_k(buf, sm.count, k, sm);
            all = sm.low == 0u;  // a worst one that is NaN lets every number pass
            low = rank_value(sm.low);
        }
    };
    for (int c = 0; c < chunks; ++c) {
#pragma unroll
        for (int j = 0; j < QUADS; ++j) v[j] = nx[j];
        if (c + 1 < chunks) fetch(nx, c + 1);
        float mx = -INFINITY;  // what lies behind the row was read as -inf
#pragma unroll
        for (int j = 0; j < QUADS; ++j) mx = fmaxf(mx, fmaxf(fmaxf(v[j].x, v[j].y), fmaxf(v[j].z, v[j].w)));
        if (c == 0 && !all) take(c, __any_sync(0xffffffffu, mx >= low), [&](float e) { return e >= low; });
        else if (all) take(c, true, [](float) { return true; });
        else take(c, __any_sync(0xffffffffu, mx > low), [&](float e) { return e > low; });
    }
    {  // the last ones (their indices are the highest, so they come last)
        const int i = head + 4 * quads + tid;
        if (i < n && (all || x[i] > low)) buf[atomicAdd(&sm.count, 1)] = make_key(x[i], lo + i);
        __syncthreads();
    }
    const int seen = sm.count;
    __syncthreads();
    if (seen > k) select_k(buf, seen, k, sm);
    if (parts > 1) {
        cluster.sync();
        if (part == 0) {
            int have = sm.count;
            for (int p = 1; p < parts; ++p) {
                const int m = *cluster.map_shared_rank(&sm.count, p);
                const u64 *other = cluster.map_shared_rank(buf, p);
                for (int i = tid; i < m; i += NT) buf[have + i] = other[i];
                have += m;
            }
            __syncthreads();
            if (have > k) select_k(buf, have, k, sm);
        }
        cluster.sync();  // the others' memory has been read
        if (part != 0) return;
    }
    // order the k by counting (short lists) or by a bitonic network
    if (k <= 128) {
        for (int c = tid; c < k; c += NT) {
            const u64 key = buf[c];
            int r = 0;
            for (int j = 0; j < k; ++j) r += buf[j] > key;
            values[row * k + r] = rank_value((uint32_t)(key >> 32));
            indices[row * k + r] = (int)(0xFFFFFFFFu - (uint32_t)key);
        }
        return;
    }
    int m = 256;
    while (m < k) m <<= 1;
    for (int i = k + tid; i < m; i += NT) buf[i] = 0;  // below every key of a token
    for (int size = 2; size <= m; size <<= 1)
        for (int d = size >> 1; d > 0; d >>= 1) {
            __syncthreads();
            for (int i = tid; i < m / 2; i += NT) {
                const int a = 2 * i - (i & (d - 1)), b = a + d;
                const u64 u = buf[a], w = buf[b];
                if ((u < w) == ((a & size) == 0)) {
                    buf[a] = w;
                    buf[b] = u;
                }
            }
        }
    __syncthreads();
    for (int i = tid; i < k; i += NT) {
        values[row * k + i] = rank_value((uint32_t)(buf[i] >> 32));
        indices[row * k + i] = (int)(0xFFFFFFFFu - (uint32_t)buf[i]);
    }
}

// Short rows: a warp each, ROWS of them a block. The bar is the k-th largest of 128
// maxima, of every lane one for each place in its groups of four, so at least k
// logits reach it; a second reading (from L1) collects those that do.
constexpr int ROWS = 4;

__global__ void __launch_bounds__(32 * ROWS)
topk_warp_kernel(const float *__restrict__ logits, long ldl, int rows, int V, int k, float *__restrict__ values,
                 int *__restrict__ indices) {
    __shared__ u64 bufs[ROWS][SMALL];
    const int lane = threadIdx.x & 31;
    const long row = (long)blockIdx.x * ROWS + (threadIdx.x >> 5);
    if (row >= rows) return;
    u64 *buf = bufs[threadIdx.x >> 5];
    const float *x = logits + row * ldl;
    const int head = min(V, (int)(((16 - (uintptr_t)x % 16) / 4) % 4)), quads = (V - head) / 4, tail = head + 4 * quads;
    const float4 *x4 = (const float4 *)(x + head);
    uint32_t key[4];
    {
        float4 m = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
#pragma unroll 4
        for (int q = lane; q < quads; q += 32) {
            const float4 v = __ldg(x4 + q);
            m.x = fmaxf(m.x, v.x);
            m.y = fmaxf(m.y, v.y);
            m.z = fmaxf(m.z, v.z);
            m.w = fmaxf(m.w, v.w);
        }
        key[0] = rank_key(m.x);
        key[1] = rank_key(m.y);
        key[2] = rank_key(m.z);
        key[3] = rank_key(m.w);
    }
    // the lowest rank that is taken, 0 with NaN
    uint32_t least = 0, top = __reduce_max_sync(0xffffffffu, max(max(key[0], key[1]), max(key[2], key[3])));
    while (least < top) {
        const uint32_t mid = least + (top - least) / 2 + 1;
        const int c = __reduce_add_sync(0xffffffffu, (key[0] >= mid) + (key[1] >= mid) + (key[2] >= mid) + (key[3] >= mid));
        if (c >= k) least = mid;
        else top = mid - 1;
        if (c == k) break;
    }
    if (least <= RANK_NEG_INF) least = 0;  // too few numbers: NaN may count
    int n = 0;
    // takes one logit of every lane, of index i
    auto take = [&](bool here, float e, int i) {
        const uint32_t r = rank_key(e), mask = __ballot_sync(0xffffffffu, here && r >= least);
        if (!mask) return;
        if (here && r >= least) buf[n + __popc(mask & ((1u << lane) - 1))] = make_key(e, (uint32_t)i);
        n += __popc(mask);
    };
    // leaves room for 128; later logits have to exceed the worst one kept
    auto room = [&] {
        __syncwarp();
        if (n + 128 <= SMALL) return;
        least = select_small(buf, n, k) + 1;
        n = k;
        __syncwarp();
    };
    take(lane < head, lane < head ? x[lane] : 0.0f, lane);
    const float bar = least > RANK_NEG_INF ? rank_value(least) : 0.0f;
    for (int q0 = 0; q0 < quads; q0 += 32) {
        const int q = q0 + lane;
        const bool here = q < quads;
        const float4 v = here ? __ldg(x4 + q) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (least > RANK_NEG_INF && !__any_sync(0xffffffffu, fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= bar)) continue;
        const int i = head + 4 * q;
        room();
        take(here, v.x, i);
        take(here, v.y, i + 1);
        take(here, v.z, i + 2);
        take(here, v.w, i + 3);
    }
    room();
    take(tail + lane < V, tail + lane < V ? x[tail + lane] : 0.0f, tail + lane);
    __syncwarp();
    if (n > k) select_small(buf, n, k);
    __syncwarp();
    for (int c = lane; c < k; c += 32) {
        const u64 mine = buf[c];
        int r = 0;
        for (int j = 0; j < k; ++j) r += buf[j] > mine;
        values[row * k + r] = rank_value((uint32_t)(mine >> 32));
        indices[row * k + r] = (int)(0xFFFFFFFFu - (uint32_t)mine);
    }
}

}  // namespace

int topk_rows(const float *logits, long ldl, int rows, int V, int k, float *values, int *indices, cudaStream_t s) {
    if (rows <= 0) return OK;
    // Short rows leave a block's warps waiting for one another. A warp each takes
    // 7000 x 500, k = 24 in 16 us where blocks take 80, 7000 x 2600 in 40, 51; but 600 x
    // 2600 in 12.8, 7.8, and 7000 x 5000, k = 64 in 83, 78.
    if (k <= 128 && (V <= 512 || (V <= 4096 && rows >= 12 * num_sms()))) {
        topk_warp_kernel<<<(rows - 1) / ROWS + 1, 32 * ROWS, 0, s>>>(logits, ldl, rows, V, k, values, indices);
        ++g_launch_count;
        CG_CUDA(cudaGetLastError());
        return OK;
    }
    // Few rows leave SMs idle: cut each among up to 8 blocks, as long as a stretch
    // is a chunk or more and the stretches' k candidates fit one block's buffer.
    int parts = 1;
    while (parts < 8 && (long)rows * parts * 2 <= num_sms() && V >= 2 * parts * CHUNK && 2 * parts * k <= k + CHUNK) parts *= 2;
    const int stretch = ((V + parts - 1) / parts + 3) / 4 * 4;
    if ((long)rows * parts > 0x7FFFFFFFL) {
        set_last_error(ERR_ARG, "topk: %d rows are too many", rows);
        return ERR_ARG;
    }
    const size_t smem = (size_t)(std::max(2 * k, TRIGGER) + CHUNK + 8) * sizeof(u64);
    static bool set_on[MAX_DEVICES];
    bool *set;
    CG_TRY(this_device(set_on, &set));
    if (!*set) {
        CG_CUDA(cudaFuncSetAttribute(topk_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)((2 * TOPK_MAX + CHUNK + 8) * sizeof(u64))));
        *set = true;
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
    CG_CUDA(cudaLaunchKernelEx(&cfg, topk_kernel, logits, ldl, V, k, values, indices, stretch));
    ++g_launch_count;
    return OK;
}

}  // namespace cg
