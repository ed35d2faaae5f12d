// Log probabilities of given tokens under rows of logits, each token's rank, the entropy of the row's distribution, and the row's most probable
// tokens, in one pass over the logits.
//
// With m the largest logit of a row, z the sum of e^{x - m} over all elements but one that is m, and w the sum of (x - m) e^{x - m}:
//   log p_i = (x_i - m) - log1p(z),   entropy = log1p(z) - w / (1 + z).
// The largest element's own term, 1, is left out of z so that a sharp distribution (z far below 1) keeps its bits.  Two such triples
// of parts of a row join exactly as one element joins a part: the smaller maximum's element becomes an ordinary term.  All sums are float32,
// in an order that depends on V alone (threads take every so many-th four elements; then trees).
//
// The `top` (at most 32) most probable tokens, ties to the lowest id: a token is a 64-bit key, the logit's bits made ordered above, the
// inverted id below; no two are equal.  Every thread knows the best key of its own elements from the pass; the top-th best of those is a
// lower bound of the top-th best of all, and only the `top` threads at or above it can own a token of the list.  Their elements are read
// again (a few percent of the row, from L2) and go, where they are above the bound, through lists of 32 sorted keys, one per warp, kept by
// bitonic sorts and merges.
//
// Bound by memory: 4 bytes an element.  A row is one block's, or, where there are few rows, shared by a cluster of 2, 4 or 8 blocks that join
// through distributed shared memory.
#include "common.cuh"
#include <cooperative_groups.h>

namespace {

namespace cg = cooperative_groups;
using u64 = unsigned long long;
constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr int UNROLL = 4;
constexpr float LOG2E = 1.4426950408889634f;
constexpr int MAX_TOP = 32;
constexpr float LEAST = -200.f;      // e^-200 is 0 here; differences stop there, so that 0 times one is 0

struct Args {
    const float* logits; const int* target;
    float* log_prob; float* entropy; int* rank; int* top_ids; float* top_log_probs;
    int V, top;
    size_t ld;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max_or_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
// ordered: a larger logit has a larger key, of equal ones the lower id; 0: no element
__device__ __forceinline__ u64 key_of(float x, int id) {
    const unsigned u = __float_as_uint(x + 0.f);       // (-0 counts as 0)
    const unsigned o = u & 0x80000000u ? ~u : u | 0x80000000u;
    return (u64)o << 32 | (0xffffffffu - (unsigned)id);
}
__device__ __forceinline__ float value_of(u64 key) {
    const unsigned o = (unsigned)(key >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ int id_of(u64 key) { return (int)(0xffffffffu - (unsigned)key); }

struct Part { float m, z, w; };
// (-infinity: a part without an element that counts)
__device__ __forceinline__ Part join(Part a, Part b) {
    if (b.m > a.m) { const Part t = a; a = b; b = t; }
    if (b.m == -INFINITY) return a;
    const float d = fmaxf(b.m - a.m, LEAST), f = ex2(d * LOG2E);
    a.z += f * (1.f + b.z);
    a.w += f * (b.w + d * (1.f + b.z));
    return a;
}

__device__ __forceinline__ u64 shfl_xor_key(u64 k, int o) { return __shfl_xor_sync(0xffffffffu, k, o); }
// a warp's 32 keys in falling order (lane 0: the best)
__device__ __forceinline__ u64 sort32(u64 k) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int o = size >> 1; o > 0; o >>= 1) {
            const u64 other = shfl_xor_key(k, o);
            const bool falling = (lane & size) == 0 || size == 32;
            const bool take_max = ((lane & o) == 0) == falling;
            k = take_max ? (k > other ? k : other) : (k < other ? k : other);
        }
    return k;
}
// the 32 best of two lists in falling order, in falling order
__device__ __forceinline__ u64 merge32(u64 a, u64 b) {
    const int lane = threadIdx.x & 31;
    const u64 r = __shfl_sync(0xffffffffu, b, 31 - lane);
    u64 k = a > r ? a : r;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const u64 other = shfl_xor_key(k, o);
        k = (lane & o) == 0 ? (k > other ? k : other) : (k < other ? k : other);
    }
    return k;
}
// the 32 best of the block's lists (one a warp), in warp 0
__device__ __forceinline__ u64 merge_warps(u64 k, u64 (*lists)[32]) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    lists[warp][lane] = k;
#pragma unroll
    for (int o = WARPS / 2; o > 0; o >>= 1) {
        __syncthreads();
        if (warp < o) {
            k = merge32(k, lists[warp + o][lane]);
            lists[warp][lane] = k;
        }
    }
    return k;
}

template <bool VEC>
__device__ __forceinline__ float4 load4(const float* row, int c, int V) {
    if (VEC && c + 4 <= V) return *reinterpret_cast<const float4*>(row + c);
    float4 v;
    v.x = c < V ? row[c] : -INFINITY; v.y = c + 1 < V ? row[c + 1] : -INFINITY;
    v.z = c + 2 < V ? row[c + 2] : -INFINITY; v.w = c + 3 < V ? row[c + 3] : -INFINITY;
    return v;
}

struct Shared {
    Part parts[WARPS];
    int counts[WARPS];
    int bad;
    u64 lists[WARPS][32];
    // the block's result, read by the cluster's first block
    Part part; int count; u64 best[32];
};

// grid: rows * blocks; a row's `blocks` blocks are one cluster.
template <bool VEC>
__global__ void __launch_bounds__(THREADS, 2)
token_probs_kernel(Args p, int blocks) {
    BW_PDL_TRIGGER();
    BW_PDL_WAIT();
    __shared__ Shared sh;
    const int r = blockIdx.x / blocks, part = blockIdx.x - r * blocks;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float* row = p.logits + (size_t)r * p.ld;
    const int target = p.target[r];
    const bool given = target >= 0 && target < p.V;
    const float xt = given ? row[target] : INFINITY;
    // the block's share: whole fours
    const int fours = (p.V + 3) / 4, each = (fours + blocks - 1) / blocks;
    const int f0 = min(fours, part * each), f1 = min(fours, f0 + each);
    if (threadIdx.x == 0) sh.bad = 0;

    Part me{-INFINITY, 0.f, 0.f};
    int id = 4 * (f0 + (int)threadIdx.x), count = 0;
    const bool any = f0 + (int)threadIdx.x < f1;
    bool bad = false;
    for (int f = f0 + threadIdx.x; f < f1; f += UNROLL * THREADS) {
        float x[UNROLL][4];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int c = 4 * (f + u * THREADS);
            const float4 v = f + u * THREADS < f1 ? load4<VEC>(row, c, p.V) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            x[u][0] = v.x; x[u][1] = v.y; x[u][2] = v.z; x[u][3] = v.w;
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int c = 4 * (f + u * THREADS);
            if (c >= 4 * f1) continue;
            const float cm = max_or_nan(max_or_nan(x[u][0], x[u][1]), max_or_nan(x[u][2], x[u][3]));
            int skip = -1;
            if (!(cm <= me.m)) {
                bad |= !(cm < INFINITY);
                skip = x[u][0] == cm ? 0 : x[u][1] == cm ? 1 : x[u][2] == cm ? 2 : 3;
                const float d = fmaxf(me.m - cm, LEAST), f2 = ex2(d * LOG2E);
                if (me.m == -INFINITY) me.z = me.w = 0.f;
                else { me.w = f2 * (me.w + d * (1.f + me.z)); me.z = f2 * (1.f + me.z); }
                me.m = cm; id = c + skip;
            }
            float z = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                // (-infinity, here or as the maximum so far, comes out as a term of 0)
                const float d = fmaxf(x[u][e] - me.m, LEAST);
                const float t = e == skip ? 0.f : ex2(d * LOG2E);
                z += t;
                me.w = fmaf(t, d, me.w);
            }
            me.z += z;
            if (c > target) {
#pragma unroll
                for (int e = 0; e < 4; ++e) count += x[u][e] > xt;
            } else if (c + 3 < target) {
#pragma unroll
                for (int e = 0; e < 4; ++e) count += x[u][e] >= xt;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) count += x[u][e] > xt || (x[u][e] == xt && c + e < target);
            }
        }
    }
    const u64 mine = any ? key_of(me.m, id) : 0;
    __syncthreads();
    if (bad) sh.bad = 1;
    // the block's triple and count
    Part all = me;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const Part other{__shfl_xor_sync(0xffffffffu, all.m, o), __shfl_xor_sync(0xffffffffu, all.z, o), __shfl_xor_sync(0xffffffffu, all.w, o)};
        // (both lanes of a pair join the same two in the same order)
        all = (lane & o) ? join(other, all) : join(all, other);
        count += __shfl_xor_sync(0xffffffffu, count, o);
    }
    if (lane == 0) { sh.parts[warp] = all; sh.counts[warp] = count; }
    u64 list = 0;
    if (p.top > 0) {
        list = merge_warps(sort32(mine), sh.lists);        // (its first barrier also stands before the reads below)
        if (p.top > 1) {
            // warp 0 has the best thread keys; the owners of the first `top` read their elements again
            if (warp == 0) sh.best[lane] = lane < p.top ? list : 0;
            __syncthreads();
            const u64 bound = sh.best[p.top - 1];
            const int rounds = (f1 - f0 + THREADS - 1) / THREADS;
            list = 0;
            for (int i0 = 0; i0 < p.top * rounds; i0 += THREADS) {       // (uniform)
                const int i = i0 + (int)threadIdx.x, who = i / rounds, it = i - who * rounds;
                const u64 owner = who < p.top ? sh.best[who] : 0;
                const int f = owner ? f0 + it * THREADS + (id_of(owner) / 4 - f0) % THREADS : f1;
                const float4 v = f < f1 ? load4<VEC>(row, 4 * f, p.V) : make_float4(0.f, 0.f, 0.f, 0.f);
                const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    u64 k = f < f1 && 4 * f + e < p.V ? key_of(x[e], 4 * f + e) : 0;
                    if (k < bound) k = 0;
                    if (__any_sync(0xffffffffu, k != 0)) list = merge32(list, sort32(k));
                }
            }
            __syncthreads();
            list = merge_warps(list, sh.lists);
        }
        if (warp == 0) sh.best[lane] = list;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        Part s = sh.parts[0];
        int n = sh.counts[0];
        for (int w = 1; w < WARPS; ++w) { s = join(s, sh.parts[w]); n += sh.counts[w]; }
        sh.part = s; sh.count = n;
    }
    if (blocks > 1) cg::this_cluster().sync();
    else __syncthreads();
    if (part == 0 && warp == 0) {
        Part s = sh.part;
        int n = sh.count, wrong = sh.bad;
        u64 best = p.top > 0 ? sh.best[lane] : 0;
        for (int b = 1; b < blocks; ++b) {
            const Shared* other = cg::this_cluster().map_shared_rank(&sh, b);
            s = join(s, other->part);
            n += other->count;
            wrong |= other->bad;
            if (p.top > 0) best = merge32(best, other->best[lane]);
        }
        const bool none = wrong || !(s.m > -INFINITY);       // no distribution: NaN, an infinite logit, or nothing but -infinity
        const float log_z = log1pf(s.z), nan = __uint_as_float(0x7fffffffu);
        if (lane == 0) {
            p.log_prob[r] = none || !given ? nan : (xt - s.m) - log_z;
            p.entropy[r] = none ? nan : log_z - s.w / (1.f + s.z);
            p.rank[r] = none || !given ? -1 : n;
        }
        if (lane < p.top) {
            p.top_ids[(size_t)r * p.top + lane] = none ? -1 : id_of(best);
            p.top_log_probs[(size_t)r * p.top + lane] = none ? nan : (value_of(best) - s.m) - log_z;
        }
    }
    if (blocks > 1) cg::this_cluster().sync();      // a block's shared memory stays until it has been read
}

}  // namespace

// logits float32, rows ld apart; target: int32 a row, outside [0, V): none is given (NaN and rank -1); top at most 32 and at most V, top_ids and
// top_log_probs [R][top].
BW_EXPORT int bw_token_probs(const float* logits, const int* target, float* log_prob, float* entropy, int* rank, int* top_ids,
                             float* top_log_probs, int R, int V, int top, long long ld, void* stream) {
    if (R <= 0) return 0;
    if (V <= 0 || V > (1 << 30) || ld < V || !logits || !target || !log_prob || !entropy || !rank) return BW_ERR_BAD_ARG;
    if (top < 0 || top > MAX_TOP || top > V || (top && (!top_ids || !top_log_probs))) return BW_ERR_BAD_ARG;
    const Args p{logits, target, log_prob, entropy, rank, top_ids, top_log_probs, V, top, (size_t)ld};
    const bool vec = ((uintptr_t)logits & 15) == 0 && ld % 4 == 0;
    // as many blocks a row as run at once (two an SM), while each has a few thousand elements
    const long long room = 2LL * bw::num_sms();
    int blocks = 1;
    while (blocks < 8 && R * 2LL * blocks <= room && V >= 8192 * blocks) blocks *= 2;
    if ((long long)R * blocks > 0x7fffffffll) return BW_ERR_UNSUPPORTED;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(R * blocks)); cfg.blockDim = dim3(THREADS); cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)blocks; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = bw::pdl_enabled() ? 2 : 1;
    const cudaError_t e = vec ? cudaLaunchKernelEx(&cfg, token_probs_kernel<true>, p, blocks)
                              : cudaLaunchKernelEx(&cfg, token_probs_kernel<false>, p, blocks);
    if (e != cudaSuccess) return (int)e;
    BW_LAUNCH_CHECK();
    return 0;
}
