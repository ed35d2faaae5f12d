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
// the 32 best of the first n warps' lists, in warp 0 (all threads of the block call it)
__device__ __forceinline__ u64 merge_warps(u64 k, u64 (*lists)[32], int n) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int o = 1;
    while (o < n) o <<= 1;
    if (warp < n) lists[warp][lane] = k;
    for (o >>= 1; o > 0; o >>= 1) {
        __syncthreads();
        if (warp < o && warp + o < n) {
            k = merge32(k, lists[warp + o][lane]);
            lists[warp][lane] = k;
        }
        n = min(n, o);
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

// What a block found in its share of a row.
struct Found { Part part; int count, bad; };
constexpr int MOST_BLOCKS = 8;
struct Shared {
    Found warps[WARPS];
    u64 lists[WARPS][32];
    u64 loose[WARPS][128];       // a warp's candidates before they are sorted
    u64 best[32];                // the block's best thread keys
    Found found[MOST_BLOCKS];    // in the cluster's first block: of every block
    u64 found_best[MOST_BLOCKS][32];
};
template <typename T> __device__ __forceinline__ T* in_first_block(T* at) { return cg::this_cluster().map_shared_rank(at, 0); }

// A thread's elements so far.  The best stays out of the sums: of four elements and the best before them, seven minima and maxima leave the best
// and four others (min and max of a pair at a time), and those are added.  The sums' exponents stand against `ref`, a best of earlier, until the
// best is more than SLACK above it: moving a reference with every new best is done by some lane of a warp nearly every time, and cost three
// quarters of the instructions.
constexpr float SLACK = 16.f;
struct Running {
    float best = -INFINITY, ref = -INFINITY;
    int four, count = 0;                     // the four where the best first stood; elements that stand before the target
    float z[2] = {0.f, 0.f}, w[2] = {0.f, 0.f};      // sums of e^(x - ref) and of (x - ref) e^(x - ref), of every other element
};
__device__ __forceinline__ void take4(Running& s, float4 x, int f, float xt, int target) {
    // (the maxima keep what is no number, and the best with them: it is looked at in the end)
    const float h0 = max_or_nan(x.x, x.y), l0 = fminf(x.x, x.y), h1 = max_or_nan(x.z, x.w), l1 = fminf(x.z, x.w);
    const float most = max_or_nan(h0, h1), l2 = fminf(h0, h1), l3 = fminf(most, s.best);
    if (!(most < xt)) {
        const int c = 4 * f;
        if (c > target) s.count += (x.x > xt) + (x.y > xt) + (x.z > xt) + (x.w > xt);
        else if (c + 3 < target) s.count += (x.x >= xt) + (x.y >= xt) + (x.z >= xt) + (x.w >= xt);
        else s.count += (x.x > xt || (x.x == xt && c < target)) + (x.y > xt || (x.y == xt && c + 1 < target)) +
                        (x.z > xt || (x.z == xt && c + 2 < target)) + (x.w > xt || (x.w == xt && c + 3 < target));
    }
    if (most > s.best) s.four = f;
    s.best = max_or_nan(s.best, most);
    if (s.best > s.ref + SLACK) {
        const float d = fmaxf(s.ref - s.best, LEAST), e = ex2(d * LOG2E);
#pragma unroll
        for (int i = 0; i < 2; ++i) { s.w[i] = e * fmaf(d, s.z[i], s.w[i]); s.z[i] *= e; }
        s.ref = s.best;
    }
    // (-infinity, here or as the reference so far, comes out as a term of 0.  One element an instruction: packed pairs, which would have to be put
    // together from what the minima leave, took twice the instructions)
    auto add = [&](float x, int i) {
        const float d = fmaxf(x - s.ref, LEAST), t = ex2(d * LOG2E);
        s.z[i] += t;
        s.w[i] = fmaf(t, d, s.w[i]);
    };
    add(l0, 0);
    add(l1, 1);
    add(l2, 0);
    add(l3, 1);
}
// the same against the best
__device__ __forceinline__ Part part_of(const Running& s) {
    if (s.ref == -INFINITY) return {s.best, 0.f, 0.f};
    const float d = fmaxf(s.ref - s.best, LEAST), e = ex2(d * LOG2E), z = s.z[0] + s.z[1];
    return {s.best, e * z, e * fmaf(d, z, s.w[0] + s.w[1])};
}

__device__ __forceinline__ Found shuffled(const Found& a, int o) {
    return {{__shfl_xor_sync(0xffffffffu, a.part.m, o), __shfl_xor_sync(0xffffffffu, a.part.z, o), __shfl_xor_sync(0xffffffffu, a.part.w, o)},
            __shfl_xor_sync(0xffffffffu, a.count, o), __shfl_xor_sync(0xffffffffu, a.bad, o)};
}
// joined over groups of n neighbouring lanes (a power of two), both lanes of a pair in the same order
__device__ __forceinline__ Found join_lanes(Found a, int n) {
    for (int o = n >> 1; o > 0; o >>= 1) {
        const Found b = shuffled(a, o);
        a.part = (threadIdx.x & o) ? join(b.part, a.part) : join(a.part, b.part);
        a.count += b.count;
        a.bad |= b.bad;
    }
    return a;
}

// grid: rows * blocks; a row's `blocks` blocks are one cluster.  AT_ONCE: blocks on an SM (three while all SMs have work for long; where few blocks are
// launched at all they would gather on some of them).
template <bool VEC, int AT_ONCE>
__global__ void __launch_bounds__(THREADS, AT_ONCE)
token_probs_kernel(Args p, int blocks) {
    BW_PDL_TRIGGER();
    __shared__ Shared sh;
    if (blocks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");     // (the cluster's blocks have begun: waited for below)
    const int r = blockIdx.x / blocks, part = blockIdx.x - r * blocks;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float* row = p.logits + (size_t)r * p.ld;
    // the block's share: whole fours
    const int fours = (p.V + 3) / 4, each = (fours + blocks - 1) / blocks;
    const int f0 = min(fours, part * each), f1 = min(fours, f0 + each);
    BW_PDL_WAIT();
    const int own = f0 + (int)threadIdx.x, target = p.target[r];
    const bool given = target >= 0 && target < p.V;
    const float xt = given ? row[target] : INFINITY;
    Running s;
    s.four = own;
    // four whole fours at a time without a look at the row's end, then what is left
    int f = own;
    const int whole = min(f1, p.V / 4);
    for (; f + (UNROLL - 1) * THREADS < whole; f += UNROLL * THREADS) {
        float4 x[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const float* at = row + 4 * (f + u * THREADS);
            x[u] = VEC ? *reinterpret_cast<const float4*>(at) : make_float4(at[0], at[1], at[2], at[3]);
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) take4(s, x[u], f + u * THREADS, xt, target);
    }
    for (; f < f1; f += THREADS) take4(s, load4<VEC>(row, 4 * f, p.V), f, xt, target);
    Found all{part_of(s), s.count, !(s.best < INFINITY)};
    all = join_lanes(all, 32);
    if (lane == 0) sh.warps[warp] = all;
    u64 list = 0;
    if (p.top > 0) {
        u64 mine = 0;
        if (own < f1) {
            const float4 v = load4<VEC>(row, 4 * s.four, p.V);          // again, for which of the four it was
            mine = key_of(s.best, 4 * s.four + (v.x == s.best ? 0 : v.y == s.best ? 1 : v.z == s.best ? 2 : 3));
        }
        list = merge_warps(sort32(mine), sh.lists, WARPS);
        if (p.top > 1) {
            // warp 0 has the best thread keys; the owners of the first `top` read their elements again
            if (warp == 0) sh.best[lane] = lane < p.top ? list : 0;
            __syncthreads();
            const u64 bound = sh.best[p.top - 1];
            const int rounds = (f1 - f0 + THREADS - 1) / THREADS, items = p.top * rounds;
            list = 0;
            for (int i0 = 0; i0 < items; i0 += THREADS) {                // (uniform)
                if (i0 + 32 * warp >= items) continue;
                const int i = i0 + (int)threadIdx.x, who = i / rounds, it = i - who * rounds;
                const u64 owner = i < items ? sh.best[who] : 0;
                const int f = owner ? f0 + it * THREADS + (id_of(owner) / 4 - f0) % THREADS : f1;
                const float4 v = f < f1 ? load4<VEC>(row, 4 * f, p.V) : make_float4(0.f, 0.f, 0.f, 0.f);
                const float y[4] = {v.x, v.y, v.z, v.w};
                // the warp's candidates side by side, then 32 of them at a time: mostly a few in all
                int n = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const u64 k = f < f1 && 4 * f + e < p.V ? key_of(y[e], 4 * f + e) : 0;
                    const bool is = k != 0 && k >= bound;
                    const unsigned b = __ballot_sync(0xffffffffu, is);
                    if (is) sh.loose[warp][n + __popc(b & ((1u << lane) - 1))] = k;
                    n += __popc(b);
                }
                __syncwarp();
                for (int j = 0; j < n; j += 32) list = merge32(list, sort32(j + lane < n ? sh.loose[warp][j + lane] : 0));
                __syncwarp();
            }
            __syncthreads();
            list = merge_warps(list, sh.lists, min(WARPS, (items + 31) / 32));
        }
    }
    __syncthreads();
    if (blocks > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (warp == 0) {
        all = join_lanes(lane < WARPS ? sh.warps[lane] : Found{{-INFINITY, 0.f, 0.f}, 0, 0}, WARPS);
        // into the cluster's first block
        if (lane == 0) *(blocks > 1 ? in_first_block(&sh.found[part]) : &sh.found[0]) = all;
        if (p.top > 0) *(blocks > 1 ? in_first_block(&sh.found_best[part][lane]) : &sh.found_best[0][lane]) = list;
    }
    if (blocks > 1) {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        if (part != 0) return;
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    } else {
        __syncwarp();
    }
    if (p.top > 0) list = blocks > 1 ? merge_warps(warp < blocks ? sh.found_best[warp][lane] : 0, sh.lists, blocks) : list;
    if (warp != 0) return;
    all = join_lanes(lane < blocks ? sh.found[lane] : Found{{-INFINITY, 0.f, 0.f}, 0, 0}, MOST_BLOCKS);
    all = Found{{__shfl_sync(0xffffffffu, all.part.m, 0), __shfl_sync(0xffffffffu, all.part.z, 0), __shfl_sync(0xffffffffu, all.part.w, 0)},
                __shfl_sync(0xffffffffu, all.count, 0), __shfl_sync(0xffffffffu, all.bad, 0)};
    const Part& q = all.part;
    const bool nothing = all.bad || !(q.m > -INFINITY);       // no distribution: NaN, an infinite logit, or nothing but -infinity
    const float log_z = log1pf(q.z), nan = __uint_as_float(0x7fffffffu);
    if (lane == 0) {
        p.log_prob[r] = nothing || !given ? nan : (xt - q.m) - log_z;
        p.entropy[r] = nothing ? nan : log_z - q.w / (1.f + q.z);
        p.rank[r] = nothing || !given ? -1 : all.count;
    }
    if (lane < p.top) {
        p.top_ids[(size_t)r * p.top + lane] = nothing ? -1 : id_of(list);
        p.top_log_probs[(size_t)r * p.top + lane] = nothing ? nan : (value_of(list) - q.m) - log_z;
    }
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
    // Few rows: as many blocks a row as run at once (two an SM), while each has a few thousand elements.  Many: a block a row; shared rows cost more in
    // sorting than they even out (1,024 rows of 128,256 with one alternative: 106 us, as two blocks each 112, as four 154).
    const long long sms = bw::num_sms();
    const bool few = R <= 2 * sms;
    int blocks = 1;
    while (few && blocks < 8 && R * 2LL * blocks <= 2 * sms && V >= 8192 * blocks) blocks *= 2;
    if ((long long)R * blocks > 0x7fffffffll) return BW_ERR_UNSUPPORTED;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(R * blocks)); cfg.blockDim = dim3(THREADS); cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)blocks; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = bw::pdl_enabled() ? 2 : 1;
    const auto kernel = few ? (vec ? token_probs_kernel<true, 2> : token_probs_kernel<false, 2>)
                            : (vec ? token_probs_kernel<true, 3> : token_probs_kernel<false, 3>);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p, blocks);
    if (e != cudaSuccess) return (int)e;
    BW_LAUNCH_CHECK();
    return 0;
}
