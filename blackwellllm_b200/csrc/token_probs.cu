// Log probabilities of given tokens under rows of logits, each token's rank, the entropy of the row's distribution, and the row's most probable
// tokens, in one pass over the logits.
//
// With m the largest logit of a row, z the sum of e^{x - m} over all elements but one that is m, and w the sum of (x - m) e^{x - m}:
//   log p_i = (x_i - m) - log1p(z),   entropy = log1p(z) - w / (1 + z).
// The largest element's own term, 1, is left out of z so that a sharp distribution (z far below 1) keeps its bits.  Two such triples
// of parts of a row join exactly as one element joins a part: the smaller maximum's element becomes an ordinary term.  All sums are float32,
// in an order that follows from V and the number of blocks that share a row (threads take every so many-th four elements; then trees).  That number
// goes by the call's rows and the GPU's SMs: a row by itself and the same row among hundreds may differ in last bits.
//
// The `top` (at most 32) most probable tokens, ties to the lowest id: a token is a 64-bit key, the logit's bits made ordered above, the
// inverted id below; no two are equal.  Every thread knows the best key of its own elements from the pass.  The top-th best of the warps' best one,
// two or four thread keys is a lower bound of the top-th best of all, and only the threads at or above it (`top` of them, or a few more)
// can own a token of the list.  Their elements are read again (a few percent of the row, from L2), those above the bound are gathered, and
// each finds its place by counting the larger ones.
// (Sorting every warp's thread keys and merging the lists, twice, as first written: 130 us for 1,024 rows of 128,256 with 20 alternatives, now
// 119; one row with five 9.7, now 7.7.)
//
// Bound by memory: 4 bytes an element (1,024 rows of 128,256 without alternatives: 96 us, 5.5 TB/s).  A row is one block's, or, where there are few
// rows, shared by a cluster of 2, 4 or 8 blocks that join through distributed shared memory; then what follows the pass over the row counts, a
// chain of short steps between barriers.  What runs once a row is kept small (not inlined, not unrolled): its instructions come from L2 first
// (one row 8.4 us with all of it in line, 7.7 so).
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
// (m -infinity: a part without an element that counts, and its factor is 0; a difference of two of them, no number, becomes LEAST)
__device__ __forceinline__ Part join(Part a, Part b) {
    const bool swap = b.m > a.m;
    const Part x = {swap ? b.m : a.m, swap ? b.z : a.z, swap ? b.w : a.w}, y = {swap ? a.m : b.m, swap ? a.z : b.z, swap ? a.w : b.w};
    const float d = fmaxf(y.m - x.m, LEAST), f = ex2(d * LOG2E), n = 1.f + y.z;
    return {x.m, x.z + f * n, x.w + f * (y.w + d * n)};
}

// a warp's largest key
__device__ __forceinline__ u64 warp_max(u64 k) {
    const unsigned hi = __reduce_max_sync(0xffffffffu, (unsigned)(k >> 32));
    return (u64)hi << 32 | __reduce_max_sync(0xffffffffu, (unsigned)(k >> 32) == hi ? (unsigned)k : 0u);
}
// The n keys, no two alike, put in falling order as far as the first `top`: a thread counts what is above its key.
__device__ __noinline__ void place_keys(const u64* keys, int n, u64* sorted, int top) {
    for (int a = threadIdx.x; a < n; a += THREADS) {
        const u64 k = keys[a];
        int above = 0;
#pragma unroll 4
        for (int b = 0; b < n; ++b) above += keys[b] > k;
        if (k != 0 && above < top) sorted[above] = k;
    }
    __syncwarp();
}
// the 32 best of two lists in falling order, in falling order
__device__ __forceinline__ u64 merge32(u64 a, u64 b) {
    const int lane = threadIdx.x & 31;
    const u64 r = __shfl_sync(0xffffffffu, b, 31 - lane);
    u64 k = a > r ? a : r;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const u64 other = __shfl_xor_sync(0xffffffffu, k, o);
        k = ((lane & o) == 0) == (k > other) ? k : other;
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
constexpr int ROOM = 256;
struct Shared {
    Found warps[WARPS];
    u64 some[4 * WARPS];         // of every warp's thread keys the best few
    u64 bound;
    int owners, gathered;        // how many
    int owner[THREADS];          // threads that can own a token of the list
    u64 keys[ROOM + 4 * THREADS];     // tokens gathered, and room for a round's
    u64 sorted[MAX_TOP];
    Found found[MOST_BLOCKS];    // in the cluster's first block: of every block
    u64 found_best[MOST_BLOCKS][MAX_TOP];
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
// joined over groups of n neighbouring lanes (a power of two); the first lane's is the result (others' may differ in a last bit)
__device__ __noinline__ Found join_lanes(Found a, int n) {
#pragma unroll 1
    for (int o = n >> 1; o > 0; o >>= 1) {
        const Found b = shuffled(a, o);
        a.part = join(a.part, b.part);
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
    __syncwarp();
    if (p.top > 0) {
        if (threadIdx.x < MAX_TOP) sh.sorted[threadIdx.x] = 0;
        if (threadIdx.x == 0) { sh.owners = sh.gathered = 0; sh.bound = 1; }        // (a short row has fewer keys: any may be in the list)
        u64 mine = 0;
        if (own < f1) {
            const float4 v = load4<VEC>(row, 4 * s.four, p.V);          // again, for which of the four it was
            mine = key_of(s.best, 4 * s.four + (v.x == s.best ? 0 : v.y == s.best ? 1 : v.z == s.best ? 2 : 3));
        }
        const int few = p.top == 1 ? 1 : p.top <= 8 ? 2 : 4;             // of a warp
        u64 left = mine;
        for (int i = 0; i < few; ++i) {
            const u64 k = warp_max(left);
            if (left == k) left = 0;
            if (lane == 0) sh.some[warp * few + i] = k;
            __syncwarp();
        }
        __syncthreads();
        const u64 a = lane < WARPS * few ? sh.some[lane] : 0, b = lane + 32 < WARPS * few ? sh.some[lane + 32] : 0;
        for (int i = 0; i < few; ++i) {
            const u64 k = sh.some[warp * few + i];
            const int above = __popc(__ballot_sync(0xffffffffu, a > k)) + __popc(__ballot_sync(0xffffffffu, b > k));
            if (lane == 0 && k != 0 && above == p.top - 1) sh.bound = k;
            __syncwarp();
        }
        __syncthreads();
        u64 bound = sh.bound;
        if (p.top == 1) {
            if (mine == bound) sh.sorted[0] = mine;
        } else {
            const bool is_owner = mine >= bound;
            const unsigned vote = __ballot_sync(0xffffffffu, is_owner);
            int to = 0;
            if (lane == 0 && vote) to = atomicAdd(&sh.owners, __popc(vote));
            __syncwarp();
            to = __shfl_sync(0xffffffffu, to, 0);
            if (is_owner) sh.owner[to + __popc(vote & ((1u << lane) - 1))] = (int)threadIdx.x;
            __syncthreads();
            const int rounds = (f1 - f0 + THREADS - 1) / THREADS, items = sh.owners * rounds;
            for (int i0 = 0; i0 < items; i0 += THREADS) {                // (uniform)
                const int i = i0 + (int)threadIdx.x, who = i / rounds, f = i < items ? f0 + (i - who * rounds) * THREADS + sh.owner[who] : f1;
                u64 k[4] = {0, 0, 0, 0};
                if (f < f1) {
                    const float4 v = load4<VEC>(row, 4 * f, p.V);
                    const float y[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const u64 key = 4 * f + e < p.V ? key_of(y[e], 4 * f + e) : 0;
                        k[e] = key >= bound ? key : 0;
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const unsigned b = __ballot_sync(0xffffffffu, k[e] != 0);
                    if (!b) continue;
                    int to = 0;
                    if (lane == 0) to = atomicAdd(&sh.gathered, __popc(b));
                    __syncwarp();
                    to = __shfl_sync(0xffffffffu, to, 0);
                    if (k[e]) sh.keys[to + __popc(b & ((1u << lane) - 1))] = k[e];
                    __syncwarp();
                }
                __syncthreads();
                const int have = sh.gathered;
                const bool last = i0 + THREADS >= items;
                if (last || have > ROOM) {
                    place_keys(sh.keys, have, sh.sorted, p.top);
                    if (last) break;
                    // (a row that is made for it) the best stay, and the last of them is the bound from here on: no element comes twice
                    __syncthreads();
                    if ((int)threadIdx.x < p.top) sh.keys[threadIdx.x] = sh.sorted[threadIdx.x];
                    if (threadIdx.x == 0) sh.gathered = p.top;
                    bound = sh.sorted[p.top - 1];
                }
                __syncthreads();
            }
        }
    }
    __syncthreads();
    if (blocks > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (warp == 0) {
        all = join_lanes(lane < WARPS ? sh.warps[lane] : Found{{-INFINITY, 0.f, 0.f}, 0, 0}, WARPS);
        // into the cluster's first block
        if (lane == 0) *(blocks > 1 ? in_first_block(&sh.found[part]) : &sh.found[0]) = all;
        if (blocks > 1 && p.top > 0) *in_first_block(&sh.found_best[part][lane]) = sh.sorted[lane];
    }
    if (blocks > 1) {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        if (part != 0) return;
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (p.top > 0) {
            // the blocks' lists, two by two
            u64 list = warp < blocks ? sh.found_best[warp][lane] : 0;
            for (int o = blocks >> 1; o > 0; o >>= 1) {
                if (warp < o) {
                    list = merge32(list, sh.found_best[warp + o][lane]);
                    sh.found_best[warp][lane] = list;
                }
                __syncthreads();
            }
            if (warp == 0) sh.sorted[lane] = list;
        }
        __syncwarp();
    } else {
        __syncwarp();
    }
    if (warp != 0) return;
    const u64 list = lane < p.top ? sh.sorted[lane] : 0;
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
    // sorting than they even out (1,024 rows of 128,256 with one alternative, in a graph: 101 us, as two blocks each 103, as four 133; 107 in a
    // stream of calls).
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
