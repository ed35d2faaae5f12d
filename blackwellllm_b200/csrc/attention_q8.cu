// Causal grouped-query attention over the 8-bit cache (quant_cache.cu): bfloat16 queries, keys and values as whole numbers with one float32
// scale a (token, kv head), head size HEAD_DIM (a compile-time multiple of 16 up to 256; the library is built per head size).
//
//   score of query i and key j = scale * ks_j * sum_c q_ic kc_jc,   out_ic = sum_j (p_ij vs_j) vc_jc / sum_j p_ij
//
// The whole numbers are widened to float16, in which they are exact, and the products run on the tensor cores (mma.sync m16n8k16, float32
// sums).  A byte b of two's complement with its top bit turned over is u = b + 128, and 0x6400 | u is the float16 1024 + u: one byte
// permutation makes two.  For V 1152 is subtracted from it; for K it is left in and 1152 times the sum of the query's channels comes off the score
// (which is then off by at most a few 2^-24 of 1152 sum |q|, a few 1e-7 of the largest score that such a key can have).
//   Queries: a row is multiplied by a power of two that brings its largest channel to 2^14 up to 2^15, so that bfloat16's eight bits
//      fit float16's eleven whatever the row's size (channels below 2^-31 of the largest lose bits); the power comes off the score.
//   Weights: w_ij = e_ij vs_j with e_ij = 2^(t_ij - m_i), t the score in powers of two.  The reference m follows the largest t + log2 vs, so what
//      counts most is near 1 and float16 rounds each weight by at most 2^-11 of itself, or of 2^-14: never more than 2^-25 of the largest.
//      The denominator is the sum of e in float32.  For the reference a scale counts as 2^-102 at least (rows of zeros have 0), so e stays
//      below 2^110 and 2^18 keys below infinity; the smallest scale that is written, 2^-117, then still has weights of 2^-15.  Where m moves far
//      (rows of zeros, then values that are large) sums are multiplied by the root of the factor twice, which never vanishes by itself.
// Everything else is float32: scores, references, sums, outputs.
//
// The products are turned around: S^T = K Q^T and O^T = V^T W^T, keys and channels in the 16 rows of an instruction, queries in its 8
// columns.  A decoding request has the G query heads of a kv head as its queries, mostly 4 to 8: so an instruction is full, and an element of
// the cache is widened once for all of them.
//   K: ldmatrix on bytes gives a lane four neighbouring channels of one key, which are taken as k indices 2q, 2q + 1, 2q + 8, 2q + 9 (a sum does
//      not mind the order of its terms; the queries' fragments take the same order);
//   V: ldmatrix.trans on bytes gives a lane two neighbouring channels of two keys; the even channel goes to row r of the instruction, the odd
//      one to row r + 8, so a lane ends with two neighbouring output channels of a query;
//   W: the scores' fragment, rounded, is turned by movmatrix.
// The eight rows of an ldmatrix lie in different banks: 16-byte units are permuted by the row's number where a row is 64, 128 or 256 bytes,
// else rows are an odd number of units apart.
#include "common.cuh"
#include <cuda_fp16.h>

#ifndef HEAD_DIM
#error "compile with -DHEAD_DIM=<multiple of 16>"
#endif

using bf16 = __nv_bfloat16;

namespace {

constexpr int HD = HEAD_DIM;
static_assert(HD % 16 == 0 && HD >= 16 && HD <= 256, "head size must be a multiple of 16 in [16, 256]");
constexpr int CHUNKS = HD / 16;                    // 16-byte units of a row
constexpr bool PERMUTED = HD == 64 || HD == 128 || HD == 256;
constexpr int STRIDE = PERMUTED ? HD : (CHUNKS | 1) * 16;      // bytes between rows of shared memory
// where unit c of row r lies in its row
__device__ __forceinline__ int unit(int r, int c) { return PERMUTED ? c ^ (HD == 64 ? r >> 1 & 3 : r & 7) : c; }
constexpr int KEYS = 16;                           // keys that a warp works on at a time
constexpr int WARPS = 4, THREADS = WARPS * 32;
constexpr int TILE = 128;                          // keys that slices are counted in: a step of a block's warps, or two
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LEAST_LOG = -102.f;                // a value's scale, in powers of two, as the reference sees it

struct Params {
    const bf16* q; bf16* out;
    const int8_t* k; const int8_t* v; const float* k_scale; const float* v_scale;
    const int* cu_q; const int* q_start; const int* kv_len; const int* table;
    const float* sink;              // float32 [nh] or null: one more term exp(sink) of a row's denominator
    float* part_o; float* part_ml;  // results of key slices: [request][kv head][slice][16][HD] and [..][2]; with `shared` [slice][kv head][16][HD]
    int max_blocks, nh, nkv, G, page_size, num_pages, window, chunk, requests;
    int per, slices;                // key slices: tiles of each, most of them that any request has
    int cluster;                    // the slices of a (request, kv head) are one cluster of blocks and join there
    int shared;                     // > 0: the requests share `slices` slices by their lengths (see deal_kernel), none counted longer than this
    int* dealt;                     // then: which slice is whose
    int slots;                      // slices of a kv head that run at once
    float scale_log2;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
    const int n = there ? 16 : 0;   // 0: nothing is read, zeros are written
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool there) {
    const int n = there ? 4 : 0;
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t turn8x8(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two bytes of r (chosen by SEL), each 128 too large, as float16: 1024 more than they are, or themselves less 128.
template <int SEL> __device__ __forceinline__ uint32_t raised2(uint32_t r) { return __byte_perm(r, 0x64646464u, SEL); }
template <int SEL> __device__ __forceinline__ uint32_t widen2(uint32_t r) {
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(raised2<SEL>(r)), "r"(0x64806480u));
    return d;
}
constexpr uint32_t TOP_BITS = 0x80808080u;
constexpr float RAISED = 1152.f;
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}

// What a warp keeps of 8 * NB queries: of block nb a lane holds columns 2 (lane & 3) and the next.
template <int NB>
struct Queries {
    uint32_t qf[CHUNKS][NB][2];
    float o[CHUNKS][NB][4];      // channels 16 mb + 2 (lane / 4) (entries 0, 1) and the next (2, 3) of the lane's two queries
    float m[NB][2], l[NB][2];    // l: this lane's keys only
    float off[NB][2], mul[NB][2];   // a score in powers of two is (product + off) * mul * key's scale
    int pos[NB][2], lo[NB][2];   // position and first visible key; pos < 0: no such query
};

// Queries row0 .. of the stacked rows (row = token * G + head of the group) of a request whose first token is `tok`.
template <int NB>
__device__ __forceinline__ void load_queries(const Params& p, Queries<NB>& s, int tok, int g, int row0, int n_rows, int q_pos0) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const int row = row0 + 8 * nb + (lane >> 2);
        const int t = row / p.G;
        const bf16* src = p.q + ((size_t)(tok + t) * p.nh + g * p.G + (row - t * p.G)) * HD + 4 * (lane & 3);
        unsigned most = 0;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const uint2 v = row < n_rows ? *reinterpret_cast<const uint2*>(src + 16 * c) : make_uint2(0, 0);
            s.qf[c][nb][0] = v.x; s.qf[c][nb][1] = v.y;
            most = max(max(most, max(v.x & 0x7fffu, v.x >> 16 & 0x7fffu)), max(v.y & 0x7fffu, v.y >> 16 & 0x7fffu));
        }
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
        // the largest channel's exponent; tiny rows as if it were 2^-112, one with an infinity or NaN as it is
        unsigned ex = max(most >> 7, 15u);
        if (ex == 255) ex = 141;
        const float up = __uint_as_float((268 - ex) << 23), down = __uint_as_float((ex - 14) << 23);
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t v = s.qf[c][nb][i];
                const uint32_t h = pack_f16x2(__uint_as_float(v << 16) * up, __uint_as_float(v & 0xffff0000u) * up);
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
                sum += f.x + f.y;
                s.qf[c][nb][i] = h;
            }
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            // (the lanes that hold the query of column 2 (lane & 3) + e)
            const int holder = 4 * (2 * (lane & 3) + e);
            s.off[nb][e] = -RAISED * __shfl_sync(0xffffffffu, sum, holder);
            s.mul[nb][e] = __shfl_sync(0xffffffffu, down, holder) * p.scale_log2;
            const int col = row0 + 8 * nb + 2 * (lane & 3) + e;
            s.pos[nb][e] = col < n_rows ? q_pos0 + col / p.G : -1;
            s.lo[nb][e] = col < n_rows ? bw::first_visible(s.pos[nb][e], p.window, p.chunk) : 0;
            s.m[nb][e] = -INFINITY; s.l[nb][e] = 0.f;
        }
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) s.o[c][nb][0] = s.o[c][nb][1] = s.o[c][nb][2] = s.o[c][nb][3] = 0.f;
    }
}

// Sixteen keys from key0 on, in shared memory: rows of K and V, their scales; bit i of `there` is set if key i has a page (what lies in the rows
// of the others is left over: whole numbers, and scales of any kind).  (Two groups of sixteen side by side in a warp's step hide each other's
// chains of products, but their registers and rings cost blocks: 64 requests at 2,048 keys 65 us where one group took 48, 8 at 8,192 34 and 32.)
// The reference follows its largest lazily: as long as nothing is more than 8 above it (a factor of 256) it stays, so most steps need one
// vote instead of a maximum over the lanes and a pass over the outputs.
template <int NB>
__device__ __forceinline__ void some_keys(Queries<NB>& s, uint32_t k_rows, uint32_t v_rows, const float* ks, const float* vs, int key0,
                                          unsigned there, bool need_mask) {
    const int lane = threadIdx.x & 31, r = lane >> 2;
    // matrices of an ldmatrix: keys 0-7 and 8-15 of one 16-byte unit, then of the next
    const int row = (lane & 7) + 8 * (lane >> 3 & 1), more = lane >> 4;
    const uint32_t at = (uint32_t)(row * STRIDE);
    float sc[NB][4];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) sc[nb][0] = sc[nb][1] = sc[nb][2] = sc[nb][3] = 0.f;
#pragma unroll
    for (int c = 0; c < CHUNKS; c += 2) {
        // (an odd last unit: its second pair of matrices reads the first's again)
        const uint32_t col = at + 16 * unit(row, c + 1 < CHUNKS ? c + more : c);
        uint32_t f[4];
        ldsm4(k_rows + col, f);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (c + i >= CHUNKS) break;
            const uint32_t x = f[2 * i] ^ TOP_BITS, y = f[2 * i + 1] ^ TOP_BITS;
            const uint32_t a[4] = {raised2<0x4140>(x), raised2<0x4140>(y), raised2<0x4342>(x), raised2<0x4342>(y)};
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) mma(sc[nb], a, s.qf[c + i][nb][0], s.qf[c + i][nb][1]);
        }
    }
    float most[NB][2], kk[2], vv[2], lv[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        // (a key that is no number, or whose value is none, has NaN as its score, and nothing else of it reaches who does not see it)
        const float k = ks[r + 8 * i], v = vs[r + 8 * i];
        const bool fine = max(__float_as_uint(k), __float_as_uint(v)) < 0x7f800000u;
        kk[i] = fine ? k : __uint_as_float(0x7fffffffu);
        vv[i] = fine ? v : 0.f;
        lv[i] = fmaxf(lg2(vv[i]), LEAST_LOG);
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        most[nb][0] = most[nb][1] = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = i & 1;
            float t = (sc[nb][i] + s.off[nb][e]) * s.mul[nb][e] * kk[i >> 1];
            if (need_mask) {
                const int j = r + 8 * (i >> 1), kp = key0 + j;
                if (!(kp <= s.pos[nb][e] && kp >= s.lo[nb][e] && (there >> j & 1))) t = -INFINITY;
            }
            sc[nb][i] = t;
            most[nb][e] = fmaxf(most[nb][e], t + lv[i >> 1]);
        }
    }
    bool grown = false;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) grown |= most[nb][0] > s.m[nb][0] + 8.f || most[nb][1] > s.m[nb][1] + 8.f;
    if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            float corr[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float mx = most[nb][e];
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                const float m_new = fmaxf(s.m[nb][e], mx);
                const float root = m_new == -INFINITY ? 0.f : ex2(0.5f * (s.m[nb][e] - m_new));     // nothing seen so far: 0
                corr[e] = root * root;
                s.m[nb][e] = m_new;
                s.l[nb][e] = s.l[nb][e] * root * root;
            }
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) {
                s.o[c][nb][0] *= corr[0]; s.o[c][nb][1] *= corr[1]; s.o[c][nb][2] *= corr[0]; s.o[c][nb][3] *= corr[1];
            }
        }
    }
    uint32_t wf[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const float ref[2] = {s.m[nb][0] == -INFINITY ? 0.f : s.m[nb][0], s.m[nb][1] == -INFINITY ? 0.f : s.m[nb][1]};
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = ex2(sc[nb][i] - ref[i & 1]);
            s.l[nb][i & 1] += x;
            w[i] = x * vv[i >> 1];
        }
        wf[nb][0] = turn8x8(pack_f16x2(w[0], w[1]));
        wf[nb][1] = turn8x8(pack_f16x2(w[2], w[3]));
    }
#pragma unroll
    for (int c = 0; c < CHUNKS; c += 2) {
        const uint32_t col = at + 16 * unit(row, c + 1 < CHUNKS ? c + more : c);
        uint32_t f[4];
        ldsm4_t(v_rows + col, f);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (c + i >= CHUNKS) break;
            const uint32_t x = f[2 * i] ^ TOP_BITS, y = f[2 * i + 1] ^ TOP_BITS;
            const uint32_t a[4] = {widen2<0x4240>(x), widen2<0x4341>(x), widen2<0x4240>(y), widen2<0x4341>(y)};
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) mma(s.o[c + i][nb], a, wf[nb][0], wf[nb][1]);
        }
    }
}

// The row (page, kv head, place) that holds a key; -1: none (behind the request's last token, or its page is not held).
__device__ __forceinline__ int key_row(const Params& p, const int* bt, int g, int key, int kv_len) {
    if (key >= kv_len) return -1;
    const int blk = key / p.page_size;
    if (blk >= p.max_blocks) return -1;
    const int page = bt[blk];
    return page >= 0 && page < p.num_pages ? (page * p.nkv + g) * p.page_size + (key - blk * p.page_size) : -1;
}

// Sixteen keys into a stage (rows of K, of V, their scales), by one warp.  What is held is looked up a step ahead of its use (`find`).
// WHOLE: pages are a multiple of sixteen keys long, so sixteen keys are one stretch of memory and need one look-up; places behind the
// request's last token are read with the others (and masked).  Otherwise every lane looks up a key of its own.
constexpr int STAGE = 2 * KEYS * (STRIDE + 4);
constexpr unsigned ALL = (1u << KEYS) - 1;         // all of them are held
template <bool WHOLE>
struct Feed {
    int row;
    __device__ __forceinline__ void find(const Params& p, const int* bt, int g, int key0, int end, int kv_len) {
        row = key0 < end ? key_row(p, bt, g, key0 + (WHOLE ? 0 : threadIdx.x & (KEYS - 1)), kv_len) : -1;
    }
    // which keys are held, as bits
    __device__ __forceinline__ unsigned fetch(const Params& p, uint8_t* stage) const {
        const int lane = threadIdx.x & 31;
        const uint32_t k_to = smem_u32(stage), v_to = k_to + KEYS * STRIDE, s_to = v_to + KEYS * STRIDE;
        const float* scales = lane < KEYS ? p.k_scale : p.v_scale;
        if constexpr (WHOLE) {
            if (row < 0) return 0;        // (uniform)
            const int8_t* k_from = p.k + (size_t)row * HD + 16 * lane;
            const int8_t* v_from = p.v + (size_t)row * HD + 16 * lane;
#pragma unroll
            for (int i = 0; i < (KEYS * CHUNKS + 31) / 32; ++i) {
                const int idx = lane + 32 * i, key = idx / CHUNKS, c = idx - key * CHUNKS;
                if ((KEYS * CHUNKS) % 32 && key >= KEYS) break;
                const uint32_t to = key * STRIDE + 16 * unit(key, c);
                cp_async16(k_to + to, k_from + 512 * i, true);
                cp_async16(v_to + to, v_from + 512 * i, true);
            }
            cp_async4(s_to + 4 * lane, scales + row + (lane & (KEYS - 1)), true);
            return ALL;
        } else {
            const unsigned got = __ballot_sync(0xffffffffu, row >= 0);
#pragma unroll
            for (int i = 0; i < (KEYS * CHUNKS + 31) / 32; ++i) {
                const int idx = lane + 32 * i, key = idx / CHUNKS, c = idx - key * CHUNKS;
                const int rw = __shfl_sync(0xffffffffu, row, key & (KEYS - 1));
                if ((KEYS * CHUNKS) % 32 && key >= KEYS) break;
                const size_t off = rw >= 0 ? (size_t)rw * HD + 16 * c : 0;
                const uint32_t to = key * STRIDE + 16 * unit(key, c);
                cp_async16(k_to + to, p.k + off, rw >= 0);
                cp_async16(v_to + to, p.v + off, rw >= 0);
            }
            cp_async4(s_to + 4 * lane, scales + (row >= 0 ? row : 0), row >= 0);
            return got & ALL;
        }
    }
};

// All (at most 16) rows of one (request, kv head) over one slice of the keys: the block's warps take sixteen keys each of every 64, each
// with a ring of its own, and are joined at the end.  How many slices a request has follows from its length on the device, so the same launch
// serves a captured step whatever the lengths become.
// Bound by memory where there is much of it: 64 requests at 2,048 keys (8 kv heads of 128) 49.3 us, 5.6 TB/s of 6.5 that a copy has.  8 at 8,192
// take 29.6, 4.7 TB/s: a block's start and the joining are a third of its eight tiles' time.  A token at 701 keys takes 6.2, the launch and
// a chain of trips (lengths, page, keys, the other blocks).
// (Two stages: other blocks' warps hide what a longer ring would, and there are more of them.  64 requests at 2,048 keys 48 us, with three
// stages 50, with four 68.)
constexpr int STAGES = 2;
constexpr int SMEM_RING = WARPS * STAGES * STAGE;
constexpr int JOIN_LD = HD + 8;
constexpr int SMEM_JOIN = (2 * WARPS * 16 + WARPS * 16 * JOIN_LD + 2 * 16) * 4;
constexpr int SMEM_FEW = SMEM_RING > SMEM_JOIN ? SMEM_RING : SMEM_JOIN;
// blocks an SM runs at once: by shared memory, and by registers (about 60 beside the queries and outputs)
constexpr int BY_SMEM = (227 * 1024) / (SMEM_FEW + 1024);
template <int NB> constexpr int BY_REGS = 512 / (((60 + NB * CHUNKS * 6) + 7) / 8 * 8);
template <int NB> constexpr int FEW_BLOCKS = BY_SMEM < BY_REGS<NB> ? (BY_SMEM > 0 ? BY_SMEM : 1) : (BY_REGS<NB> > 0 ? BY_REGS<NB> : 1);

constexpr int MOST_CLUSTER = 8;
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// from another block of the cluster, at the place where it is in this one's shared memory
template <typename T> __device__ __forceinline__ T read_block(uint32_t at, int rank) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(at), "r"(rank));
    T v;
    if constexpr (sizeof(T) == 16)
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
    else
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
    return v;
}

// Where only the device knows the lengths of a step (it was captured), and where lengths are so uneven that a place for every request's every
// slice would be mostly empty, the slices are dealt out by it: of one length for all requests, the shortest with which all run at once, or
// (slice_tiles) an even share of all tiles.  item: of which request a slice is, which one, how many the request has and where they
// begin (x -1: there are fewer slices); first: where a request's slices begin, and how many.  One warp, 32 requests at a time.
// Tiles of a slice, given all tiles of a step and `count(per)`, the slices that its requests have then: the shortest with which no more than
// `slots` slices are made, and so run at once.  Many short requests make that many slices by themselves, and a long one beside them would stay in
// few or one (one request at 65,536 keys beside 79 at 500: 512 tiles in a row): where it is more than twice an even share the share it is, and
// slices run after one another.  count is at most slots + requests, and at most slots where requests are no more than half of that.
#pragma nv_exec_check_disable      // (count is a lambda of the host's or of the device's)
template <typename Int, typename Count>
__host__ __device__ __forceinline__ Int slice_tiles(Int all, Int slots, Count count) {
    const Int even = all > 0 ? (all - 1) / slots + 1 : 1;
    if (const Int n = count(2 * even); n > slots) return n == count(all) ? 2 * even : even;      // (the same: none is longer than that)
    Int lo = even, hi = 2 * even;
    while (lo < hi) {
        const Int mid = lo + (hi - lo) / 2;
        if (count(mid) <= slots) hi = mid; else lo = mid + 1;
    }
    return lo;
}
struct Dealt { int4* item; int2* first; };
__host__ __device__ __forceinline__ Dealt dealt_at(int* at, int slices) { return {(int4*)at, (int2*)(at + 4 * (size_t)slices)}; }
__global__ void __launch_bounds__(32)
deal_kernel(Params p) {
    BW_PDL_TRIGGER();
    const int lane = threadIdx.x;
    const Dealt to = dealt_at(p.dealt, p.slices);
    BW_PDL_WAIT();
    auto tiles_of = [&](int r) {
        if (r >= p.requests) return 0;
        const int n_tok = p.cu_q[r + 1] - p.cu_q[r], pos = p.q_start[r];
        if (n_tok <= 0 || n_tok * p.G > 16) return 0;
        // (one that is longer than was planned for gets longer slices, not more)
        return min((pos + n_tok - 1) / TILE + 1 - bw::first_visible(pos, p.window, p.chunk) / TILE, p.shared);
    };
    const int mine = tiles_of(lane);
    int all = mine;
    for (int r = lane + 32; r < p.requests; r += 32) all += tiles_of(r);
    all = __reduce_add_sync(0xffffffffu, all);
    const int per = slice_tiles(all, p.slots, [&](int per) {
        int n = (mine + per - 1) / per;
        for (int r = lane + 32; r < p.requests; r += 32) n += (tiles_of(r) + per - 1) / per;
        return __reduce_add_sync(0xffffffffu, n);
    });
    int before = 0;
    for (int r0 = 0; r0 < p.requests; r0 += 32) {
        const int n = ((r0 ? tiles_of(r0 + lane) : mine) + per - 1) / per;
        int upto = n;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) { const int x = __shfl_up_sync(0xffffffffu, upto, d); if (lane >= d) upto += x; }
        const int at = before + upto - n;
        if (r0 + lane < p.requests) to.first[r0 + lane] = make_int2(at, n);
        for (int i = 0; i < n; ++i) to.item[at + i] = make_int4(r0 + lane, i, n, at);
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    for (int i = before + lane; i < p.slices; i += 32) to.item[i] = make_int4(-1, 0, 1, 0);
}

struct Walk { int first, tiles, per, live; };   // in tiles of TILE keys: where it begins, how many, of a slice; slices that have any
__device__ __forceinline__ Walk walk_of(const Params& p, int q_pos0, int last, int of) {
    Walk w;
    w.first = bw::first_visible(q_pos0, p.window, p.chunk) / TILE;
    w.tiles = last / TILE + 1 - w.first;
    // (a request that is longer than the plan was made for gets longer slices, not more of them)
    w.per = max(p.cluster || p.shared ? 1 : p.per, (w.tiles + of - 1) / of);
    w.live = (w.tiles + w.per - 1) / w.per;
    return w;
}

// Outputs and a sum that stand against the reference m, added to others against M >= m.
__device__ __forceinline__ void add_part(float4& acc, float& L, float4 v, float m, float l, float M) {
    const float root = m == -INFINITY ? 0.f : ex2(0.5f * (m - M)), f = root * root;
    acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
    L += l * root * root;
}
__device__ __forceinline__ void write_row(const Params& p, size_t token, int head, int c, float4 v, float L) {
    // (a row that sees nothing is zeros; a sum that is no number stays one)
    const float inv = L == 0.f ? 0.f : 1.f / L;
    if (L == 0.f) v = make_float4(0.f, 0.f, 0.f, 0.f);
    *reinterpret_cast<uint2*>(p.out + (token * p.nh + head) * HD + c) =
        make_uint2(bw::pack_bf16x2(v.x * inv, v.y * inv), bw::pack_bf16x2(v.z * inv, v.w * inv));
}
__device__ __forceinline__ float sink_term(const Params& p, int head, float M) { return p.sink ? exp2f(p.sink[head] * LOG2E - M) : 0.f; }

template <int NB, bool WHOLE>
__global__ void __launch_bounds__(THREADS, FEW_BLOCKS<NB>)
few_kernel(Params p) {
    BW_PDL_TRIGGER();
    extern __shared__ __align__(16) uint8_t smem[];
    // (dealt slices: a slice's kv heads one after the other, so that places left over come last)
    const int g = p.shared ? blockIdx.x % p.nkv : blockIdx.y, place = p.shared ? blockIdx.x / p.nkv : blockIdx.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    BW_PDL_WAIT();
    const int4 item = p.shared ? dealt_at(p.dealt, p.slices).item[place] : make_int4(blockIdx.z, blockIdx.x, p.slices, 0);
    const int r = item.x, slice = item.y;
    if (r < 0) return;
    const int tok = p.cu_q[r], n_tok = p.cu_q[r + 1] - tok, n_rows = n_tok * p.G;
    if (n_tok <= 0 || n_rows > 8 * NB || (NB == 2 && n_rows <= 8)) return;
    const int q_pos0 = p.q_start[r], last = q_pos0 + n_tok - 1, kv_len = p.kv_len[r];
    const Walk walk = walk_of(p, q_pos0, last, item.z);
    if (slice >= walk.live) return;        // (a cluster's barrier waits for no block that has left)
    const int t0 = walk.first + slice * walk.per, t1 = min(walk.first + walk.tiles, t0 + walk.per);
    const int* bt = p.table + (size_t)r * p.max_blocks;
    uint8_t* ring = smem + warp * STAGES * STAGE;
    // a warp's steps: every fourth sixteen keys of the slice
    const int first = t0 * TILE + warp * KEYS, end = min(t1 * TILE, last + 1);
    Feed<WHOLE> next;
    next.find(p, bt, g, first, end, kv_len);
    unsigned there[STAGES];
    auto feed = [&](int key0, int st) {
        if (key0 < end) {
            there[st] = next.fetch(p, ring + st * STAGE);
            next.find(p, bt, g, key0 + WARPS * KEYS, end, kv_len);
        }
        cp_async_commit();
    };
#pragma unroll
    for (int st = 0; st < STAGES - 1; ++st) feed(first + st * WARPS * KEYS, st);
    Queries<NB> s;
    load_queries<NB>(p, s, tok, g, 0, n_rows, q_pos0);
    const int see_all = bw::first_visible(last, p.window, p.chunk);      // from here on every query of the segment sees keys up to q_pos0
    for (int base = first; base < end; base += STAGES * WARPS * KEYS) {
#pragma unroll
        for (int st = 0; st < STAGES; ++st) {
            const int key0 = base + st * WARPS * KEYS;
            if (key0 >= end) break;
            cp_async_wait<STAGES - 2>();
            __syncwarp();
            feed(key0 + (STAGES - 1) * WARPS * KEYS, (st + STAGES - 1) % STAGES);
            const uint32_t at = smem_u32(ring + st * STAGE);
            const float* sc = reinterpret_cast<const float*>(ring + st * STAGE + 2 * KEYS * STRIDE);
            const bool need_mask = there[st] != ALL || key0 + KEYS - 1 > q_pos0 || key0 < see_all;
            some_keys<NB>(s, at, at + KEYS * STRIDE, sc, sc + KEYS, key0, there[st], need_mask);
            __syncwarp();
        }
    }
    cp_async_wait<0>();
    __syncthreads();
    // the warps' shares joined through shared memory (over the rings)
    float* ms = reinterpret_cast<float*>(smem);
    float* ls = ms + WARPS * 16;
    float* os = ls + WARPS * 16;
    float* ml = os + WARPS * 16 * JOIN_LD;      // [16][2]: the block's reference and sum of a row, for its cluster
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float l = s.l[nb][e];
            l += __shfl_xor_sync(0xffffffffu, l, 4);
            l += __shfl_xor_sync(0xffffffffu, l, 8);
            l += __shfl_xor_sync(0xffffffffu, l, 16);
            const int col = 8 * nb + 2 * (lane & 3) + e;
            if ((lane >> 2) == 0) { ms[warp * 16 + col] = s.m[nb][e]; ls[warp * 16 + col] = l; }
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c)
                *reinterpret_cast<float2*>(os + (warp * 16 + col) * JOIN_LD + 16 * c + 2 * (lane >> 2)) = make_float2(s.o[c][nb][e], s.o[c][nb][2 + e]);
        }
    }
    __syncthreads();
    for (int idx = threadIdx.x; idx < n_rows * (HD / 4); idx += THREADS) {
        const int row = idx / (HD / 4), c = (idx - row * (HD / 4)) * 4;
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) M = fmaxf(M, ms[w * 16 + row]);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float4 v = *reinterpret_cast<const float4*>(os + (w * 16 + row) * JOIN_LD + c);
            add_part(acc, L, v, ms[w * 16 + row], ls[w * 16 + row], M);
        }
        if (walk.live == 1) {
            const int t = row / p.G, head = g * p.G + row - t * p.G;
            write_row(p, (size_t)(tok + t), head, c, acc, L + sink_term(p, head, M));
        } else if (p.cluster) {
            // (in the place of the first warp's, which this thread alone reads)
            *reinterpret_cast<float4*>(os + row * JOIN_LD + c) = acc;
            if (c == 0) { ml[2 * row] = M; ml[2 * row + 1] = L; }
        } else {
            const size_t at = (p.shared ? (size_t)place * p.nkv + g : ((size_t)r * p.nkv + g) * p.slices + slice) * 16 + row;
            *reinterpret_cast<float4*>(p.part_o + at * HD + c) = acc;
            if (c == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(M, L);
        }
    }
    if (!p.cluster || walk.live == 1) return;
    // every block takes its share of (row, four channels) from all the cluster's blocks, in the order of the keys
    cluster_sync();
    const uint32_t os_at = smem_u32(os), ml_at = smem_u32(ml);
    for (int idx = slice * THREADS + threadIdx.x; idx < n_rows * (HD / 4); idx += walk.live * THREADS) {
        const int row = idx / (HD / 4), c = (idx - row * (HD / 4)) * 4;
        float4 v[MOST_CLUSTER];
        float2 x[MOST_CLUSTER];
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int i = 0; i < MOST_CLUSTER; ++i) {
            if (i >= walk.live) break;
            x[i] = read_block<float2>(ml_at + 8 * row, i);
            v[i] = read_block<float4>(os_at + 4 * (row * JOIN_LD + c), i);
        }
#pragma unroll
        for (int i = 0; i < MOST_CLUSTER; ++i) if (i < walk.live) M = fmaxf(M, x[i].x);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < MOST_CLUSTER; ++i) {
            if (i >= walk.live) break;
            add_part(acc, L, v[i], x[i].x, x[i].y, M);
        }
        const int t = row / p.G, head = g * p.G + row - t * p.G;
        write_row(p, (size_t)(tok + t), head, c, acc, L + sink_term(p, head, M));
    }
    cluster_sync();      // a block's shared memory stays until it has been read
}

// Joins the slices of every request that has more than one: blocks for the rows of a (kv head, request), groups of HD / 4 threads that take every
// so many-th slice, then the groups' sums in order: the same sum in every run of a step.  (How long the slices are follows from the lengths of all the
// step's requests: beside others a request's last bits may differ.)
constexpr int QUADS = HD / 4;
constexpr int JOIN_GROUPS = 256 / QUADS;
__global__ void __launch_bounds__(256)
join_kernel(Params p) {
    BW_PDL_TRIGGER();
    BW_PDL_WAIT();
    const int g = blockIdx.y, r = blockIdx.z;
    const int2 mine = p.shared ? dealt_at(p.dealt, p.slices).first[r] : make_int2(0, p.slices);
    if (mine.y <= 1) return;        // (of many requests most have one slice)
    const int tok = p.cu_q[r], n_tok = p.cu_q[r + 1] - tok, n_rows = n_tok * p.G;
    if (n_tok <= 0 || n_rows > 16) return;
    const int q_pos0 = p.q_start[r];
    const int live = walk_of(p, q_pos0, q_pos0 + n_tok - 1, mine.y).live;
    if (live <= 1) return;
    __shared__ float4 red[JOIN_GROUPS][QUADS];
    __shared__ float red_l[JOIN_GROUPS];
    __shared__ float scratch[32];
    for (int row = blockIdx.x; row < n_rows; row += gridDim.x) {
        // from one slice's row to the next one's
        const size_t step = p.shared ? (size_t)p.nkv * 16 : 16;
        const size_t base = (p.shared ? (size_t)mine.x * p.nkv + g : ((size_t)r * p.nkv + g) * p.slices) * 16 + row;
        const float2* ml = reinterpret_cast<const float2*>(p.part_ml);
        float M = -INFINITY;
        for (int i = threadIdx.x; i < live; i += 256) M = fmaxf(M, ml[base + i * step].x);
        M = bw::block_max(M, scratch);
        const int group = threadIdx.x / QUADS, quad = threadIdx.x - group * QUADS;
        if (group < JOIN_GROUPS) {
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            float L = 0.f;
#pragma unroll 4
            for (int i = group; i < live; i += JOIN_GROUPS) {
                const float2 x = ml[base + i * step];
                const float4 v = reinterpret_cast<const float4*>(p.part_o + (base + i * step) * HD)[quad];
                add_part(acc, L, v, x.x, x.y, M);
            }
            red[group][quad] = acc;
            if (quad == 0) red_l[group] = L;
        }
        __syncthreads();
        if (threadIdx.x < QUADS) {
            float4 acc = red[0][threadIdx.x];
            float L = red_l[0];
            for (int i = 1; i < JOIN_GROUPS; ++i) {
                const float4 v = red[i][threadIdx.x];
                acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
                L += red_l[i];
            }
            const int t = row / p.G, head = g * p.G + row - t * p.G;
            write_row(p, (size_t)(tok + t), head, 4 * threadIdx.x, acc, L + sink_term(p, head, M));
        }
        __syncthreads();
    }
}

}  // namespace

// Clusters of `size` blocks of the key-slice kernel that run at once on the current device (0: none, or not known), looked up once.
template <int NB, bool WHOLE>
static int clusters_at_once(int size) {
    static int known[bw::MAX_DEVICES][MOST_CLUSTER + 1];      // one more than the number
    int& n = known[bw::current_device()][size];
    if (n == 0) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)size); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = SMEM_FEW;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)size; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr; cfg.numAttrs = 1;
        int got = 0;
        if (cudaFuncSetAttribute(few_kernel<NB, WHOLE>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_FEW) != cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&got, few_kernel<NB, WHOLE>, &cfg) != cudaSuccess) { cudaGetLastError(); got = 0; }
        n = got + 1;
    }
    return n - 1;
}

// Key slices of the requests with at most 16 rows.  Lengths are the host's: of the step, or, for a step that is captured, the longest that may
// come (`bound` > 0: for every request).  `per`: tiles of a slice, so that the slices of all requests fill the GPU about once; `slices`: the
// most of any request (0: there is no such request).
// Where requests are about equally long, up to eight slices that all run at once are a cluster and join there; a join of its own (a launch,
// and a trip through memory: about a tile's time) serves more slices, and requests of many lengths, whose clusters would be half empty:
// us with clusters and without, a token at 701 keys 6.2 and 7.8, 2 at 2,000 9.0 and 10.3, 4 at 4,000 16.1 and 14.7, 8 at 8,192 29.6 and 32.5; 31 at 512 to 4,096
// with a prompt's portion beside them 55.3 and 53.1, 8 at 8,192 with 2 kv heads of 64 (which want 32 slices) 16.1 and 12.0.
// A step whose lengths only the device will know, and may be long, gets the slices that run at once, to share by what the lengths are then; and so does
// one whose longest request has so many slices that a place for as many of each would be far more than there are (scratch, and blocks that
// leave at once): 217 MB of scratch for one request at 131,072 keys and 50 short ones on 1 kv head of 128 are 5 so.
constexpr int CLUSTER_EXTRA = 1;
struct Plan { int per, slices, cluster, shared, slots; };
static Plan plan_slices(const int* q_len, const int* q_start, int requests, int G, int nkv, int window, int chunk, int bound, bool whole) {
    auto tiles_of = [&](int r) -> long long {
        if (q_len[r] <= 0 || (long long)q_len[r] * G > 16) return 0;
        const long long first = bound > 0 ? 0 : bw::first_visible(q_start[r], window, chunk), end = bound > 0 ? bound : (long long)q_start[r] + q_len[r];
        long long n = (end - 1) / TILE + 1 - first / TILE;
        if (bound > 0) {      // wherever the token stands, it sees no more than this
            long long span = bound;
            if (window > 0 && window + q_len[r] < span) span = window + q_len[r];
            if (chunk > 0 && chunk + q_len[r] < span) span = chunk + q_len[r];
            const long long m = (span + TILE - 1) / TILE + 1;
            if (m < n) n = m;
        }
        return n;
    };
    long long most = 0, least = 0x7fffffff, few = 0, all = 0;
    bool wide = false;                        // more than eight rows: the larger kernel, of which fewer run at once
    for (int r = 0; r < requests; ++r) {
        const long long n = tiles_of(r);
        if (n == 0) continue;
        ++few;
        all += n;
        wide |= q_len[r] * G > 8;
        if (n > most) most = n;
        if (n < least) least = n;
    }
    if (most == 0) return {1, 0, 0, 0, 0};
    const long long room = (long long)(wide ? FEW_BLOCKS<2> : FEW_BLOCKS<1>) * bw::num_sms();          // blocks that run at once
    const long long slots = room > nkv ? room / nkv : 1;
    auto count = [&](long long per) {
        long long n = 0;
        for (int r = 0; r < requests; ++r) n += (tiles_of(r) + per - 1) / per;
        return n;
    };
    long long lo = slice_tiles(all, slots, count);
    if (lo > most) lo = most;
    const long long slices = (most + lo - 1) / lo;
    if (slices > 1 && 4 * least >= 3 * most && (bound <= 0 || few == 1 || most <= MOST_CLUSTER)) {
        for (int size = slices < MOST_CLUSTER ? (int)slices : MOST_CLUSTER; size > 1; --size) {
            const long long per = (most + size - 1) / size;
            if (per > lo + CLUSTER_EXTRA) break;
            const int at_once = wide ? (whole ? clusters_at_once<2, true>(size) : clusters_at_once<2, false>(size))
                                     : (whole ? clusters_at_once<1, true>(size) : clusters_at_once<1, false>(size));
            if (few * nkv <= at_once) return {(int)per, (int)((most + per - 1) / per), 1, 0, 0};
        }
    }
    if (bound > 0 && requests == 1 && slices > 1) return {1, (int)slots, 0, 0, 0};
    // (what slice_tiles says of its count.  Captured requests of which as many run at once as there are stay whole while none is long)
    const long long shared = 2LL * requests <= slots ? slots : slots + requests;
    const bool captured = bound > 0 && requests > 1 && (slices > 1 || most > MOST_CLUSTER), 
               uneven = bound <= 0 && requests * slices > 4 * count(lo) && requests * slices * nkv > 8 * room;
    if ((captured || uneven) && most * requests <= 0x1fffffffll && shared * nkv <= 0x7fffffffll)
        return {1, (int)shared, 0, (int)most, (int)slots};
    return {(int)lo, (int)slices, 0, 0, 0};
}

template <int NB, bool WHOLE>
static int launch_few(const Params& p, dim3 grid, cudaStream_t s) {
    static bool done[bw::MAX_DEVICES];
    if (cudaError_t e = bw::allow_dynamic_smem(few_kernel<NB, WHOLE>, SMEM_FEW, done); e != cudaSuccess) return (int)e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = SMEM_FEW; cfg.stream = s;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (p.cluster) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = grid.x; attr[n].val.clusterDim.y = 1; attr[n].val.clusterDim.z = 1;
        ++n;
    }
    if (bw::pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = attr; cfg.numAttrs = n;
    if (const cudaError_t e = cudaLaunchKernelEx(&cfg, few_kernel<NB, WHOLE>, p); e != cudaSuccess) return (int)e;
    BW_LAUNCH_CHECK();
    return 0;
}

// Segments as the kernels may take them: positions that stay clear of 2^31 by more than a tile.
static bool segments_ok(const int* h_q_len, const int* h_q_start, int requests) {
    for (int r = 0; r < requests; ++r)
        if (h_q_len[r] < 0 || h_q_start[r] < 0 || (long long)h_q_start[r] + h_q_len[r] > 0x7fffff00ll) return false;
    return true;
}
static void deal(const Params& p, cudaStream_t s) { bw::launch(deal_kernel, dim3(1), dim3(32), 0, s, p); }

// For a step that is captured: which slice is whose, for any number of bw_attention_q8 calls on the same lengths, in *need ints of `dealt`.  With
// none given (null) *need is set alone (0: the step needs none); it depends on what lies on the host only.
BW_EXPORT int bw_attention_q8_deal(const int* cu_q, const int* q_start, const int* h_q_len, const int* h_q_start, int requests, int nh, int nkv,
                                   int page_size, int window, int chunk, int bound, int* dealt, long long* need, void* stream) {
    if (requests < 0 || nkv <= 0 || nh <= 0 || nh % nkv || page_size <= 0 || !segments_ok(h_q_len, h_q_start, requests)) return BW_ERR_BAD_ARG;
    window = window > 0 ? window : 0; chunk = chunk > 0 ? chunk : 0;
    const Plan plan = plan_slices(h_q_len, h_q_start, requests, nh / nkv, nkv, window, chunk, bound, page_size % KEYS == 0);
    *need = plan.shared ? 4ll * plan.slices + 2ll * requests : 0;
    if (!dealt || !plan.shared) return 0;
    if ((uintptr_t)dealt & 15) return BW_ERR_BAD_ARG;
    Params p{};
    p.cu_q = cu_q; p.q_start = q_start; p.window = window; p.chunk = chunk; p.requests = requests; p.G = nh / nkv;
    p.slices = plan.slices; p.shared = plan.shared; p.dealt = dealt; p.slots = plan.slots;
    deal(p, (cudaStream_t)stream);
    BW_LAUNCH_CHECK();
    return 0;
}

// q, out: bfloat16 [tokens][nh][HD]; h_q_len, h_q_start: lengths on the host; bound: see plan_slices.  Requests with more than 16 rows
// are left out (attention_q8_tc.cu has them).  room: where the joining needs memory, for *need floats; with none given (null), or too little (room_floats), *need is set, the call
// returns BW_ERR_ROOM and has launched nothing.  dealt: what bw_attention_q8_deal left for these lengths, or null (then it is done here).
#define BW_ERR_ROOM (-11)
BW_EXPORT int bw_attention_q8(const void* q, const void* k, const void* v, const float* k_scale, const float* v_scale, void* out,
                              const int* cu_q, const int* q_start, const int* kv_len, const int* table, int max_blocks, const int* h_q_len,
                              const int* h_q_start, int requests, int nh, int nkv, int page_size, int num_pages, int window, int chunk, int bound,
                              float scale, const float* sink, float* room, long long room_floats, long long* need, int* dealt,
                              void* stream) {
    if (requests < 0 || nkv <= 0 || nh <= 0 || nh % nkv || page_size <= 0 || num_pages <= 0 || max_blocks <= 0) return BW_ERR_BAD_ARG;
    if (!segments_ok(h_q_len, h_q_start, requests)) return BW_ERR_BAD_ARG;
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k | (uintptr_t)v | (uintptr_t)room | (uintptr_t)dealt) & 15) return BW_ERR_BAD_ARG;
    if ((long long)num_pages * nkv * page_size > 0x7fffffffll || nkv > 65535 || requests > 65535) return BW_ERR_UNSUPPORTED;
    const int G = nh / nkv;
    window = window > 0 ? window : 0; chunk = chunk > 0 ? chunk : 0;
    const bool whole = page_size % KEYS == 0;
    const Plan plan = plan_slices(h_q_len, h_q_start, requests, G, nkv, window, chunk, bound, whole);
    const long long rows = plan.slices > 1 && !plan.cluster ? (long long)(plan.shared ? 1 : requests) * nkv * plan.slices * 16 : 0;
    const long long wanted = rows * (HD + 2) + (plan.shared && !dealt ? 4ll * plan.slices + 2ll * requests : 0);
    if (wanted > room_floats) { *need = wanted; return BW_ERR_ROOM; }
    const bool deal_here = plan.shared && !dealt;
    if (deal_here) dealt = reinterpret_cast<int*>(room + rows * (HD + 2));       // (rows is a multiple of 16)
    const int slices = plan.slices;
    Params p{(const bf16*)q, (bf16*)out, (const int8_t*)k, (const int8_t*)v, k_scale, v_scale, cu_q, q_start, kv_len, table, sink, room, room + rows * HD,
             max_blocks, nh, nkv, G, page_size, num_pages, window, chunk, requests, plan.per, slices, plan.cluster, plan.shared, dealt, plan.slots, scale * LOG2E};
    cudaStream_t s = (cudaStream_t)stream;
    int most_rows = 0;
    bool few1 = false, few2 = false;
    for (int r = 0; r < requests; ++r) {
        const long long rows = (long long)h_q_len[r] * G;
        if (rows <= 0 || rows > 16) continue;
        (rows <= 8 ? few1 : few2) = true;
        if (rows > most_rows) most_rows = (int)rows;
    }
    if (!most_rows) return 0;
    if (slices < 1) return BW_ERR_BAD_ARG;
    const dim3 grid = plan.shared ? dim3((unsigned)slices * (unsigned)nkv) : dim3((unsigned)slices, (unsigned)nkv, (unsigned)requests);
    if (deal_here) {
        deal(p, s);
        BW_LAUNCH_CHECK();
    }
    if (few1) if (const int e = whole ? launch_few<1, true>(p, grid, s) : launch_few<1, false>(p, grid, s)) return e;
    if (few2) if (const int e = whole ? launch_few<2, true>(p, grid, s) : launch_few<2, false>(p, grid, s)) return e;
    if (slices > 1 && !plan.cluster) {
        // (a block for every row, for few requests; for many, whose rows have mostly nothing to join, about 512 blocks: 64 at 2,048 keys, captured,
        // 54.4 us with a block each and 51.2 so)
        long long cols = 512 / ((long long)nkv * requests);
        cols = cols < 1 ? 1 : cols > most_rows ? most_rows : cols;
        bw::launch(join_kernel, dim3((unsigned)cols, (unsigned)nkv, (unsigned)requests), dim3(256), 0, s, p);
        BW_LAUNCH_CHECK();
    }
    return 0;
}
