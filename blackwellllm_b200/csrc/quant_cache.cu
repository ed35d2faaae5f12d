// The 8-bit cache of keys and values: rows written as a step makes them, and read back.
//
// A row is the head size of one (token, kv head), key or value: whole numbers c of -127 to 127 (int8) and one float32 scale s, the value
// of a channel being c * s.  With a the row's largest magnitude s = a / 127 and c = x * (127 / a) rounded to nearest.  The scale belongs to
// one token: a row's bits depend on that row alone, so a prompt cut anywhere, a request computed again after a preemption and a sequence
// that was put back leave the same cache (a scale of several tokens would have to grow while they arrive, which rewrites rows).  int8 and
// not a float of 8 bits: against the row's root mean square, N(0, 1) channels come back with an error of 0.6 percent, e4m3's three
// fraction bits leave 2.6; the attention kernels multiply the scale to scores and probabilities, so whole numbers cost them nothing more.
//   a below 2^-110: zeros (127 / a would overflow near 2^-121, and beside a bfloat16 query such a key scores nothing);
//   a infinite or no number: c = 0, s = NaN, so the row reads back as NaN in every channel and whatever attends to it is NaN.
// Pages are [pages, kv heads, page size, head size], scales [pages, kv heads, page size].
//
// A lane takes eight channels of a row (two float4 of the projection; eight bytes of the cache), so whole sectors move whatever the head size,
// and nothing is staged.  Reading back is bound by memory: 65,536 tokens of 8 kv heads of 128 as bfloat16 in 72 us, 5.7 TB/s of 6.5 that a
// copy has.  Writing has about as many instructions as bytes (rotation, rounding and packing of every channel: 72 percent of the issue
// slots): 2,048 tokens of 32 + 16 heads of 128, float32, in 17.8 us by itself and from memory, 71 MB, where a copy would take 11; held to 32
// registers a thread eight blocks are on an SM and hide its trips (2,048 tokens written and read back 32 us before, 19 so).
#include "common.cuh"

namespace {

using bf16 = __nv_bfloat16;
constexpr int THREADS = 256;
constexpr float LEAST = 7.7037197775489434e-34f;   // 2^-110

struct Rows {
    int8_t* k; int8_t* v; float* k_scale; float* v_scale;
    const int* positions; const int* req; const int* table;
    int tokens, requests, max_blocks, page_size, num_pages, nkv, hd;
    unsigned per_page;           // the page size's reciprocal (divide)
};

// n / d for d whose reciprocal `inv` is 2^32 / d rounded down (2^32 - 1 for 1): that is at most one too low.
__device__ __forceinline__ unsigned divide(unsigned n, unsigned d, unsigned inv) {
    const unsigned q = __umulhi(n, inv);
    return q + (n - q * d >= d ? 1u : 0u);
}
inline unsigned reciprocal_of(unsigned d) { return d == 1 ? 0xffffffffu : (unsigned)((1ull << 32) / d); }

// Where the row of (token t, kv head 0) lies, in rows (head g's: g pages' length behind); -1: the table names no page for its position.
__device__ __forceinline__ long long row_of(const Rows& p, int t) {
    const int pos = p.positions[t], r = p.req[t];
    if (pos < 0 || r < 0 || r >= p.requests) return -1;
    const int blk = (int)divide((unsigned)pos, (unsigned)p.page_size, p.per_page);
    if (blk >= p.max_blocks) return -1;
    const int page = p.table[(size_t)r * p.max_blocks + blk];
    if (page < 0 || page >= p.num_pages) return -1;
    return (long long)page * p.nkv * p.page_size + (pos - blk * p.page_size);
}

template <typename T> __device__ __forceinline__ void load4(const T* src, float (&v)[4]);
template <> __device__ __forceinline__ void load4<float>(const float* src, float (&v)[4]) {
    const float4 t = *reinterpret_cast<const float4*>(src);
    v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
}
template <> __device__ __forceinline__ void load4<bf16>(const bf16* src, float (&v)[4]) {
    const uint2 t = *reinterpret_cast<const uint2*>(src);
    v[0] = __uint_as_float(t.x << 16); v[1] = __uint_as_float(t.x & 0xffff0000u);
    v[2] = __uint_as_float(t.y << 16); v[3] = __uint_as_float(t.y & 0xffff0000u);
}

__device__ __forceinline__ uint32_t pack4(const int (&c)[4]) {
    return (uint32_t)(c[0] & 255) | (uint32_t)(c[1] & 255) << 8 | (uint32_t)(c[2] & 255) << 16 | (uint32_t)(c[3] & 255) << 24;
}

// The q/k/v rows of a step: planes [planes][tokens][(nh + 2 nkv) * hd] that add up to them (one plane: the rows themselves).  A group of
// `lanes` neighbouring lanes (a power of two) makes one head of one token; lane l has units 4 l to 4 l + 3, a unit being a pair of channels
// that turn together, (u, u + rd / 2) for u < rd / 2, or the two channels 2 u, 2 u + 1 that do not turn.  `paired`: the two of a rotated
// pair stand side by side in the source.  VEC: rd is a multiple of 8 and the rows are aligned, so a lane's units are of one kind and their
// channels come as two vectors.
template <typename T, bool VEC, int LANES>
__global__ void __launch_bounds__(THREADS, 8)
append_kernel(const T* qkv, int planes, long long plane_stride, const float* turns, int rd, int paired,
              bf16* q_out, int nh, Rows p, unsigned per_heads, int append) {
    BW_PDL_TRIGGER();
    BW_PDL_WAIT();
    const int heads = nh + 2 * p.nkv, half = rd >> 1;
    const unsigned group = (blockIdx.x * (unsigned)THREADS + threadIdx.x) / LANES;
    const int l = threadIdx.x & (LANES - 1);
    const int t = (int)divide(group, (unsigned)heads, per_heads), head = (int)(group - (unsigned)t * heads);
    const bool live = t < p.tokens && 8 * l < p.hd;
    const bool is_q = head < nh, is_v = head >= nh + p.nkv;
    // (where the row goes is looked up while the row itself is on its way)
    long long row = append && live && !is_q ? row_of(p, t) : -1;
    float a[4] = {0.f, 0.f, 0.f, 0.f}, b[4] = {0.f, 0.f, 0.f, 0.f};
    bool turned[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) turned[i] = !is_v && 4 * l + i < half;
    if (live) {
        const T* src = qkv + ((size_t)t * heads + head) * p.hd;
#pragma unroll 1
        for (int pl = 0; pl < planes; ++pl, src += plane_stride) {
            float u[4], w[4];
            if constexpr (VEC) {
                const bool apart = turned[0] && !paired;
                load4(src + (apart ? 4 * l : 8 * l), u);
                load4(src + (apart ? half + 4 * l : 8 * l + 4), w);
                if (!apart) {      // neighbours: the first of each two belongs to u
                    const float u1 = u[1], u2 = u[2], u3 = u[3];
                    u[1] = u2; u[2] = w[0]; u[3] = w[2];
                    w[2] = w[1]; w[0] = u1; w[1] = u3;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int c = 4 * l + i;
                    const bool apart = turned[i] && !paired;
                    u[i] = bw::to_f32(src[apart ? c : 2 * c]);
                    w[i] = bw::to_f32(src[apart ? c + half : 2 * c + 1]);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) { a[i] += u[i]; b[i] += w[i]; }
        }
        float c[4] = {1.f, 1.f, 1.f, 1.f}, s[4] = {0.f, 0.f, 0.f, 0.f};
        if (VEC && turned[0]) {
            load4(turns + (size_t)t * rd + 4 * l, c);
            load4(turns + (size_t)t * rd + half + 4 * l, s);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (turned[i]) { c[i] = turns[(size_t)t * rd + 4 * l + i]; s[i] = turns[(size_t)t * rd + half + 4 * l + i]; }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (!turned[i]) continue;
            const float x = a[i], y = b[i];
            a[i] = x * c[i] - y * s[i];
            b[i] = y * c[i] + x * s[i];
        }
    }
    // a lane's channels: 4 l + i and 4 l + i + rd / 2 where they turn, else 8 l + 2 i and the next
    if (live && is_q) {
        bf16* dst = q_out + ((size_t)t * nh + head) * p.hd;
        if (VEC && turned[0]) {
            *reinterpret_cast<uint2*>(dst + 4 * l) = make_uint2(bw::pack_bf16x2(a[0], a[1]), bw::pack_bf16x2(a[2], a[3]));
            *reinterpret_cast<uint2*>(dst + half + 4 * l) = make_uint2(bw::pack_bf16x2(b[0], b[1]), bw::pack_bf16x2(b[2], b[3]));
        } else if (VEC) {
            *reinterpret_cast<uint4*>(dst + 8 * l) = make_uint4(bw::pack_bf16x2(a[0], b[0]), bw::pack_bf16x2(a[1], b[1]),
                                                                bw::pack_bf16x2(a[2], b[2]), bw::pack_bf16x2(a[3], b[3]));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = 4 * l + i;
                dst[turned[i] ? c : 2 * c] = __float2bfloat16_rn(a[i]);
                dst[turned[i] ? c + half : 2 * c + 1] = __float2bfloat16_rn(b[i]);
            }
        }
    }
    if (!__any_sync(0xffffffffu, row >= 0)) return;          // nothing of this warp's is written to the cache
    // the largest magnitude as an ordered whole number: what is no number stands above infinity and stays
    unsigned most = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) most = max(most, max(__float_as_uint(a[i]) & 0x7fffffffu, __float_as_uint(b[i]) & 0x7fffffffu));
#pragma unroll
    for (int o = LANES >> 1; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (row < 0) return;
    row += (long long)(is_v ? head - nh - p.nkv : head - nh) * p.page_size;
    const float big = __uint_as_float(most);
    const bool fine = most < 0x7f800000u, some = big >= LEAST;
    const float inv = fine && some ? 127.f / big : 0.f;
    int ca[4], cb[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        // (the product is at most 127 and a rounding of it; a value that is no number is never converted)
        ca[i] = fine ? __float2int_rn(a[i] * inv) : 0;
        cb[i] = fine ? __float2int_rn(b[i] * inv) : 0;
    }
    int8_t* dst = (is_v ? p.v : p.k) + (size_t)row * p.hd;
    if (VEC && turned[0]) {
        *reinterpret_cast<uint32_t*>(dst + 4 * l) = pack4(ca);
        *reinterpret_cast<uint32_t*>(dst + half + 4 * l) = pack4(cb);
    } else if (VEC) {
        const int lo[4] = {ca[0], cb[0], ca[1], cb[1]}, hi[4] = {ca[2], cb[2], ca[3], cb[3]};
        *reinterpret_cast<uint2*>(dst + 8 * l) = make_uint2(pack4(lo), pack4(hi));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = 4 * l + i;
            dst[turned[i] ? c : 2 * c] = (int8_t)ca[i];
            dst[turned[i] ? c + half : 2 * c + 1] = (int8_t)cb[i];
        }
    }
    if (l == 0) (is_v ? p.v_scale : p.k_scale)[row] = !fine ? __uint_as_float(0x7fffffffu) : (some ? big / 127.f : 0.f);
}

// Four whole numbers times s.  A byte with its top bit turned over, in the lowest place of 2^23, is 2^23 + 128 more than the number (the
// converting instruction runs at an eighth of this).
__device__ __forceinline__ void widen(uint32_t c, float s, float (&v)[4]) {
    c ^= 0x80808080u;
    v[0] = (__uint_as_float(__byte_perm(c, 0x4b000000u, 0x7650)) - 8388736.f) * s;
    v[1] = (__uint_as_float(__byte_perm(c, 0x4b000000u, 0x7651)) - 8388736.f) * s;
    v[2] = (__uint_as_float(__byte_perm(c, 0x4b000000u, 0x7652)) - 8388736.f) * s;
    v[3] = (__uint_as_float(__byte_perm(c, 0x4b000000u, 0x7653)) - 8388736.f) * s;
}
__device__ __forceinline__ void store8(bf16* dst, const float (&u)[4], const float (&w)[4]) {
    *reinterpret_cast<uint4*>(dst) = make_uint4(bw::pack_bf16x2(u[0], u[1]), bw::pack_bf16x2(u[2], u[3]),
                                                bw::pack_bf16x2(w[0], w[1]), bw::pack_bf16x2(w[2], w[3]));
}
__device__ __forceinline__ void store8(float* dst, const float (&u)[4], const float (&w)[4]) {
    reinterpret_cast<float4*>(dst)[0] = make_float4(u[0], u[1], u[2], u[3]);
    reinterpret_cast<float4*>(dst)[1] = make_float4(w[0], w[1], w[2], w[3]);
}

// Keys and values of the listed tokens, [tokens, kv heads, head size] each; zeros where the table names no page.  A block takes `each` tokens:
// their places are looked up once, by a thread a token, and then eight channels a thread are read and written (with a look-up and three
// divisions of its own for every thread, arithmetic was what the kernel took its time for).
constexpr int MOST_EACH = 32;
template <typename T>
__global__ void __launch_bounds__(THREADS)
read_kernel(Rows p, T* k_out, T* v_out, int each, unsigned per_token, unsigned per_units) {
    BW_PDL_TRIGGER();
    BW_PDL_WAIT();
    __shared__ long long place[MOST_EACH];
    const int t0 = blockIdx.x * each, n = min(each, p.tokens - t0);
    if ((int)threadIdx.x < n) place[threadIdx.x] = row_of(p, t0 + threadIdx.x);
    __syncthreads();
    const unsigned units = (unsigned)p.hd >> 3, items = units * p.nkv;
    for (unsigned i = threadIdx.x; i < items * n; i += THREADS) {
        const unsigned j = divide(i, items, per_token), rest = i - j * items, g = divide(rest, units, per_units), l = rest - g * units;
        const long long at = place[j];
        uint2 kc = make_uint2(0, 0), vc = make_uint2(0, 0);
        float ks = 0.f, vs = 0.f;
        if (at >= 0) {
            const size_t row = (size_t)at + (size_t)g * p.page_size, from = row * p.hd + 8 * l;
            kc = *reinterpret_cast<const uint2*>(p.k + from);
            vc = *reinterpret_cast<const uint2*>(p.v + from);
            ks = p.k_scale[row]; vs = p.v_scale[row];
        }
        float u[4], w[4];
        const size_t to = (size_t)t0 * items * 8 + (size_t)i * 8;
        widen(kc.x, ks, u); widen(kc.y, ks, w);
        store8(k_out + to, u, w);
        widen(vc.x, vs, u); widen(vc.y, vs, w);
        store8(v_out + to, u, w);
    }
}

bool sizes_ok(const Rows& p) {
    return p.tokens >= 0 && p.requests > 0 && p.max_blocks > 0 && p.page_size > 0 && p.num_pages > 0 && p.nkv > 0 && p.hd > 0 &&
           p.hd % 16 == 0 && p.hd <= 256;
}

}  // namespace

// qkv: BW_F32 or BW_BF16 (code `type`).  turns: float32 [tokens][rd] (cosines, then sines), null with rd == 0.  append == 0: nothing is
// written to the cache.  A call whose groups do not fit 32-bit thread numbers is refused.
BW_EXPORT int bw_quant_append(const void* qkv, int type, int planes, long long plane_stride, const float* turns, int rd, int paired,
                              void* q_out, int nh, void* k, void* v, float* k_scale, float* v_scale, const int* positions,
                              const int* req, const int* table, int tokens, int requests, int max_blocks, int page_size, int num_pages,
                              int nkv, int hd, int append, void* stream) {
    Rows p{(int8_t*)k, (int8_t*)v, k_scale, v_scale, positions, req, table, tokens, requests, max_blocks, page_size, num_pages, nkv, hd, 0};
    if (!sizes_ok(p) || nh < 0 || planes < 1 || rd < 0 || rd > hd || (rd & 1) || (rd && !turns)) return BW_ERR_BAD_ARG;
    if (tokens == 0) return 0;
    int lanes = 2;
    while (8 * lanes < hd) lanes *= 2;
    const int heads = nh + 2 * nkv;
    const long long threads = (long long)tokens * heads * lanes;
    if (threads + THREADS > 0xffffffffll) return BW_ERR_UNSUPPORTED;
    p.per_page = reciprocal_of((unsigned)page_size);
    const int es = type == BW_F32 ? 4 : 2;
    const bool vec = rd % 8 == 0 && ((uintptr_t)turns & 15) == 0 && (((uintptr_t)qkv | (uintptr_t)(plane_stride * es)) & (4 * es - 1)) == 0 &&
                     (((uintptr_t)q_out | (uintptr_t)k | (uintptr_t)v) & 15) == 0;
    const dim3 grid((unsigned)((threads + THREADS - 1) / THREADS)), block(THREADS);
    cudaStream_t s = (cudaStream_t)stream;
#define BW_APPEND(T, VEC, LANES) bw::launch(append_kernel<T, VEC, LANES>, grid, block, 0, s, (const T*)qkv, planes, plane_stride, turns, rd, paired, \
                                            (bf16*)q_out, nh, p, reciprocal_of((unsigned)heads), append)
#define BW_APPEND_LANES(T, VEC) switch (lanes) { case 2: BW_APPEND(T, VEC, 2); break; case 4: BW_APPEND(T, VEC, 4); break; case 8: BW_APPEND(T, VEC, 8); break; \
                                                 case 16: BW_APPEND(T, VEC, 16); break; default: BW_APPEND(T, VEC, 32); }
    if (type == BW_F32) { if (vec) BW_APPEND_LANES(float, true) else BW_APPEND_LANES(float, false) }
    else if (type == BW_BF16) { if (vec) BW_APPEND_LANES(bf16, true) else BW_APPEND_LANES(bf16, false) }
    else return BW_ERR_UNSUPPORTED;
#undef BW_APPEND_LANES
#undef BW_APPEND
    BW_LAUNCH_CHECK();
    return 0;
}

BW_EXPORT int bw_quant_read(const void* k, const void* v, const float* k_scale, const float* v_scale, const int* positions, const int* req,
                            const int* table, void* k_out, void* v_out, int type, int tokens, int requests, int max_blocks,
                            int page_size, int num_pages, int nkv, int hd, void* stream) {
    Rows p{(int8_t*)k, (int8_t*)v, (float*)k_scale, (float*)v_scale, positions, req, table, tokens, requests, max_blocks, page_size,
           num_pages, nkv, hd, 0};
    if (!sizes_ok(p) || (((uintptr_t)k | (uintptr_t)v) & 7) || (((uintptr_t)k_out | (uintptr_t)v_out) & 15)) return BW_ERR_BAD_ARG;
    if (tokens == 0) return 0;
    p.per_page = reciprocal_of((unsigned)page_size);
    // a block's tokens: about four rounds of its threads (65,536 tokens of 8 kv heads of 128: one round 88 us, two 76, four and eight 72), fewer
    // where the blocks would not fill the GPU
    const int items = nkv * (hd / 8);
    if ((long long)items * MOST_EACH > 0x7fffffffll) return BW_ERR_UNSUPPORTED;
    int each = (4 * THREADS + items - 1) / items;
    if (each > MOST_EACH) each = MOST_EACH;
    while (each > 1 && tokens < (long long)each * 4 * bw::num_sms()) each = (each + 1) / 2;
    const dim3 grid((unsigned)((tokens + each - 1) / each)), block(THREADS);
    const unsigned per_token = reciprocal_of((unsigned)items), per_units = reciprocal_of((unsigned)hd / 8);
    cudaStream_t s = (cudaStream_t)stream;
    if (type == BW_F32) bw::launch(read_kernel<float>, grid, block, 0, s, p, (float*)k_out, (float*)v_out, each, per_token, per_units);
    else if (type == BW_BF16) bw::launch(read_kernel<bf16>, grid, block, 0, s, p, (bf16*)k_out, (bf16*)v_out, each, per_token, per_units);
    else return BW_ERR_UNSUPPORTED;
    BW_LAUNCH_CHECK();
    return 0;
}
