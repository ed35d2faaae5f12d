// Attention over the 8-bit cache for portions of prompts, on the 5th-generation tensor cores (head size HEAD_DIM: a compile-time multiple
// of 16 up to 256; what attention_q8.cu says of the formula holds here).
//
// A block works on 256 stacked rows (row = token * G + head of the group) of one (request, kv head) as two tiles of 128 (one, of head sizes
// above 128: tensor memory holds no more) against tiles of 64 keys:
//   * eight warps widen, four keys and four values: whole numbers from the cache (16 bytes a load, straight into registers) become bfloat16 (keys) and
//     float16 (values), exact in both, and are written as the 128-byte-swizzled operands of the tensor cores.  Both tiles of rows use them:
//     widening is a third of the block's instructions, and the reason why a block has 256 rows and is alone on its SM;
//   * one warp issues S = Q K^T (M 128, N 64) into one of two buffers a tile of rows, another O += P V with P from tensor memory (one warp for
//     both spent two thirds of its time between its products);
//   * eight warps make P: products times the keys' scales, the values' scales inside the exponent, maximum, exponentials, sums; P is written as
//     float16 pairs over the S that it came from.  A lane has 16 columns of four rows and not 64 of one: what it reads of the 64 keys' scales
//     serves four rows (a row a thread would read four times as many bytes from shared memory).
// Roundings: P to float16 (2^-11 of a weight, or 2^-25 of the row's largest), and the result to bfloat16.  Whole numbers and queries are exact, the
// scales are multiplied or added in float32: a row's result has nothing of a key that the row does not see.  (Scales inside the operands, over
// the largest scale of the 64 keys beside them, are a twentieth faster for 2,048 tokens and a tenth behind a long context, but a row then depends
// on later tokens: one value 2^18 times as loud leaves float16's subnormals to those beside it.)  Scores, sums and outputs are float32.  Sums
// of products stay below infinity for queries up to 2^112.  The exponents' reference follows the largest t + log2 vs that the row sees
// lazily (RISE), so O is seldom rescaled.  With the scale inside the exponent, weights 2^126 below the reference vanish, and their part of the sum with
// them: value scales that a row sees are to lie within 2^100 of each other (the key-slice kernel, which has instructions to spare, takes any).
// A key that is no number (its scale, or its value's, is NaN) has NaN as its score: rows that see it become NaN, masked rows do not.  Keys behind
// the request's end or on a page that is not held are masked, whatever stands in their place.
//
// Work is the list of all (rows, tile of keys) steps of the launch, cut into equal stretches, one a block, so that the last wave is not mostly
// empty and a few rows over many keys still fill the GPU.  A stretch that begins or ends inside a block of rows leaves its sums in
// memory; join_kernel adds them in the order of the keys.  Every wait is bounded: one that gives up sets the status word, and the rows that it left out, and
// all rows of later launches until the status is read, are NaN.
//
// 2,048 tokens of 32 heads of 128 on 8 kv heads: 73.5 us, 467 TFLOP/s; 2,048 behind 13,312 (40 heads on 8) 740 us, 812 of 1,652 that a large product
// has, in bursts (790 in a stream of calls, whose clock falls).  A step (256 rows, 64 keys) takes about 2,750 cycles, and nothing alone bounds it: the softmax's warps are busy for most of
// them, the products need 1,500 (N 64 reads as many bytes of Q as it has work for).  Late piece without the exponentials 4 percent less, with
// keys widened at the cost of values 2, where no reference ever moves 5.  An item costs about five steps beside (its queries come, the first
// scores, the outputs): of the 74 us a third.
#include "tcgen05.cuh"
#include <cuda_fp16.h>

#ifndef HEAD_DIM
#error "compile with -DHEAD_DIM=<multiple of 16>"
#endif

using bf16 = __nv_bfloat16;

namespace {

constexpr int HD = HEAD_DIM;
static_assert(HD % 16 == 0 && HD >= 16 && HD <= 256, "head size must be a multiple of 16 in [16, 256]");
constexpr int CHUNKS = HD / 16;             // 16-byte units of a row of the cache
constexpr int NS = (HD + 63) / 64;          // 128-byte slices of a widened row, of which the last may be filled in part (no product reads the rest)
constexpr int O_COLS = NS * 64;             // columns of tensor memory between the tiles' outputs
constexpr int O_STEP = HD % 32 ? 16 : 32;   // columns of outputs that a thread reads at a time
constexpr int BM = 128, BN = 64;
constexpr int NQ = HD <= 128 ? 2 : 1;       // tiles of rows a block
constexpr int ROWS = NQ * BM;
constexpr int STAGES = 2;
constexpr int Q_SLICE = BM * 128, KV_SLICE = BN * 128;
constexpr int Q_BYTES = NS * Q_SLICE, KV_BYTES = NS * KV_SLICE;
constexpr int RING = STAGES + 2;            // what the softmax reads of a tile of keys: a widening warp is at most that far ahead of it
// Groups of four warps: NQ of the softmax, one that widens keys, one that widens values, and one whose first two warps issue products.  A block is
// launched with 96 registers a thread (128 with four groups) and the groups trade them: 256 * 144 + 256 * 72 + 128 * 48 = 61,440, all of them,
// and 128 * 168 + 256 * 112 + 128 * 48 = 56,320 of 65,536.
constexpr int KEY_WARP = 4 * NQ, VALUE_WARP = KEY_WARP + 4, QK_WARP = VALUE_WARP + 4, PV_WARP = QK_WARP + 1;
constexpr int THREADS = 32 * (QK_WARP + 4);
constexpr int SOFTMAX_REGS = NQ == 2 ? 144 : 168, WIDEN_REGS = NQ == 2 ? 72 : 112, ISSUE_REGS = 48;
template <int N> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
// What the softmax needs of a tile of keys.
struct TileInfo {
    float kl[BN / 2][4];            // of two neighbouring keys: ks, then lv; a weight in powers of two is the product times ks plus lv (a value's scale)
    float per_v[BN];                // what makes of a weight its part of the sum: the scale comes off, and SUM_SHIFT
    unsigned there[2], bad[2];      // bits: keys that are held, and that are no number
};
constexpr int SMEM_BYTES = NQ * Q_BYTES + 2 * STAGES * KV_BYTES + RING * (int)sizeof(TileInfo) + 32 * 8 + 16;
constexpr uint32_t TMEM_COLS = 512;
// float16 operands, B's rows the keys (the values), beside bw::umma_idesc_bf16 (queries and keys)
constexpr uint32_t IDESC_PV = (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
constexpr float ZERO_LOG = -60.f;           // a value's scale of 0, in powers of two (its whole numbers are zeros)
constexpr float SUM_SHIFT = -20.f, SUM_UNIT = 1.f / (1 << 20);          // sums are kept times 2^this: of scales of 2^-117 they would reach infinity
constexpr float RISE = 14.f;                // a reference moves when a weight is 2^this times what it was taken from (float16 ends at 2^16)
constexpr float LOG2E = 1.4426950408889634f;
constexpr int MOST_BLOCKS = 160;            // blocks of a launch
constexpr int MOST_PORTIONS = 16;           // requests of a launch

__device__ int g_status = 0;

struct Params {
    const bf16* q; bf16* out;
    const int8_t* k; const int8_t* v; const float* k_scale; const float* v_scale;
    const int* kv_len; const int* table; const float* sink;
    float* part_o; float* part_ml;          // [2 x blocks][HD / 4][ROWS][4] and [2 x blocks][ROWS][2]
    int max_blocks, nh, nkv, G, page_size, num_pages, window, chunk, blocks, portions;
    float scale_log2;
    unsigned per_page;                      // 2^32 / page_size, rounded down
};
struct Portion { int request, tok, n_tok, q_pos0, first, n_blocks; };      // first: the first of its n_blocks * nkv items
struct Work {
    Portion portion[MOST_PORTIONS];
    int item[MOST_BLOCKS], offset[MOST_BLOCKS], steps[MOST_BLOCKS];        // where a block's stretch begins, and its length
};
struct Splits { int n; int item[MOST_BLOCKS]; short from[MOST_BLOCKS], to[MOST_BLOCKS]; };   // items that several blocks share: from .. to

// An item: 256 rows of one (request, kv head).
struct Item {
    int request, tok, g, row0, n_rows, q_pos0, t0, tiles;    // tok: its request's first token; t0, tiles: the tiles of keys that its rows see
};
__host__ __device__ __forceinline__ void tiles_of(int q_pos0, int row0, int n_rows, int G, int window, int chunk, int& t0, int& n) {
    const int first = q_pos0 + row0 / G, last = q_pos0 + (row0 + n_rows - 1) / G;
    t0 = bw::first_visible(first, window, chunk) / BN;
    n = last / BN + 1 - t0;
}
__host__ __device__ __forceinline__ Item item_of(const Portion* portions, int count, int index, int nkv, int G, int window, int chunk) {
    int i = 0;
    while (i + 1 < count && index >= portions[i + 1].first) ++i;
    const Portion& p = portions[i];
    const int local = index - p.first, block = p.n_blocks - 1 - local / nkv;      // the latest rows first: they have the most keys
    Item it;
    it.request = p.request; it.tok = p.tok; it.g = local % nkv; it.row0 = block * ROWS; it.q_pos0 = p.q_pos0;
    const int all = p.n_tok * G;
    it.n_rows = all - it.row0 < ROWS ? all - it.row0 : ROWS;
    tiles_of(it.q_pos0, it.row0, it.n_rows, G, window, chunk, it.t0, it.tiles);
    return it;
}

// A block's walk over its stretch: tiles of one item after another.
struct Walk {
    int index, offset, left;     // the item, tiles of it that lie before, steps to go (with the current one)
    Item it;
    int tile, end;               // of the current item's part: the tile, and the first behind the part
    bool opens, closes;          // the part begins, or ends, with the item
    __device__ __forceinline__ void open(const Params& p, const Work& w) {
        it = item_of(w.portion, p.portions, index, p.nkv, p.G, p.window, p.chunk);
        const int n = min(left, it.tiles - offset);
        tile = it.t0 + offset;
        end = tile + n;
        opens = offset == 0; closes = offset + n == it.tiles;
    }
    __device__ __forceinline__ void start(const Params& p, const Work& w) {
        index = w.item[blockIdx.x]; offset = w.offset[blockIdx.x]; left = w.steps[blockIdx.x];
        if (left > 0) open(p, w);
    }
    // to the next step; true if it is the first of another item
    __device__ __forceinline__ bool step(const Params& p, const Work& w) {
        --left; ++tile;
        if (tile < end || left == 0) return false;
        ++index; offset = 0;
        open(p, w);
        return true;
    }
    // past the whole part
    __device__ __forceinline__ void pass(const Params& p, const Work& w) {
        left -= end - tile;
        if (left == 0) return;
        ++index; offset = 0;
        open(p, w);
    }
};
__device__ __forceinline__ int q_tiles(const Item& it) { return NQ == 2 && it.n_rows > BM ? 2 : 1; }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
__device__ __forceinline__ bw::f32x2 add2(bw::f32x2 a, bw::f32x2 b) {
    bw::f32x2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two bytes of r (chosen by SEL) as bfloat16, exact: 0x4300 | the lower seven bits is 128 more than they are, and what comes off is 128, or with
// the sign's bit 256 (0x4380).
template <int SEL> __device__ __forceinline__ uint32_t key2(uint32_t r) {
    const uint32_t x = __byte_perm(r, 0x43434343u, SEL);
    uint32_t d;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(x & 0xff7fff7fu), "r"(x & 0xff80ff80u));
    return d;
}
// As float16: a byte with its top bit turned over is 128 more, 0x6400 | byte 1024 more.
template <int SEL> __device__ __forceinline__ uint32_t value2(uint32_t r) {
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(__byte_perm(r, 0x64646464u, SEL)), "r"(0x64806480u));
    return d;
}
// 16 channels, as the two units of a row of operands
__device__ __forceinline__ void widen_key(uint8_t* first, uint8_t* second, uint4 x) {
    *reinterpret_cast<uint4*>(first) = make_uint4(key2<0x4140>(x.x), key2<0x4342>(x.x), key2<0x4140>(x.y), key2<0x4342>(x.y));
    *reinterpret_cast<uint4*>(second) = make_uint4(key2<0x4140>(x.z), key2<0x4342>(x.z), key2<0x4140>(x.w), key2<0x4342>(x.w));
}
__device__ __forceinline__ void widen_value(uint8_t* first, uint8_t* second, uint4 x) {
    const uint32_t w[4] = {x.x ^ 0x80808080u, x.y ^ 0x80808080u, x.z ^ 0x80808080u, x.w ^ 0x80808080u};
    *reinterpret_cast<uint4*>(first) = make_uint4(value2<0x4140>(w[0]), value2<0x4342>(w[0]), value2<0x4140>(w[1]), value2<0x4342>(w[1]));
    *reinterpret_cast<uint4*>(second) = make_uint4(value2<0x4140>(w[2]), value2<0x4342>(w[2]), value2<0x4140>(w[3]), value2<0x4342>(w[3]));
}

// 16 lanes of tensor memory by 64 columns: a lane of the warp gets columns 8 j + 2 (lane & 3) and the next of row lane / 4 (v[4 j], v[4 j + 1]) and of
// row lane / 4 + 8 (v[4 j + 2], v[4 j + 3]).
__device__ __forceinline__ void tmem_ld_16x64(uint32_t at, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
          "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
          "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(at) : "memory");
}
// The same lanes' float16 pairs: column 4 j + (lane & 3) of row lane / 4 from v[2 j], of row lane / 4 + 8 from v[2 j + 1].
__device__ __forceinline__ void tmem_st_16x32(uint32_t at, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        :: "r"(at),
           "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
           "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}

template <int N>
__device__ __forceinline__ void outputs_at(uint32_t at, uint32_t (&o)[N]) {
    if constexpr (N == 32) bw::tmem_ld_32x32(at, o);
    else bw::tmem_ld_32x16(at, o);
}
template <int N>
__device__ __forceinline__ void outputs_to(uint32_t at, const uint32_t (&o)[N]) {
    if constexpr (N == 32) bw::tmem_st_32x32(at, o);
    else bw::tmem_st_32x16(at, o);
}

__global__ void __launch_bounds__(THREADS, 1)
attn_q8_tc_kernel(const __grid_constant__ Params p, const __grid_constant__ Work work) {
    BW_PDL_TRIGGER();
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* q_s = smem;                                // [NQ][Q_BYTES]
    uint8_t* k_s = q_s + NQ * Q_BYTES;                  // [STAGES][KV_BYTES]
    uint8_t* v_s = k_s + STAGES * KV_BYTES;
    TileInfo* info = reinterpret_cast<TileInfo*>(v_s + STAGES * KV_BYTES);
    uint64_t* bars = reinterpret_cast<uint64_t*>(info + RING);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 32);
    const uint32_t bar0 = bw::smem_u32(bars);
    const uint32_t q_full = bar0, k_full = bar0 + 8 * NQ, k_empty = k_full + 8 * STAGES, v_full = k_empty + 8 * STAGES, v_empty = v_full + 8 * STAGES;
    const uint32_t s_full = v_empty + 8 * STAGES, p_full = s_full + 16 * NQ, pv_done = p_full + 16 * NQ;     // [tile of rows][buffer]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int q = 0; q < NQ; ++q) bw::mbar_init(q_full + 8 * q, 4);
        for (int s = 0; s < STAGES; ++s) {
            bw::mbar_init(k_full + 8 * s, 4); bw::mbar_init(v_full + 8 * s, 4);
            bw::mbar_init(k_empty + 8 * s, 1); bw::mbar_init(v_empty + 8 * s, 1);
        }
        for (int s = 0; s < 2 * NQ; ++s) {
            bw::mbar_init(s_full + 8 * s, 1); bw::mbar_init(p_full + 8 * s, 4); bw::mbar_init(pv_done + 8 * s, 1);
        }
        bw::fence_barrier_init();
        tmem_slot[1] = (uint32_t)g_status;
    }
    if (warp == QK_WARP) bw::tmem_alloc(bw::smem_u32(tmem_slot), TMEM_COLS);
    bw::tc_fence_before();
    __syncthreads();
    bw::tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const uint32_t tmem_O = tmem_base + 128 * NQ;        // S: [tile of rows][buffer] of 64 columns, then O: [tile of rows] of O_COLS
    auto all = [](bool ok) { return __all_sync(0xffffffffu, ok) != 0; };

    Walk w;
    w.start(p, work);                                    // (of the launch's own numbers, while the kernel before is still at work)
    BW_PDL_WAIT();
    bool ok = tmem_slot[1] == 0;                         // else an earlier launch gave up: nothing is done, and the rows are no numbers
    if (!ok && warp >= KEY_WARP) w.left = 0;

    if (warp >= QK_WARP) {
        fewer_registers<ISSUE_REGS>();
        const uint32_t tmem0 = __shfl_sync(0xffffffffu, tmem_base, 0);
        // descriptors of the first operands; others lie a multiple of 16 bytes behind (added to the low word: addresses stay below its field)
        auto behind = [](uint64_t d, uint32_t units) { return (d & 0xffffffff00000000ull) | (uint32_t)((uint32_t)d + units); };
        int n[NQ] = {};                                  // steps of each tile of rows so far
        if (warp == QK_WARP) {
            const uint64_t dq = bw::umma_smem_desc_sw128(bw::smem_u32(q_s)), dk = bw::umma_smem_desc_sw128(bw::smem_u32(k_s));
            int loaded[NQ] = {};                         // times that a tile's queries came
            bool begins = true;
            for (int it = 0; ok && w.left > 0; ++it) {
                const int s = it % STAGES, tiles_q = q_tiles(w.it);
                if (begins) {
#pragma unroll
                    for (int q = 0; q < NQ; ++q)
                        if (ok && q < tiles_q) {
                            ok = all(bw::mbar_wait(q_full + 8 * q, loaded[q] & 1, &g_status, 36));
                            ++loaded[q];
                        }
                    // whoever was in the item before has read what it needs of its keys' tiles (`info` holds them a few steps long)
#pragma unroll
                    for (int q = 0; q < NQ; ++q)
                        if (ok && n[q] > 0) ok = all(bw::mbar_wait(pv_done + 8 * (2 * q + ((n[q] - 1) & 1)), ((n[q] - 1) >> 1) & 1, &g_status, 42));
                    if (!ok) break;
                }
                if (!all(bw::mbar_wait(k_full + 8 * s, (it / STAGES) & 1, &g_status, 32))) break;
                const uint64_t dks = behind(dk, s * (KV_BYTES >> 4));
#pragma unroll
                for (int q = 0; q < NQ; ++q) {
                    if (q >= tiles_q) break;
                    const int b = n[q] & 1;
                    // the buffer holds P of the step before last, which the P V issued for it may still read
                    if (n[q] >= 2) ok = all(bw::mbar_wait(pv_done + 8 * (2 * q + b), ((n[q] >> 1) - 1) & 1, &g_status, 33));
                    if (!ok) break;
                    bw::tc_fence_after();
                    if (bw::elect_one()) {
#pragma unroll
                        for (int ks = 0; ks < HD / 16; ++ks)
                            bw::umma_bf16(tmem0 + 128 * q + 64 * b, behind(dq, (q * Q_BYTES + (ks >> 2) * Q_SLICE) / 16 + 2 * (ks & 3)),
                                          behind(dks, (ks >> 2) * (KV_SLICE / 16) + 2 * (ks & 3)), bw::umma_idesc_bf16(BM, BN), ks != 0);
                        bw::umma_commit(s_full + 8 * (2 * q + b));
                        if (q == tiles_q - 1) bw::umma_commit(k_empty + 8 * s);
                    }
                    __syncwarp();
                    ++n[q];
                }
                begins = w.step(p, work);
            }
        } else if (warp == PV_WARP) {
            const uint64_t dv = bw::umma_smem_desc_mn_sw128(bw::smem_u32(v_s), KV_SLICE);
            bool begins = true;
            for (int it = 0; ok && w.left > 0; ++it) {
                const int s = it % STAGES, tiles_q = q_tiles(w.it);
                if (!all(bw::mbar_wait(v_full + 8 * s, (it / STAGES) & 1, &g_status, 34))) break;
                const uint64_t dvs = behind(dv, s * (KV_BYTES >> 4));
#pragma unroll
                for (int q = 0; q < NQ; ++q) {
                    if (q >= tiles_q) break;
                    const int b = n[q] & 1;
                    ok = all(bw::mbar_wait(p_full + 8 * (2 * q + b), (n[q] >> 1) & 1, &g_status, 35));
                    if (!ok) break;
                    bw::tc_fence_after();
                    if (bw::elect_one()) {
#pragma unroll
                        for (int kk = 0; kk < BN / 16; ++kk)
                            bw::umma_bf16_ts(tmem0 + 128 * NQ + q * O_COLS, tmem0 + 128 * q + 64 * b + 8 * kk, behind(dvs, kk * (2048 / 16)), IDESC_PV,
                                             !(begins && kk == 0));
                        bw::umma_commit(pv_done + 8 * (2 * q + b));
                        if (q == tiles_q - 1) bw::umma_commit(v_empty + 8 * s);
                    }
                    __syncwarp();
                    ++n[q];
                }
                begins = w.step(p, work);
            }
        }
    } else if (warp >= KEY_WARP) {
        // ---------------------------------------------------------------- widening
        fewer_registers<WIDEN_REGS>();
        const bool keys = warp < VALUE_WARP;
        // This lane's keys of a tile are mine and mine + 32.  Eight lanes, whose 16 bytes move together, take units 0 to 3 of a slice of one key and
        // of the other slice of the next (of the same slice, where rows are an odd number of slices long): in the cache that is 128 bytes from
        // different banks, and among the operands, whose units are permuted by the key's number, too.  (Eight keys' units with the same
        // number, as first written, took eight turns: two thirds of the data pipe's time.)
        const int ww = (warp - KEY_WARP) & 3, odd = lane >> 2 & 1, mine = 8 * ww + 2 * (lane >> 3) + odd;
        constexpr bool SWAP = NS % 2 == 0;
        const int8_t* from = keys ? p.k : p.v;
        uint8_t* tiles = keys ? k_s : v_s;
        const uint32_t full = keys ? k_full : v_full, empty = keys ? k_empty : v_empty;
        constexpr int PER = NS;                                          // units of 16 channels a key
        struct Rows { int a, b; };                                       // of the keys lane and lane + 32; -1: none
        // the pages of the keys lane and lane + 32 as the table has them (-1: none); made into rows only a step later, so that nothing waits
        struct Pages { int page[2], slot[2], g; };
        int item_seen = -1, len = 0;
        const int* bt = nullptr;
        auto look_up = [&](const Walk& x) {
            if (x.index != item_seen) {
                item_seen = x.index;
                len = p.kv_len[x.it.request];
                bt = p.table + (size_t)x.it.request * p.max_blocks;
            }
            Pages got{{-1, -1}, {0, 0}, x.it.g};
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                // the key's block: by a reciprocal that is at most one too low
                const int key = x.tile * BN + lane + 32 * i;
                int blk = (int)__umulhi((unsigned)key, p.per_page), slot = key - blk * p.page_size;
                if (slot >= p.page_size) { slot -= p.page_size; ++blk; }
                got.slot[i] = slot;
                if (key < len && blk < p.max_blocks) got.page[i] = bt[blk];
            }
            return got;
        };
        auto rows_of = [&](const Pages& x) {
            int got[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) got[i] = (unsigned)x.page[i] < (unsigned)p.num_pages ? (x.page[i] * p.nkv + x.g) * p.page_size + x.slot[i] : -1;
            return Rows{got[0], got[1]};
        };
        if (w.left > 0) {
            Walk ahead = w;
            Rows rows = rows_of(look_up(ahead));
            Pages next{{-1, -1}, {0, 0}, 0};
            if (ahead.left > 1) { ahead.step(p, work); next = look_up(ahead); }
            // A unit of the next step is loaded as soon as this step's is widened, into the same registers: it has a whole step to come.  Where no
            // row is, the pool's first is read, and masked.
            uint4 x[2][PER];
            const int8_t* base = from + 16 * (lane & 3);
            const int swap = SWAP && odd ? 1 : 0;            // slice j of this lane is slice j ^ swap of the row
            auto has = [&](int j) { return HD % 64 == 0 || 4 * (j ^ swap) + (lane & 3) < CHUNKS; };
            auto unit_of = [&](const int8_t* row, int j) {
                return has(j) ? *reinterpret_cast<const uint4*>(row + 64 * j + (j & 1 ? -64 : 64) * swap) : make_uint4(0, 0, 0, 0);
            };
            {
                const int8_t *a = base + (size_t)max(__shfl_sync(0xffffffffu, rows.a, mine), 0) * HD, *b = base + (size_t)max(__shfl_sync(0xffffffffu, rows.b, mine), 0) * HD;
#pragma unroll
                for (int j = 0; j < PER; ++j) { x[0][j] = unit_of(a, j); x[1][j] = unit_of(b, j); }
            }
            // of the keys' warps: each looks after the scales of 16 keys, keys' in the lower lanes, values' in the upper ones
            const int own_key = 16 * ww + (lane & 15);
            auto scale_of = [&](const Rows& x) {
                const int row = __shfl_sync(0xffffffffu, ww < 2 ? x.a : x.b, own_key & 31);
                return keys && row >= 0 ? (lane < 16 ? p.k_scale : p.v_scale)[row] : 0.f;
            };
            float own = scale_of(rows);
            unsigned there0 = __ballot_sync(0xffffffffu, rows.a >= 0), there1 = __ballot_sync(0xffffffffu, rows.b >= 0);
            // where this lane's units go: rows mine and mine + 32, units 2 (lane & 3) and the next of every slice, permuted by the row
            uint8_t* first = tiles + mine * 128 + (((2 * (lane & 3)) ^ (mine & 7)) << 4);
            uint8_t* second = tiles + mine * 128 + (((2 * (lane & 3) + 1) ^ (mine & 7)) << 4);
            const int total = w.left;
            for (int it = 0; it < total; ++it) {
                const int s = it % STAGES;
                rows = rows_of(next);                                                     // of the next step (behind the last: none)
                const int8_t *a = base + (size_t)max(__shfl_sync(0xffffffffu, rows.a, mine), 0) * HD, *b = base + (size_t)max(__shfl_sync(0xffffffffu, rows.b, mine), 0) * HD;
                // (into the first-level cache now; loaded only behind the fence below, which waits for loads under way)
                if (it >= STAGES && !all(bw::mbar_wait(empty + 8 * s, ((it / STAGES) - 1) & 1, &g_status, keys ? 37 : 38))) break;
                if (keys) {
                    TileInfo& t = info[it % RING];
                    const bool fine = __float_as_uint(own) < 0x7f800000u;
                    const unsigned bad = __ballot_sync(0xffffffffu, !fine);
                    float* kl = &t.kl[own_key >> 1][own_key & 1];
                    // (ks positive and finite: a masked product, -infinity, stays that)
                    if (lane < 16) kl[0] = fine ? fminf(fmaxf(own * p.scale_log2, 1.17549435e-38f), 3.402823466e38f) : 1.f;
                    else {
                        const float lv = fine && own > 0.f ? fmaxf(lg2(own), -126.f) : ZERO_LOG;
                        kl[2] = lv;
                        t.per_v[own_key] = ex2(SUM_SHIFT - lv);
                    }
                    if (lane == 0) {
                        reinterpret_cast<unsigned short*>(t.bad)[ww] = (unsigned short)(bad | bad >> 16);
                        if (ww == 0) { t.there[0] = there0; t.there[1] = there1; }
                    }
                    __syncwarp();
                }
                there0 = __ballot_sync(0xffffffffu, rows.a >= 0); there1 = __ballot_sync(0xffffffffu, rows.b >= 0);
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    if (!has(j)) continue;
                    const int to = s * KV_BYTES + j * KV_SLICE + (j & 1 ? -KV_SLICE : KV_SLICE) * swap;
                    if (keys) {
                        widen_key(first + to, second + to, x[0][j]);
                        widen_key(first + to + 32 * 128, second + to + 32 * 128, x[1][j]);
                    } else {
                        widen_value(first + to, second + to, x[0][j]);
                        widen_value(first + to + 32 * 128, second + to + 32 * 128, x[1][j]);
                    }
                }
                bw::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) bw::mbar_arrive(full + 8 * s);
                __syncwarp();
                own = scale_of(rows);
#pragma unroll
                for (int j = 0; j < PER; ++j) { x[0][j] = unit_of(a, j); x[1][j] = unit_of(b, j); }
                next = Pages{{-1, -1}, {0, 0}, 0};
                if (it + 2 < total) { ahead.step(p, work); next = look_up(ahead); }
            }
        }
    } else {
        // ---------------------------------------------------------------- softmax: tile of rows `q`
        more_registers<SOFTMAX_REGS>();
        const int q = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tmem_S = tmem_base + 128 * q + lanes, tmem_Oq = tmem_O + q * O_COLS + lanes;
        int it = 0, c = 0;              // steps of the walk, and those of them that this tile of rows has
        constexpr int UNITS = HD / 8;   // of 16 bytes: a row of queries or outputs
        uint8_t* rows32 = q_s + q * Q_BYTES + (warp & 3) * 32 * 128;        // the warp's rows of the queries' tile
        auto unit_at = [&](int r, int u) { return reinterpret_cast<uint4*>(rows32 + (u >> 3) * Q_SLICE + r * 128 + (((u & 7) ^ (r & 7)) << 4)); };
        // Every unit of the warp's rows once: f(row of the warp, unit, element of the queries or outputs, whether the row exists).  Rolled up, as
        // everything that runs once an item, or nearly: code that is not in the instruction cache costs more than it does (a row's load,
        // conversion and store, unrolled, took 13,000 cycles).
        auto move_rows = [&](int own_row, bool row_ok, auto f) {
#pragma unroll 4
            for (int i = 0; i < UNITS; ++i) {
                const int idx = lane + 32 * i, r = idx / UNITS, u = idx - r * UNITS;
                const int at = __shfl_sync(0xffffffffu, row_ok ? own_row : -1, r);
                f(r, u, (size_t)(at >= 0 ? at : 0) * HD + 8 * u, at >= 0);
            }
        };
        while (ok && w.left > 0) {
            const Item item = w.it;
            const bool mine = q < q_tiles(item);
            const int gr = item.row0 + q * BM + row;                    // the row among the request's
            const bool row_ok = q * BM + row < item.n_rows;
            const int tok = gr / p.G, head = item.g * p.G + gr - tok * p.G;
            const int own_row = (item.tok + tok) * p.nh + head;         // of the queries and outputs
            if (mine) {
                // The warp's 32 rows come together (16 bytes a lane, neighbours of a row side by side: a row a lane would touch 32 lines with every
                // load) and lie in their place in shared memory as they are.
                move_rows(own_row, row_ok, [&](int r, int u, size_t from, bool live) {
                    const int bytes = live ? 16 : 0;       // 0: zeros are written
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(bw::smem_u32(unit_at(r, u))), "l"(p.q + from), "r"(bytes) : "memory");
                });
                asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory");
                bw::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) bw::mbar_arrive(q_full + 8 * q);
                __syncwarp();
            } else {
                it += w.end - w.tile;
                w.pass(p, work);
                continue;
            }

            // the warp's rows that exist: positions of the first and the last
            const int warp_row = item.row0 + q * BM + (warp & 3) * 32, end_row = item.row0 + item.n_rows - 1;
            const int first_pos = item.q_pos0 + min(warp_row, end_row) / p.G, last_pos = item.q_pos0 + min(warp_row + 31, end_row) / p.G;
            const int see_all = bw::first_visible(last_pos, p.window, p.chunk);
            // The lane's rows of the 32: lane / 4 and every eighth from there (columns: tmem_ld_16x64).  A row that does not exist stands against
            // infinity: its weights are zeros, and no maximum moves it.
            int pos[4];
            float m4[4];
            bw::f32x2 l4[4];            // this lane's columns only, even and odd ones
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = warp_row + 8 * i + (lane >> 2);
                pos[i] = item.q_pos0 + r / p.G;
                m4[i] = r <= end_row ? -INFINITY : INFINITY;
                l4[i] = 0ull;
            }
            // from a lane's rows to row `lane` of the warp: row 8 i + k lies in lanes 4 k to 4 k + 3
            auto own_row_of = [&](const float (&x)[4]) {
                float got = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float y = __shfl_sync(0xffffffffu, x[i], 4 * (lane & 7));
                    if (lane >> 3 == i) got = y;
                }
                return got;
            };
            const int t_first = w.tile, t_end = w.end;
            for (int t = t_first; t < t_end; ++t, ++it, ++c) {
                const int b = c & 1;
                if (!all(bw::mbar_wait(s_full + 8 * (2 * q + b), (c >> 1) & 1, &g_status, 39))) { ok = false; break; }
                bw::tc_fence_after();
                const TileInfo& ti = info[it % RING];
                const int key0 = t * BN;
                uint32_t v[2][32];
                tmem_ld_16x64(tmem_S + 64 * b, v[0]);
                tmem_ld_16x64(tmem_S + 64 * b + (16u << 16), v[1]);
                bw::tmem_ld_wait();
                const unsigned bad = ti.bad[0] | ti.bad[1];
                const bool gone = (ti.there[0] & ti.there[1]) != 0xffffffffu;
                if (gone || bad || key0 + BN - 1 > first_pos || key0 < see_all) {      // one branch a tile
                    const unsigned long long held = (unsigned long long)ti.there[1] << 32 | ti.there[0], none = (unsigned long long)ti.bad[1] << 32 | ti.bad[0];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        // key j is seen for j <= position - key0 and j >= lo - key0, if it is there: a mask of 64 bits
                        const int hi_j = pos[i] - key0, lo_j = bw::first_visible(pos[i], p.window, p.chunk) - key0;
                        unsigned long long seen = held;
                        if (hi_j < 0 || lo_j > 63) seen = 0;
                        else {
                            if (hi_j < 63) seen &= (2ull << hi_j) - 1;
                            if (lo_j > 0) seen &= ~0ull << lo_j;
                        }
                        const unsigned long long mine = seen >> (2 * (lane & 3)), nan = none >> (2 * (lane & 3));
#pragma unroll
                        for (int j = 0; j < 8; ++j)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                uint32_t& x = v[i >> 1][4 * j + 2 * (i & 1) + e];
                                if (!(mine >> (8 * j + e) & 1)) x = 0xff800000u;
                                else if (nan >> (8 * j + e) & 1) x = 0x7fffffffu;
                            }
                    }
                }
                // weights in powers of two, and the largest of each row
                auto pair = [&](int i, int j) {
                    const uint32_t* x = &v[i >> 1][4 * j + 2 * (i & 1)];
                    return bw::pack2(__uint_as_float(x[0]), __uint_as_float(x[1]));
                };
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const ulonglong2 kl = *reinterpret_cast<const ulonglong2*>(ti.kl[4 * j + (lane & 3)]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float a, d;
                        bw::unpack2(bw::fma2(pair(i, j), kl.x, kl.y), a, d);
                        v[i >> 1][4 * j + 2 * (i & 1)] = __float_as_uint(a);
                        v[i >> 1][4 * j + 2 * (i & 1) + 1] = __float_as_uint(d);
                        mx[i] = fmaxf(mx[i], fmaxf(a, d));
                    }
                }
                bool grow = false;
#pragma unroll
                for (int i = 0; i < 4; ++i) grow |= mx[i] > m4[i] + RISE;
                grow = __any_sync(0xffffffffu, grow);
                float shrink = 1.f;
                if (grow) {
                    float factor[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
                        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
                        float root = 1.f;          // (attention_q8.cu: squares of roots)
                        if (mx[i] > m4[i] + RISE) {
                            if (m4[i] != -INFINITY) root = ex2(0.5f * (m4[i] - mx[i]));
                            m4[i] = mx[i];
                        }
                        factor[i] = root * root;
                        l4[i] = bw::mul2(bw::mul2(l4[i], bw::pack2(root, root)), bw::pack2(root, root));
                    }
                    shrink = own_row_of(factor);
                }
                bw::f32x2 less[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x = m4[i] == -INFINITY ? 0.f : -m4[i];
                    less[i] = bw::pack2(x, x);
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const bw::f32x2 per_v = *reinterpret_cast<const bw::f32x2*>(ti.per_v + 8 * j + 2 * (lane & 3));
#pragma unroll
                        for (int i = 2 * h; i < 2 * h + 2; ++i) {
                            float a, d;
                            bw::unpack2(add2(pair(i, j), less[i]), a, d);
                            a = ex2(a);
                            d = ex2(d);
                            l4[i] = bw::fma2(bw::pack2(a, d), per_v, l4[i]);
                            v[h][2 * j + (i & 1)] = pack_f16x2(a, d);      // (a place whose score is done with)
                        }
                    }
                    tmem_st_16x32(tmem_S + 64 * b + (uint32_t)h * (16u << 16), v[h]);
                }
                if (grow && t > t_first) {
                    // O may be read once the P V of the step before is done; the next one waits for this warp.  (Behind the weights, whose registers are
                    // free for 64 columns at a time; ahead of them, sixteen by sixteen, the late piece took 3 percent more.)
                    if (!all(bw::mbar_wait(pv_done + 8 * (2 * q + (b ^ 1)), ((c - 1) >> 1) & 1, &g_status, 40))) { ok = false; break; }
                    bw::tc_fence_after();
                    constexpr int COLS = HD % 64 == 0 ? 2 : 1;
#pragma unroll 1
                    for (int c0 = 0; c0 < HD; c0 += COLS * O_STEP) {
                        uint32_t o[COLS][O_STEP];
#pragma unroll
                        for (int h = 0; h < COLS; ++h) outputs_at(tmem_Oq + c0 + h * O_STEP, o[h]);
                        bw::tmem_ld_wait();
#pragma unroll
                        for (int h = 0; h < COLS; ++h) {
#pragma unroll
                            for (int j = 0; j < O_STEP; ++j) o[h][j] = __float_as_uint(__uint_as_float(o[h][j]) * shrink);
                            outputs_to(tmem_Oq + c0 + h * O_STEP, o[h]);
                        }
                    }
                }
                bw::tmem_st_wait();
                bw::tc_fence_before();
                __syncwarp();
                if (lane == 0) bw::mbar_arrive(p_full + 8 * (2 * q + b));
                __syncwarp();
            }
            if (!ok || !(ok = all(bw::mbar_wait(pv_done + 8 * (2 * q + ((c - 1) & 1)), ((c - 1) >> 1) & 1, &g_status, 41)))) break;
            bw::tc_fence_after();
            float sums[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sums[i] = bw::sum2(l4[i]);
                sums[i] += __shfl_xor_sync(0xffffffffu, sums[i], 1);
                sums[i] += __shfl_xor_sync(0xffffffffu, sums[i], 2);
            }
            float l = own_row_of(sums);
            const float m = own_row_of(m4);
            if (w.opens && w.closes) {
                if (p.sink && row_ok) l += ex2(p.sink[head] * LOG2E - m + SUM_SHIFT);
                const float inv = l == 0.f ? 0.f : SUM_UNIT / l;
                // (the queries are done with: the warp's outputs take their place, and go out 16 bytes a lane, a row's side by side)
#pragma unroll 1
                for (int c0 = 0; c0 < HD; c0 += O_STEP) {
                    uint32_t o[O_STEP];
                    outputs_at(tmem_Oq + c0, o);
                    bw::tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < O_STEP; j += 8) {
                        auto two = [&](int i) { return bw::pack_bf16x2(__uint_as_float(o[j + i]) * inv, __uint_as_float(o[j + i + 1]) * inv); };
                        *unit_at(lane, (c0 + j) >> 3) = make_uint4(two(0), two(2), two(4), two(6));
                    }
                }
                __syncwarp();
                move_rows(own_row, row_ok, [&](int r, int u, size_t to, bool live) {
                    if (live) *reinterpret_cast<uint4*>(p.out + to) = *unit_at(r, u);
                });
                __syncwarp();
            } else {
                // a part of the item: the block's first part (1 if it begins with the item, so it is its last) leaves its sums
                const size_t slot = 2 * (size_t)blockIdx.x + (w.opens ? 1 : 0);
                const int r = q * BM + row;
                float4* dst = reinterpret_cast<float4*>(p.part_o) + slot * (HD / 4) * ROWS + r;
#pragma unroll 1
                for (int c0 = 0; c0 < HD; c0 += O_STEP) {
                    uint32_t o[O_STEP];
                    outputs_at(tmem_Oq + c0, o);
                    bw::tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < O_STEP; j += 4)
                        dst[(size_t)((c0 + j) >> 2) * ROWS] = make_float4(__uint_as_float(o[j]), __uint_as_float(o[j + 1]), __uint_as_float(o[j + 2]), __uint_as_float(o[j + 3]));
                }
                reinterpret_cast<float2*>(p.part_ml)[slot * ROWS + r] = make_float2(m, l);
            }
            // (the queries' place is written again, and O: both are done with)
            bw::tc_fence_before();
            w.pass(p, work);
        }
        // a wait gave up, here or in a launch before: what is left of the stretch must not pass for a result
        for (; w.left > 0; w.pass(p, work)) {
            const Item item = w.it;
            const int r = q * BM + row, gr = item.row0 + r, tok = gr / p.G;
            if (q >= q_tiles(item) || r >= item.n_rows) continue;
            if (w.opens && w.closes) {
                uint4* dst = reinterpret_cast<uint4*>(p.out + ((size_t)(item.tok + tok) * p.nh + item.g * p.G + gr - tok * p.G) * HD);
#pragma unroll 1
                for (int u = 0; u < UNITS; ++u) dst[u] = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
            } else {
                reinterpret_cast<float2*>(p.part_ml)[(2 * (size_t)blockIdx.x + (w.opens ? 1 : 0)) * ROWS + r] = make_float2(0.f, __uint_as_float(0x7fffffffu));
            }
        }
    }
    bw::tc_fence_before();
    __syncthreads();
    if (warp == QK_WARP) bw::tmem_dealloc(tmem_base, TMEM_COLS);
}

// The items that several blocks share: a thread for four channels of a row.  A warp has eight rows of sixteen channels, so it reads whole lines of
// the parts and writes whole sectors (a row a lane, four channels a block, wrote a quarter of each).  Four parts are read at a time, sums and
// outputs together: mostly that is all of them, and the kernel is one trip to memory long.
constexpr int JOIN_THREADS = 256, JOIN_ROWS = JOIN_THREADS / 4;
__global__ void __launch_bounds__(JOIN_THREADS)
join_kernel(const __grid_constant__ Params p, const __grid_constant__ Work work, const __grid_constant__ Splits splits) {
    BW_PDL_TRIGGER();
    const int i = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int quad = 4 * blockIdx.y + (lane >> 3), r = blockIdx.z * JOIN_ROWS + 8 * warp + (lane & 7);
    const Item it = item_of(work.portion, p.portions, splits.item[i], p.nkv, p.G, p.window, p.chunk);
    BW_PDL_WAIT();
    if (r >= it.n_rows) return;
    const int from = splits.from[i], to = splits.to[i];
    // the first block's part begins with the item: its slot is the second
    auto slot_of = [&](int b) { return (size_t)(2 * b + (b == from ? 1 : 0)); };
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + r;
    const float4* part = reinterpret_cast<const float4*>(p.part_o) + (size_t)quad * ROWS + r;
    float M = -INFINITY, L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int b = from; b <= to; b += 4) {
        float2 x[4];
        float4 o[4];
        float most = M;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const size_t at = slot_of(min(b + j, to));
            x[j] = ml[at * ROWS];
            o[j] = part[at * (HD / 4) * ROWS];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) if (b + j <= to) most = fmaxf(most, x[j].x);
        // (factors as the squares of their roots, which never vanish by themselves: attention_q8.cu)
        const float root = M == -INFINITY ? 0.f : ex2(0.5f * (M - most)), less = root * root;
        M = most;
        acc.x *= less; acc.y *= less; acc.z *= less; acc.w *= less; L = L * root * root;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float part = b + j > to || x[j].x == -INFINITY ? 0.f : ex2(0.5f * (x[j].x - M)), f = part * part;
            acc.x = fmaf(o[j].x, f, acc.x); acc.y = fmaf(o[j].y, f, acc.y); acc.z = fmaf(o[j].z, f, acc.z); acc.w = fmaf(o[j].w, f, acc.w);
            L = fmaf(x[j].y * part, part, L);
        }
    }
    const int gr = it.row0 + r, tok = gr / p.G, head = it.g * p.G + gr - tok * p.G;
    if (p.sink) L += ex2(p.sink[head] * LOG2E - M + SUM_SHIFT);
    const float inv = L == 0.f ? 0.f : SUM_UNIT / L;
    *reinterpret_cast<uint2*>(p.out + ((size_t)(it.tok + tok) * p.nh + head) * HD + 4 * quad) =
        make_uint2(bw::pack_bf16x2(acc.x * inv, acc.y * inv), bw::pack_bf16x2(acc.z * inv, acc.w * inv));
}

// Blocks of a launch: one an SM, but no fewer steps a block than pay for its start (queries, tensor memory) and its part of the joining (100
// tokens alone 21 us; with eight steps at least, and so fewer blocks, 28; two steps make no difference).
constexpr int LEAST_STEPS = 4;
// what an item costs beside its steps (its queries, the first scores, its outputs), in steps: 2,048 tokens 74 us counted as five, 78 as four, 87 as three
constexpr int ITEM_COST = 5;
int blocks_for(long long cost) {
    const long long sms = bw::num_sms() < MOST_BLOCKS ? bw::num_sms() : MOST_BLOCKS;
    const long long n = (cost + LEAST_STEPS + ITEM_COST - 1) / (LEAST_STEPS + ITEM_COST);
    return (int)(n < sms ? n : sms);
}

}  // namespace

// The launches of a call, handed one after the other to `run(work, portions, items, cost)`, which returns 0 or an error: the requests whose segments
// have more than `min_rows` stacked rows, sixteen at a time.
template <typename Run>
static int launches(const int* h_q_len, const int* h_q_start, int requests, int min_rows, int G, int nkv, int window, int chunk, Run run) {
    Work work{};
    int count = 0, items = 0, tok = 0;
    auto flush = [&]() -> int {
        if (!count) return 0;
        long long cost = 0;
        for (int i = 0; i < items; ++i) cost += item_of(work.portion, count, i, nkv, G, window, chunk).tiles + ITEM_COST;
        const int e = run(work, count, items, cost);
        count = items = 0;
        return e;
    };
    for (int r = 0; r < requests; ++r) {
        const int n = h_q_len[r];
        // (positions stay clear of 2^31 by more than a tile)
        if (n < 0 || h_q_start[r] < 0 || (long long)h_q_start[r] + n > 0x7fffff00ll) return BW_ERR_BAD_ARG;
        const long long rows = (long long)n * G, blocks = (rows + ROWS - 1) / ROWS;
        if (rows > min_rows) {
            // (items, and rows of the queries, are counted in 32 bits)
            if (rows > 0x3fffffffll || items + blocks * nkv > 0x3fffffffll || (tok + (long long)n) * G * nkv > 0x7fffffffll) return BW_ERR_UNSUPPORTED;
            work.portion[count] = {r, tok, n, h_q_start[r], items, (int)blocks};
            items += (int)blocks * nkv;
            if (++count == MOST_PORTIONS) if (const int e = flush()) return e;
        }
        tok += n;
    }
    return flush();
}

// Room that a call needs for the sums of shared items, in floats (negative: an error).
BW_EXPORT long long bw_attention_q8_tc_room(const int* h_q_len, const int* h_q_start, int requests, int min_rows, int G, int nkv, int window, int chunk) {
    if (requests < 0 || G <= 0 || nkv <= 0) return BW_ERR_BAD_ARG;
    long long most = 0;
    const int e = launches(h_q_len, h_q_start, requests, min_rows, G, nkv, window > 0 ? window : 0, chunk > 0 ? chunk : 0,
                           [&](Work&, int, int, long long cost) { const int n = blocks_for(cost); if (n > most) most = n; return 0; });
    return e ? e : 2 * most * ROWS * (HD + 2);
}

// q, out: bfloat16 [tokens][nh][HD]; h_q_len, h_q_start: on the host; room: what bw_attention_q8_tc_room says (kept until the call's kernels are
// done; the launches of one call follow one another and share it).
BW_EXPORT int bw_attention_q8_tc(const void* q, const void* k, const void* v, const float* k_scale, const float* v_scale, void* out,
                                 const int* kv_len, const int* table, int max_blocks, const int* h_q_len, const int* h_q_start, int requests,
                                 int min_rows, int nh, int nkv, int page_size, int num_pages, int window, int chunk, float scale,
                                 const float* sink, float* room, long long room_floats, void* stream) {
    if (requests < 0 || nkv <= 0 || nh <= 0 || nh % nkv || page_size <= 0 || num_pages <= 0 || max_blocks <= 0 || !room) return BW_ERR_BAD_ARG;
    if (!(scale > 0.f)) return BW_ERR_UNSUPPORTED;
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k | (uintptr_t)v | (uintptr_t)room) & 15) return BW_ERR_BAD_ARG;
    if ((long long)num_pages * nkv * page_size > 0x7fffffffll) return BW_ERR_UNSUPPORTED;
    static bool done[bw::MAX_DEVICES];
    if (cudaError_t e = bw::allow_dynamic_smem(attn_q8_tc_kernel, SMEM_BYTES, done); e != cudaSuccess) return (int)e;
    const int G = nh / nkv;
    window = window > 0 ? window : 0; chunk = chunk > 0 ? chunk : 0;
    cudaStream_t s = (cudaStream_t)stream;
    return launches(h_q_len, h_q_start, requests, min_rows, G, nkv, window, chunk, [&](Work& work, int count, int items, long long cost) -> int {
        const int blocks = blocks_for(cost);
        if (room_floats < 2ll * blocks * ROWS * (HD + 2)) return BW_ERR_BAD_ARG;
        const Params p{(const bf16*)q, (bf16*)out, (const int8_t*)k, (const int8_t*)v, k_scale, v_scale, kv_len, table, sink, room,
                       room + 2ll * blocks * ROWS * HD, max_blocks, nh, nkv, G, page_size, num_pages, window, chunk, blocks, count, scale * LOG2E,
                       page_size == 1 ? 0xffffffffu : (unsigned)((1ull << 32) / (unsigned)page_size)};
        // Stretches of equal cost, and the items that they cut.  A cut that falls on what an item costs beside its steps falls before the item.
        Splits splits{};
        int b = 0;
        long long at = 0;                          // cost of the items before
        int open = -1, open_offset = 0;            // the block that has steps up to here, and the offset in this item where it began (if in it)
        for (int i = 0; i < items; ++i) {
            const int n = item_of(work.portion, count, i, nkv, G, window, chunk).tiles;
            int from = b - 1;                      // the block that has the item's first step, unless one begins with it
            open_offset = 0;
            for (; b < blocks && cost * b / blocks < at + n + ITEM_COST; ++b) {
                long long offset = cost * b / blocks - at - ITEM_COST;
                if (offset < 0) offset = 0;
                if (open >= 0) work.steps[open] += (int)offset - open_offset;
                if (offset == 0) from = b;         // (a block whose cut falls here too begins where the next does: it has no steps)
                work.item[b] = i; work.offset[b] = (int)offset; work.steps[b] = 0;
                open = b; open_offset = (int)offset;
            }
            if (open >= 0) work.steps[open] += n - open_offset;
            if (from != b - 1) {
                splits.item[splits.n] = i; splits.from[splits.n] = (short)from; splits.to[splits.n] = (short)(b - 1);
                ++splits.n;
            }
            at += n + ITEM_COST;
        }
        bw::launch(attn_q8_tc_kernel, dim3((unsigned)blocks), dim3(THREADS), SMEM_BYTES, s, p, work);
        BW_LAUNCH_CHECK();
        if (splits.n) {
            bw::launch(join_kernel, dim3((unsigned)splits.n, HD / 16, ROWS / JOIN_ROWS), dim3(JOIN_THREADS), 0, s, p, work, splits);
            BW_LAUNCH_CHECK();
        }
        return 0;
    });
}

// Sets the status as a wait that gives up does, for a test of what follows from that (synchronises the device).
BW_EXPORT int bw_attention_q8_tc_give_up(int code) { return (int)cudaMemcpyToSymbol(g_status, &code, sizeof(int)); }

// 0 if no bounded wait ever gave up; clears the status (synchronises the device).
BW_EXPORT int bw_attention_q8_tc_status() {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_status, sizeof(int)) != cudaSuccess) return -1;
    if (v) cudaMemcpyToSymbol(g_status, &zero, sizeof(int));
    return v;
}
