// Causal grouped-query attention over a paged cache in four bits (kv4.cuh), for decoded tokens and short portions, bfloat16 or float32
// queries, head sizes up to 256.
//
// For the query at position p, head h, kv head h / (H/K):  s_t = (q . k_t) * scale over the keys it sees (attention_mask.cuh: causal, a
// window, kept first keys), with a cap c tanh(s / c) or a bias by distance as options, a = softmax(s) (a sink joins its denominator),
// o = sum_t a_t v_t; k_t and v_t are the held values, c s with c of four bits and s a bfloat16.  (src/model.c:3548-3589, 3409-3415;
// the reference attends over its eight-bit cache in k_attn_dec, src/kernels.cu:2171-2270.)
//
// The keys are the M side of the matrix instruction (m16n8k16), the packed query rows (row i: token i / G, head i % G) the N side: eight
// rows cost one instruction where rows on M would cost a half empty one.  S^T = K Q^T has a key's scores for two rows in a thread;
// O^T = V^T P^T has two neighbouring elements of the value for the same two rows, so that the running maximum's factor is one number a
// column in both.  P^T as the second product's operand is S^T turned by movmatrix.  A block takes eight rows, or sixteen where some request has more
// than eight; a request with more rows than a block takes several (and reads its keys as often).
//
// Codes become operands without leaving the thread that loads them.  Two shifts and four masks bring a word's eight codes into the mantissas of float16
// numbers, 256 + u and 16 + u by turns (u the code plus 8).  Keys are multiplied as that, exactly, into sums that start at what takes the bias off; a
// group of 32 elements is two k-steps, and its scale a factor on their float32 result.  (bfloat16 operands, which hold one code at a time, want four
// shifts and a fused product and sum a pair.)  The bias costs the sums log2(264 / 8) bits of 24; scores
// are off by less than the weights' rounding.  q is scaled by a power of two a row, so that its eight bits are whole in float16.  Values are
// scaled ahead of the product, where a thread's elements share a scale and its keys do not: (256 + u) s - 264 s in one rounding, which is none, because c s
// has eight bits.  They are in units of a power of two, one a group of elements, that follows the largest scale (2^-23 of it is what keeps all its bits); weights are rounded
// to float16 (2^-11) once.
// The words of two keys, their halves brought together by two byte permutations, give the pairs over KEYS that the second product wants.  The
// order of elements along k and of keys along k is free as long as both operands share it: a4_key.
//
// A warp walks tiles of its own (64 keys, 32 at head size 256) through a ring of asynchronous copies, 16 bytes a lane; the next page's number is asked
// for a tile ahead.  The warps of a block interleave the tiles of a span and meet once, at its end.  Spans of a request meet in a cluster of up to
// eight blocks through its shared memory, or leave partial sums to k_kv4_merge; either way in ascending order.
//
// What bounds it: 55 requests of 8,192 keys, 32 heads on 8 of 128 elements, one block a pair and three an SM, take 3.0 us a tile of every warp: 0.83 of the copy
// peak (6.54 TB/s), and as long where the cache fits in L2, with issue slots 44 to 62 % and the integer pipe 35 to 57 % busy and the tensor cores at 19 %: what
// is left is warps waiting for one another's results.  Around that stand what a launch costs before its first tiles are there (about 9 us
// with all SMs' first tiles on their way at once, 5.6 with a few) and what the last round of blocks leaves idle.
// Measured and left: four blocks an SM (64 ragged requests of 40 heads 253 us against 214: 128 registers a thread, where three leave 168 and spill 24 bytes), tiles of 32 keys at three (230), the next tile's scores
// interleaved with this tile's values (55 requests of 8,192 keys 119.9 against 107.8), bulk copies instead of cp.async (equal), e4m3 operands (the
// instruction runs at 0.16 a cycle and SM), equal shares of all tiles for resident blocks (268 and a second kernel against 214).
//
// float32: a float32 number is the exact sum of three bfloat16 numbers, the held values are bfloat16 numbers, so that three products on
// the tensor cores (q in pieces, p in pieces) give float32's precision.
#include "kv4.cuh"
#include "attention_mask.cuh"
#include <cuda_fp16.h>
#include <math.h>

#define A4_WARPS 4
#define A4_THREADS (32 * A4_WARPS)
#define A4_LOG2E 1.4426950408889634f
#define A4_SLACK 8.0f
#define A4_CLUSTER 8                  // most spans that a cluster combines (the portable cluster size)

struct A4Args {
    const void* q; void* out;
    Kv4Cache c;
    const int* seg_start; const int* seg_len; const int* seg_pos0; const int* block_tables;
    float* part_acc;                  // [blocks][K][splits][rows][hs]
    float* part_ml;                   // [blocks][K][splits][rows][2]
    int blocks;                       // row blocks of all portions, one after another (a4_place)
    long long q_stride;
    int H, G, D, max_pages, window, keep, splits, span_tiles, row_blocks, most_rows;
    float scale, softcap;
    const float* sink;
    XrBias bias;
    int wide, wide_out;               // 16-byte loads of q; four neighbouring outputs at once
    int early;                        // what earlier steps left, and the step's description, are at rest
    int clustered;                    // a request's spans are the blocks of a cluster, which combines them
    int tile_shift;                   // pages of 2^tile_shift whole tiles (-1: pages of other sizes)
};

// Four neighbouring elements of an output row: divided by the row's sum, to which a sink adds exp(sink - maximum).
template <bool F32>
__device__ __forceinline__ void a4_out(const A4Args& a, int tok0, int kvh, int row, int d, float4 v, float m, float sum) {
    if (d >= a.D) return;
    const int head = kvh * a.G + row % a.G;
    if (a.sink != nullptr) { float e; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fmaf(a.sink[head], A4_LOG2E, -m))); sum += e; }
    const float inv = 1.0f / sum;
    const float x[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
    const long long at = ((long long)(tok0 + row / a.G) * a.H + head) * a.D + d;
    if constexpr (F32) {
        float* dst = (float*)a.out + at;
        if (a.wide_out) *reinterpret_cast<float4*>(dst) = make_float4(x[0], x[1], x[2], x[3]);
        else
            for (int e = 0; e < 4; e++) if (d + e < a.D) dst[e] = x[e];
    } else {
        __nv_bfloat16* dst = (__nv_bfloat16*)a.out + at;
        if (a.wide_out) {
            const __nv_bfloat162 lo = __floats2bfloat162_rn(x[0], x[1]), hi = __floats2bfloat162_rn(x[2], x[3]);
            *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
        } else
            for (int e = 0; e < 4; e++) if (d + e < a.D) dst[e] = __float2bfloat16_rn(x[e]);
    }
}

__device__ __forceinline__ uint32_t a4_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// 16 bytes from global to shared memory without a register between; `bytes` 0: zeros instead.
__device__ __forceinline__ void a4_copy(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// Shared memory of another block of the cluster, and the cluster's barrier.
__device__ __forceinline__ uint32_t a4_of_rank(const void* mine, uint32_t rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(a4_smem(mine)), "r"(rank));
    return at;
}
__device__ __forceinline__ float4 a4_far4(uint32_t at) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ float2 a4_far2(uint32_t at) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
    return v;
}
// (The barrier is defined for warps whose lanes run it together, and loops of other lengths a lane lie ahead of it.)
__device__ __forceinline__ void a4_cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void a4_mma(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void a4_mma_half(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// d = A B + (c0, c1, c0, c1): what a key's row starts from hangs on its column alone
__device__ __forceinline__ void a4_mma_from(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, float c0, float c1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %10, %11};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ uint32_t a4_pack_half(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// A word's four pairs of neighbouring codes as float16 numbers: a mantissa of ten bits takes two codes side by side, so that two shifts serve four pairs.
// Pairs 0 and 2 are 256 + u, pairs 1 and 3 are 16 + u.
__device__ __forceinline__ void a4_pairs(uint32_t w, uint32_t* p) {
    const uint32_t l = w * 4u, r = w >> 6;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(p[0]) : "r"(l), "r"(0x003C003Cu), "r"(0x5C005C00u));
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(p[1]) : "r"(l), "r"(0x03C003C0u), "r"(0x4C004C00u));
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(p[2]) : "r"(r), "r"(0x003C003Cu), "r"(0x5C005C00u));
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(p[3]) : "r"(r), "r"(0x03C003C0u), "r"(0x4C004C00u));
}
__device__ __forceinline__ uint32_t a4_fma_half(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
__device__ __forceinline__ uint32_t a4_mul_half(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ void a4_ldsm4(uint32_t* r, uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
template <int W> __device__ __forceinline__ void a4_lds(uint32_t* r, uint32_t at) {
    if constexpr (W == 1) asm volatile("ld.shared.b32 %0, [%1];" : "=r"(r[0]) : "r"(at));
    else if constexpr (W == 2) asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(at));
    else {
#pragma unroll
        for (int i = 0; i < W; i += 4) asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]) : "r"(at + 4 * i));
    }
}
__device__ __forceinline__ uint32_t a4_lds16(uint32_t at) {
    unsigned short r;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(r) : "r"(at));
    return r;
}
__device__ __forceinline__ uint32_t a4_turn(uint32_t x) {            // transpose of an 8 x 8 matrix of 16-bit numbers over the warp
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ float a4_exp2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ uint32_t a4_pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// Takes the leading bfloat16 piece off a pair: returns it, leaves the (exact) rest.
__device__ __forceinline__ uint32_t a4_piece(float& lo, float& hi) {
    const uint32_t r = a4_pack(lo, hi);
    lo -= __uint_as_float(r << 16);
    hi -= __uint_as_float(r & 0xffff0000u);
    return r;
}
// Row r of a 16-key subtile's S^T, and equally place r along k of the second product, is key 8 (r / 8) + at_key(r % 8): the places 2t of a
// group of four threads are four neighbouring keys, and so are the places 2t + 1.
__device__ __forceinline__ int a4_key(int r) { return (r & 8) + 4 * (r & 1) + (((r & 7) >> 1) ^ (r & 1)); }

template <int NG> struct A4Tile { static constexpr int KEYS = NG <= 4 ? 64 : 32, STAGES = NG == 4 ? 2 : 3; };

// The tiles that the rows of a block see: those of the kept first keys, then those of the window.
struct A4Walk { int lo, hi, t_lo, kept, n; };
__device__ __forceinline__ A4Walk a4_walk(int first_pos, int last_pos, int window, int keep, int tile) {
    A4Walk w;
    w.lo = window > 0 ? max(0, first_pos - window + 1) : 0;
    w.hi = last_pos;
    w.t_lo = w.lo / tile;
    // (xr_kept_tiles in unsigned numbers: with sixteen rows of 128 elements the compiler spills less, 1,087 us instead of 1,150 at 200 single tokens beside a portion)
    w.kept = min((int)(((unsigned)keep + tile - 1) / tile), w.t_lo);
    w.n = w.kept + w.hi / tile - w.t_lo + 1;
    return w;
}
// Spans of a request: a.span_tiles tiles each, the last of the grid's takes what is left (a captured launch may meet longer requests
// than the one it was planned for).
__device__ __forceinline__ int a4_spans(const A4Args& a, const A4Walk& w) { return min((w.n + a.span_tiles - 1) / a.span_tiles, a.splits); }

// Row blocks of the portions ahead of portion `seg`, of those that are taken.  All lanes of a warp.  (Not inlined: it costs the loop over tiles no register.)
__device__ __noinline__ int a4_blocks_ahead(const int* seg_len, int seg, int G, int most_rows, int rows) {
    int ahead = 0;
#pragma unroll 4
    for (int s = threadIdx.x & 31; s < seg; s += 32) {
        const long long r = (long long)seg_len[s] * G;
        if (r > 0 && r <= most_rows) ahead += (int)((r + rows - 1) / rows);
    }
    return __reduce_add_sync(0xffffffffu, ahead);
}
// The place of a row block in the scratch for partial sums: row blocks of all portions that are taken lie one after another.  (One a portion: a place for every
// portion, empty ones too.)
__device__ __forceinline__ int a4_place(const A4Args& a, int seg, int rb, int rows) {
    return a.row_blocks == 1 ? seg : a4_blocks_ahead(a.seg_len, seg, a.G, a.most_rows, rows) + rb;
}

// NG: groups of 32 elements a held head (2, 4, 8); NT: eight-row tiles a block; F32: float32 queries and outputs, in pieces (NT 1);
// EXTRA: a cap or a bias on the scores
template <int NG, int NT, bool F32, bool EXTRA> struct A4Shape {
    static constexpr int HS = NG * 32, TK = A4Tile<NG>::KEYS, SUB = TK / 16, STAGES = A4Tile<NG>::STAGES, KS = 2 * NG, RB = 8 * NT, P = F32 ? 3 : 1;
    static constexpr int CODES = HS / 2, SCALES = HS / 16;           // bytes of a token's keys (or values)
    static constexpr int STAGE = TK * 2 * (CODES + SCALES);
    static constexpr int VW = NG / 2, MT = 4 * VW;                   // words of a value's row a thread takes; m-tiles of O^T
    static constexpr bool Q_REGS = KS * 2 * NT * P <= 48;            // q's fragments in registers, else in shared memory
    static constexpr int SMEM = A4_WARPS * STAGES * STAGE + (Q_REGS ? 0 : P * NT * KS * 32 * 8) + 16;
    // Blocks an SM: by registers, and by its 228 KB of shared memory, of which a block takes one more.  (Heads of 256 elements: two of eight bfloat16 rows, one of
    // sixteen or of float32.)
    static constexpr int BY_REGS = NG <= 4 && NT == 1 && !F32 ? 3 : 2, BY_SMEM = 228 * 1024 / (SMEM + 1024), BLOCKS = BY_REGS < BY_SMEM ? BY_REGS : BY_SMEM;
};

template <int NG, int NT, bool F32, bool EXTRA>
__global__ void __launch_bounds__(A4_THREADS, (A4Shape<NG, NT, F32, EXTRA>::BLOCKS))
k_kv4_attention(A4Args a) {
    xr_pdl_launch();
    using S = A4Shape<NG, NT, F32, EXTRA>;
    constexpr int HS = S::HS, TK = S::TK, SUB = S::SUB, STAGES = S::STAGES, KS = S::KS, RB = S::RB, P = S::P, CODES = S::CODES, SCALES = S::SCALES, STAGE = S::STAGE;
    constexpr int VW = S::VW, MT = S::MT;
    extern __shared__ __align__(128) uint8_t smem[];
    uint2* q_sm = (uint2*)(smem + A4_WARPS * STAGES * STAGE);                        // [P][NT][KS][32]
    const int seg = blockIdx.z, kvh = blockIdx.y, rb = blockIdx.x / a.splits, span = blockIdx.x - rb * a.splits;
    // (a.early: portions, block tables and the rows of earlier steps are at rest, so that tiles of such rows set out before the kernel ahead is complete.  It
    // takes more than that kernel's wait to say so, for kernels here let the next one start before they wait themselves: an engine's step begins with
    // the copy of its description, which waits for all of the last step, and stores no rows but its own.  Blocks without work leave without a wait;
    // a launch has one that waits, or it is not made.)
    if (!a.early) xr_pdl_wait();
    const int L = a.seg_len[seg];
    const long long rows_all = (long long)L * a.G;
    if (L < 1 || rows_all > a.most_rows || (long long)rb * RB >= rows_all) return;
    const int row0 = rb * RB, rows = (int)min((long long)RB, rows_all - row0);
    const int pos0 = a.seg_pos0[seg], tok0 = a.seg_start[seg];
    const int first_pos = pos0 + row0 / a.G, last_pos = pos0 + (row0 + rows - 1) / a.G;
    const A4Walk walk = a4_walk(first_pos, last_pos, a.window, a.keep, TK);
    const int n_spans = a4_spans(a, walk);
    if (span >= n_spans) {
        if (a.clustered) { a4_cluster_sync(); a4_cluster_sync(); }       // (nothing to do, but the cluster's barriers count every block)
        return;
    }
    const int i_begin = span * a.span_tiles, i_end = span == n_spans - 1 ? walk.n : i_begin + a.span_tiles;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int* bt = a.block_tables + (size_t)seg * a.max_pages;
    const int ps = a.c.page_size;
    uint8_t* my_ring = smem + warp * STAGES * STAGE;              // a stage: keys' codes, values' codes, keys' scales, values' scales
    const uint32_t ring_at = a4_smem(my_ring);
    const uint8_t* head_run = a.c.base + a.c.layer_at + (long long)kvh * a.c.block();
    auto page_of = [&](int pi) -> int {
        const int page = pi < a.max_pages ? __ldg(bt + pi) : -1;
        return page < a.c.n_pages ? page : -1;
    };
    // The page of tile i, where pages hold whole tiles (2^tile_shift of them); asked for a tile ahead of its fetch: one trip to L1 that nobody waits for.
    auto tiles_page = [&](int i) { return a.tile_shift >= 0 && i < i_end ? page_of(xr_walk_tile(i, walk.kept, walk.t_lo) >> a.tile_shift) : -1; };
    // The warp fetches tile i of the walk into stage s, 16 bytes a lane at a time; rows on a page that is not held become zeros.
    auto fetch = [&](int i, int s, int page) {
        const int tile = xr_walk_tile(i, walk.kept, walk.t_lo);
        const uint32_t st = ring_at + s * STAGE + 16 * lane;
        if (a.tile_shift >= 0) {
            const int in = (tile & ((1 << a.tile_shift) - 1)) * TK;
            const uint32_t n = page >= 0 ? 16 : 0;
            const uint8_t* run = head_run + max(page, 0) * a.c.page_bytes;
            const uint8_t* codes = run + in * CODES + 16 * lane;
            const uint8_t* scales = run + a.c.scales_at(0) + in * SCALES;
            const int far = a.c.codes_at(1);
#pragma unroll
            for (int e = 0; e < TK * CODES / 512; e++) {
                a4_copy(st + 512 * e, codes + 512 * e, n);
                a4_copy(st + TK * CODES + 512 * e, codes + far + 512 * e, n);
            }
#pragma unroll
            for (int e = 0; e < TK * SCALES / 256; e++) {
                // (half the lanes the keys' scales, half the values')
                const int b = 16 * (lane & 15) + 256 * e;
                a4_copy(ring_at + s * STAGE + 2 * TK * CODES + (lane >> 4) * TK * SCALES + b, scales + (lane >> 4) * (ps * SCALES) + b, n);
            }
        } else {
            const long long k0 = (long long)tile * TK;
            auto piece = [&](uint32_t to, int at, int token, int bytes) {         // the 16 bytes at `at` behind the first token's in a part, `bytes` a token
                const int r = at / bytes, pi = (int)((k0 + r) / ps), held = page_of(pi);
                const uint8_t* run = head_run + max(held, 0) * a.c.page_bytes + token;
                a4_copy(to, run + (k0 + r - (long long)pi * ps) * bytes + at % bytes, held >= 0 ? 16 : 0);
            };
#pragma unroll 1
            for (int b = 16 * lane; b < TK * CODES; b += 512) {
                piece(ring_at + s * STAGE + b, b, a.c.codes_at(0), CODES);
                piece(ring_at + s * STAGE + TK * CODES + b, b, a.c.codes_at(1), CODES);
            }
#pragma unroll 1
            for (int b = 16 * (lane & 15); b < TK * SCALES; b += 256)
                piece(ring_at + s * STAGE + 2 * TK * CODES + (lane >> 4) * TK * SCALES + b, b, a.c.scales_at(lane >> 4), SCALES);
        }
    };
    // (a group of copies a stage, empty ones behind the last tile: the wait counts groups)
    int next_page;
    {
        int first[STAGES];
#pragma unroll
        for (int s = 0; s < STAGES; s++) first[s] = tiles_page(i_begin + warp + s * A4_WARPS);
        next_page = tiles_page(i_begin + warp + STAGES * A4_WARPS);
        // (this step's own rows are stored by a kernel ahead; the span's last tile is the furthest)
        const bool old_rows = ((long long)xr_walk_tile(i_end - 1, walk.kept, walk.t_lo) + 1) * TK <= pos0;
        if (a.early && !old_rows) xr_pdl_wait();
#pragma unroll
        for (int s = 0; s < STAGES; s++) {
            if (i_begin + warp + s * A4_WARPS < i_end) fetch(i_begin + warp + s * A4_WARPS, s, first[s]);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        if (a.early && old_rows) xr_pdl_wait();
    }
    // (where the block's sums will lie, while its first tiles are on their way)
    int* place_s = reinterpret_cast<int*>(smem + S::SMEM - 16);
    if (warp == 0 && n_spans > 1 && !a.clustered) {
        const int place = a4_place(a, seg, rb, RB);
        if (lane == 0) *place_s = place;
    }

    // q.  float32: thread (row g, t) holds the elements that its words of a key hold, 8 NG t ..; k-step 2 w + half: elements 8 w + 4 half ..  bfloat16: thread
    // (row g, t) holds the elements of word t of every group; k-steps 2 grp and 2 grp + 1.
    uint32_t qf[S::Q_REGS ? P : 1][S::Q_REGS ? NT : 1][S::Q_REGS ? KS : 1][2];
    float q_sum[F32 ? 1 : NT][F32 ? 1 : NG][2], q_unit[NT][2];       // of the thread's two columns: what takes a group's bias off; a score's unit
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const int row = row0 + nt * 8 + g, live = nt * 8 + g < rows;
        const long long base = live ? (long long)(tok0 + row / a.G) * a.q_stride + (long long)(kvh * a.G + row % a.G) * a.D : 0;
        if constexpr (F32) {
            q_unit[nt][0] = q_unit[nt][1] = 1.f;
#pragma unroll
            for (int w = 0; w < NG; w++) {
                const int d = 8 * (NG * t + w);
                float x[8];
                const float* src = (const float*)a.q + base + d;
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = live && d + e < a.D ? src[e] : 0.f;
#pragma unroll
                for (int p = 0; p < 3; p++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const uint32_t u = a4_piece(x[4 * h], x[4 * h + 1]), v = a4_piece(x[4 * h + 2], x[4 * h + 3]);
                        if constexpr (S::Q_REGS) { qf[p][nt][2 * w + h][0] = u; qf[p][nt][2 * w + h][1] = v; }
                        else if (warp == 0) q_sm[((p * NT + nt) * KS + 2 * w + h) * 32 + lane] = make_uint2(u, v);
                    }
            }
        } else {
            auto word_of = [&](int w, uint32_t* x) {
                const int d = 32 * w + 8 * t;
                const __nv_bfloat16* src = (const __nv_bfloat16*)a.q + base + d;
                x[0] = x[1] = x[2] = x[3] = 0;
                if (a.wide) {
                    if (live && d < a.D) { const uint4 v = *reinterpret_cast<const uint4*>(src); x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w; }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (live && d + e < a.D) x[e >> 1] |= (uint32_t)reinterpret_cast<const unsigned short*>(src)[e] << (16 * (e & 1));
                }
            };
            uint32_t top = 0;                                        // the largest magnitude, by its bits: a NaN is above all others
#pragma unroll
            for (int w = 0; w < NG; w++) {
                uint32_t x[4];
                word_of(w, x);
#pragma unroll
                for (int e = 0; e < 4; e++) top = max(top, max((x[e] << 16) & 0x7fff0000u, x[e] & 0x7fff0000u));
            }
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // The row in float16, times a power of two: largest magnitude in [2^13, 2^14), every element's eight bits whole down to 2^-31 of it.  A row
            // with an infinity or a NaN has no unit.
            const int ex = max((int)(top >> 23), 20) - 127;
            const float up = __int_as_float((127 + 13 - ex) << 23), unit = ex == 128 ? __int_as_float(0x7fc00000) : __int_as_float((127 - 13 + ex) << 23);
            q_unit[nt][0] = __shfl_sync(0xffffffffu, unit, 8 * t);
            q_unit[nt][1] = __shfl_sync(0xffffffffu, unit, 8 * t + 4);
#pragma unroll
            for (int w = 0; w < NG; w++) {
                uint32_t x[4];
                word_of(w, x);
                uint32_t y[4];
                float sum = 0.f;                                     // the pairs' biases: 256 + 8 and 16 + 8
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    y[e] = a4_pack_half(__uint_as_float(x[e] << 16) * up, __uint_as_float(x[e] & 0xffff0000u) * up);
                    const float2 z = __half22float2(*reinterpret_cast<const __half2*>(&y[e]));
                    sum = fmaf(e & 1 ? -24.f : -264.f, z.x + z.y, sum);
                }
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    if constexpr (S::Q_REGS) { qf[0][nt][2 * w + h][0] = y[2 * h]; qf[0][nt][2 * w + h][1] = y[2 * h + 1]; }
                    else if (warp == 0) q_sm[(nt * KS + 2 * w + h) * 32 + lane] = make_uint2(y[2 * h], y[2 * h + 1]);
                }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                q_sum[nt][w][0] = __shfl_sync(0xffffffffu, sum, 8 * t);
                q_sum[nt][w][1] = __shfl_sync(0xffffffffu, sum, 8 * t + 4);
            }
        }
    }
    if (!S::Q_REGS) __syncthreads();

    int pos_r[NT][2];                                                // positions of this thread's two columns (rows of q) of each tile
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 2; e++) pos_r[nt][e] = pos0 + (row0 + min(nt * 8 + 2 * t + e, rows - 1)) / a.G;
    const float sl = a.scale * A4_LOG2E;
    // (float16 weights: 2^LIFT times larger, so that they are whole numbers of 2^-11 of themselves down to 2^-19 of the largest; at most 2^13)
    constexpr float LIFT = F32 ? 0.f : 5.f;
    float unit[NT][2];                                               // what turns a column's scores into exponents of two
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            unit[nt][e] = EXTRA ? 1.f : sl * q_unit[nt][e];
            if (unit[nt][e] == 0.f) unit[nt][e] = __int_as_float(1);       // (below float32: a hidden key's minus infinity times it is to stay that)
        }
    float o[NT][MT][4], m[NT][2], l[NT][2];
    float v_unit = 1.f, v_inv = 1.f, v_most = F32 ? INFINITY : 0.f;  // the sums' unit, its inverse, the largest scale that it takes
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int i = 0; i < MT; i++) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
        m[nt][0] = m[nt][1] = -INFINITY; l[nt][0] = l[nt][1] = 0.f;
    }
    const int key_a = a4_key(g);                                     // a subtile's key of row g (row g + 8: 8 further)
    const int place_a = t, place_b = 4 + (t ^ 1);                    // ... of places 2t and 2t + 1
    // where a thread reads in a stage: keys' codes (bfloat16: the row that it names to ldmatrix; float32: its words) and scales, values' codes and
    // scales of places 2t and 2t + 1
    const uint32_t k_at = F32 ? key_a * CODES + 4 * NG * t
                        : NG == 2 ? (8 * (lane >> 4) + a4_key(lane & 7)) * CODES + 16 * ((lane >> 3) & 1) : a4_key(lane & 7) * CODES + 16 * (lane >> 3);
    const uint32_t ks_at = 2 * TK * CODES + key_a * SCALES + (F32 ? 2 * (NG * t / 4) : 0);
    const uint32_t va_at = TK * CODES + place_a * CODES + 4 * VW * g, vb_at = TK * CODES + place_b * CODES + 4 * VW * g;
    const uint32_t vsa_at = 2 * TK * CODES + TK * SCALES + place_a * SCALES + 2 * (g * VW / 4), vsb_at = vsa_at + (place_b - place_a) * SCALES;
    int stage = 0;
    for (int i = i_begin + warp; i < i_end; i += A4_WARPS) {
        const int k0 = xr_walk_tile(i, walk.kept, walk.t_lo) * TK;
        const uint32_t st = ring_at + stage * STAGE;
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        __syncwarp();
        float s[SUB][NT][4];
#pragma unroll
        for (int sub = 0; sub < SUB; sub++) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++) s[sub][nt][0] = s[sub][nt][1] = s[sub][nt][2] = s[sub][nt][3] = 0.f;
            if constexpr (!F32) {
                // A group's codes are multiplied as they are, with their bias, from sums that start at what takes it off; the group's scale is a factor on the
                // result.  All four threads of a key have a word of the same group: ldmatrix deals a 16-byte row's words to them.
                uint32_t w[2][NG];                                   // word t of every group, of the keys of rows g and g + 8
                uint32_t sc[2][NG / 2];
                if constexpr (NG == 2) {
                    uint32_t r[4];
                    a4_ldsm4(r, st + k_at + sub * 16 * CODES);
                    w[0][0] = r[0]; w[0][1] = r[1]; w[1][0] = r[2]; w[1][1] = r[3];
                } else {
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int c = 0; c < NG; c += 4) a4_ldsm4(&w[h][c], st + k_at + (sub * 16 + 8 * h) * CODES + 16 * c);
                }
#pragma unroll
                for (int h = 0; h < 2; h++) a4_lds<NG / 2>(sc[h], st + ks_at + (sub * 16 + 8 * h) * SCALES);
#pragma unroll
                for (int grp = 0; grp < NG; grp++) {
                    uint32_t pa[4], pb[4];
                    a4_pairs(w[0][grp], pa);
                    a4_pairs(w[1][grp], pb);
                    const float fa = __uint_as_float(grp & 1 ? sc[0][grp >> 1] & 0xffff0000u : sc[0][grp >> 1] << 16);
                    const float fb = __uint_as_float(grp & 1 ? sc[1][grp >> 1] & 0xffff0000u : sc[1][grp >> 1] << 16);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        float d[4];
                        uint2 qa, qb;
                        if constexpr (S::Q_REGS) { qa = make_uint2(qf[0][nt][2 * grp][0], qf[0][nt][2 * grp][1]); qb = make_uint2(qf[0][nt][2 * grp + 1][0], qf[0][nt][2 * grp + 1][1]); }
                        else { qa = q_sm[(nt * KS + 2 * grp) * 32 + lane]; qb = q_sm[(nt * KS + 2 * grp + 1) * 32 + lane]; }
                        a4_mma_from(d, pa[0], pb[0], pa[1], pb[1], qa.x, qa.y, q_sum[nt][grp][0], q_sum[nt][grp][1]);
                        a4_mma_half(d, pa[2], pb[2], pa[3], pb[3], qb.x, qb.y);
#pragma unroll
                        for (int e = 0; e < 4; e++) s[sub][nt][e] = grp == 0 ? (e < 2 ? fa : fb) * d[e] : fmaf(e < 2 ? fa : fb, d[e], s[sub][nt][e]);
                    }
                }
            } else {
                uint32_t wa[NG], wb[NG];
                a4_lds<NG>(wa, st + k_at + sub * 16 * CODES);
                a4_lds<NG>(wb, st + k_at + (sub * 16 + 8) * CODES);
#pragma unroll
                for (int w0 = 0; w0 < NG; w0 += NG == 2 ? 2 : 4) {
                    // (a thread's words of one group share a scale)
                    uint32_t sa = a4_lds16(st + ks_at + sub * 16 * SCALES + w0 / 2), sb = a4_lds16(st + ks_at + (sub * 16 + 8) * SCALES + w0 / 2);
                    sa *= 0x10001u; sb *= 0x10001u;
                    const uint32_t ma = kv4_m24(sa), mb = kv4_m24(sb);
#pragma unroll
                    for (int w = w0; w < w0 + (NG == 2 ? 2 : 4); w++) {
                        const uint32_t a0 = kv4_scaled(kv4_pair<0>(wa[w]), sa, ma), a1 = kv4_scaled(kv4_pair<0>(wb[w]), sb, mb);
                        const uint32_t a2 = kv4_scaled(kv4_pair<1>(wa[w]), sa, ma), a3 = kv4_scaled(kv4_pair<1>(wb[w]), sb, mb);
                        const uint32_t b0 = kv4_scaled(kv4_pair<2>(wa[w]), sa, ma), b1 = kv4_scaled(kv4_pair<2>(wb[w]), sb, mb);
                        const uint32_t b2 = kv4_scaled(kv4_pair<3>(wa[w]), sa, ma), b3 = kv4_scaled(kv4_pair<3>(wb[w]), sb, mb);
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            float d[4] = {0.f, 0.f, 0.f, 0.f};         // (see A4_VALUES)
#pragma unroll
                            for (int p = P - 1; p >= 0; p--) {
                                uint2 qa, qb;
                                if constexpr (S::Q_REGS) { qa = make_uint2(qf[p][nt][2 * w][0], qf[p][nt][2 * w][1]); qb = make_uint2(qf[p][nt][2 * w + 1][0], qf[p][nt][2 * w + 1][1]); }
                                else { qa = q_sm[((p * NT + nt) * KS + 2 * w) * 32 + lane]; qb = q_sm[((p * NT + nt) * KS + 2 * w + 1) * 32 + lane]; }
                                a4_mma(d, a0, a1, a2, a3, qa.x, qa.y);
                                a4_mma(d, b0, b1, b2, b3, qb.x, qb.y);
                            }
#pragma unroll
                            for (int e = 0; e < 4; e++) s[sub][nt][e] += d[e];
                        }
                    }
                }
            }
        }
        // a tile that not every row sees whole
        const bool edge = k0 + TK - 1 > first_pos || (a.window > 0 && k0 <= last_pos - a.window && k0 + TK > a.keep);
        if constexpr (EXTRA) {
#pragma unroll
            for (int sub = 0; sub < SUB; sub++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        float& x = s[sub][nt][e];
                        // (exponents of two, so that `unit` is one: scores that are equal and huge, a bias of the lowest number for one, differ by exactly zero)
                        if (a.softcap > 0.f) {
                            // c tanh(x scale / c), through one exponential: tanh(y) = 1 - 2 / (exp(2 y) + 1)
                            const float cap = a.softcap * A4_LOG2E, y = x * q_unit[nt][e & 1] * (a.scale / a.softcap);
                            x = F32 ? cap * tanhf(y) : cap * (1.0f - __fdividef(2.0f, __expf(2.0f * y) + 1.0f));
                        } else {
                            const int row = row0 + min(nt * 8 + 2 * t + (e & 1), rows - 1);
                            const float y = x * q_unit[nt][e & 1] + xr_bias_at(a.bias.table + (size_t)(kvh * a.G + row % a.G) * a.bias.len, a.bias.len, pos_r[nt][e & 1] - (k0 + sub * 16 + key_a + 4 * (e & 2)));
                            x = y * sl;
                            // (a score that is a number stays one: a scale above ln 2 takes the largest ones out of float32)
                            if (sl > 1.f && fabsf(x) == INFINITY && fabsf(y) < INFINITY) x = copysignf(3.402823466e38f, y);
                        }
                    }
        }
        if (edge) {
#pragma unroll
            for (int sub = 0; sub < SUB; sub++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int key = k0 + sub * 16 + key_a + 4 * (e & 2), pos = pos_r[nt][e & 1];
                        if (!xr_sees(key, pos, a.window > 0 ? pos - a.window + 1 : 0, a.keep)) s[sub][nt][e] = -INFINITY;
                    }
        }
        // The running maximum is followed loosely: weights are exp2(score - m), and m is raised (to the columns' maxima over all lanes) only where a score
        // is 2^A4_SLACK times above it, or is the first.  Weights up to 2^A4_SLACK change no relative error, and most tiles pay neither for shuffles nor
        // for another pass over the sums.
        bool grown = false;
        float mx[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                mx[nt][e] = fmaxf(s[0][nt][e], s[0][nt][e + 2]);
#pragma unroll
                for (int sub = 1; sub < SUB; sub++) mx[nt][e] = fmaxf(mx[nt][e], fmaxf(s[sub][nt][e], s[sub][nt][e + 2]));
                grown |= mx[nt][e] * unit[nt][e] > m[nt][e] + A4_SLACK;
            }
        if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                float f[2];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float x = mx[nt][e];
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                    const float was = m[nt][e];
                    m[nt][e] = fmaxf(was, x * unit[nt][e]);
                    f[e] = was == m[nt][e] ? 1.f : a4_exp2(was - m[nt][e]);            // (both -infinity: no key seen yet)
                    l[nt][e] *= f[e];
                }
#pragma unroll
                for (int d = 0; d < MT; d++) { o[nt][d][0] *= f[0]; o[nt][d][1] *= f[1]; o[nt][d][2] *= f[0]; o[nt][d][3] *= f[1]; }
            }
        }
        float off[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 2; e++) off[nt][e] = m[nt][e] == -INFINITY ? 0.f : m[nt][e] - LIFT;
        // the values' scales: of places 2t, 2t + 1, 2t + 8, 2t + 9 of every subtile
        uint32_t sv[SUB][4];
#pragma unroll
        for (int sub = 0; sub < SUB; sub++)
#pragma unroll
            for (int c = 0; c < 4; c++) sv[sub][c] = a4_lds16(st + (c & 1 ? vsb_at : vsa_at) + (sub * 16 + 8 * (c >> 1)) * SCALES);
        if (edge) {
            // What lies behind the last key or ahead of the window may be anything, scales that are no numbers too: no row sees it.
            const bool several = first_pos != last_pos;
#pragma unroll
            for (int sub = 0; sub < SUB; sub++) {
                uint32_t none = 0;
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const int at = (c & 1 ? place_b : place_a) + 8 * (c >> 1);
                    if (!xr_sees(k0 + sub * 16 + at, walk.hi, walk.lo, a.keep)) sv[sub][c] = 0;
                    if (several && (sv[sub][c] & 0x7f80) == 0x7f80) { none |= 1u << at; sv[sub][c] = 0; }
                }
                if (__any_sync(0xffffffffu, none != 0)) {
                    // A value that is no number, and rows of several positions, some of which may not see it: it is left out of the products, and the
                    // elements of its group become NaN for the rows that do see it.
                    none |= __shfl_xor_sync(0xffffffffu, none, 1);
                    none |= __shfl_xor_sync(0xffffffffu, none, 2);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            bool hit = false;
                            for (int b = 0; b < 16; b++)
                                hit |= (none >> b & 1) && xr_sees(k0 + sub * 16 + b, pos_r[nt][e], a.window > 0 ? pos_r[nt][e] - a.window + 1 : 0, a.keep);
                            if (hit) {
#pragma unroll
                                for (int d = 0; d < MT; d++) o[nt][d][e] = o[nt][d][e + 2] = __int_as_float(0x7fc00000);
                            }
                        }
                }
            }
            __syncwarp();                                             // (lanes parted in there, and the matrix instructions want them together)
        }
        // bfloat16 queries: values are multiplied in float16, in units of a power of two: scales within 2^-20 .. 248 units make values that are exact.  A unit belongs
        // to the elements that four lanes share (of one group: a head's groups may differ in size as they like).  It is chosen by the first tile with values
        // that are not zero, so that the largest scale is 8 to 16 of it, and again where a scale outgrows it.  So a value keeps all its bits down to 2^-23 of the
        // largest one of its elements, and is zero from 2^-29 on: beside weights of the same size nothing, and what a hidden or hardly seen row takes from the others.
        // Units are compared and changed by the scales' own bits: the range of what is held is wider than that of a float32 quotient.
        uint32_t v_scale[F32 ? 1 : SUB][2];                            // pairs of scales in float16
        if constexpr (!F32) {
            float vs[SUB][4], top = 0.f;
#pragma unroll
            for (int sub = 0; sub < SUB; sub++)
#pragma unroll
                for (int c = 0; c < 4; c++) { vs[sub][c] = __uint_as_float(sv[sub][c] << 16); top = fmaxf(top, fabsf(vs[sub][c])); }
            if (__any_sync(0xffffffffu, top > v_most)) {
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                float less = 1.f;
                if (top > v_most) {
                    const int e = min(max((int)(__float_as_uint(top) >> 23) - 3, 1), 253);
                    const float inv = __int_as_float((254 - e) << 23);
                    less = v_unit * inv;                               // (the first time there is nothing but zeros to change)
                    v_unit = __int_as_float(e << 23); v_inv = inv; v_most = 248.f * v_unit;
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int d = 0; d < MT; d++) { o[nt][d][0] *= less; o[nt][d][1] *= less; o[nt][d][2] *= less; o[nt][d][3] *= less; }
            }
#pragma unroll
            for (int sub = 0; sub < SUB; sub++)
#pragma unroll
                for (int c = 0; c < 4; c++) vs[sub][c] *= v_inv;
#pragma unroll
            for (int sub = 0; sub < SUB; sub++) { v_scale[sub][0] = a4_pack_half(vs[sub][0], vs[sub][1]); v_scale[sub][1] = a4_pack_half(vs[sub][2], vs[sub][3]); }
        }
#pragma unroll
        for (int sub = 0; sub < SUB; sub++) {
            uint32_t pb[P][NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                float x[4];
#pragma unroll
                for (int e = 0; e < 4; e++) { x[e] = a4_exp2(fmaf(s[sub][nt][e], unit[nt][e & 1], -off[nt][e & 1])); l[nt][e & 1] += x[e]; }
#pragma unroll
                for (int p = 0; p < P; p++) {
                    pb[p][nt][0] = a4_turn(F32 ? a4_piece(x[0], x[1]) : a4_pack_half(x[0], x[1]));
                    pb[p][nt][1] = a4_turn(F32 ? a4_piece(x[2], x[3]) : a4_pack_half(x[2], x[3]));
                }
            }
            uint32_t w[4][VW];
#pragma unroll
            for (int c = 0; c < 4; c++) a4_lds<VW>(w[c], st + (c & 1 ? vb_at : va_at) + (sub * 16 + 8 * (c >> 1)) * CODES);
            if constexpr (!F32) {
                const uint32_t s0 = v_scale[sub][0], s1 = v_scale[sub][1];
                // -264 s and -24 s (11 and 7 bits: exact)
                const uint32_t m0[2] = {a4_mul_half(s0, 0xDC20DC20u), a4_mul_half(s0, 0xCE00CE00u)}, m1[2] = {a4_mul_half(s1, 0xDC20DC20u), a4_mul_half(s1, 0xCE00CE00u)};
#pragma unroll
                for (int j = 0; j < VW; j++) {
                    // the halves of two keys' words side by side: pair i of them is element 2i (low halves) or 2i + 1 of both keys
                    uint32_t lo0[4], hi0[4], lo1[4], hi1[4];
                    a4_pairs(__byte_perm(w[0][j], w[1][j], 0x5410), lo0);
                    a4_pairs(__byte_perm(w[0][j], w[1][j], 0x7632), hi0);
                    a4_pairs(__byte_perm(w[2][j], w[3][j], 0x5410), lo1);
                    a4_pairs(__byte_perm(w[2][j], w[3][j], 0x7632), hi1);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t a0 = a4_fma_half(lo0[i], s0, m0[i & 1]), a1 = a4_fma_half(hi0[i], s0, m0[i & 1]);
                        const uint32_t a2 = a4_fma_half(lo1[i], s1, m1[i & 1]), a3 = a4_fma_half(hi1[i], s1, m1[i & 1]);
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) a4_mma_half(o[nt][4 * j + i], a0, a1, a2, a3, pb[0][nt][0], pb[0][nt][1]);
                    }
                }
            } else {
                const uint32_t s0 = sv[sub][1] * 65536u + sv[sub][0], s1 = sv[sub][3] * 65536u + sv[sub][2], m0 = kv4_m24(s0), m1 = kv4_m24(s1);
#pragma unroll
                for (int j = 0; j < VW; j++) {
                    const uint32_t lo0 = __byte_perm(w[0][j], w[1][j], 0x5410), hi0 = __byte_perm(w[0][j], w[1][j], 0x7632);
                    const uint32_t lo1 = __byte_perm(w[2][j], w[3][j], 0x5410), hi1 = __byte_perm(w[2][j], w[3][j], 0x7632);
                    // The matrix instruction does not round its sums to nearest: what it adds to a long sum is off to one side every time.  So its sums begin
                    // at zero, the small pieces ahead of the large, and the long ones are the float32 additions'.  (27,777 keys: 4.6e-7 off instead of 1.9e-6,
                    // 256 elements: 2.3e-7 instead of 1.4e-6; no time.)
#define A4_VALUES(I)                                                                                                                              \
                    {                                                                                                                             \
                        const uint32_t a0 = kv4_scaled(kv4_pair<I>(lo0), s0, m0), a1 = kv4_scaled(kv4_pair<I>(hi0), s0, m0);                      \
                        const uint32_t a2 = kv4_scaled(kv4_pair<I>(lo1), s1, m1), a3 = kv4_scaled(kv4_pair<I>(hi1), s1, m1);                      \
                        _Pragma("unroll") for (int nt = 0; nt < NT; nt++) {                                                                       \
                            float d[4] = {0.f, 0.f, 0.f, 0.f};                                                                                    \
                            _Pragma("unroll") for (int p = P - 1; p >= 0; p--) a4_mma(d, a0, a1, a2, a3, pb[p][nt][0], pb[p][nt][1]);             \
                            _Pragma("unroll") for (int e = 0; e < 4; e++) o[nt][4 * j + I][e] += d[e];                                            \
                        }                                                                                                                         \
                    }
                    A4_VALUES(0) A4_VALUES(1) A4_VALUES(2) A4_VALUES(3)
#undef A4_VALUES
                }
            }
        }
        __syncwarp();
        if (i + STAGES * A4_WARPS < i_end) {
            fetch(i + STAGES * A4_WARPS, stage, next_page);
            next_page = tiles_page(i + (STAGES + 1) * A4_WARPS);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (++stage == STAGES) stage = 0;
    }
    // the warps' sums meet in the ring's memory: [warp][row][HS], then [warp][row] (maximum, sum)
    __syncthreads();
    float* acc_s = reinterpret_cast<float*>(smem);
    float* ml_s = acc_s + A4_WARPS * RB * HS;
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int r = nt * 8 + 2 * t + e;
            float sum = l[nt][e];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            float* dst = acc_s + (warp * RB + r) * HS + 8 * VW * g;
#pragma unroll
            for (int j = 0; j < VW; j++) {
                *reinterpret_cast<float4*>(dst + 8 * j) = make_float4(o[nt][4 * j][e] * v_unit, o[nt][4 * j][e + 2] * v_unit, o[nt][4 * j + 1][e] * v_unit, o[nt][4 * j + 1][e + 2] * v_unit);
                *reinterpret_cast<float4*>(dst + 8 * j + 4) = make_float4(o[nt][4 * j + 2][e] * v_unit, o[nt][4 * j + 2][e + 2] * v_unit, o[nt][4 * j + 3][e] * v_unit, o[nt][4 * j + 3][e + 2] * v_unit);
            }
            if (g == 0) { ml_s[(warp * RB + r) * 2] = m[nt][e] - LIFT; ml_s[(warp * RB + r) * 2 + 1] = sum; }
        }
    __syncthreads();
    size_t item = 0;
    if (n_spans > 1 && !a.clustered) {
        const int place = *place_s;
        if ((unsigned)place >= (unsigned)a.blocks) return;           // (lengths that the launch was not made for: nothing is written beyond the scratch)
        item = ((size_t)place * a.c.K + kvh) * a.splits + span;
    }
    for (int q = threadIdx.x; q < rows * (HS / 4); q += A4_THREADS) {
        const int r = q / (HS / 4), d = (q % (HS / 4)) * 4;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < A4_WARPS; w++) mm = fmaxf(mm, ml_s[(w * RB + r) * 2]);
        const float at = mm == -INFINITY ? 0.f : mm;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < A4_WARPS; w++) {
            const float k = a4_exp2(ml_s[(w * RB + r) * 2] - at);
            const float4 u = *reinterpret_cast<const float4*>(acc_s + (w * RB + r) * HS + d);
            v.x += u.x * k; v.y += u.y * k; v.z += u.z * k; v.w += u.w * k;
            sum += ml_s[(w * RB + r) * 2 + 1] * k;
        }
        if (n_spans == 1) a4_out<F32>(a, tok0, kvh, row0 + r, d, v, at, sum);
        else if (a.clustered) {
            // the block's own sums, where its first warp's were (this thread alone reads them), and behind all others (maximum, sum)
            *reinterpret_cast<float4*>(acc_s + r * HS + d) = v;
            if (d == 0) *reinterpret_cast<float2*>(ml_s + (A4_WARPS * RB + r) * 2) = make_float2(mm, sum);
        } else {
            *reinterpret_cast<float4*>(a.part_acc + (item * RB + r) * HS + d) = v;
            if (d == 0) *reinterpret_cast<float2*>(a.part_ml + (item * RB + r) * 2) = make_float2(mm, sum);
        }
    }
    if (a.clustered) {
        // Every block of the cluster finishes a share of the rows' quadruples out of all blocks' shared memory, in ascending order of spans.
        a4_cluster_sync();
        if (n_spans > 1)
            for (int q = span + threadIdx.x * n_spans; q < rows * (HS / 4); q += A4_THREADS * n_spans) {
                const int r = q / (HS / 4), d = (q % (HS / 4)) * 4;
                float2 ml[A4_CLUSTER];
                float4 acc[A4_CLUSTER];
#pragma unroll
                for (int s = 0; s < A4_CLUSTER; s++) {
                    const uint32_t rank = min(s, n_spans - 1);       // (clamped: no load is conditional)
                    ml[s] = a4_far2(a4_of_rank(ml_s + (A4_WARPS * RB + r) * 2, rank));
                    acc[s] = a4_far4(a4_of_rank(acc_s + r * HS + d, rank));
                }
                float mm = -INFINITY;
#pragma unroll
                for (int s = 0; s < A4_CLUSTER; s++) mm = fmaxf(mm, ml[s].x);
                const float at = mm == -INFINITY ? 0.f : mm;
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                float sum = 0.f;
#pragma unroll
                for (int s = 0; s < A4_CLUSTER; s++) {
                    if (s >= n_spans) break;
                    const float k = a4_exp2(ml[s].x - at);
                    v.x += acc[s].x * k; v.y += acc[s].y * k; v.z += acc[s].z * k; v.w += acc[s].w * k;
                    sum += ml[s].y * k;
                }
                a4_out<F32>(a, tok0, kvh, row0 + r, d, v, at, sum);
            }
        a4_cluster_sync();                                           // (nobody leaves while another reads its memory)
    }
}

// ---------------------------------------------------------------------------------------------
// The spans of one (request, kv head, row block) in ascending order: grid (K * row blocks, requests).  A thread owns four neighbouring elements of
// a row and every `groups`-th span; the groups' sums meet in shared memory in ascending order.
// ---------------------------------------------------------------------------------------------
#define A4_MERGE_THREADS 512
#define A4_MAX_SPLITS 256
#define A4_MAX_FLOATS (1LL << 26)      // of scratch for partial sums (256 MB): spans are made longer until they fit
#define A4_START 1.5
#define A4_MEET 0.5
#define A4_MERGE 1.3
template <int NG, int RB, bool F32>
__global__ void __launch_bounds__(A4_MERGE_THREADS)
k_kv4_merge(A4Args a) {
    xr_pdl_launch();
    constexpr int HS = NG * 32, QUADS = HS / 4, TK = A4Tile<NG>::KEYS;
    __shared__ float wgt[RB][A4_MAX_SPLITS];
    __shared__ float row_max[RB], row_sum[RB];
    __shared__ float4 part[A4_MERGE_THREADS];
    const int seg = blockIdx.y, kvh = blockIdx.x / a.row_blocks, rb = blockIdx.x - kvh * a.row_blocks;
    xr_pdl_wait();
    const int L = a.seg_len[seg];
    const long long rows_all = (long long)L * a.G;
    if (L < 1 || rows_all > a.most_rows || (long long)rb * RB >= rows_all) return;
    const int row0 = rb * RB, rows = (int)min((long long)RB, rows_all - row0), pos0 = a.seg_pos0[seg];
    const int n_spans = a4_spans(a, a4_walk(pos0 + row0 / a.G, pos0 + (row0 + rows - 1) / a.G, a.window, a.keep, TK));
    if (n_spans == 1) return;                                        // (written already)
    const int place = a4_place(a, seg, rb, RB);
    if ((unsigned)place >= (unsigned)a.blocks) return;
    const size_t item = ((size_t)place * a.c.K + kvh) * a.splits;
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + item * RB;
    const float4* acc = reinterpret_cast<const float4*>(a.part_acc) + item * RB * QUADS;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int r = warp; r < rows; r += A4_MERGE_THREADS / 32) {
        float mm = -INFINITY;
        for (int s = lane; s < n_spans; s += 32) mm = fmaxf(mm, __ldcg(&ml[(size_t)s * RB + r]).x);
        mm = xr_warp_max(mm);
        const float at = mm == -INFINITY ? 0.f : mm;
        float sum = 0.f;
        for (int s = lane; s < n_spans; s += 32) {
            const float2 x = __ldcg(&ml[(size_t)s * RB + r]);
            const float k = a4_exp2(x.x - at);
            wgt[r][s] = k;
            sum += x.y * k;
        }
        sum = xr_warp_sum(sum);
        if (lane == 0) { row_max[r] = at; row_sum[r] = sum; }
    }
    __syncthreads();
    for (int q0 = 0; q0 < rows * QUADS; q0 += A4_MERGE_THREADS) {
        const int owned = min(A4_MERGE_THREADS, rows * QUADS - q0), groups = A4_MERGE_THREADS / owned;
        const int grp = threadIdx.x / owned, e = q0 + threadIdx.x % owned, r = e / QUADS;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (grp < groups) {
#pragma unroll 4
            for (int s = grp; s < n_spans; s += groups) {
                const float4 u = __ldcg(acc + (size_t)s * RB * QUADS + e);
                const float k = wgt[r][s];
                v.x += u.x * k; v.y += u.y * k; v.z += u.z * k; v.w += u.w * k;
            }
        }
        __syncthreads();
        part[threadIdx.x] = v;
        __syncthreads();
        if (threadIdx.x < owned) {
            for (int k = 1; k < groups; k++) {
                const float4 u = part[k * owned + threadIdx.x];
                v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
            }
            a4_out<F32>(a, a.seg_start[seg], kvh, row0 + r, (e % QUADS) * 4, v, row_max[r], row_sum[r]);
        }
    }
}

// ---------------------------------------------------------------------------------------------
// Blocks that are resident at once, and a row block's size, for a head size and type.  wide_rows: some request has more than eight packed rows.
static int a4_rows(int f32, int wide_rows) { return f32 || !wide_rows ? 8 : 16; }
template <int NG> static int a4_blocks(int f32, int wide_rows) {
    return f32 ? A4Shape<NG, 1, true, false>::BLOCKS : wide_rows ? A4Shape<NG, 2, false, false>::BLOCKS : A4Shape<NG, 1, false, false>::BLOCKS;
}
static int a4_resident(int hs, int f32, int wide_rows) {
    return (hs == 64 ? a4_blocks<2>(f32, wide_rows) : hs == 128 ? a4_blocks<4>(f32, wide_rows) : a4_blocks<8>(f32, wide_rows)) * xr_sm_count();
}
static int a4_tile(int hs) { return hs <= 128 ? 64 : 32; }

// How a step is cut: row blocks of the longest portion that is taken (at most `most_rows` packed rows), tiles a span, spans of the longest
// request.  len, pos0: the portions on the HOST; max_kv: how far requests may get by the time the launch runs (0: as far as they say).  A captured launch is cut for
// the lengths that it may meet: all portions as far on as brings the furthest to max_kv.  (Cut for the lengths at capture, 64 requests of 200 keys ran
// up to 1,024 keys in four spans and a second kernel, where one span is planned for 1,024.)  Beyond the grid's spans the last one takes the rest.
struct A4Plan { int row_blocks, wide, span_tiles, splits, clustered, blocks; };
static A4Plan a4_plan(const int* len, const int* pos0, int n_seg, int K, int G, int hs, int f32, int window, int keep, int most_rows, int max_kv) {
    const int tile = a4_tile(hs);
    long long rows = 0;
    for (int s = 0; s < n_seg; s++) {
        const long long r = (long long)len[s] * G;
        if (r <= most_rows && r > rows) rows = r;
    }
    A4Plan p{0, rows > 8, A4_WARPS, 1, 0, n_seg};
    if (rows < 1) return p;
    const int rb = a4_rows(f32, p.wide);
    p.row_blocks = (int)((rows + rb - 1) / rb);
    const long long resident = a4_resident(hs, f32, p.wide);
    auto taken = [&](int s) { return len[s] >= 1 && (long long)len[s] * G <= most_rows; };
    int ahead = 0;
    if (max_kv > 0) {
        int furthest = 0;
        for (int s = 0; s < n_seg; s++)
            if (taken(s) && pos0[s] + len[s] > furthest) furthest = pos0[s] + len[s];
        ahead = max_kv > furthest ? max_kv - furthest : 0;
    }
    auto tiles_of = [&](int s) {                                     // (of the last row block, whose window is the furthest)
        const int end = pos0[s] + len[s] + ahead, lo = window > 0 ? (end - len[s] - window + 1 > 0 ? end - len[s] - window + 1 : 0) : 0;
        // (a window that moves begins inside a tile nearly always)
        const int seen = max_kv > 0 && lo > 0 ? (int)((end - (long long)lo + tile - 2) / tile) + 1 : (end - 1) / tile - lo / tile + 1;
        return seen + xr_kept_tiles(keep, lo, tile);
    };
    int longest = 1;
    for (int s = 0; s < n_seg; s++)
        if (taken(s)) { const int t = tiles_of(s); longest = t > longest ? t : longest; }
    // blocks by the tiles that they would have whole, in at most 32 classes (each taken for its upper end)
    constexpr int CLASSES = 32;
    long long of[CLASSES] = {};
    double tiles = 0.0;
    for (int s = 0; s < n_seg; s++)
        if (taken(s)) {
            const int t = tiles_of(s);
            const long long blocks = K * (((long long)len[s] * G + rb - 1) / rb);
            of[((long long)t * CLASSES - 1) / longest] += blocks;
            tiles += (double)blocks * t;
        }
    // Tiles a warp of a span takes: the number whose last block is done first, in the time of a tile (a warp's, all others at work).  Up to `resident` blocks
    // run at once; blocks of one length go in rounds, blocks of many lengths as slots fall free, half a block of which is idle at the end.  A block
    // costs A4_START beside its tiles (its first tiles are on their way), combining spans A4_MEET inside a cluster and A4_MERGE in a kernel of its own.
    const int most = (longest + A4_WARPS - 1) / A4_WARPS, least = (longest + A4_MAX_SPLITS * A4_WARPS - 1) / (A4_MAX_SPLITS * A4_WARPS);
    int best = most;
    double best_cost = -1.0;
    for (int n = most; n >= least && n >= 1; n = n > 48 ? n - n / 24 : n - 1) {
        const int span = n * A4_WARPS;
        long long blocks = 0;
        for (int c = 0; c < CLASSES; c++)
            if (of[c]) blocks += of[c] * (((long long)(c + 1) * longest / CLASSES + span - 1) / span);
        const int splits = (longest + span - 1) / span;
        const double work = tiles / A4_WARPS + A4_START * blocks;
        const bool alike = tiles > 0.85 * (double)blocks * span;
        double cost = blocks <= resident ? n + A4_START : alike ? (double)((blocks + resident - 1) / resident) * (n + A4_START) : work / resident + 0.5 * (n + A4_START);
        const bool meet = splits <= A4_CLUSTER && blocks + 8LL * (splits - 1) <= resident;
        if (splits > 1) cost += meet ? A4_MEET : A4_MERGE;
        if (best_cost < 0.0 || cost < best_cost) { best_cost = cost; best = n; p.clustered = splits > 1 && meet; }
        if (work / resident > 1.5 * best_cost) break;
    }
    p.span_tiles = best * A4_WARPS;
    p.splits = (longest + p.span_tiles - 1) / p.span_tiles;
    if (p.row_blocks > 1) {
        p.blocks = 0;
        for (int s = 0; s < n_seg; s++)
            if (taken(s)) p.blocks += (int)(((long long)len[s] * G + rb - 1) / rb);
    }
    const long long span_floats = (long long)p.blocks * K * rb * (hs + 2);
    if (p.splits > 1 && !p.clustered && p.splits * span_floats > A4_MAX_FLOATS) {
        // (many row blocks beside a long request: nearly all of them are one span, but each has room for as many as the longest)
        const long long most_spans = A4_MAX_FLOATS / span_floats > 1 ? A4_MAX_FLOATS / span_floats : 1;
        p.span_tiles = (int)((longest + most_spans * A4_WARPS - 1) / (most_spans * A4_WARPS)) * A4_WARPS;
        p.splits = (longest + p.span_tiles - 1) / p.span_tiles;
    }
    return p;
}

template <int NG, int NT, bool F32, bool EXTRA>
static int a4_launch(const A4Args& a, int n_seg, cudaStream_t stream) {
    using S = A4Shape<NG, NT, F32, EXTRA>;
    static_assert((A4_WARPS * S::RB * (S::HS + 2) + 2 * S::RB) * 4 <= A4_WARPS * S::STAGES * S::STAGE, "the warps' sums lie in the ring");
    static bool ready[XR_DEVICES];
    if (!xr_once_per_device(ready, [] { return xr_allow_smem(k_kv4_attention<NG, NT, F32, EXTRA>, S::SMEM); })) return XR_ERR_LAUNCH;
    const dim3 grid(a.splits * a.row_blocks, a.c.K, n_seg);          // (a cluster is a row block's spans)
    if (a.clustered) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = grid; cfg.blockDim = dim3(A4_THREADS); cfg.dynamicSmemBytes = S::SMEM; cfg.stream = stream;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = a.splits; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = xr_pdl_enabled() ? 2 : 1;
        cudaLaunchKernelEx(&cfg, k_kv4_attention<NG, NT, F32, EXTRA>, a);
        return xr_launch_status();
    }
    xr_launch((k_kv4_attention<NG, NT, F32, EXTRA>), grid, dim3(A4_THREADS), S::SMEM, stream, a);
    if (xr_launch_status() != XR_OK) return XR_ERR_LAUNCH;
    if (a.splits > 1) xr_launch((k_kv4_merge<NG, S::RB, F32>), dim3(a.c.K * a.row_blocks, n_seg), dim3(A4_MERGE_THREADS), 0, stream, a);
    return xr_launch_status();
}
template <int NG, int NT, bool F32>
static int a4_launch(const A4Args& a, int n_seg, cudaStream_t stream) {
    return a.softcap > 0.f || a.bias.table != nullptr ? a4_launch<NG, NT, F32, true>(a, n_seg, stream) : a4_launch<NG, NT, F32, false>(a, n_seg, stream);
}
template <int NG>
static int a4_launch(const A4Args& a, int n_seg, int f32, int wide, cudaStream_t stream) {
    return f32 ? a4_launch<NG, 1, true>(a, n_seg, stream) : wide ? a4_launch<NG, 2, false>(a, n_seg, stream) : a4_launch<NG, 1, false>(a, n_seg, stream);
}

// Whether a step's longer portions go by the codes or through the prompt kernels.  By the codes every 16 rows of a kv head are a row block that walks
// the keys for itself: time follows the number of blocks, 0.045 to 0.051 ns a key and block once the SMs are busy.  The prompt kernels read the rows back once and
// walk the keys once for 128 rows: 11.4 ns a key while tiles are fewer than SMs, 22 where a tile is part full and the mask is asked for every
// score.  So the border is a number of row blocks, one for full tiles and one for others.  32 heads on 8 of 128 elements, codes / prompt kernels in us:
// full tiles, 256 blocks: 20.5 / 21.8 (2 requests, 1,000 keys), 100.7 / 101.0 (2, 8,192), 101.0 / 116.3 (4, 8,192); 320: 33.5 / 22.5, 144.4 / 94.3 (1 request);
// part full, 384 blocks: 35.3 / 33.3 (4, 1,000), 160.2 / 207.9 (4, 8,192), 36.5 / 35.9 (8, 1,000); 400: 37.5 / 31.4 (2, 1,000), 37.9 / 29.7 (1, 1,000), but
// 163.8 / 183.2 (1, 8,192).  Of 64 elements a block is cheaper: full tiles, 320: 84.4 / 90.6 (1, 8,192), 22.2 / 20.8 (1, 1,000), 384: 92.5 / 90.5, 23.6 / 20.8; part
// full, 448: 62.5 / 97.8, 640: 91.1 / 98.3 (4, 4,096).  Near the borders the wrong side is at most 1.18 times slower.  The rule asks nothing of positions, so
// that a replayed graph may have others.
static bool a4_by_codes(long long row_blocks, bool full, int hs) { return row_blocks <= (hs == 64 ? (full ? 320 : 576) : (full ? 256 : 384)); }

// What a step's portions ask for, from their lengths and first positions on the HOST: said[0] portions that attend to the codes, [1] ones that go through the
// prompt kernels (of more than `most_rows` packed rows, all or none of them: a4_by_codes), [2] float32 values of scratch that xr_kv4_attention needs
// for the first; of the others [3] the pages that xr_kv4_read writes for them, [4] the most tokens, [5], [6] the row tiles of 128 and 64 packed rows, [7] the
// furthest end; [8] the most packed rows of a portion that attends to the codes; [9] .. [14] how those are cut, as xr_kv4_attention takes it.
// n: tokens of the step; max_kv: how far requests may get by the time the launches run (0: as far as the portions go); rule: whether a4_by_codes is asked, or
// most_rows stands as it is (some portions of a step whose rule has been asked).
XR_EXPORT int xr_kv4_plan(const int* len, const int* pos0, int n_seg, int n, int K, int G, int D, int page_size, int dtype, int window, int keep_first,
                          int most_rows, int max_kv, int rule, long long* said) {
    if (n_seg < 1 || n < 0 || K < 1 || G < 1 || D < 1 || D > 256 || page_size < 1 || window < 0 || keep_first < 0 || most_rows < 0 || max_kv < 0) return XR_ERR_ARG;
    long long tokens = 0, row_blocks = 0;
    bool full = true;
    for (int i = 0; i < 15; i++) said[i] = 0;
    for (int s = 0; s < n_seg; s++) {
        const long long l = len[s], p = pos0[s], rows = l * G;
        if (l < 0 || p < 0 || p + l > 0x7fffffffLL) return XR_ERR_ARG;
        tokens += l;
        if (rows > most_rows) { row_blocks += (rows + 15) / 16 * K; full = full && rows % 128 == 0; }
    }
    if (tokens > n) return XR_ERR_ARG;
    if (rule && row_blocks > 0 && a4_by_codes(row_blocks, full, kv4_held(D))) most_rows = 1 << 30;
    said[8] = most_rows;
    for (int s = 0; s < n_seg; s++) {
        const long long l = len[s], p = pos0[s], rows = l * G;
        if (l == 0) continue;
        if (rows <= most_rows) { said[0]++; continue; }
        said[1]++;
        const long long first = window > 0 && p - window + 1 > 0 ? p - window + 1 : 0, from = first / page_size, end = p + l > max_kv ? p + l : max_kv;
        const long long kept = ((long long)keep_first + page_size - 1) / page_size, all = (end - 1) / page_size + 1;
        // (with max_kv the portion may lie anywhere up to there: a window's rows touch one page more where they begin inside one)
        const long long seen = window > 0 ? kept + ((long long)window + l - 2) / page_size + 2 : all;
        if (max_kv > 0) said[3] += seen < all ? seen : all;
        else said[3] += (window > 0 ? (kept < from ? kept : from) : 0) + (p + l - 1) / page_size - from + 1;
        if (l > said[4]) said[4] = l;
        said[5] += (rows + 127) / 128;
        said[6] += (rows + 63) / 64;
        if (end > said[7]) said[7] = end;
    }
    if (said[0] > 0) {
        const int hs = kv4_held(D), f32 = dtype == XR_F32;
        const A4Plan p = a4_plan(len, pos0, n_seg, K, G, hs, f32, window, xr_keep(window, keep_first), most_rows, max_kv);
        said[9] = p.row_blocks; said[10] = p.wide; said[11] = p.span_tiles; said[12] = p.splits; said[13] = p.clustered; said[14] = p.blocks;
        if (p.splits > 1 && !p.clustered) said[2] = (long long)p.blocks * K * p.splits * a4_rows(f32, p.wide) * (hs + 2);
    }
    return XR_OK;
}

// q: token t, head h at q + t * q_stride + h * D; out [n][H * D], both of `dtype`.  Portions of at most `most_rows` packed rows (tokens x heads per
// kv head) are computed, longer ones passed over.  row_blocks, wide, span_tiles, splits, clustered, blocks: xr_kv4_plan's answer for the portions' lengths on the
// host (they cut the work; what is computed goes by seg_len and seg_pos0 on the device, of at most row_blocks row blocks).  early: nothing that is still
// running writes the portions, the block tables or rows before a portion's first.
XR_EXPORT int xr_kv4_attention(const void* q, void* out, int dtype, const void* cache, long long n_pages, int layers, int layer, int K, int block, int page_size,
                               const int* seg_start, const int* seg_len, const int* seg_pos0, const int* block_tables, float* scratch, long long floats,
                               long long q_stride, int n_seg, int H, int D, int max_pages, int window, float scale, const float* sink, float softcap,
                               int keep_first, const float* bias, int bias_len, int most_rows, int early, int row_blocks, int wide, int span_tiles,
                               int splits, int clustered, int blocks, cudaStream_t stream) {
    if (n_seg < 1 || n_seg > 65535 || H < 1 || K < 1 || H % K != 0 || max_pages < 1 || window < 0 || keep_first < 0 || !(scale > 0.f) || !(softcap >= 0.f) ||
        (bias != nullptr && (bias_len < 1 || softcap > 0.f)) || most_rows < 1 || q_stride < (long long)H * D || (dtype != XR_F32 && dtype != XR_BF16) ||
        !kv4_cache_ok(cache, n_pages, layers, layer, K, block, page_size, D) || (long long)max_pages * page_size > 0x7fffffffLL - 64 || row_blocks < 1 ||
        span_tiles < 1 || blocks < 1 || splits < 1 || splits > A4_MAX_SPLITS || (clustered && splits > A4_CLUSTER) || (long long)splits * row_blocks > 0x7fffffffLL || (long long)K * row_blocks > 0x7fffffffLL)
        return XR_ERR_ARG;
    const int G = H / K, f32 = dtype == XR_F32, hs = kv4_held(D), keep = xr_keep(window, keep_first);
    const bool spans = splits > 1 && !clustered;
    const long long items = spans ? (long long)blocks * K * splits : 0, rb = a4_rows(f32, wide);
    if (spans && (scratch == nullptr || ((uintptr_t)scratch & 15) || floats < items * rb * (hs + 2))) return XR_ERR_ARG;
    A4Args a{q, out, kv4_cache(cache, n_pages, layers, layer, K, page_size, D), seg_start, seg_len, seg_pos0, block_tables, scratch,
             spans ? scratch + items * rb * hs : nullptr, blocks, q_stride, H, G, D, max_pages, window, keep, splits, span_tiles, row_blocks, most_rows,
             scale, softcap, sink, {bias, bias_len}, 0, 0, early, clustered && splits > 1, -1};
    const int lot = f32 ? 4 : 8;                                     // elements of 16 bytes
    a.wide = D % 8 == 0 && q_stride % lot == 0 && !((uintptr_t)q & 15);
    a.wide_out = D % 4 == 0 && !((uintptr_t)out & 15);
    const int tile = a4_tile(hs);
    if (page_size % tile == 0 && ((page_size / tile) & (page_size / tile - 1)) == 0)
        for (a.tile_shift = 0; (tile << a.tile_shift) < page_size;) a.tile_shift++;
    return hs == 64 ? a4_launch<2>(a, n_seg, f32, wide, stream) : hs == 128 ? a4_launch<4>(a, n_seg, f32, wide, stream) : a4_launch<8>(a, n_seg, f32, wide, stream);
}
