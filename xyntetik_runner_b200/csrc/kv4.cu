// Writing rows of keys and values into a cache in four bits, and reading them back (the layout and its numbers: kv4.cuh).
// The reference's counterpart is its cache in eight bits (`--kv q8_0`; k_store_kv, src/kernels.cu:2008-2022).
#include "kv4.cuh"
#include <math.h>

// ---------------------------------------------------------------------------------------------
// store: rows k [n][K][D] and v [n][K][Vd] (strided by rows) -> the token's page.
//
// A thread owns one word: eight neighbouring elements, 16 (bfloat16) or 32 bytes read and 4 written.  A group is four neighbouring threads;
// its largest and smallest element meet by two shuffles.  Its elements are asked for ahead of its token's page, so that a step of a few tokens waits for one
// chain of loads.  2,048 tokens of 8 heads of 128 elements: 5.4 us (8.4 MB read, 2.4 written: 1.65 us at the copy peak; about 100 instructions a
// word are 1.5), 8 tokens 1.5 us, a launch.
// ---------------------------------------------------------------------------------------------
struct Kv4StoreArgs {
    const void* k; const void* v;
    long long k_stride, v_stride;        // elements between rows
    const int* positions; const int* tok_seg; const int* block_tables;
    Kv4Cache c;
    int n, D, Vd, n_seg, max_pages;
    int wide;                            // rows, heads and addresses allow 16-byte loads
    int word_shift;                      // log2 of the words of a held head
};

// A maximum and a minimum that keep a NaN.
__device__ __forceinline__ float kv4_max(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float kv4_min(float a, float b) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }

// s of a group from its largest and smallest element (kv4.cuh)
__device__ __forceinline__ float kv4_scale_of(float hi, float lo) {
    const float e = hi >= -lo ? hi : lo;
    const float size = fabsf(e);
    if (!(size < 1.329227995784916e36f)) return __int_as_float(0x7fc00000);       // 2^120
    if (size < 1.262177448353619e-29f) return 0.f;                                 // 2^-96
    int b = __float_as_int(e);
    b = (b + 0x3ffff + ((b >> 19) & 1)) & ~0x7ffff;
    return -0.125f * __int_as_float(b);
}

// Eight elements in two steps, so that a thread's loads are all on their way before the first is used.
template <typename T> struct Kv4Row8;
template <> struct Kv4Row8<__nv_bfloat16> {
    uint4 r;
    __device__ __forceinline__ void load(const __nv_bfloat16* src, int live, bool wide) {
        r = make_uint4(0, 0, 0, 0);
        if (wide) { if (live > 0) r = *reinterpret_cast<const uint4*>(src); return; }
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < live) w[i >> 1] |= (uint32_t)reinterpret_cast<const unsigned short*>(src)[i] << (16 * (i & 1));
        r = make_uint4(w[0], w[1], w[2], w[3]);
    }
    __device__ __forceinline__ void get(float* x) const {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; i++) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    }
};
template <> struct Kv4Row8<float> {
    float4 p, q;
    __device__ __forceinline__ void load(const float* src, int live, bool wide) {
        p = q = make_float4(0.f, 0.f, 0.f, 0.f);
        if (wide) {                                        // (a head ends with a whole or half a word)
            if (live > 0) p = reinterpret_cast<const float4*>(src)[0];
            if (live > 4) q = reinterpret_cast<const float4*>(src)[1];
            return;
        }
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = i < live ? src[i] : 0.f;
        p = make_float4(x[0], x[1], x[2], x[3]); q = make_float4(x[4], x[5], x[6], x[7]);
    }
    __device__ __forceinline__ void get(float* x) const { x[0] = p.x; x[1] = p.y; x[2] = p.z; x[3] = p.w; x[4] = q.x; x[5] = q.y; x[6] = q.z; x[7] = q.w; }
};

// The word of eight elements with scale s (finite, not zero).  The codes hang on x / s rounded to the nearest whole number, and quotients of exactly n + 1/2 are
// common (x has eight bits, s five), so the quotient has to be the correctly rounded one: r the correctly rounded 1 / s, q = x r, and q + (x - q s) r
// with fused operations is it (Markstein, IBM J. Res. Dev. 34, 1990).  Codes come out of the low bits of 1.5 2^23 + 8 + c; the constant's bits, shifted
// and added up like the codes', are taken off at the end.
__device__ __forceinline__ uint32_t kv4_word(const float* x, float s) {
    const float r = __frcp_rn(s);
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float q = x[i] * r, c = fmaf(fmaf(-q, s, x[i]), r, q);
        word += __float_as_uint(fminf(fmaxf(c, -8.f), 7.f) + 12582920.f) << (4 * (i >> 1) + 16 * (i & 1));
    }
    return word - 0x4B400000u * 0x11111111u;
}

// grid (tokens, 256 words of a token)
template <typename T>
__global__ void __launch_bounds__(256)
k_kv4_store(Kv4StoreArgs a) {
    xr_pdl_launch();
    const int words = 1 << a.word_shift, per = 2 * a.c.K << a.word_shift;       // words of a head; of a token
    const int u = blockIdx.y * 256 + threadIdx.x, t = blockIdx.x;
    // (groups are whole: a token's words are a multiple of four)
    const bool live = u < per;
    const int w = u & (words - 1), r = u >> a.word_shift, plane = r >= a.c.K, kvh = r - (plane ? a.c.K : 0), D = plane ? a.Vd : a.D;
    const T* src = plane ? (const T*)a.v + (long long)t * a.v_stride + (long long)kvh * D + 8 * w : (const T*)a.k + (long long)t * a.k_stride + (long long)kvh * D + 8 * w;
    xr_pdl_wait();
    Kv4Row8<T> row;
    row.load(src, live ? min(8, max(0, D - 8 * w)) : 0, a.wide);
    const int pos = a.positions[t], seg = a.tok_seg[t];
    const int pi = pos / a.c.page_size, tok = pos - pi * a.c.page_size;
    int page = -1;
    if (pos >= 0 && seg >= 0 && seg < a.n_seg && pi < a.max_pages) page = a.block_tables[(size_t)seg * a.max_pages + pi];
    float x[8];
    row.get(x);
    float hi = x[0], lo = x[0];
#pragma unroll
    for (int i = 1; i < 8; i++) { hi = kv4_max(hi, x[i]); lo = kv4_min(lo, x[i]); }
#pragma unroll
    for (int o = 1; o <= 2; o <<= 1) {
        hi = kv4_max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        lo = kv4_min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    }
    if (!live || page < 0 || page >= a.c.n_pages) return;  // (a token whose page is not held is not written)
    const float s = kv4_scale_of(hi, lo);
    const uint32_t word = s != 0.f && s == s ? kv4_word(x, s) : 0x88888888u;       // (c = 0 everywhere)
    uint8_t* run = const_cast<uint8_t*>(a.c.run(page, kvh));
    reinterpret_cast<uint32_t*>(run + a.c.codes_at(plane))[(tok << a.word_shift) + w] = word;
    if ((w & 3) == 0) reinterpret_cast<__nv_bfloat16*>(run + a.c.scales_at(plane))[((tok << a.word_shift) + w) >> 2] = __float2bfloat16_rn(s);
}

XR_EXPORT int xr_kv4_store(const void* k, const void* v, int dtype, long long k_stride, long long v_stride, const int* positions, const int* tok_seg,
                           const int* block_tables, void* cache, long long n_pages, int layers, int layer, int K, int block, int page_size, int n, int D,
                           int Vd, int n_seg, int max_pages, cudaStream_t stream) {
    if (n < 1 || Vd < 1 || Vd > 256 || n_seg < 1 || max_pages < 1 || K > 16384 || k_stride < (long long)K * D || v_stride < (long long)K * Vd ||
        !kv4_cache_ok(cache, n_pages, layers, layer, K, block, page_size, D > Vd ? D : Vd) || D < 1)
        return XR_ERR_ARG;
    Kv4StoreArgs a{k, v, k_stride, v_stride, positions, tok_seg, block_tables, kv4_cache(cache, n_pages, layers, layer, K, page_size, D > Vd ? D : Vd),
                   n, D, Vd, n_seg, max_pages, 0};
    const int even = dtype == XR_F32 ? 4 : 8;              // elements of 16 bytes
    a.wide = !(((uintptr_t)k | (uintptr_t)v) & 15) && D % even == 0 && Vd % even == 0 && k_stride % even == 0 && v_stride % even == 0;
    a.word_shift = a.c.hs == 64 ? 3 : a.c.hs == 128 ? 4 : 5;
    const dim3 grid(n, (unsigned)(((2LL * K << a.word_shift) + 255) / 256));
    if (dtype == XR_F32) xr_launch((k_kv4_store<float>), grid, dim3(256), 0, stream, a);
    else if (dtype == XR_BF16) xr_launch((k_kv4_store<__nv_bfloat16>), grid, dim3(256), 0, stream, a);
    else return XR_ERR_ARG;
    return xr_launch_status();
}

// ---------------------------------------------------------------------------------------------
// read: the rows first .. end - 1 of every request (and its first `keep` rows, where they lie before them) as values, in pages
// [page of the output][keys, values][kv head][token][D]: the requests one after another, the kept rows' pages of a request first.
// Rows of those pages that are not asked for are zeros, and so are rows whose page is not held.  tables (optional) [n_seg][max_pages]: where
// a request's pages lie in the output (-1: not there), a block table for kernels that read values from pages.
//
// A block takes one page of the output and some of its kv heads and finds its request by adding up the requests' pages, 32 at a time; a thread owns words,
// four bytes read and 16 (bfloat16) or 32 written, eight of them side by side.  Bound by the writes: 4 requests of 8,192 rows (134 MB out, 38 in) 35.7 us, 0.74
// of the copy peak; 2,048 rows 4.6 us; 8 pages 2.6 us.
// ---------------------------------------------------------------------------------------------
struct Kv4ReadArgs {
    Kv4Cache c;
    const int* first; const int* end; const int* block_tables;
    void* out;
    int* tables;
    int n_seg, max_pages, D, keep, out_pages;
    int wide;
};

// pages of the output that a request takes: kept ones, then those of first .. end - 1
__device__ __forceinline__ void kv4_pages_of(const Kv4ReadArgs& a, int seg, int& kept, int& from, int& count) {
    const int P = a.c.page_size, f = max(0, a.first[seg]), e = (int)min((long long)a.end[seg], (long long)a.max_pages * P);
    from = f / P;
    kept = f < e ? min((int)(((unsigned)a.keep + P - 1) / P), from) : 0;
    count = f < e ? (e - 1) / P - from + 1 : 0;
}

__device__ __forceinline__ void kv4_values(uint32_t word, uint32_t s, uint32_t* v) {
    const uint32_t s2 = s * 0x10001u, m = kv4_m24(s2);
    v[0] = kv4_scaled(kv4_pair<0>(word), s2, m); v[1] = kv4_scaled(kv4_pair<1>(word), s2, m);
    v[2] = kv4_scaled(kv4_pair<2>(word), s2, m); v[3] = kv4_scaled(kv4_pair<3>(word), s2, m);
}
// A word's eight values to a 16-byte border.
template <typename T>
__device__ __forceinline__ void kv4_eight(uint32_t word, uint32_t s, T* to) {
    uint32_t v[4];
    kv4_values(word, s, v);
    if constexpr (sizeof(T) == 2) *reinterpret_cast<uint4*>(to) = make_uint4(v[0], v[1], v[2], v[3]);
    else {
        reinterpret_cast<uint4*>(to)[0] = make_uint4(v[0] << 16, v[0] & 0xffff0000u, v[1] << 16, v[1] & 0xffff0000u);
        reinterpret_cast<uint4*>(to)[1] = make_uint4(v[2] << 16, v[2] & 0xffff0000u, v[3] << 16, v[3] & 0xffff0000u);
    }
}

// WS: log2 of a held head's words where a head is held as it is (D is 8 << WS, on 16-byte borders); 0: any head.
template <typename T, int WS>
__global__ void __launch_bounds__(256)
k_kv4_read(Kv4ReadArgs a) {
    __shared__ int found[2];
    xr_pdl_wait();
    // Behind the wait, not ahead of it: the prompt kernels walk the portions' lengths before they wait themselves, and on the route of attention_kv4
    // those lengths are k_kv4_long's.  Nothing behind this kernel starts before that one is complete.
    xr_pdl_launch();
    const int j = blockIdx.x;
    if (threadIdx.x < 32) {
        int before = 0;
        bool done = false;
        for (int s0 = 0; s0 < a.n_seg && !done; s0 += 32) {
            const int seg = s0 + threadIdx.x;
            int kept = 0, from = 0, count = 0;
            if (seg < a.n_seg) kv4_pages_of(a, seg, kept, from, count);
            int sum = kept + count;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const int u = __shfl_up_sync(0xffffffffu, sum, o); if (threadIdx.x >= o) sum += u; }
            const int at = before + sum - kept - count;                  // this request's first page of the output
            const bool mine = seg < a.n_seg && j >= at && j < at + kept + count;
            if (mine) {
                const int i = j - at, pi = i < kept ? i : from + i - kept;
                found[0] = seg; found[1] = pi;
                if (blockIdx.y == 0 && a.tables != nullptr) a.tables[(size_t)seg * a.max_pages + pi] = j;
            }
            done = __ballot_sync(0xffffffffu, mine) != 0;
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (!done && threadIdx.x == 0) found[0] = -1;
    }
    __syncthreads();
    const int seg = found[0];
    if (seg < 0) return;                                                 // (more pages of output than the requests take: left as they were)
    const int pi = found[1], P = a.c.page_size, first = max(0, a.first[seg]), end = a.end[seg];
    int page = a.block_tables[(size_t)seg * a.max_pages + pi];
    if (page >= a.c.n_pages) page = -1;
    const int words = a.c.hs >> 3, used = (a.D + 7) >> 3, p0 = pi * P;
    const size_t plane_step = (size_t)a.c.K * P * a.D;
    // what of the page is asked for: tokens a0 .. a1 - 1, and the first `kept`
    const int a0 = max(first - p0, 0), a1 = page >= 0 ? min(end - p0, P) : 0, kept = page >= 0 ? min(a.keep - p0, a1) : 0;
    for (int kvh = blockIdx.y; kvh < a.c.K; kvh += gridDim.y) {
        const uint8_t* run = a.c.run(max(page, 0), kvh);
        T* dst = (T*)a.out + ((size_t)j * 2 * a.c.K + kvh) * P * a.D;
        if constexpr (WS > 0) {
            // four words of the keys and four of the values a thread, their loads side by side
            constexpr int N = 4;
            for (int i0 = threadIdx.x; i0 < P << WS; i0 += N * 256) {
                uint32_t word[2][N], s[2][N];
#pragma unroll
                for (int plane = 0; plane < 2; plane++)
#pragma unroll
                    for (int e = 0; e < N; e++) {
                        const int i = i0 + e * 256, tok = i >> WS;
                        word[plane][e] = s[plane][e] = 0;
                        if (tok < a1 && (tok >= a0 || tok < kept)) {
                            word[plane][e] = __ldcs(reinterpret_cast<const uint32_t*>(run + a.c.codes_at(plane)) + i);
                            s[plane][e] = __ldg(reinterpret_cast<const unsigned short*>(run + a.c.scales_at(plane)) + (i >> 2));
                        }
                    }
#pragma unroll
                for (int plane = 0; plane < 2; plane++)
#pragma unroll
                    for (int e = 0; e < N; e++) {
                        const int i = i0 + e * 256;
                        if (i >= P << WS) break;
                        kv4_eight<T>(word[plane][e], s[plane][e], dst + plane * plane_step + 8 * (size_t)i);
                    }
            }
            continue;
        }
#pragma unroll
        for (int plane = 0; plane < 2; plane++) {
            const uint32_t* codes = reinterpret_cast<const uint32_t*>(run + a.c.codes_at(plane));
            const unsigned short* scales = reinterpret_cast<const unsigned short*>(run + a.c.scales_at(plane));
            T* to = dst + plane * plane_step;
            for (int i = threadIdx.x; i < P * used; i += 256) {
                const int tok = i / used, w = i - tok * used;
                uint32_t word = 0, s = 0;
                if (tok < a1 && (tok >= a0 || tok < kept)) { word = __ldg(codes + tok * words + w); s = __ldg(scales + tok * (words >> 2) + (w >> 2)); }
                if (a.wide && 8 * w + 8 <= a.D) { kv4_eight<T>(word, s, to + (size_t)tok * a.D + 8 * w); continue; }
                uint32_t v[4];
                kv4_values(word, s, v);
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (8 * w + e < a.D) to[(size_t)tok * a.D + 8 * w + e] = xr_from_f32<T>(__uint_as_float(e & 1 ? v[e >> 1] & 0xffff0000u : v[e >> 1] << 16));
            }
        }
    }
}

template <typename T>
static void kv4_launch_read(const Kv4ReadArgs& a, cudaStream_t stream) {
    // A block takes one page and as many of its kv heads as leave six blocks an SM: what a block works out about its page costs more than a head's values.
    const long long want = 6LL * xr_sm_count();
    const int heads = (int)(a.out_pages * (long long)a.c.K / want < 1 ? 1 : a.out_pages * (long long)a.c.K / want > a.c.K ? a.c.K : a.out_pages * (long long)a.c.K / want);
    const dim3 grid(a.out_pages, (a.c.K + heads - 1) / heads);
    const bool whole = a.wide && a.D == a.c.hs;
    if (whole && a.D == 64) xr_launch((k_kv4_read<T, 3>), grid, dim3(256), 0, stream, a);
    else if (whole && a.D == 128) xr_launch((k_kv4_read<T, 4>), grid, dim3(256), 0, stream, a);
    else if (whole) xr_launch((k_kv4_read<T, 5>), grid, dim3(256), 0, stream, a);
    else xr_launch((k_kv4_read<T, 0>), grid, dim3(256), 0, stream, a);
}

XR_EXPORT int xr_kv4_read(const void* cache, long long n_pages, int layers, int layer, int K, int block, int page_size, const int* block_tables,
                          const int* first, const int* end, void* out, int dtype, int* tables, int n_seg, int max_pages, int D, int keep, int out_pages,
                          cudaStream_t stream) {
    if (n_seg < 1 || max_pages < 1 || keep < 0 || out_pages < 1 || !kv4_cache_ok(cache, n_pages, layers, layer, K, block, page_size, D) ||
        (long long)max_pages * page_size > 0x7fffffffLL)
        return XR_ERR_ARG;
    Kv4ReadArgs a{kv4_cache(cache, n_pages, layers, layer, K, page_size, D), first, end, block_tables, out, tables, n_seg, max_pages, D, keep, out_pages, 0};
    a.wide = D % (dtype == XR_F32 ? 4 : 8) == 0 && !((uintptr_t)out & 15);
    if (dtype == XR_F32) kv4_launch_read<float>(a, stream);
    else if (dtype == XR_BF16) kv4_launch_read<__nv_bfloat16>(a, stream);
    else return XR_ERR_ARG;
    return xr_launch_status();
}

// ---------------------------------------------------------------------------------------------
// Which portions of a step go through values that are read back: those of more than `most_rows` packed rows (tokens x query heads per kv
// head).  first, end: the rows such a portion sees (none for the others); long_len: its tokens (0 for the others, which the prompt kernels then
// pass over); tables is filled with -1 for the reader.
// ---------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(256)
k_kv4_long(const int* __restrict__ seg_len, const int* __restrict__ seg_pos0, int* __restrict__ first, int* __restrict__ end, int* __restrict__ long_len,
           int* __restrict__ tables, int n_seg, int max_pages, int G, int window, int most_rows) {
    xr_pdl_launch();
    xr_pdl_wait();
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    int f = 0, e = 0, l = 0;
    if (i < n_seg) {
        l = seg_len[i];
        const int p = seg_pos0[i];
        if ((long long)l * G <= most_rows) l = 0;
        else { f = window > 0 ? max(0, p - window + 1) : 0; e = p + l; }
    }
    if (i < n_seg) { first[i] = f; end[i] = e; long_len[i] = l; }
    if (i < (long long)n_seg * max_pages) tables[i] = -1;
}

XR_EXPORT int xr_kv4_long(const int* seg_len, const int* seg_pos0, int* first, int* end, int* long_len, int* tables, int n_seg, int max_pages, int G,
                          int window, int most_rows, cudaStream_t stream) {
    if (n_seg < 1 || max_pages < 1 || G < 1 || window < 0 || most_rows < 0) return XR_ERR_ARG;
    const long long blocks = ((long long)n_seg * max_pages + 255) / 256;
    if (blocks > 0x7fffffffLL) return XR_ERR_ARG;
    xr_launch(k_kv4_long, dim3((unsigned)blocks), dim3(256), 0, stream, seg_len, seg_pos0, first, end, long_len, tables, n_seg, max_pages, G, window, most_rows);
    return xr_launch_status();
}
