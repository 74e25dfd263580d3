// Writing rows of keys and values into a cache in four bits, and reading them back (the layout and its numbers: kv4.cuh).
// The reference's counterpart is its cache in eight bits (`--kv q8_0`; k_store_kv, src/kernels.cu:2008-2022); the format here is its own.
#include "kv4.cuh"
#include <math.h>

// ---------------------------------------------------------------------------------------------
// store: rows k [n][K][D] and v [n][K][Vd] (strided by rows) -> the token's page.
//
// A thread owns one word: eight neighbouring elements, 16 (bfloat16) or 32 bytes read and 4 written.  A group is four neighbouring threads;
// its largest and smallest element meet by two shuffles.  Bound by memory at many tokens, by the launch at few.
// ---------------------------------------------------------------------------------------------
struct Kv4StoreArgs {
    const void* k; const void* v;
    long long k_stride, v_stride;        // elements between rows
    const int* positions; const int* tok_seg; const int* block_tables;
    Kv4Cache c;
    int n, D, Vd, n_seg, max_pages;
    int wide;                            // rows, heads and addresses allow 16-byte loads
};

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

template <typename T>
__device__ __forceinline__ void kv4_load8(const T* src, int live, bool wide, float* x) {
    if (wide && live == 8) {
        if constexpr (sizeof(T) == 2) {
            const uint4 r = *reinterpret_cast<const uint4*>(src);
            const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
            for (int i = 0; i < 4; i++) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
        } else {
            const float4 a = reinterpret_cast<const float4*>(src)[0], b = reinterpret_cast<const float4*>(src)[1];
            x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = i < live ? xr_to_f32<T>(src[i]) : 0.f;
}

template <typename T>
__global__ void __launch_bounds__(256)
k_kv4_store(Kv4StoreArgs a) {
    xr_pdl_launch();
    xr_pdl_wait();
    const int words = a.c.hs >> 3;
    const long long at = (long long)blockIdx.x * 256 + threadIdx.x, total = (long long)a.n * 2 * a.c.K * words;
    const bool live = at < total;
    // (groups are whole: a head's words are a multiple of four, and so are the threads behind the last one)
    const int w = (int)(at % words);
    const long long head = live ? at / words : 0;
    const int t = (int)(head / (2 * a.c.K)), r = (int)(head % (2 * a.c.K)), plane = r >= a.c.K, kvh = r - plane * a.c.K;
    const int pos = a.positions[t], seg = a.tok_seg[t];
    const int pi = pos / a.c.page_size;
    int page = -1;
    if (live && pos >= 0 && seg >= 0 && seg < a.n_seg && pi < a.max_pages) page = a.block_tables[(size_t)seg * a.max_pages + pi];
    if (page >= a.c.n_pages) page = -1;                    // (a token whose page is not held is not written)
    const int D = plane ? a.Vd : a.D;
    float x[8];
    const T* src = plane ? (const T*)a.v + (long long)t * a.v_stride + (long long)kvh * D + 8 * w : (const T*)a.k + (long long)t * a.k_stride + (long long)kvh * D + 8 * w;
    kv4_load8<T>(src, page >= 0 ? min(8, max(0, D - 8 * w)) : 0, a.wide, x);
    float hi = x[0], lo = x[0];
    bool none = !(fabsf(x[0]) <= 3.402823466e38f);
#pragma unroll
    for (int i = 1; i < 8; i++) { hi = fmaxf(hi, x[i]); lo = fminf(lo, x[i]); none |= !(fabsf(x[i]) <= 3.402823466e38f); }
    // (maximum and minimum pass a NaN over: it is looked for apart, and an infinity with it)
    if (none) hi = INFINITY;
#pragma unroll
    for (int o = 1; o <= 2; o <<= 1) {
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    }
    if (page < 0) return;
    const float s = kv4_scale_of(hi, lo);
    uint32_t word = 0x88888888u;                           // c = 0 everywhere
    if (s != 0.f && s == s) {
        word = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            // a true division: x has eight bits (or 24), s five, and halves between two codes occur; a product with 1 / s may land on their other side
            const int c = (int)fminf(fmaxf(rintf(__fdiv_rn(x[i], s)), -8.f), 7.f);
            word |= (uint32_t)(c + 8) << (4 * (i >> 1) + 16 * (i & 1));
        }
    }
    uint8_t* run = const_cast<uint8_t*>(a.c.run(page, kvh));
    const int tok = pos % a.c.page_size;
    reinterpret_cast<uint32_t*>(run + a.c.codes_at(plane))[(long long)tok * words + w] = word;
    if ((w & 3) == 0) reinterpret_cast<__nv_bfloat16*>(run + a.c.scales_at(plane))[(long long)tok * (words >> 2) + (w >> 2)] = __float2bfloat16_rn(s);
}

XR_EXPORT int xr_kv4_store(const void* k, const void* v, int dtype, long long k_stride, long long v_stride, const int* positions, const int* tok_seg,
                           const int* block_tables, void* cache, long long n_pages, int layers, int layer, int K, int block, int page_size, int n, int D,
                           int Vd, int n_seg, int max_pages, cudaStream_t stream) {
    if (n < 1 || Vd < 1 || Vd > 256 || n_seg < 1 || max_pages < 1 || k_stride < (long long)K * D || v_stride < (long long)K * Vd ||
        !kv4_cache_ok(cache, n_pages, layers, layer, K, block, page_size, D > Vd ? D : Vd) || D < 1)
        return XR_ERR_ARG;
    Kv4StoreArgs a{k, v, k_stride, v_stride, positions, tok_seg, block_tables, kv4_cache(cache, n_pages, layers, layer, K, page_size, D > Vd ? D : Vd),
                   n, D, Vd, n_seg, max_pages, 0};
    a.wide = !(((uintptr_t)k | (uintptr_t)v) & 15) && D % 8 == 0 && Vd % 8 == 0 && k_stride % 8 == 0 && v_stride % 8 == 0;
    const long long blocks = ((long long)n * 2 * K * (a.c.hs >> 3) + 255) / 256;
    if (blocks > 0x7fffffffLL) return XR_ERR_ARG;
    if (dtype == XR_F32) xr_launch((k_kv4_store<float>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
    else if (dtype == XR_BF16) xr_launch((k_kv4_store<__nv_bfloat16>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
    else return XR_ERR_ARG;
    return xr_launch_status();
}

// ---------------------------------------------------------------------------------------------
// read: the rows first .. end - 1 of every request (and its first `keep` rows, where they lie before them) as values, in pages
// [page of the output][keys, values][kv head][token][D]: the requests one after another, the kept rows' pages of a request first.
// Rows of those pages that are not asked for are zeros, and so are rows whose page is not held.  tables (optional) [n_seg][max_pages]: where
// a request's pages lie in the output (-1: not there), a block table for kernels that read values from pages.
//
// A block owns one page and kv head of the output and finds its request by adding up the requests' pages, 32 at a time; a thread owns words,
// four bytes read and 16 (bfloat16) or 32 written.  Bound by the writes.
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
    kept = f < e ? min((a.keep + P - 1) / P, from) : 0;
    count = f < e ? (e - 1) / P - from + 1 : 0;
}

template <typename T>
__global__ void __launch_bounds__(256)
k_kv4_read(Kv4ReadArgs a) {
    xr_pdl_launch();
    __shared__ int found[4];
    xr_pdl_wait();
    const int j = blockIdx.x, kvh = blockIdx.y;
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
            if (mine) { const int i = j - at; found[0] = seg; found[1] = i < kept ? i : from + i - kept; }
            done = __ballot_sync(0xffffffffu, mine) != 0;
            if (kvh == 0 && a.tables != nullptr && mine) a.tables[(size_t)seg * a.max_pages + (j - at < kept ? j - at : from + j - at - kept)] = j;
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (!done && threadIdx.x == 0) found[0] = -1;
    }
    __syncthreads();
    const int seg = found[0];
    if (seg < 0) return;                                                 // (more pages of output than the requests take: left as they were)
    const int pi = found[1], P = a.c.page_size, words = a.c.hs >> 3, used = (a.D + 7) >> 3;
    const int first = a.first[seg], end = a.end[seg];
    int page = a.block_tables[(size_t)seg * a.max_pages + pi];
    if (page >= a.c.n_pages) page = -1;
    const uint8_t* run = a.c.run(max(page, 0), kvh);
    T* dst = (T*)a.out + ((size_t)j * 2 * a.c.K + kvh) * P * a.D;
    const size_t plane_step = (size_t)a.c.K * P * a.D;
    const int per_plane = P * used;
#pragma unroll 4
    for (int i = threadIdx.x; i < 2 * per_plane; i += 256) {
        const int plane = i >= per_plane, u = i - plane * per_plane, tok = u / used, w = u - tok * used;
        const int p = pi * P + tok;
        const bool seen = page >= 0 && p < end && (p >= first || p < a.keep);
        uint32_t word = 0, s = 0;
        if (seen) {
            word = __ldg(reinterpret_cast<const uint32_t*>(run + a.c.codes_at(plane)) + tok * words + w);
            s = __ldg(reinterpret_cast<const unsigned short*>(run + a.c.scales_at(plane)) + tok * (words >> 2) + (w >> 2));
        }
        const uint32_t s2 = s | (s << 16), m = kv4_m24(s2);
        const uint32_t v[4] = {kv4_scaled(kv4_pair<0>(word), s2, m), kv4_scaled(kv4_pair<1>(word), s2, m), kv4_scaled(kv4_pair<2>(word), s2, m),
                               kv4_scaled(kv4_pair<3>(word), s2, m)};
        T* to = dst + plane * plane_step + (size_t)tok * a.D + 8 * w;
        if (a.wide) {
            if constexpr (sizeof(T) == 2) *reinterpret_cast<uint4*>(to) = make_uint4(v[0], v[1], v[2], v[3]);
            else {
                reinterpret_cast<uint4*>(to)[0] = make_uint4(v[0] << 16, v[0] & 0xffff0000u, v[1] << 16, v[1] & 0xffff0000u);
                reinterpret_cast<uint4*>(to)[1] = make_uint4(v[2] << 16, v[2] & 0xffff0000u, v[3] << 16, v[3] & 0xffff0000u);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (8 * w + e < a.D) to[e] = xr_from_f32<T>(__uint_as_float(e & 1 ? v[e >> 1] & 0xffff0000u : v[e >> 1] << 16));
        }
    }
}

XR_EXPORT int xr_kv4_read(const void* cache, long long n_pages, int layers, int layer, int K, int block, int page_size, const int* block_tables,
                          const int* first, const int* end, void* out, int dtype, int* tables, int n_seg, int max_pages, int D, int keep, int out_pages,
                          cudaStream_t stream) {
    if (n_seg < 1 || max_pages < 1 || keep < 0 || out_pages < 1 || !kv4_cache_ok(cache, n_pages, layers, layer, K, block, page_size, D) ||
        (long long)max_pages * page_size > 0x7fffffffLL)
        return XR_ERR_ARG;
    Kv4ReadArgs a{kv4_cache(cache, n_pages, layers, layer, K, page_size, D), first, end, block_tables, out, tables, n_seg, max_pages, D, keep, out_pages, 0};
    a.wide = D % 8 == 0 && !((uintptr_t)out & 15);
    if (dtype == XR_F32) xr_launch((k_kv4_read<float>), dim3(out_pages, K), dim3(256), 0, stream, a);
    else if (dtype == XR_BF16) xr_launch((k_kv4_read<__nv_bfloat16>), dim3(out_pages, K), dim3(256), 0, stream, a);
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
