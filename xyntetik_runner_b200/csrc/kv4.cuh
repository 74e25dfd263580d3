// How a cache in four bits holds keys and values.  (A scale from the signed element of largest magnitude is the idea of the q4_0 format; a scale of five
// bits, which makes every held value a bfloat16, and the bytes' order are this format's own.)
//
// A group is 32 neighbouring elements of one token's head; a head of D elements is held as 64, 128 or 256 of them, zeros behind D.
// With e the group's element of largest magnitude (the positive one of two), s = -e / 8, e rounded to five significant bits (ties
// to even).  An element x is held as c = x / s, rounded to the nearest whole number (ties to even) and brought into -8 .. 7, and stands for
// c s.  e itself becomes -8 s: the side of the largest element has eight steps, the other one seven (mean square error of normal
// values 0.0074 of their square; a scale of e / 7 and codes -7 .. 7 have 0.0094, e / 7.5 0.0089).
//
// c has at most three significant bits (or is -8, a power of two) and s five, so that c s has eight: a bfloat16, EXACTLY.  What the
// attention multiplies, what is read back for the prompt kernels and what a float32 model reads are the same numbers.  No kernel rounds a
// held value but one: the attention of bfloat16 queries has values in float16 units of the largest ones, token by token, and those below 2^-23 of them lose
// bits (attention_kv4.cu).  s has its sign and its exponent: bfloat16 holds it.
//
// Groups whose largest magnitude is below 2^-96 are held as zeros (s = 0), groups with an element of 2^120 or more, or one that is no number,
// as NaN (s = NaN: every value of the group is NaN): between those borders s, c s and 24 s are normal bfloat16 numbers.
//
// Bytes.  A page of one layer and kv head is one run: [codes of the keys | codes of the values | scales of the keys | scales of the
// values], token after token.  Eight codes, plus 8 each, are one little-endian word, element 2i at bit 4i and element 2i + 1 at bit
// 16 + 4i: one shift and one mask bring a PAIR of neighbouring elements into the halves of a register.  A token costs (hs / 2 + hs / 16) x 2 bytes a
// kv head: 144 at 128 elements, where bfloat16 has 512.  Pages of a multiple of eight tokens keep every part of a run, from any
// multiple of eight tokens on, on a 16-byte border, as bulk copies want it.
#pragma once
#include "common.cuh"

struct Kv4Cache {
    const uint8_t* base;         // [pages][layers][kv heads][block]
    long long page_bytes;        // layers * K * block
    long long layer_at;          // layer * K * block
    int n_pages, K, page_size, hs;
    __host__ __device__ int block() const { return page_size * (hs + hs / 8); }
    __host__ __device__ int codes_at(int plane) const { return plane * page_size * (hs / 2); }
    __host__ __device__ int scales_at(int plane) const { return page_size * hs + plane * page_size * (hs / 16); }
    __host__ __device__ const uint8_t* run(long long page, int kvh) const { return base + page * page_bytes + layer_at + (long long)kvh * block(); }
};

static inline int kv4_held(int head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }

// What every entry point asks of a cache.  `layer` of `layers`; block: bytes of one page, layer and kv head.
static inline bool kv4_cache_ok(const void* base, long long n_pages, int layers, int layer, int K, int block, int page_size, int D) {
    if (base == nullptr || ((uintptr_t)base & 15) || n_pages < 1 || n_pages > 0x7fffffffLL || layers < 1 || layer < 0 || layer >= layers || K < 1 ||
        K > 65535 || page_size < 8 || page_size % 8 || page_size > 65536 || D < 1 || D > 256)
        return false;
    return block == page_size * (kv4_held(D) + kv4_held(D) / 8);
}
static inline Kv4Cache kv4_cache(const void* base, long long n_pages, int layers, int layer, int K, int page_size, int D) {
    Kv4Cache c{(const uint8_t*)base, 0, 0, (int)n_pages, K, page_size, kv4_held(D)};
    c.page_bytes = (long long)layers * K * c.block();
    c.layer_at = (long long)layer * K * c.block();
    return c;
}

// The pair of neighbouring codes i (elements 2i and 2i + 1) of a word as bfloat16 numbers 16 + u: u (three bits up) is the top of the
// mantissa of 16.0.
template <int I>
__device__ __forceinline__ uint32_t kv4_pair(uint32_t w) {
    const uint32_t at = I == 0 ? w << 3 : w >> (4 * I - 3);
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(at), "r"(0x00780078u), "r"(0x41804180u));      // (at & mask) | 16.0
    return r;
}
// (16 + u) s - 24 s = c s for both halves; m24s = -24 s.  The fused product and sum rounds once, and c s is a bfloat16: exact.
__device__ __forceinline__ uint32_t kv4_scaled(uint32_t pair, uint32_t s2, uint32_t m24s2) {
    uint32_t r;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(pair), "r"(s2), "r"(m24s2));
    return r;
}
// -24 s for both halves: 24 s has 2 + 5 bits, exact.
__device__ __forceinline__ uint32_t kv4_m24(uint32_t s2) {
    uint32_t r;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(s2), "r"(0xC1C0C1C0u), "r"(0x80008000u));       // -24.0, -0.0
    return r;
}
