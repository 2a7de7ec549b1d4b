// What the attention kernels over the 8-bit cache share: their arguments, which tile a block works on, and conversions.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace {
constexpr int D = HEAD_DIM;
constexpr float LOG2E = 1.4426950408889634f;
constexpr int NO_SCALE = -300;     // stands for log2 of a value scale of zero

struct Kv8Args {
    const unsigned char* k_cache;
    const unsigned char* v_cache;
    const float* k_scale;    // [num_pages, KV]
    const float* v_scale;
    const int* cu_q;         // [n + 1] start of each request's new tokens
    const int* ctx_lens;     // [n] tokens in the cache, the new ones among them
    const int* block_table;  // [n, table_width]
    int n, n_tokens, table_width, page_size, num_pages;
    int page_shift;          // log2(page_size) when it is a power of two, else -1
    long long page_stride;   // bytes from page to page
    long long q_stride;      // entries from token to token
    int H, KV;
    int heads_per_tile;      // query heads of one KV head that a tile handles
    int tokens_per_tile;
    int head_groups;         // tiles that the heads of one KV head make
    float scale;
    int window;              // 0: unlimited
    int min_q, max_q;        // requests of so many new tokens are worked on
    int any_q;               // no request brings more
    int* status;

    __device__ __forceinline__ int page_of(int key) const { return page_shift >= 0 ? key >> page_shift : key / page_size; }
    __device__ __forceinline__ int in_page(int key) const { return page_shift >= 0 ? key & (page_size - 1) : key % page_size; }
    // bytes from the start of its page to a key's row of a KV head (a page may be of more than 2^31)
    __device__ __forceinline__ long long row_in_page(int key, int kvh) const { return ((long long)in_page(key) * KV + kvh) * D; }
};

// A call as the host lays it out in one block of memory (its parts one by one cost the host 2 us more).
struct Kv8Call {
    void* out;                      // [n_tokens, H, D]
    const void* q;                  // [n_tokens, H, D], tokens q_stride entries apart
    const void *k_cache, *v_cache;  // e4m3 codes: pages page_stride bytes apart, each [page_size, KV, D]
    const float *k_scale, *v_scale; // [num_pages, KV]
    const int* cu_q;                // [n + 1]
    const int* ctx_lens;            // [n]
    const int* block_table;         // [n, table_width]
    float* scratch;                 // of the split-key kernel: 8 * blocks * tile_rows * (D + 3) + 32 * blocks words
    int* status;
    cudaStream_t stream;
    long long page_stride, q_stride;
    int n, n_tokens, table_width, page_size, num_pages, H, KV, window;
    int min_q, max_q;               // requests of so many new tokens are worked on
    int any_q;                      // the most that any request may bring
    int tile_rows;                  // split-key kernel: rows of its tiles, 8 or 16
    int blocks;                     // split-key kernel: blocks of four warps that share the work; prompt kernel: at least as many tiles as the requests make
    int dtype;                      // of q and out: 0 fp32, 1 bf16
    float scale;
};

inline bool kv8_call_ok(const Kv8Call& c) {
    return c.n >= 0 && c.n_tokens >= 0 && c.KV > 0 && (long long)c.KV * D <= 0x7fffffffll && c.H > 0 && c.H % c.KV == 0 && c.page_size > 0 && c.table_width >= 0 && c.num_pages >= 0 && c.window >= 0 &&
           c.any_q >= 1 && c.min_q >= 1 && (c.dtype == 0 || c.dtype == 1);
}

inline Kv8Args kv8_args(const Kv8Call& c, int tile_rows) {
    Kv8Args a;
    a.k_cache = (const unsigned char*)c.k_cache;
    a.v_cache = (const unsigned char*)c.v_cache;
    a.k_scale = c.k_scale;
    a.v_scale = c.v_scale;
    a.cu_q = c.cu_q;
    a.ctx_lens = c.ctx_lens;
    a.block_table = c.block_table;
    a.n = c.n;
    a.n_tokens = c.n_tokens;
    a.table_width = c.table_width;
    a.page_size = c.page_size;
    a.num_pages = c.num_pages;
    a.page_shift = -1;
    for (int s = 0; s < 30; ++s)
        if (c.page_size == 1 << s) a.page_shift = s;
    a.page_stride = c.page_stride;
    a.q_stride = c.q_stride;
    a.H = c.H;
    a.KV = c.KV;
    const int group = c.H / c.KV;
    a.heads_per_tile = group < tile_rows ? group : tile_rows;
    a.tokens_per_tile = tile_rows / a.heads_per_tile;
    a.head_groups = (group + a.heads_per_tile - 1) / a.heads_per_tile;
    a.scale = c.scale;
    a.window = c.window;
    a.min_q = c.min_q;
    a.max_q = c.max_q;
    a.any_q = c.any_q;
    a.status = c.status;
    return a;
}

struct Kv8Tile {
    int req;       // -1: no such tile
    int q_begin;   // the request's first row of q
    int q_len;
    int tok0;      // the tile's first token, counted from the request's first new one
};

// The `index`-th tile over all requests, in their order: each warp of a block finds it for itself from the boundaries, so that neither host nor
// an earlier kernel has to make a list. `look`: this block also checks that no request brings more than `any_q` tokens.
__device__ __forceinline__ Kv8Tile kv8_find_tile(const Kv8Args& a, int index, int tokens_per_tile, bool look) {
    Kv8Tile t = {-1, 0, 0, 0};
    const int lane = threadIdx.x & 31;
    int before = 0;
    for (int r0 = 0; r0 < a.n; r0 += 32) {
        const int r = r0 + lane;
        const int from = r < a.n ? __ldg(a.cu_q + r) : 0, len = r < a.n ? __ldg(a.cu_q + r + 1) - from : 0;
        const bool bad = len > a.any_q || (len > 0 && (from < 0 || (long long)from + len > a.n_tokens));
        if (look && bad && threadIdx.x < 32) oxr_report(a.status, OXR_BAD_ARGUMENT, r);
        const int count = (!bad && len >= a.min_q && len <= a.max_q) ? (len + tokens_per_tile - 1) / tokens_per_tile : 0;
        int upto = count;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const int mine = index - before - (upto - count);
        const unsigned hit = __ballot_sync(0xffffffffu, mine >= 0 && mine < count);
        if (hit && t.req < 0) {
            const int src = __ffs(hit) - 1;
            t.req = r0 + src;
            t.q_begin = __shfl_sync(0xffffffffu, from, src);
            t.q_len = __shfl_sync(0xffffffffu, len, src);
            t.tok0 = __shfl_sync(0xffffffffu, mine, src) * tokens_per_tile;
            if (!look) break;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return t;
}

// Two e4m3 codes (the low or the high 16 bits) as two fp16 numbers: exact, NaN stays NaN.
__device__ __forceinline__ uint32_t codes_to_f16(uint32_t w) {
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(w));
    return r;
}
__device__ __forceinline__ uint32_t codes_to_f16_high(uint32_t w) {
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(w));
    return r;
}
// The integer e with 2^(e - 1) < s <= 2^e for a positive finite s (subnormal ones count as 2^-126).
__device__ __forceinline__ int scale_exponent(float s) {
    const uint32_t b = __float_as_uint(s);
    return max((int)(b >> 23) - 127 + ((b & 0x7fffffu) != 0), -126);
}
__device__ __forceinline__ float exp2_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^e as the product of two powers: x * a * b, and what comes between, stays in range where the result does.
struct Power { float a, b; };
__device__ __forceinline__ Power power_of(float e) {
    const float half = floorf(0.5f * e);
    return {exp2_of(half), exp2_of(e - half)};
}
}  // namespace
