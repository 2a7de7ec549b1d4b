// Attention of long portions of prompts over the 8-bit paged cache on tcgen05, for bf16 queries and head sizes up to 128. Compiled once per head size.
//
// The formula is that of attention_kv8.cu, and so are the tricks with the scales. A tile is 256 rows, (token, query head) pairs of one KV head, in two
// halves of 128 (a row is a lane of tensor memory). Per block of 128 keys and half
//     S = Q K^T      tcgen05.mma on fp16 operands in shared memory, fp32 sums in tensor memory;
//     softmax        a thread per row: P = exp2(S - m), fp16, back into tensor memory over the columns that S came from;
//     O += P V       tcgen05.mma with P from tensor memory.
// kind::f8f6f4 would take the codes as they are, but its other operand would have to have 8 bits too, and two e4m3 numbers for each weight cost the
// softmax threads more than what is done instead: seven warps turn the codes of a block, while it passes from global to shared memory, into fp16
// numbers, times the ratio of their scale to the block's largest where that is a power of two and the products are exact: for keys from 2^-14 on, for values
// from 2^-4 on, which leaves the weights their bits; elsewhere times 1. There are three kinds of blocks:
//     EVEN   all ratios are such, as mostly among the store's scales: the largest key scale goes into the factor of the scores, the largest value scale, as its
//            logarithm, into the exponent of the weights, and neither costs the softmax an instruction per key;
//     NEAR   the value scales lie within 2^4 of the largest all the same (and key scales below 2^64): scores and weights are multiplied by what is left of their
//            keys' scales, in fp32;
//     ODD    any others, and blocks whose value scales are 2^60 off the last page's or below some met before: keys one by one, with two exponentials each.
// As in the split-key kernel the maximum is that of score and value scale, in whole numbers, and the sum of the weights a double: a row's result does not hang on
// scales that it does not see or gives no weight.
// Weights are kept as 2^7 P against a maximum that is raised in steps of 2^8: below 2^15 in
// fp16, with their eleven bits down to 2^-21 of the largest (2^-17 where one power stands for a block's scales).
// Warps: 0 issues the products and owns the tensor memory, 1 to 3 and 12 to 15 bring in keys and values, 4 to 7 and 8 to 11 are the
// softmax of the first and the second half; setmaxnreg gives those 160 registers (128 scores and what goes with them) and the others 96 (with 64 the
// codes on their way were spilled: 404 us instead of 146 in the case below).
// What bounds it: per block of 128 keys the products take 2,048 cycles of the tensor pipe and about as much shared-memory bandwidth, the exponentials 2,048 of
// theirs. 2,048 tokens on 2,048 cached ones, 32 / 8 heads of 128, take 148 us (697 TFLOP/s, 0.42 of measured): 2.9 us a block. Without the loaders' work it would be 120,
// without the softmax's arithmetic 133: two chains of latencies that are equally long and share the issue slots. With all blocks NEAR, scales of any mantissa, it takes 170, with
// all ODD 325. (NEAR and EVEN in one piece of code: 165 for EVEN blocks, whose registers were spilled.)
// Every wait on an mbarrier is bounded.
#include <cuda_fp16.h>

#include <type_traits>

#include "umma.cuh"

#ifndef HEAD_DIM
#error "compile with -DHEAD_DIM=<head size>"
#endif

#include "attention_kv8.cuh"

#if HEAD_DIM <= 128
namespace {
constexpr int HALF_ROWS = 128, TILE_ROWS = 2 * HALF_ROWS, KEYS = 128, STAGES = 2;
constexpr int THREADS = 512, LOADERS = 224;
constexpr int PANELS = (D + 63) / 64;                    // of 64 entries: 128 bytes a row, 128-byte swizzle
constexpr int PANEL_BYTES = 128 * 128;
constexpr int TENSOR_BYTES = PANELS * PANEL_BYTES;       // a half's queries, a block's keys, a block's values
constexpr int O_COLS = PANELS * 64;                      // whole panels: what the columns behind D hold is not looked at
constexpr int WORDS = D / 16;                            // 16 codes of a key: what a loader thread takes at a time
constexpr int PASSES = (KEYS * WORDS + LOADERS - 1) / LOADERS;
constexpr int INFO = 4;                                  // blocks whose pages and scales are at hand
constexpr int ODD = 0, NEAR = 1, EVEN = 2;
constexpr float RAISE = 8.f;
constexpr float P_SHIFT = 7.f;
constexpr uint32_t TMEM_COLS = 512;                      // S | P of half h at 128 h, O of half h at 256 + h O_COLS

struct __align__(16) BlockInfo {
    union {
        long long row[KEYS];   // byte offset of each key's row in the pools; -1: zeros stand for it
        float v_exp[KEYS];     // of an ODD block, once its codes have been asked for
    };
    // Scales; of blocks that are not EVEN then what is left of them beside the ratios: a factor of a key's scores, and of its values a factor of up to 1 and in an ODD
    // block a power of two, as its exponent relative to the last page's.
    float k_scale[KEYS], v_scale[KEYS];
    __half2 k_ratio[KEYS], v_ratio[KEYS];   // what codes are multiplied by: a scale over the block's largest, or 1 where that is not exact
    float k_most[4], v_most[4];   // of each 32 keys: the largest scale
    int kind;                  // EVEN: all of them are exact; NEAR: the value scales lie within 2^4 of the largest all the same; else ODD
    float factor, shift;       // of the block: its largest key scale; log2 of its largest value scale, relative to the last page's
};
struct Shared {
    BlockInfo info[INFO];
    uint64_t k_full[STAGES], k_empty[STAGES], v_full[STAGES], v_empty[STAGES], s_full[2], p_full[2], o_done[2], q_ready;
    uint32_t tmem;
    int nan_values;            // a block that not every row sees in full has a NaN among its values
};
constexpr size_t SMEM = (2 + 2 * STAGES) * (size_t)TENSOR_BYTES + sizeof(Shared);
static_assert(SMEM <= 227 * 1024, "shared memory of a block");

// rows are keys (the products' depth), 64 entries in 128 bytes; the next 64 entries a panel on
__device__ __forceinline__ uint64_t desc_mnmajor(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)(PANEL_BYTES >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// kind::f16, fp32 sums, both operands fp16, A K-major, B K-major or MN-major (the product itself is the one that umma_bf16 issues: the descriptor has the types)
__host__ __device__ constexpr uint32_t idesc_of(int m, int n, bool b_mn_major) {
    return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t ta, uint64_t db, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}"
                 ::"r"(d), "r"(ta), "l"(db), "r"(idesc), "r"(accumulate), "r"(0u) : "memory");
}
#define KV8_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define KV8_I8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
__device__ __forceinline__ void ld32(uint32_t taddr, uint32_t (&r)[32]) {   // tcgen05.wait::ld has to follow
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : KV8_R8(r, 0), KV8_R8(r, 8), KV8_R8(r, 16), KV8_R8(r, 24) : "r"(taddr));
}
__device__ __forceinline__ void ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : KV8_R8(r, 0), KV8_R8(r, 8) : "r"(taddr));
}
__device__ __forceinline__ void st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(taddr), KV8_I8(r, 0), KV8_I8(r, 8) : "memory");
}
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Two fp32 numbers in a pair of registers, for the packed fp32 instructions.
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// Four numbers by four others.
__device__ __forceinline__ void by_four(uint32_t* x, const float4& k) {
    float z[4];
    unpair(fma2(pair_of(__uint_as_float(x[0]), __uint_as_float(x[1])), pair_of(k.x, k.y), 0ull), z[0], z[1]);
    unpair(fma2(pair_of(__uint_as_float(x[2]), __uint_as_float(x[3])), pair_of(k.z, k.w), 0ull), z[2], z[3]);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __float_as_uint(z[i]);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ void loaders_meet() { asm volatile("bar.sync 1, %0;" ::"n"(LOADERS) : "memory"); }
__device__ __forceinline__ bool has_nan(uint4 w) {
    constexpr uint32_t M = 0x7f7f7f7fu;
    return (__vcmpeq4(w.x & M, M) | __vcmpeq4(w.y & M, M) | __vcmpeq4(w.z & M, M) | __vcmpeq4(w.w & M, M)) != 0;
}
__device__ __forceinline__ float usable(float scale) { return scale > 0.f && scale < INFINITY ? scale : 0.f; }

// A row's running maximum (see the head of the file; a whole number), and the sum of its weights 2^(score - m).
struct Row {
    float m;
    double l;
};
// A block's largest score with its value scale is `mx`: the maximum is raised to it, if it is 2^RAISE above, and with it go the sums. By whole warps.
__device__ __forceinline__ void raise_row(Row& row, float mx, uint32_t tmem_o, bool begun) {
    float alpha = 1.f;
    const bool raise = mx > row.m + RAISE || (row.m == -INFINITY && mx != -INFINITY);
    if (raise) {
        const float n = ceilf(mx);
        alpha = row.m == -INFINITY ? 0.f : exp2_of(row.m - n);
        row.l *= __hiloint2double((int)(fmaxf(row.m - n, -1022.f) + 1023.f) << 20, 0);
        row.m = n;
    }
    // S(b) complete means that O += P(b - 1) V(b - 1), issued before it, is complete: O may be rescaled
    if (__any_sync(0xffffffffu, raise && begun)) {
#pragma unroll 1
        for (int c = 0; c < D / 16; ++c) {
            uint32_t ov[16];
            ld16(tmem_o + (uint32_t)(c * 16), ov);
            wait_ld();
#pragma unroll
            for (int j = 0; j < 16; ++j) ov[j] = __float_as_uint(__uint_as_float(ov[j]) * alpha);
            st16(tmem_o + (uint32_t)(c * 16), ov);
        }
        wait_st();
    }
}
// The softmax of an ODD block, key by key; a row sees keys row_lo .. row_pos. By whole warps. (A function of its own: inlined it took registers from the ordinary
// block's softmax.)
__device__ __noinline__ Row one_by_one(const BlockInfo& f, uint32_t tmem_s, uint32_t tmem_o, float row_factor, int key0, int row_lo, int row_pos, bool begun, Row row) {
    // The scores of 32 keys, the hidden ones' -inf.
    auto scores_of = [&](int c, float (&x)[32]) {
        uint32_t v[32];
        ld32(tmem_s + (uint32_t)(c * 32), v);
        const int low = max(row_lo - key0 - c * 32, 0), high = min(row_pos - key0 - c * 32, 31);      // the first and the last that the row sees
        const uint32_t seen = row_pos >= row_lo && low <= high ? (0xffffffffu >> (31 - high)) & (0xffffffffu << low) : 0u;
        wait_ld();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float4 k = reinterpret_cast<const float4*>(f.k_scale)[c * 8 + i];
            const float kp[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) x[4 * i + j] = seen >> (4 * i + j) & 1u ? __uint_as_float(v[4 * i + j]) * (row_factor * kp[j]) : -INFINITY;
        }
    };
    float mx = -INFINITY, sc = -INFINITY;      // the largest score + log2 of the value scale; the largest score
#pragma unroll 1
    for (int c = 0; c < KEYS / 32; ++c) {
        float x[32];
        scores_of(c, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float4 e = reinterpret_cast<const float4*>(f.v_exp)[c * 8 + i];
            sc = fmaxf(max3(sc, x[4 * i], x[4 * i + 1]), fmaxf(x[4 * i + 2], x[4 * i + 3]));
            mx = fmaxf(max3(mx, x[4 * i] + e.x, x[4 * i + 1] + e.y), fmaxf(x[4 * i + 2] + e.z, x[4 * i + 3] + e.w));
        }
    }
    raise_row(row, mx, tmem_o, begun);
    const float most = sc == -INFINITY ? 0.f : ceilf(sc), off = (row.m == -INFINITY ? 0.f : -row.m) + P_SHIFT;
    float sum = 0.f;
#pragma unroll 1
    for (int c = 0; c < KEYS / 32; ++c) {      // (the columns that 32 weights go to held scores that have been read)
        float x[32];
        uint32_t pv[16];
        scores_of(c, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float4 e4 = reinterpret_cast<const float4*>(f.v_exp)[c * 8 + i], p4 = reinterpret_cast<const float4*>(f.v_scale)[c * 8 + i];
            const float e[4] = {e4.x, e4.y, e4.z, e4.w}, p[4] = {p4.x, p4.y, p4.z, p4.w};
            float w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float y = x[4 * i + j];
                sum += exp2_of(y - most);
                w[j] = y == -INFINITY ? 0.f : exp2_of(y + (e[j] + off)) * p[j];      // (a hidden key's scale may be anything)
            }
            const __half2 h0 = __floats2half2_rn(w[0], w[1]), h1 = __floats2half2_rn(w[2], w[3]);
            pv[2 * i] = *reinterpret_cast<const uint32_t*>(&h0);
            pv[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&h1);
        }
        st16(tmem_s + (uint32_t)(c * 16), pv);
    }
    if (sum != 0.f) row.l += (double)sum * __hiloint2double((int)(fminf(fmaxf(most - row.m, -1000.f), 1000.f) + 1023.f) << 20, 0);
    return row;
}

__global__ void __launch_bounds__(THREADS, 1)
attn_kv8_prompt_kernel(__nv_bfloat16* __restrict__ out, const __nv_bfloat16* __restrict__ q, const Kv8Args a, const int tiles) {
    extern __shared__ __align__(1024) unsigned char smem[];     // nothing static stands before it
    unsigned char* q_tiles = smem;                              // [half] queries
    unsigned char* k_ring = q_tiles + 2 * TENSOR_BYTES;         // [STAGES]
    unsigned char* v_ring = k_ring + STAGES * TENSOR_BYTES;
    Shared& sh = *reinterpret_cast<Shared*>(v_ring + STAGES * TENSOR_BYTES);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_wait();
    pdl_trigger();

    // later tiles of a prompt see more keys: the long ones first, the heads of a tile side by side
    const int per_tile = a.KV * a.head_groups, y = (int)(blockIdx.x % (unsigned)per_tile);
    const int kvh = y / a.head_groups, hg = y % a.head_groups, G = a.H / a.KV;
    const Kv8Tile t = kv8_find_tile(a, tiles - 1 - (int)(blockIdx.x / (unsigned)per_tile), a.tokens_per_tile, blockIdx.x == 0);
    if (t.req < 0) return;
    const int tokens = min(a.tokens_per_tile, t.q_len - t.tok0), rows = tokens * a.heads_per_tile;
    const int first_pos = __ldg(a.ctx_lens + t.req) - t.q_len + t.tok0, last_pos = first_pos + tokens - 1;
    int hi = last_pos + 1;
    const int lo = a.window > 0 ? max(0, first_pos - a.window + 1) : 0;
    if (hi > (long long)a.table_width * a.page_size) {
        if (threadIdx.x == 0) oxr_report(a.status, OXR_BAD_PAGE, t.req);
        hi = a.table_width * a.page_size;
    }
    const int block0 = lo / KEYS, count = hi > lo ? (hi + KEYS - 1) / KEYS - block0 : 0;
    const bool half1_live = rows > HALF_ROWS;
    const int* table_row = a.block_table + (size_t)t.req * a.table_width;
    const int last_lo = a.window > 0 ? last_pos - a.window + 1 : 0;
    auto partial = [&](int b) { return (block0 + b) * KEYS < last_lo || (block0 + b) * KEYS + KEYS - 1 > first_pos; };   // not every row sees all of it

    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) { mbar_init(sh.k_full + i, LOADERS / 32); mbar_init(sh.k_empty + i, 1); mbar_init(sh.v_full + i, LOADERS / 32); mbar_init(sh.v_empty + i, 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(sh.s_full + i, 1); mbar_init(sh.p_full + i, 4); mbar_init(sh.o_done + i, 1); }
        mbar_init(&sh.q_ready, 8);
        mbar_fence_init();
        sh.nan_values = 0;
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&sh.tmem)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = sh.tmem;
    int base_exp = 0;       // what value scales are relative to: the last visible page's
    if (count > 0) {
        const int page = __ldg(table_row + a.page_of(hi - 1));
        if (page >= 0 && page < a.num_pages) {
            const float s = usable(__ldg(a.v_scale + (size_t)page * a.KV + kvh));
            if (s > 0.f) base_exp = scale_exponent(s);
        }
    }

    if (warp < 4 || warp >= 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
        if (warp > 0) {
            // ------------------------------------------------------------------ keys and values come in
            const int lt = warp < 4 ? threadIdx.x - 32 : threadIdx.x - 12 * 32 + 96;      // 0 .. 223
            // The first 128 threads look after a key of a block each: its page two blocks ahead, its scales one block ahead.
            auto page_for = [&](int b) -> int {        // -1: none to be read
                const int key = (block0 + b) * KEYS + lt;
                if (lt >= KEYS || b >= count || key < lo || key >= hi) return -1;
                const int page = __ldg(table_row + a.page_of(key));
                if (page >= 0 && page < a.num_pages) return page;
                oxr_report(a.status, OXR_BAD_PAGE, t.req);
                return -1;
            };
            auto put_info = [&](int b, int page, float ks, float vs) {
                if (lt >= KEYS) return;
                BlockInfo& f = sh.info[b % INFO];
                const int key = (block0 + b) * KEYS + lt;
                f.k_scale[lt] = ks;
                f.v_scale[lt] = vs;
                f.row[lt] = page >= 0 ? (long long)page * a.page_stride + a.row_in_page(key, kvh) : -1;
                if (lt == 0) f.kind = EVEN;
                // (positive floats compare as integers do)
                const uint32_t km = __reduce_max_sync(0xffffffffu, __float_as_uint(usable(ks))), vm = __reduce_max_sync(0xffffffffu, __float_as_uint(usable(vs)));
                if (lane == 0) { f.k_most[lt / 32] = __uint_as_float(km); f.v_most[lt / 32] = __uint_as_float(vm); }
            };
            auto scale_of = [&](const float* scales, int page) { return page >= 0 ? __ldg(scales + (size_t)page * a.KV + kvh) : 0.f; };
            // Which 16 codes a thread takes in each pass: mostly the same columns of a key so many further on.
            constexpr bool SAME_COLUMNS = LOADERS % WORDS == 0;
            const int first_key = lt / WORDS, first_col = lt % WORDS;
            auto key_of = [&](int p) { return SAME_COLUMNS ? first_key + p * (LOADERS / WORDS) : (lt + p * LOADERS) / WORDS; };
            auto col_of = [&](int p) { return SAME_COLUMNS ? first_col : (lt + p * LOADERS) % WORDS; };
            uint4 kc[PASSES], vc[PASSES];
            auto ask = [&](uint4 (&c)[PASSES], const unsigned char* pool, int b) {
                if (b >= count) return;
                const BlockInfo& f = sh.info[b % INFO];
#pragma unroll
                for (int p = 0; p < PASSES; ++p) {
                    const long long row = key_of(p) < KEYS ? f.row[key_of(p)] : -1;
                    c[p] = row >= 0 ? __ldg(reinterpret_cast<const uint4*>(pool + row + col_of(p) * 16)) : make_uint4(0, 0, 0, 0);
                }
            };
            // A NaN that some row does not see is taken out here and put into the rows that see it at the end.
            auto take_out = [&](uint4 (&c)[PASSES]) {
#pragma unroll 1
                for (int p = 0; p < PASSES; ++p) {
                    uint4 w = make_uint4(0, 0, 0, 0);
#pragma unroll
                    for (int x = 0; x < PASSES; ++x)
                        if (x == p) w = c[x];
                    if (!has_nan(w)) continue;
                    sh.nan_values = 1;
                    w.x &= ~__vcmpeq4(w.x & 0x7f7f7f7fu, 0x7f7f7f7fu);
                    w.y &= ~__vcmpeq4(w.y & 0x7f7f7f7fu, 0x7f7f7f7fu);
                    w.z &= ~__vcmpeq4(w.z & 0x7f7f7f7fu, 0x7f7f7f7fu);
                    w.w &= ~__vcmpeq4(w.w & 0x7f7f7f7fu, 0x7f7f7f7fu);
#pragma unroll
                    for (int x = 0; x < PASSES; ++x)
                        if (x == p) c[x] = w;
                }
            };
            // The codes of a block as fp16 numbers, times the ratio of their scale to the block's largest, into a stage.
            auto put = [&](const uint4 (&c)[PASSES], unsigned char* stage, const __half2* ratios) {
#pragma unroll
                for (int p = 0; p < PASSES; ++p) {
                    const int key = key_of(p), col = col_of(p);
                    if (key >= KEYS) continue;
                    const __half2 r = ratios[key];
                    unsigned char* dst = stage + (col >> 2) * PANEL_BYTES + key * 128;
                    // threads of the second panel begin with the second of their two 16-byte words: the eight of a key then write to different banks
                    const int second = (col >> 2) & 1;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int word = (col & 3) * 2 + (i ^ second);
                        const uint32_t x = i ^ second ? c[p].z : c[p].x, z = i ^ second ? c[p].w : c[p].y;
                        uint32_t h[4] = {codes_to_f16(x), codes_to_f16_high(x), codes_to_f16(z), codes_to_f16_high(z)};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(h + j), r);
                            h[j] = *reinterpret_cast<const uint32_t*>(&v);
                        }
                        *reinterpret_cast<uint4*>(dst + ((word ^ (key & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
                    }
                }
                fence_proxy_async();
                __syncwarp();
            };
            // A key's ratios, by its thread: a power of two of 2^-14 and more for keys and 2^-4 and more for values, else 1. (The mantissas are the same but for the
            // rounding of the quotient.)
            auto most_of = [&](const float (&m)[4]) { return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])); };
            auto exact = [](float x, uint32_t least) {
                const uint32_t bits = __float_as_uint(x) + 4u;
                return bits - least <= 0x3f800008u - least && (bits & 0x7ffff0u) == 0u;
            };
            constexpr uint32_t K_LEAST = 0x38800000u, V_LEAST = 0x3d800000u;
            float top = -1e9f;       // the largest of the blocks' shifts so far
            auto put_ratios = [&](int b, int page, float ks, float vs) {
                if (lt >= KEYS || b >= count) return;
                BlockInfo& f = sh.info[b % INFO];
                const float km = most_of(f.k_most), vm = most_of(f.v_most);
                const float kr = __fdividef(ks, km), vr = __fdividef(vs, vm);
                const bool k_exact = exact(kr, K_LEAST) || ks == 0.f, v_none = vm == 0.f && vs == 0.f, v_exact = exact(vr, V_LEAST) || v_none;
                f.k_ratio[lt] = __float2half2_rn(k_exact ? (ks == 0.f ? 0.f : kr) : 1.f);
                f.v_ratio[lt] = __float2half2_rn(v_exact ? (v_none ? 0.f : vr) : 1.f);
                const float shift = vm > 0.f ? log2f(vm) - (float)base_exp : -60.f;      // (values of zero alone count as of 2^-60)
                top = fmaxf(top, shift);
                if (page >= 0) {
                    const bool near = v_none || (vr >= 0.0625f && vr <= 1.00001f);
                    const bool fits = !(fmaxf(km, fabsf(ks)) > 1.8e19f);      // 2^64: a score times it stays a float
                    if (!(near && fabsf(shift) <= 60.f && shift >= top - 60.f)) atomicMin(&f.kind, ODD);
                    else if (!k_exact || !v_exact) atomicMin(&f.kind, fits ? NEAR : ODD);
                }
                if (lt == 0) {
                    f.factor = km > 0.f ? km : 1.f;
                    f.shift = shift;
                }
            };
            // What the softmax needs for the keys of a block that is not EVEN.
            auto put_parts = [&](BlockInfo& f) {
                const float km = most_of(f.k_most), vm = most_of(f.v_most), ks = f.k_scale[lt], vs = f.v_scale[lt];
                if (exact(__fdividef(ks, km), K_LEAST)) f.k_scale[lt] = km;
                if (exact(__fdividef(vs, vm), V_LEAST)) {
                    f.v_exp[lt] = f.shift;
                    f.v_scale[lt] = 1.f;
                } else if (f.kind == NEAR) {
                    f.v_scale[lt] = vm > 0.f ? __fdividef(vs, vm) : 0.f;
                } else {
                    const int up = fabsf(vs) < INFINITY ? scale_exponent(fabsf(vs)) : base_exp;
                    const Power unit = power_of(-(float)up);
                    f.v_exp[lt] = (float)(vs == 0.f ? NO_SCALE : up - base_exp);
                    f.v_scale[lt] = vs * unit.a * unit.b;
                }
            };
            // of the block behind the present one
            int page1 = page_for(1);
            float ks1 = scale_of(a.k_scale, page1), vs1 = scale_of(a.v_scale, page1);
            int page2 = page_for(2);
            {
                const int page0 = page_for(0);
                const float ks0 = scale_of(a.k_scale, page0), vs0 = scale_of(a.v_scale, page0);
                put_info(0, page0, ks0, vs0);
                put_info(1, page1, ks1, vs1);
                loaders_meet();
                put_ratios(0, page0, ks0, vs0);
                loaders_meet();
            }
            ask(kc, a.k_cache, 0);
            ask(vc, a.v_cache, 0);
            loaders_meet();        // the first block's rows have been read: an ODD one's exponents come over them
            bool ok = true;        // (a thread that has given up keeps meeting the others)
            for (int b = 0; b < count; ++b) {
                BlockInfo& f = sh.info[b % INFO];
                const int st = b % STAGES;
                const float ks = scale_of(a.k_scale, page2), vs = scale_of(a.v_scale, page2);      // of block b + 2
                const int page3 = page_for(b + 3);
                if (lt < KEYS && f.kind != EVEN) put_parts(f);      // (its rows have been asked for)
                ok = ok && mbar_wait(sh.k_empty + st, ((b / STAGES) & 1) ^ 1);
                put(kc, k_ring + st * TENSOR_BYTES, f.k_ratio);
                if (lane == 0) mbar_arrive(sh.k_full + st);
                ask(kc, a.k_cache, b + 1);
                ok = ok && mbar_wait(sh.v_empty + st, ((b / STAGES) & 1) ^ 1);
                if (partial(b)) take_out(vc);
                put(vc, v_ring + st * TENSOR_BYTES, f.v_ratio);
                if (lane == 0) mbar_arrive(sh.v_full + st);
                ask(vc, a.v_cache, b + 1);
                put_ratios(b + 1, page1, ks1, vs1);      // (here rather than at the loop's start, which delays the keys: 4 us less in the case above)
                put_info(b + 2, page2, ks, vs);
                page1 = page2; ks1 = ks; vs1 = vs;
                page2 = page3;
                loaders_meet();
            }
            if (!ok && lane == 0) oxr_report(a.status, OXR_WAIT_EXPIRED, 41);
        } else if (elect_one()) {
            // ------------------------------------------------------------------ the products
            constexpr uint32_t idesc_s = idesc_of(HALF_ROWS, KEYS, false), idesc_o = idesc_of(HALF_ROWS, O_COLS, true);
            const int halves = half1_live ? 2 : 1;
            bool ok = count > 0;
            auto wait_for = [&](uint64_t* bar, uint32_t parity, int where) -> bool {
                if (!mbar_wait(bar, parity)) { oxr_report(a.status, OXR_WAIT_EXPIRED, where); return false; }
                fence_after();
                return true;
            };
            auto issue_s = [&](int b, int h) {
                const uint32_t ka = smem_addr(k_ring + (b % STAGES) * TENSOR_BYTES), qa = smem_addr(q_tiles + h * TENSOR_BYTES);
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk)
                    umma_bf16(tmem + (uint32_t)(h * KEYS), umma_desc(qa + (kk >> 2) * PANEL_BYTES + (kk & 3) * 32), umma_desc(ka + (kk >> 2) * PANEL_BYTES + (kk & 3) * 32),
                             idesc_s, kk > 0 ? 1u : 0u);
                umma_commit(sh.s_full + h);
                if (h == halves - 1) umma_commit(sh.k_empty + b % STAGES);
            };
            ok = ok && wait_for(&sh.q_ready, 0, 42) && wait_for(sh.k_full, 0, 43);
            if (ok)
                for (int h = 0; h < halves; ++h) issue_s(0, h);
            // block by block and half by half: O_h += P_h(b) V(b), and at once S_h(b + 1) over the columns that P_h(b) was in (the pipe keeps their order)
            for (int b = 0; b < count && ok; ++b) {
                const uint32_t va = smem_addr(v_ring + (b % STAGES) * TENSOR_BYTES);
                for (int h = 0; h < halves && ok; ++h) {
                    ok = wait_for(sh.p_full + h, b & 1, 44) && (h > 0 || wait_for(sh.v_full + b % STAGES, (b / STAGES) & 1, 45));
                    if (!ok) break;
#pragma unroll
                    for (int kk = 0; kk < KEYS / 16; ++kk)
                        mma_tmem(tmem + 256 + (uint32_t)(h * O_COLS), tmem + (uint32_t)(h * KEYS + kk * 8), desc_mnmajor(va + kk * 16 * 128), idesc_o, (b > 0 || kk > 0) ? 1u : 0u);
                    umma_commit(sh.o_done + h);
                    if (h == halves - 1) umma_commit(sh.v_empty + b % STAGES);
                    if (b + 1 < count) {
                        ok = h > 0 || wait_for(sh.k_full + (b + 1) % STAGES, ((b + 1) / STAGES) & 1, 43);
                        if (ok) issue_s(b + 1, h);
                    }
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 160;");
        // ---------------------------------------------------------------------- softmax: a thread per row
        const int half = (warp - 4) >> 2, quarter = warp & 3, rr = quarter * 32 + lane, r = half * HALF_ROWS + rr;
        const int tok = r / a.heads_per_tile, head = hg * a.heads_per_tile + r % a.heads_per_tile;
        const bool row_ok = r < rows && head < G;
        const int row_pos = first_pos + tok, row_lo = a.window > 0 ? row_pos - a.window + 1 : 0;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        const uint32_t tmem_s = tmem + lanes + (uint32_t)(half * KEYS), tmem_o = tmem + lanes + 256 + (uint32_t)(half * O_COLS);
        float row_factor;
        {   // the row as fp16 numbers, times the power of two that brings its largest entry to [2^14, 2^15)
            const uint4* src = reinterpret_cast<const uint4*>(q + (size_t)(t.q_begin + t.tok0 + (row_ok ? tok : 0)) * a.q_stride + (size_t)(kvh * G + (row_ok ? head : 0)) * D);
            uint4 v[D / 8];
            float most = 0.f;
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
                v[c] = row_ok ? __ldg(src + c) : make_uint4(0, 0, 0, 0);
                const uint32_t w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) most = fmaxf(most, fmaxf(fabsf(__uint_as_float(w[i] << 16)), fabsf(__uint_as_float(w[i] & 0xffff0000u))));
            }
            const int up = (most > 0.f && most < INFINITY) ? min(14 - (int)((__float_as_uint(most) >> 23) & 255) + 127, 126) : 0;
            const float f = __uint_as_float((uint32_t)(up + 127) << 23);
            row_factor = a.scale * LOG2E * __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
                const uint32_t w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
                uint32_t h[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const __half2 x = __floats2half2_rn(__uint_as_float(w[i] << 16) * f, __uint_as_float(w[i] & 0xffff0000u) * f);
                    h[i] = *reinterpret_cast<const uint32_t*>(&x);
                }
                *reinterpret_cast<uint4*>(q_tiles + half * TENSOR_BYTES + (c >> 3) * PANEL_BYTES + rr * 128 + (((c & 7) ^ (rr & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.q_ready);
        }
        if (half == 0 || half1_live) {
            Row row = {-INFINITY, 0.};
            bool alive = true;
            for (int b = 0; b < count; ++b) {
                if (!mbar_wait(sh.s_full + half, b & 1)) { if (lane == 0) oxr_report(a.status, OXR_WAIT_EXPIRED, 46); alive = false; break; }
                fence_after();
                const int key0 = (block0 + b) * KEYS;
                const BlockInfo& f = sh.info[b % INFO];
                const int kind = f.kind;
                // (never zero: a hidden score of -inf has to stay one)
                const float factor = fmaxf(row_factor * (kind == EVEN ? f.factor : 1.f), 1e-37f), shift = f.shift;
                // Rows without a token or head see what comes (their queries are zero); the others see keys row_lo .. row_pos.
                const bool some_hidden = key0 < row_lo || key0 + KEYS - 1 > row_pos;
                const int from = row_lo - key0;
                const unsigned span = row_pos >= row_lo ? (unsigned)(row_pos - row_lo) : 0u;
                auto hidden = [&](int j) { return (unsigned)(j - from) > span || row_pos < row_lo; };
                auto in_registers = [&](auto by_key) {
                    constexpr bool BY_KEY = decltype(by_key)::value;
                    uint32_t sv[KEYS / 32][32];
#pragma unroll
                    for (int c = 0; c < KEYS / 32; ++c) ld32(tmem_s + (uint32_t)(c * 32), sv[c]);
                    wait_ld();
                    if constexpr (BY_KEY) {      // each score by its key's scale
#pragma unroll
                        for (int c = 0; c < KEYS / 32; ++c)
#pragma unroll
                            for (int i = 0; i < 8; ++i) by_four(&sv[c][4 * i], reinterpret_cast<const float4*>(f.k_scale)[c * 8 + i]);
                    }
                    if (some_hidden) {
#pragma unroll
                        for (int c = 0; c < KEYS / 32; ++c)
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (hidden(c * 32 + j)) sv[c][j] = __float_as_uint(-INFINITY);
                    }
                    float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int c = 0; c < KEYS / 32; ++c)
#pragma unroll
                        for (int j = 0; j < 16; ++j) mx4[j & 3] = max3(mx4[j & 3], __uint_as_float(sv[c][2 * j]), __uint_as_float(sv[c][2 * j + 1]));
                    const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * factor + shift;
                    raise_row(row, mx, tmem_o, b > 0);
                    const float off = (row.m == -INFINITY ? 0.f : shift - row.m) + P_SHIFT;
                    const uint64_t factor2 = pair_of(factor, factor), off2 = pair_of(off, off);
                    uint64_t sum2[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
                    for (int c = 0; c < KEYS / 32; ++c) {
                        uint32_t pv[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            float x0, x1;
                            unpair(fma2(pair_of(__uint_as_float(sv[c][2 * e]), __uint_as_float(sv[c][2 * e + 1])), factor2, off2), x0, x1);
                            const float p0 = exp2_of(x0), p1 = exp2_of(x1);
                            sum2[e & 3] = add2(sum2[e & 3], pair_of(p0, p1));
                            if constexpr (BY_KEY) {
                                sv[c][2 * e] = __float_as_uint(p0);
                                sv[c][2 * e + 1] = __float_as_uint(p1);
                            } else {
                                const __half2 pk = __floats2half2_rn(p0, p1);
                                pv[e] = *reinterpret_cast<const uint32_t*>(&pk);
                            }
                        }
                        if constexpr (BY_KEY) {      // each weight by its key's value scale over the largest
#pragma unroll
                            for (int i = 0; i < 8; ++i) by_four(&sv[c][4 * i], reinterpret_cast<const float4*>(f.v_scale)[c * 8 + i]);
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                const __half2 pk = __floats2half2_rn(__uint_as_float(sv[c][2 * e]), __uint_as_float(sv[c][2 * e + 1]));
                                pv[e] = *reinterpret_cast<const uint32_t*>(&pk);
                            }
                        }
                        st16(tmem_s + (uint32_t)(c * 16), pv);
                    }
                    float sum4[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) { float x, z; unpair(sum2[i], x, z); sum4[i] = x + z; }
                    row.l += (double)(((sum4[0] + sum4[1]) + (sum4[2] + sum4[3])) * exp2_of(-shift - P_SHIFT));
                };
                if (kind == EVEN) in_registers(std::false_type{});
                else if (kind == NEAR) in_registers(std::true_type{});
                else {
                    row = one_by_one(f, tmem_s, tmem_o, row_factor, key0, row_lo, row_pos, b > 0, row);
                }
                wait_st();
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(sh.p_full + half);
            }
            // ---- O / l
            if (alive && count > 0 && !mbar_wait(sh.o_done + half, (count - 1) & 1)) { if (lane == 0) oxr_report(a.status, OXR_WAIT_EXPIRED, 47); alive = false; }
            alive = __all_sync(0xffffffffu, alive);
            if (alive) {
                fence_after();
                const int l_exp = (__double2hiint(row.l) >> 20 & 0x7ff) - 1023;       // the sum is a number from 1 up to 2, times 2^l_exp
                const bool none = row.l == 0.;
                const Power unit = power_of((float)(base_exp - l_exp) - P_SHIFT);
                const float inverse = unit.a / (float)(l_exp == 1024 ? row.l : __hiloint2double(__double2hiint(row.l) - (l_exp << 20), __double2loint(row.l)));
                __nv_bfloat16* dst = out + ((size_t)(t.q_begin + t.tok0 + tok) * a.H + (size_t)kvh * G + head) * D;
#pragma unroll 1
                for (int c = 0; c < D / 16; ++c) {
                    uint32_t ov[16];
                    if (count > 0) {
                        ld16(tmem_o + (uint32_t)(c * 16), ov);
                        wait_ld();
                    }
                    uint4 o4[2];
                    __nv_bfloat162* op = reinterpret_cast<__nv_bfloat162*>(o4);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        op[e] = none ? __floats2bfloat162_rn(0.f, 0.f)
                                     : __floats2bfloat162_rn(__uint_as_float(ov[2 * e]) * inverse * unit.b, __uint_as_float(ov[2 * e + 1]) * inverse * unit.b);
                    if (row_ok) {
                        reinterpret_cast<uint4*>(dst + 16 * c)[0] = o4[0];
                        reinterpret_cast<uint4*>(dst + 16 * c)[1] = o4[1];
                    }
                }
                // values that were taken out of blocks which not every row sees: NaN to the rows that do
                if (*reinterpret_cast<volatile int*>(&sh.nan_values) && row_ok) {
                    for (int key = max(row_lo, block0 * KEYS); key <= min(row_pos, hi - 1); ++key) {
                        if (!partial(key / KEYS - block0)) { key = key / KEYS * KEYS + KEYS - 1; continue; }
                        const int page = __ldg(table_row + a.page_of(key));
                        if (page < 0 || page >= a.num_pages) continue;
                        const unsigned char* codes = a.v_cache + (long long)page * a.page_stride + a.row_in_page(key, kvh);
                        for (int d = 0; d < D; ++d)
                            if ((__ldg(codes + d) & 0x7f) == 0x7f) dst[d] = __float2bfloat16_rn(__uint_as_float(0x7fffffffu));
                    }
                }
            }
        }
    }
    fence_before();
    __syncthreads();
    if (warp == 0) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}
}  // namespace
#endif

// Whether the kernel may run at all. setmaxnreg deals out what the block is launched with: 128 registers a thread, or the softmax warps would wait for
// theirs in vain.
OXR_API int oxr_kv8_prompt_ready() {
#if HEAD_DIM <= 128
    cudaFuncAttributes attrs;
    if (cudaFuncGetAttributes(&attrs, attn_kv8_prompt_kernel) == cudaSuccess) return attrs.numRegs == 128;
    cudaGetLastError();
#endif
    return 0;
}
// For bf16 queries, head sizes up to 128 and a positive scale.
OXR_API int oxr_kv8_prompt_attention(const Kv8Call* c) {
#if HEAD_DIM <= 128
    if (!kv8_call_ok(*c) || c->any_q < 2 || c->blocks < 0 || c->dtype != 1 || !(c->scale > 0.f)) return OXR_BAD_ARGUMENT;
    if (c->blocks == 0 || c->n == 0 || c->n_tokens == 0) return 0;
    const Kv8Args a = kv8_args(*c, TILE_ROWS);
    const long long grid = (long long)c->blocks * c->KV * a.head_groups;
    if (grid > 0x7fffffffll) return OXR_BAD_ARGUMENT;
    static thread_local int ready = -1;
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return oxr_launch_status();
    if (ready != device) {
        if (!oxr_kv8_prompt_ready()) return OXR_BAD_ARGUMENT;
        if (cudaFuncSetAttribute(attn_kv8_prompt_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM) != cudaSuccess) return oxr_launch_status();
        ready = device;
    }
    oxr_launch(attn_kv8_prompt_kernel, dim3((unsigned)grid), dim3(THREADS), SMEM, c->stream, true, (__nv_bfloat16*)c->out, (const __nv_bfloat16*)c->q, a, c->blocks);
    return oxr_launch_status();
#else
    return OXR_BAD_ARGUMENT;
#endif
}
