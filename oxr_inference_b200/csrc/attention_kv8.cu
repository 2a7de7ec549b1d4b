// Paged grouped-query attention over a cache of 8-bit floating-point numbers (e4m3) with one scale for each page and KV head. Compiled once
// per head size: -DHEAD_DIM=<multiple of 16, at most 256>.
//
// A cached key is ks * K and a cached value vs * V, with e4m3 codes K, V and the fp32 scales of the page that holds them. A query q at position p
// of its request sees the keys j <= p (j > p - window behind a window):
//     s_j = scale * ks_j * (q . K_j),     o = sum_j exp(s_j) vs_j V_j / sum_j exp(s_j).
//
// The codes go through the tensor cores as they are (mma.sync, fp32 sums) and both scales stay outside the products: ks multiplies the fp32 score,
// vs the weight. Keys and values are the left operands (16 keys, or 16 entries of the values, by the products' depth) and the queries the right one (8
// of them): a decode step has as few queries per KV head as that, and scores, weights and sums then come in fragments of 8 columns, a half of what
// 16 rows of queries would take.
// Every code is an fp16 number (a pair costs one conversion, 64 lanes a clock), so both products are m16n8k16 on fp16 operands. (m16n8k32 takes codes
// as they are, but converts them itself, again for each product: scores that way, with the queries as two e4m3 numbers, took 76 us where fp16 took 68.)
// A bf16 query is an fp16 number too once its row is multiplied by a power of two that brings its largest entry to 2^14 (what lies 2^-39 below that is
// lost); an fp32 query is the sum of two fp16 numbers to 22 bits. The weights are rounded to fp16 (11 bits) against the row's running maximum, times
// 2^15 so that they keep their bits down to 2^-29 of it; with fp32 queries they are two numbers as well.
//
// The running maximum m of a row is that of s_j + log2(vs_j), with 2^log2(vs) the power of two above a key's value scale, rounded up to a whole number (all
// factors between blocks and pieces are powers of two then). Weights times scales never exceed one against it, and the largest of them is at least 2^-6, however
// much the scales of pages differ and whatever scales pages have that the row does not see or gives no weight. The sum of the weights without their
// scales may lie as far from m as scales reach, 2^+-250.
// The ordinary walk over a tile's blocks takes one power for the value scales of a block, so that the sum follows from the weighted weights, and a float for the
// sum. That is good while the scales of a block lie within 2^4 of each other, and all of them within 2^30 of the last page's, which is their unit (and not below 2^-110); blocks of zeros alone count as of 2^-60. A warp that
// meets others begins its part of the tile anew in a careful walk, where the sum has a power of two beside it and a block is gone through once for each 2^4 that its
// scales span. (One walk for both issued 14 % more instructions: 64 requests of 2,048 keys 64 us instead of 61.)
//
// The work is a row of items, one for each block of 32 keys of each tile (rows of queries of one KV head) of each request, and every warp of the
// grid takes an equal stretch of it, so that requests of any lengths keep all of them busy to the end; the boundaries are worked out on the GPU, from
// the lengths. A warp is on its own: a ring of stages filled by TMA (with cp.async where pages are not multiples of eight keys), one online softmax,
// no barrier. What it has of a tile that it does not have whole goes to scratch memory, and a second kernel joins those pieces. What bounds it
// is reading the cache: 2 D bytes per key and KV head. 64 requests of 2,048 keys, 32 / 8 heads of 128: 55 us (4.9 TB/s, 0.75 of measured) and 6 for
// the join; the rest is the latency of a warp's chain of conversions, products and softmax at the twelve warps that an SM's registers hold.
#include <cuda_fp16.h>
#include <type_traits>

#include "tma.cuh"

#ifndef HEAD_DIM
#error "compile with -DHEAD_DIM=<head size>"
#endif
static_assert(HEAD_DIM % 16 == 0 && HEAD_DIM >= 16 && HEAD_DIM <= 256, "head size: a multiple of 16 up to 256");

#include "attention_kv8.cuh"

namespace {
constexpr int WARPS = 4;
constexpr int THREADS = WARPS * 32;
constexpr int KEYS = 32;                       // keys of a block: one per lane while addresses are worked out
// A stage holds K and V as panels of PW bytes a key. Where a row is an odd number of 16-byte words it is a panel of its own and eight rows lie on
// different banks as they are; elsewhere panels are the largest power of two up to 128 bytes and swizzled as TMA does it.
constexpr bool SWIZZLED = (D / 16) % 2 == 0;
constexpr int PW = !SWIZZLED ? D : (D % 128 == 0 ? 128 : D % 64 == 0 ? 64 : 32);
constexpr int PANELS = D / PW;
constexpr int TENSOR_BYTES = KEYS * D;
constexpr int STAGE_BYTES = 2 * TENSOR_BYTES;      // a multiple of 1,024: swizzled panels start where the pattern does
constexpr int SCALE_BYTES = 2 * KEYS * 4;
constexpr int KSTEPS = D / 16;
constexpr float P_LOG2 = 15.f;                 // weights are kept as 2^15 w
constexpr int GROUPS = 2 * THREADS, GROUP_BYTES = (GROUPS + 2 + WARPS) * 8;   // see Items
// Of a kernel whose tiles have 8 NQ rows, (token, query head) pairs of one KV head:
template <typename T, int NQ> struct Shape {
    static constexpr int PIECES = sizeof(T) == 4 ? 2 : 1;             // fp16 numbers that make a query's entry or a weight
    static constexpr int ROWS = 8 * NQ;
    static constexpr int Q_WORDS = NQ * KSTEPS * PIECES * 2;          // of a lane
    static constexpr bool Q_IN_REGS = Q_WORDS + NQ * D / 4 <= 160;    // beside the sums
    // Blocks of four warps on an SM: with 8 rows of bf16 queries the registers suffice for three, which hide more of each other's waits than a third
    // stage does (64 requests of 2,048 keys: 59 against 68 us); the ring takes what shared memory that leaves, four stages at most.
    static constexpr int BLOCKS = D > 128 ? 1 : NQ == 1 && PIECES == 1 ? 3 : 2;
    static constexpr int FIT = (225 * 1024 / BLOCKS - 4096 - (Q_IN_REGS ? 0 : WARPS * Q_WORDS * 128)) / (WARPS * (STAGE_BYTES + SCALE_BYTES));
    static constexpr int STAGES = FIT < 4 ? FIT : 4;
    static_assert(STAGES >= 2, "room for a ring");
    static constexpr int RING_BYTES = WARPS * STAGES * STAGE_BYTES;
    static constexpr int AT_BARS = RING_BYTES + WARPS * STAGES * SCALE_BYTES, AT_GROUPS = AT_BARS + WARPS * STAGES * 8, AT_POWERS = AT_GROUPS + GROUP_BYTES, AT_Q = AT_POWERS + THREADS * 2 * NQ * 2;
    static constexpr size_t SMEM = AT_Q + (Q_IN_REGS ? 0 : WARPS * Q_WORDS * 128);
    static_assert(SMEM <= 227 * 1024, "shared memory of a block");
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool take) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
// What the swizzle of a panel's row changes in the address of its 16-byte words.
__device__ __forceinline__ uint32_t row_swizzle(int row) {
    return !SWIZZLED ? 0u : PW == 128 ? (uint32_t)(row & 7) << 4 : PW == 64 ? (uint32_t)((row >> 1) & 3) << 4 : (uint32_t)((row >> 2) & 1) << 4;
}
// The address of 16-byte word `w` of a row, from that of the row in the first panel with the row's swizzle in it.
__device__ __forceinline__ uint32_t word_at(uint32_t row, int w) {
    if constexpr (!SWIZZLED) return row + w * 16;
    return (row ^ (uint32_t)(w % (PW / 16) * 16)) + (uint32_t)(w / (PW / 16) * KEYS * PW);
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool take) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(take ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// An 8 x 8 matrix of 16-bit numbers, two of a row per lane, turned over.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
// Four entries of a query row.
__device__ __forceinline__ float4 load4(const float* p) { return __ldg(reinterpret_cast<const float4*>(p)); }
__device__ __forceinline__ float4 load4(const __nv_bfloat16* p) {
    const uint2 w = __ldg(reinterpret_cast<const uint2*>(p));
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
}
__device__ __forceinline__ void store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void store4(__nv_bfloat16* p, float4 v) {
    uint2 w;
    reinterpret_cast<__nv_bfloat162*>(&w)[0] = __floats2bfloat162_rn(v.x, v.y);
    reinterpret_cast<__nv_bfloat162*>(&w)[1] = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(p) = w;
}
__device__ __forceinline__ void store2(float* p, float2 v) { *reinterpret_cast<float2*>(p) = v; }
__device__ __forceinline__ void store2(__nv_bfloat16* p, float2 v) { *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(v.x, v.y); }
// A sum of weights, times 2^k. k is 0 unless the sum lies further than 2^30 from 1 (and it does not come near the ends of a float).
struct Sum { float f; int k; };
__device__ __forceinline__ double whole_of(const Sum& s) { return (double)s.f * __hiloint2double((1023 + max(s.k, -1022)) << 20, 0); }
__device__ __forceinline__ Sum sum_of(double x) {
    const int e = (__double2hiint(x) >> 20 & 0x7ff) - 1023;
    if (e < -1000 || e > 1000 || abs(e) <= 30) return {(float)x, 0};      // 0, NaN, infinity; what a float holds well
    return {(float)__hiloint2double(__double2hiint(x) - (e << 20), __double2loint(x)), e};
}
// What a row's sums are relative to, and the sum of its weights; of nothing: -inf and 0. A sum with a power of two beside it has a minus sign. (A NaN may have
// a sum without a maximum.)
struct __align__(8) RowSum { float m, total; };
// (s, v) += N pieces of a row, powers left aside.
template <int N> __device__ __forceinline__ void add_pieces(RowSum& s, float4& v, const RowSum (&y)[N], const float4 (&u)[N]) {
    float n = s.m;
    bool powers = s.total < 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) { n = fmaxf(n, y[i].m); powers |= y[i].total < 0.f; }
    const float f0 = s.m == n ? 1.f : exp2_of(s.m - n);
    float total = fabsf(s.total) * f0, f[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        f[i] = y[i].m == n ? 1.f : exp2_of(y[i].m - n);
        total += fabsf(y[i].total) * f[i];
    }
    v.x *= f0; v.y *= f0; v.z *= f0; v.w *= f0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (y[i].total == 0.f) continue;
        v.x += u[i].x * f[i]; v.y += u[i].y * f[i]; v.z += u[i].z * f[i]; v.w += u[i].w * f[i];
    }
    s = {n, powers ? -1.f : total};
}
__device__ __forceinline__ float times(float x, const Power& p) { return x * p.a * p.b; }
// What a row's sums are multiplied by at the end, 2^(base_exp - 15) / total.
__device__ __forceinline__ Power final_unit(const Sum& total, int base_exp) { return power_of((float)(base_exp - total.k) - P_LOG2); }
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// What rounding a pair to fp16 left over, as fp16 again.
__device__ __forceinline__ uint32_t pack_rest(float lo, float hi, uint32_t packed) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&packed));
    return pack_f16(lo - f.x, hi - f.y);
}

// ---- the row of work items
// Request after request; of a request tile after tile, of a tile each group of query heads (`per_tile` of them), of that the blocks of 32 keys behind
// TILE_COST items that stand for the time a warp needs to begin a tile and to put its result away (without them a warp whose stretch is a dozen of
// requests of a few tokens works twice as long as the others: 24 requests of 1 to 32,768 keys 118 us without,
// 79 with one, 66 with three). All tiles of a request count as many blocks as the widest; what a tile lacks of them is empty. A block of threads sums up the items of 256 groups of neighbouring
// requests (each request is its own group up to 256 of them); a warp finds the request of an item by bisection and a scan of the group.
constexpr int TILE_COST = 3;
struct Items {
    const Kv8Args& a;
    long long* upto;        // [GROUPS + 1] in shared memory: items of the groups before
    int group, per_tile;

    struct Request { int q_begin, q_len, ctx, tiles, blocks; long long items; };
    __device__ __forceinline__ Request request(int r, bool look) const {
        Request x = {0, 0, 0, 0, 1, 0};
        if (r >= a.n) return x;
        x.q_begin = __ldg(a.cu_q + r);
        x.q_len = __ldg(a.cu_q + r + 1) - x.q_begin;
        x.ctx = __ldg(a.ctx_lens + r);
        if (x.q_len < 1) return x;
        if (x.q_len > a.any_q || x.q_begin < 0 || (long long)x.q_begin + x.q_len > a.n_tokens) {
            if (look) oxr_report(a.status, OXR_BAD_ARGUMENT, r);
            return x;
        }
        if (x.q_len < a.min_q || x.q_len > a.max_q) return x;
        x.tiles = (x.q_len + a.tokens_per_tile - 1) / a.tokens_per_tile;
        const int keys = min((long long)max(x.ctx, 0), (long long)a.table_width * a.page_size);
        x.blocks = max(1, (keys + KEYS - 1) / KEYS);
        if (a.window > 0) x.blocks = min(x.blocks, (int)(((long long)a.window + a.tokens_per_tile + KEYS - 2) / KEYS) + 1);
        x.blocks += TILE_COST;
        x.items = (long long)x.tiles * per_tile * x.blocks;
        return x;
    }
    // All items; by every thread of the block. `sums`: a word of shared memory per warp.
    __device__ long long prepare(long long* sums) {
        group = (a.n + GROUPS - 1) / GROUPS;
        per_tile = a.KV * a.head_groups;
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        long long mine[2] = {0, 0};                // a thread's two groups, side by side
#pragma unroll
        for (int k = 0; k < 2; ++k)
            for (int r = 0; r < group; ++r) mine[k] += request((threadIdx.x * 2 + k) * group + r, blockIdx.x == 0).items;
        long long v = mine[0] + mine[1];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long w = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += w;
        }
        if (lane == 31) sums[warp] = v;
        __syncthreads();
        long long before = v - mine[0] - mine[1], all = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const long long s = sums[w];
            if (w < warp) before += s;
            all += s;
        }
        upto[threadIdx.x * 2] = before;
        upto[threadIdx.x * 2 + 1] = before + mine[0];
        if (threadIdx.x == 0) upto[GROUPS] = all;
        __syncthreads();
        return all;
    }
    struct Place { int req; Request of; int tile, y, block; };
    // Of item `i`, which is one; by a whole warp.
    __device__ __forceinline__ Place find(int i) const {
        int low = 0, high = GROUPS;               // the last group that begins at or before it (those without items share their start with the next)
        while (high - low > 1) {
            const int mid = (low + high) >> 1;
            if (upto[mid] <= i) low = mid; else high = mid;
        }
        int rest = i - (int)upto[low];
        Place p;
        p.req = low * group;
        p.of = request(p.req, false);
        for (int r = 1; r < group && rest >= p.of.items; ++r) {
            rest -= (int)p.of.items;
            p.of = request(++p.req, false);
        }
        const int per = p.of.blocks * per_tile;
        p.tile = rest / per;
        const int in_tile = rest - p.tile * per;
        p.y = in_tile / p.of.blocks;
        p.block = in_tile % p.of.blocks;
        return p;
    }
};

// Scratch: a warp leaves what it has of a tile in its first place when the tile began before its stretch, else in its second.
struct Cut {         // what the join has to know of a tile that a stretch ends in and that began in it
    int last;        // the warp with its last piece; -1: the stretch ends in no such tile
    int token, head; // first row of q and first head
    int rows, heads; // (token, head) pairs of the tile, and how many heads of them there are
    int base_exp;    // what the pieces are relative to
    int spare[2];
};
struct Pieces {
    float* sums;     // [2 * warps][ROWS][D]
    RowSum* rows;    // [2 * warps][ROWS]
    int* powers;     // [2 * warps][ROWS], of sums that have one
    Cut* cuts;       // [warps]
};

// TMA: pages hold whole pieces of 8, 16 or 32 keys (2^piece_shift), which come in as boxes; otherwise each lane copies 16 bytes at a time.
template <typename T, bool TMA, int NQ>
__global__ void __launch_bounds__(THREADS, Shape<T, NQ>::BLOCKS)
attn_kv8_kernel(T* __restrict__ out, const T* __restrict__ q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                const int piece_shift, const Kv8Args a, const Pieces left) {
    using S = Shape<T, NQ>;
    constexpr int ROWS = S::ROWS, PIECES = S::PIECES, STAGES = S::STAGES, SCALES_AT = S::RING_BYTES;
    extern __shared__ __align__(1024) unsigned char smem[];   // nothing static stands before it: it starts on a 1,024-byte boundary
    long long* groups = reinterpret_cast<long long*>(smem + S::AT_GROUPS);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, quad = lane & 3;
    if (TMA && threadIdx.x == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
    }
    const uint32_t ring = smem_addr(smem) + warp * STAGES * STAGE_BYTES, my_scales = smem_addr(smem) + SCALES_AT + warp * STAGES * SCALE_BYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::AT_BARS) + warp * STAGES;   // a stage's rows have arrived
    [[maybe_unused]] uint32_t* q_smem = reinterpret_cast<uint32_t*>(smem + S::AT_Q) + warp * S::Q_WORDS * 32;   // [Q_WORDS][32 lanes]
    if (TMA && lane == 0) {
        for (int i = 0; i < STAGES; ++i) mbar_init(bars + i, 1);
        mbar_fence_init();
        fence_proxy_async();
    }
    pdl_wait();
    pdl_trigger();
    Items items = {a, groups};
    const long long all = items.prepare(groups + GROUPS + 2);
    const int G = a.H / a.KV, me = (int)blockIdx.x * WARPS + warp;
    const int warps = (int)gridDim.x * WARPS;
    if (all > 0x7fffffffll - warps) {      // some thousands of the longest sequences: more than a step can mean
        if (blockIdx.x == 0 && threadIdx.x == 0) oxr_report(a.status, OXR_BAD_ARGUMENT, -1);
        if (lane == 0) left.cuts[me].last = -1;
        return;
    }
    const int share = max(1, ((int)all + warps - 1) / warps), end = (int)min(all, (me + 1ll) * share);
    int turn = 0;      // stages filled before this tile: the ring and its barriers go on from there
    Cut cut = {-1, 0, 0, 0, 0, 0, {0, 0}};

    // The items from `item` on: where it came to, -1 if a wait ran out. An ordinary walk comes to `end` or to a tile whose scales it is not for.
    auto stretch = [&](int item, auto careful) -> int {
    constexpr bool CAREFUL = decltype(careful)::value;
    while (item < end) {
    const Items::Place at = items.find(item);
    const int count = min(end - item, at.of.blocks - at.block);   // items of this tile that are this warp's
    item += count;

    // ---- which rows
    const int kvh = at.y / a.head_groups, hg = at.y % a.head_groups;
    const int q_begin = at.of.q_begin, tok0 = at.tile * a.tokens_per_tile;
    const int tokens = min(a.tokens_per_tile, at.of.q_len - tok0);
    const int rows = tokens * a.heads_per_tile;
    const int first_pos = at.of.ctx - at.of.q_len + tok0, last_pos = first_pos + tokens - 1;
    int hi = last_pos + 1;
    const int lo = a.window > 0 ? max(0, first_pos - a.window + 1) : 0;
    if (hi > (long long)a.table_width * a.page_size) {
        if (lane == 0) oxr_report(a.status, OXR_BAD_PAGE, at.req);
        hi = a.table_width * a.page_size;
    }
    const int block0 = lo / KEYS + max(0, at.block - TILE_COST), blocks_end = min(lo / KEYS + at.block + count - TILE_COST, hi > lo ? (hi + KEYS - 1) / KEYS : 0);
    const int mine = max(0, blocks_end - block0);      // blocks of keys to visit
    const int* table_row = a.block_table + (size_t)at.req * a.table_width;

    // the scale that scales are relative to: the last visible page's
    int base_exp = 0;
    if (hi > lo) {
        const int page = __ldg(table_row + a.page_of(hi - 1));
        if (page >= 0 && page < a.num_pages) {
            const float s = __ldg(a.v_scale + (size_t)page * a.KV + kvh);
            if (s > 0.f && s < INFINITY) base_exp = scale_exponent(s);
        }
    }

    // ---- the keys' way into the ring
    bool bad_page = false;                    // the request's table named one: the result is void
    auto page_for = [&](int i) -> int {       // of this lane's key of the i-th block; -1: nothing to fetch
        const int key = (block0 + i) * KEYS + lane;
        if (i >= mine || key < lo || key >= hi) return -1;
        return __ldg(table_row + a.page_of(key));
    };
    // By TMA a lane sends for one panel of one piece of K or V, and a barrier counts what arrives; the scales of the lane's own key are a copy group.
    auto fetch = [&](int i, int page) {
        if (i < mine) {
            const int key0 = (block0 + i) * KEYS, key = key0 + lane, slot = (turn + i) % STAGES;
            const bool wanted = key >= lo && key < hi, good = wanted && page >= 0 && page < a.num_pages;
            if (wanted && !good) oxr_report(a.status, OXR_BAD_PAGE, at.req);
            if (TMA) bad_page |= __any_sync(0xffffffffu, wanted && !good);
            const uint32_t st = ring + slot * STAGE_BYTES;
            const int place = good ? page : -1;
            if constexpr (TMA) {
                // a piece is on one page: whichever of its keys are wanted name it
                const unsigned some = __ballot_sync(0xffffffffu, good);
                const int pieces = KEYS >> piece_shift, piece = 1 << piece_shift, ops = 2 * PANELS * pieces;
                const unsigned mine = some >> ((lane & (pieces - 1)) << piece_shift) & (0xffffffffu >> (32 - piece));   // of the piece that this lane sends for
                const int there = __popc(__ballot_sync(0xffffffffu, lane < pieces && mine));
                uint64_t* bar = bars + slot;
                if (lane == 0) {
                    if (there) mbar_expect_tx(bar, (uint32_t)(there * piece * 2 * D));
                    else mbar_arrive(bar);
                }
                __syncwarp();
                for (int x0 = 0; x0 < ops; x0 += 32) {
                    const int x = x0 + lane, pc = x & (pieces - 1), of = x >> (5 - piece_shift), pnl = of % PANELS;
                    const bool is_v = of >= PANELS;
                    const int from = __shfl_sync(0xffffffffu, place, pc * piece + (mine ? __ffs(mine) - 1 : 0));
                    if (x < ops && mine)
                        tma_load_3d(smem + (st - smem_addr(smem)) + is_v * TENSOR_BYTES + pnl * KEYS * PW + pc * piece * PW, is_v ? &map_v : &map_k,
                                    kvh * D + pnl * PW, a.in_page(key0 + pc * piece), from, bar);
                }
            } else {
                const long long row = good ? (long long)page * a.page_stride + a.row_in_page(key, kvh) : -1;
#pragma unroll
                for (int c = 0; c < KSTEPS; ++c) {
                    const int chunk = c * 32 + lane, r = chunk / KSTEPS, col = chunk % KSTEPS;
                    const long long from = __shfl_sync(0xffffffffu, row, r);
                    const bool take = from >= 0;
                    const long long off = (take ? from : 0) + col * 16;
                    const uint32_t dst = word_at(st + r * PW ^ row_swizzle(r), col);
                    cp_async16(dst, a.k_cache + off, take);
                    cp_async16(dst + TENSOR_BYTES, a.v_cache + off, take);
                }
            }
            const size_t sc = good ? (size_t)page * a.KV + kvh : 0;      // pools of small pages have more scales than 32 bits count
            const uint32_t scale_at = my_scales + slot * SCALE_BYTES + lane * 4;
            cp_async4(scale_at, a.k_scale + sc, good);
            cp_async4(scale_at + KEYS * 4, a.v_scale + sc, good);
        }
        cp_async_commit();
    };
    int next_page;
    auto prime = [&] {
        next_page = page_for(0);
#pragma unroll
        for (int i = 0; i < STAGES - 1; ++i) {
            const int page = next_page;
            next_page = page_for(i + 1);
            fetch(i, page);
        }
    };
    prime();

    // ---- the queries: lane (g, quad) holds entries 16 c + 4 quad .. + 3 of rows g, g + 8, ...
    uint32_t q_regs[S::Q_IN_REGS ? S::Q_WORDS : 1];
    auto put_q = [&](int word, uint32_t v) {
        if constexpr (S::Q_IN_REGS) q_regs[word] = v;
        else q_smem[word * 32 + lane] = v;      // (a lane reads what it has written)
    };
    float row_factor[NQ][2];       // of rows 2 quad and 2 quad + 1, as the scores come
    uint32_t row_toks = 0u;        // the tokens of rows 2 quad and 2 quad + 1 of each eight, a byte each
    auto row_pos = [&](int nq, int e) { return first_pos + (int)(row_toks >> 8 * (2 * nq + e) & 255u); };
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq) {
        const int r = g + 8 * nq, tok = r / a.heads_per_tile, head = hg * a.heads_per_tile + r % a.heads_per_tile;
        const bool row_ok = r < rows && head < G;   // (rows of the tile without a token or head hold zeros; what they compute goes nowhere)
        const T* src = q + (size_t)(q_begin + tok0 + tok) * a.q_stride + (size_t)(kvh * G + head) * D + 4 * quad;
        float4 v[KSTEPS];
        float most = 0.f;
#pragma unroll
        for (int c = 0; c < KSTEPS; ++c) {
            v[c] = row_ok ? load4(src + 16 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
            most = fmaxf(fmaxf(most, fmaxf(fabsf(v[c].x), fabsf(v[c].y))), fmaxf(fabsf(v[c].z), fabsf(v[c].w)));
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        // a power of two: the largest entry of the row goes to [2^14, 2^15)
        const int shift = (most > 0.f && most < INFINITY) ? min(14 - (int)((__float_as_uint(most) >> 23) & 255) + 127, 126) : 0;
        const float f = __uint_as_float((uint32_t)(shift + 127) << 23);
        const float factor = a.scale * LOG2E * __uint_as_float((uint32_t)(127 - shift) << 23);
#pragma unroll
        for (int c = 0; c < KSTEPS; ++c) {      // word 0: entries 4 quad, + 1; word 1: + 2, + 3
            const float4 x = make_float4(v[c].x * f, v[c].y * f, v[c].z * f, v[c].w * f);
            const uint32_t w0 = pack_f16(x.x, x.y), w1 = pack_f16(x.z, x.w);
            put_q((nq * KSTEPS + c) * 2 * PIECES, w0);
            put_q((nq * KSTEPS + c) * 2 * PIECES + 1, w1);
            if constexpr (PIECES == 2) {
                put_q((nq * KSTEPS + c) * 4 + 2, pack_rest(x.x, x.y, w0));
                put_q((nq * KSTEPS + c) * 4 + 3, pack_rest(x.z, x.w, w1));
            }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            row_factor[nq][e] = __shfl_sync(0xffffffffu, factor, (2 * quad + e) * 4);
            row_toks |= (uint32_t)__shfl_sync(0xffffffffu, tok, (2 * quad + e) * 4) << 8 * (2 * nq + e);
        }
    }
    auto get_q = [&](int word) -> uint32_t {
        if constexpr (S::Q_IN_REGS) return q_regs[word];
        else return q_smem[word * 32 + lane];
    };
    const int last_lo = a.window > 0 ? last_pos - a.window + 1 : 0;   // the latest start of a row's window

    // sums: o[nq][m] holds entries 16 m + 2 g (words 0, 1) and 16 m + 2 g + 1 (words 2, 3) of rows 2 quad and 2 quad + 1
    float o[NQ][KSTEPS][4];
    float m[NQ][2];
    float l[NQ][2];
    short* sum_k = reinterpret_cast<short*>(smem + S::AT_POWERS) + threadIdx.x * 2 * NQ;     // [NQ][2] a careful walk's powers of two of the sums
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq) {
#pragma unroll
        for (int i = 0; i < KSTEPS; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[nq][i][e] = 0.f;
        m[nq][0] = m[nq][1] = -INFINITY;
        l[nq][0] = l[nq][1] = 0.f;
        if constexpr (CAREFUL) sum_k[2 * nq] = sum_k[2 * nq + 1] = 0;
    }

    // the blocks from `first` up to `end`, which are on their way, arrive: before the stages are another's
    auto arrived = [&](int first, int end) {
        bool all = true;
        if constexpr (TMA)
            for (int k = first; k < min(end, mine); ++k) all = mbar_wait(bars + (turn + k) % STAGES, ((turn + k) / STAGES) & 1) && all;
        cp_async_wait<0>();
        return all;
    };
    // ---- the walk
    [[maybe_unused]] int top_exp = -(1 << 20);      // the largest value scale so far, as the power above it
    for (int i = 0; i < mine; ++i) {
        cp_async_wait<STAGES - 2>();
        const int slot = (turn + i) % STAGES;
        if (TMA && !mbar_wait(bars + slot, ((turn + i) / STAGES) & 1)) {
            if (lane == 0) oxr_report(a.status, OXR_WAIT_EXPIRED, 40);
            arrived(i + 1, i + STAGES - 1);
            return -1;
        }
        __syncwarp();
        {   // the stage that the block before this one has left
            const int page = next_page;
            next_page = page_for(i + STAGES);
            fetch(i + STAGES - 1, page);
        }
        const uint32_t st = ring + slot * STAGE_BYTES;
        const float* scales = reinterpret_cast<const float*>(smem + SCALES_AT + (warp * STAGES + slot) * SCALE_BYTES);
        unsigned char* values = smem + (st - smem_addr(smem)) + TENSOR_BYTES;
        const int key0 = (block0 + i) * KEYS;
        const uint32_t seen = __ballot_sync(0xffffffffu, key0 + lane >= lo && key0 + lane < hi);      // by any row
        if constexpr (TMA) {
            // Values that no row sees but that lie in a piece which one does, or in one that was not fetched, become zero: a weight of zero does not
            // undo a NaN. (Their scores are masked whatever the keys hold.)
            if (seen != 0xffffffffu || bad_page) {
                if (!(seen >> lane & 1u) || bad_page) {
#pragma unroll
                    for (int c = 0; c < KSTEPS; ++c) *reinterpret_cast<uint4*>(values + c / (PW / 16) * KEYS * PW + lane * PW + c % (PW / 16) * 16) = make_uint4(0, 0, 0, 0);
                }
                __syncwarp();
            }
        }

        const uint32_t my_vs = __float_as_uint(scales[KEYS + lane]) & 0x7fffffffu;
        uint32_t left_keys = seen;       // to be gone through
        const bool whole = key0 >= last_lo && key0 + KEYS - 1 <= min(first_pos, hi - 1);
        do {
        // (asked for here, looked at behind the scores)
        const bool is_left = left_keys >> lane & 1u;
        const uint32_t most_vs = __reduce_max_sync(0xffffffffu, is_left ? my_vs : 0u), least_vs = __reduce_min_sync(0xffffffffu, is_left ? my_vs : 0xffffffffu);

        // scores: two tiles of 16 keys by 8 rows; c[..][mt]: key 16 mt + g (words 0, 1) and + 8 (words 2, 3) of rows 2 quad and 2 quad + 1
        float c[NQ][2][4];
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int e = 0; e < 4; ++e) c[nq][mt][e] = 0.f;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
            // lanes 0-7, 8-15, 16-23, 24-31 name keys 0-7 and 8-15 at 16-byte word 2 kk and again at 2 kk + 1
            const uint32_t k_row = (st + (16 * mt + (lane & 15)) * PW) ^ row_swizzle(lane & 15) ^ (SWIZZLED ? (lane >> 4) * 16 : 0);
#pragma unroll
            for (int kk = 0; kk < (KSTEPS + 1) / 2; ++kk) {
                uint32_t w[4];
                ldsm4(w, word_at(k_row, 2 * kk) + (!SWIZZLED && 2 * kk + 1 < KSTEPS ? (lane >> 4) * 16 : 0));
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    if (2 * kk + half >= KSTEPS) break;
                    const uint32_t x = w[2 * half], z = w[2 * half + 1];
                    const uint32_t kf[4] = {codes_to_f16(x), codes_to_f16(z), codes_to_f16_high(x), codes_to_f16_high(z)};
#pragma unroll
                    for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
                        for (int pc = 0; pc < PIECES; ++pc) {
                            const int word = ((nq * KSTEPS + 2 * kk + half) * PIECES + pc) * 2;
                            mma_f16(c[nq][mt], kf, get_q(word), get_q(word + 1));
                        }
                }
            }
        }
        // 2^lv: the power above the largest value scale, relative to the last page's scale; `now`: the keys whose scales lie within 2^4 of it
        const bool finite = most_vs < 0x7f800000u;
        const int most_exp = !finite ? base_exp : most_vs ? scale_exponent(__uint_as_float(most_vs)) : 0, lv = most_vs ? most_exp - base_exp : CAREFUL ? NO_SCALE : -60;
        uint32_t now = left_keys;
        if constexpr (!CAREFUL) {
            if (!finite || (most_vs && (least_vs == 0u || most_vs - least_vs > 4u << 23 || lv > 30 || lv < -30 || most_exp < -110))) {
                const bool all = arrived(i + 1, i + STAGES);
                if (!all && lane == 0) oxr_report(a.status, OXR_WAIT_EXPIRED, 40);
                fence_proxy_async();
                __syncwarp();
                turn += min(mine, i + STAGES);
                return all ? item - count : -1;
            }
            left_keys = 0u;
        } else {
            now = __ballot_sync(0xffffffffu, is_left && (finite ? (my_vs > 0u || most_vs == 0u) && most_vs - my_vs <= 4u << 23 : my_vs >= 0x7f800000u));
            left_keys &= ~now;
            if (finite) top_exp = max(top_exp, lv);
        }
        const float lvf = (float)lv;
        float ks[4], vf[4];     // of keys g, g + 8, g + 16, g + 24
        [[maybe_unused]] const float inverse = exp2_of(P_LOG2 - (float)most_exp);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            ks[j] = scales[g + 8 * j];
            const float vs = scales[KEYS + g + 8 * j];
            if constexpr (!CAREFUL) vf[j] = vs * inverse;      // at most 2^15
            else vf[j] = now >> (8 * j + g) & 1u ? times(vs, power_of(P_LOG2 - (float)most_exp)) : 0.f;
        }
        [[maybe_unused]] const float down = CAREFUL ? 0.f : exp2_of(-lvf);
        auto hidden = [&](int nq, int e, int j) {       // key g + 8 j to row 2 quad + e
            const int key = key0 + 8 * j + g, pos = row_pos(nq, e);
            return !(now >> (8 * j + g) & 1u) || key > pos || (a.window > 0 && key <= pos - a.window);
        };
        uint32_t p[NQ][PIECES][2][2];    // weights: [..][key tile][keys 0-7 or 8-15 of it]
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) {
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float& s = c[nq][j >> 1][(j & 1) * 2 + e];
                    s *= row_factor[nq][e] * ks[j];
                }
            if (CAREFUL || !whole) {
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (hidden(nq, e, j)) c[nq][j >> 1][(j & 1) * 2 + e] = -INFINITY;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) mx[e] = fmaxf(mx[e], c[nq][j >> 1][(j & 1) * 2 + e]);
            bool raise = false;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], x));
                raise |= mx[e] + lvf > m[nq][e];
            }
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float n = fmaxf(m[nq][e], ceilf(mx[e] + lvf)), f = n > m[nq][e] ? exp2_of(m[nq][e] - n) : 1.f;
                    if (!CAREFUL) l[nq][e] *= f;
                    else if (n > m[nq][e]) sum_k[2 * nq + e] = (short)max(sum_k[2 * nq + e] + (int)fmaxf(m[nq][e] - n, -2000.f), -2000);
#pragma unroll
                    for (int x = 0; x < KSTEPS; ++x) { o[nq][x][e] *= f; o[nq][x][2 + e] *= f; }
                    m[nq][e] = n;
                }
            }
            // weights: exp2(s - m) carries 2^lv into the products and none of it into the sum
            float off[2], sum[2] = {0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 2; ++e) off[e] = m[nq][e] == -INFINITY ? 0.f : lvf - m[nq][e];
            [[maybe_unused]] int up[2] = {-lv, -lv};
            if (CAREFUL && lv < top_exp - 60) {
                // a row may have met products to which these add nothing, although their weights count: those are taken by themselves
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (mx[e] > -INFINITY && mx[e] + off[e] < -60.f) {
                        off[e] = -ceilf(mx[e]);
                        up[e] = (int)fmaxf(-off[e] - m[nq][e], -1000.f);
                    }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float& w = c[nq][j >> 1][(j & 1) * 2 + e];
                    w = exp2_of(w + off[e]);
                    sum[e] += w;
                    w *= vf[j];
                }
            if constexpr (!CAREFUL) {
                l[nq][0] += sum[0] * down;
                l[nq][1] += sum[1] * down;
            } else {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (up[e] != -lv || hidden(nq, e, j)) c[nq][j >> 1][(j & 1) * 2 + e] = 0.f;      // (a hidden key's scale may be anything)
                    const Sum all = sum_of(whole_of({l[nq][e], sum_k[2 * nq + e]}) + whole_of({sum[e], up[e]}));
                    l[nq][e] = all.f;
                    sum_k[2 * nq + e] = (short)all.k;
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float w0 = c[nq][j >> 1][(j & 1) * 2], w1 = c[nq][j >> 1][(j & 1) * 2 + 1];
                const uint32_t packed = pack_f16(w0, w1);
                p[nq][0][j >> 1][j & 1] = transposed(packed);
                if constexpr (PIECES == 2) p[nq][PIECES - 1][j >> 1][j & 1] = transposed(pack_rest(w0, w1, packed));
            }
        }

        // o += values x weights. Lanes 0-7 and 8-15 of an ldmatrix name keys 0-7 and 8-15 of a tile at 16-byte word n, lanes 16-31 the same keys at word
        // n + 1 (or, for an odd number of words, at the last one again). Bytes of keys 2 quad and 2 quad + 1 at entries 2 g and 2 g + 1 come
        // back: in another order they are the pairs of rows g and g + 8 of a left operand whose rows g are the even and g + 8 the odd entries.
        const uint32_t v_row = (st + TENSOR_BYTES + (lane & 15) * PW) ^ row_swizzle(lane & 15);
        bool apart = false;
        if (!whole && tokens > 1) {   // a NaN among the values must not reach the rows that do not see it
            bool nan = false;
            for (int x = lane; x < KEYS * D / 4; x += 32) {
                const uint32_t w = *reinterpret_cast<const uint32_t*>(values + x * 4);
                nan |= __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu) != 0;
            }
            apart = __any_sync(0xffffffffu, nan);
        }
        if (!apart) {
#pragma unroll
            for (int n = 0; n < KSTEPS; n += 2) {
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    uint32_t w[4];
                    ldsm4_trans(w, word_at(v_row ^ (SWIZZLED ? (lane >> 4) * 16 : 0), n) + s * 16 * PW + (!SWIZZLED && n + 1 < KSTEPS ? (lane >> 4) * 16 : 0));
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        if (n + half >= KSTEPS) break;
                        const uint32_t x = __byte_perm(w[2 * half], 0, 0x3120), z = __byte_perm(w[2 * half + 1], 0, 0x3120);
                        const uint32_t vt[4] = {codes_to_f16(x), codes_to_f16_high(x), codes_to_f16(z), codes_to_f16_high(z)};
#pragma unroll
                        for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
                            for (int pc = 0; pc < PIECES; ++pc) mma_f16(o[nq][n + half], vt, p[nq][pc][s][0], p[nq][pc][s][1]);
                    }
                }
            }
        } else {
            // one pass per token of the tile with the keys that it does not see taken out; its rows alone keep the result
            for (int tk = 0; tk < tokens; ++tk) {
                const int pos = first_pos + tk, from = a.window > 0 ? pos - a.window + 1 : 0;
                uint32_t keep[2][2];
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int key = key0 + 16 * s + 8 * e + 2 * quad;
                        keep[s][e] = (key <= pos && key >= from ? 0x00ff00ffu : 0u) | (key + 1 <= pos && key + 1 >= from ? 0xff00ff00u : 0u);
                    }
#pragma unroll
                for (int n = 0; n < KSTEPS; ++n) {
#pragma unroll
                    for (int nq = 0; nq < NQ; ++nq) {
                        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int s = 0; s < 2; ++s) {
                            uint32_t w[4];
                            ldsm4_trans(w, word_at(v_row, n) + s * 16 * PW);
                            const uint32_t x = __byte_perm(w[0], 0, 0x3120) & keep[s][0], z = __byte_perm(w[1], 0, 0x3120) & keep[s][1];
                            const uint32_t vt[4] = {codes_to_f16(x), codes_to_f16_high(x), codes_to_f16(z), codes_to_f16_high(z)};
#pragma unroll
                            for (int pc = 0; pc < PIECES; ++pc) mma_f16(sum, vt, p[nq][pc][s][0], p[nq][pc][s][1]);
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (row_pos(nq, e & 1) == pos) o[nq][n][e] += sum[e];
                    }
                }
            }
        }
        } while (CAREFUL && left_keys);
        fence_proxy_async();   // every lane has read the stage before the next turn's copies fill it
        __syncwarp();
    }
    turn += mine;

    // ---- the tile's result, or what this warp has of it
    const bool whole_tile = at.block == 0 && count == at.of.blocks;
    if (at.block == 0 && !whole_tile)
        cut = {(item - count + at.of.blocks - 1) / share, q_begin + tok0, kvh * G + hg * a.heads_per_tile, rows, min(a.heads_per_tile, G - hg * a.heads_per_tile), base_exp, {0, 0}};
    const size_t place = (size_t)2 * me + (at.block == 0 ? 1 : 0);
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            Sum total = {l[nq][e], 0};      // (every lane of a row has the same m)
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) total.f += __shfl_xor_sync(0xffffffffu, total.f, x);
            if constexpr (CAREFUL) {
                double all = whole_of({l[nq][e], sum_k[2 * nq + e]});
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) all += __shfl_xor_sync(0xffffffffu, all, x);
                total = sum_of(all);
            }
            const int r = 8 * nq + 2 * quad + e, tok = r / a.heads_per_tile, head = hg * a.heads_per_tile + r % a.heads_per_tile;
            if (r >= rows || head >= G) continue;
            if (whole_tile) {
                const bool none = total.f == 0.f;
                const Power unit = final_unit(total, base_exp);
                const float f = 1.f / total.f * unit.a;
                T* row = out + ((size_t)(q_begin + tok0 + tok) * a.H + (size_t)kvh * G + head) * D + 2 * g;
#pragma unroll
                for (int n = 0; n < KSTEPS; ++n)
                    store2(row + 16 * n, none ? make_float2(0.f, 0.f) : make_float2(o[nq][n][e] * f * unit.b, o[nq][n][2 + e] * f * unit.b));
            } else {
                // (all pieces of a tile are relative to the same scale)
                if (g == 0) {
                    left.rows[place * ROWS + r] = {m[nq][e], total.k != 0 ? -total.f : fabsf(total.f)};
                    if (total.k != 0) left.powers[place * ROWS + r] = total.k;
                }
                float* row = left.sums + (place * ROWS + r) * D + 2 * g;
#pragma unroll
                for (int n = 0; n < KSTEPS; ++n) *reinterpret_cast<float2*>(row + 16 * n) = make_float2(o[nq][n][e], o[nq][n][2 + e]);
            }
        }
    __syncwarp();
    }
    return item;
    };
    int item = stretch((int)min(all, (long long)me * share), std::false_type{});
    if (item >= 0 && item < end) item = stretch(item, std::true_type{});
    if (lane == 0) {
        if (item < 0) cut.last = -1;      // nothing of this stretch is to be joined
        left.cuts[me] = cut;
    }
}

// Joins the pieces of the tiles that lie in more than one warp's stretch. A block looks at some of the stretches and, of each that ends in a tile
// which began in it, takes eight rows of the tile. A thread has four entries of a row; where the rows leave threads over, they take the pieces in turn.
constexpr int JOIN_THREADS = 256, JOIN_ROWS = D <= 128 ? 8 : 4, JOIN_BLOCKS = 592;
template <typename T, int NQ>
__global__ void __launch_bounds__(JOIN_THREADS, 3) attn_kv8_join_kernel(T* __restrict__ out, const Pieces left, const int warps, const int H, const int heads_per_tile) {
    constexpr int ROWS = 8 * NQ, WORDS = D / 4;
    __shared__ float4 sums[JOIN_THREADS];
    __shared__ RowSum rows[JOIN_THREADS];
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, r0 = (int)blockIdx.y * JOIN_ROWS;
    for (int w0 = blockIdx.x; w0 < warps; w0 += 32 * (int)gridDim.x) {
        const int mine = w0 + lane * (int)gridDim.x;
        for (unsigned valid = __ballot_sync(0xffffffffu, mine < warps && __ldcg(&left.cuts[mine < warps ? mine : 0].last) >= 0); valid; valid &= valid - 1) {
            const int first = w0 + (__ffs(valid) - 1) * (int)gridDim.x;       // the same in every warp
            const int4 c0 = __ldcg(reinterpret_cast<const int4*>(left.cuts + first)), c1 = __ldcg(reinterpret_cast<const int4*>(left.cuts + first) + 1);
            const Cut cut = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, {0, 0}};
            if (r0 >= cut.rows) continue;
            const int all = min(JOIN_ROWS, cut.rows - r0) * WORDS;
            int ways = 1;      // threads that share an entry's pieces
            while (ways * 2 * all <= JOIN_THREADS) ways *= 2;
            const int x = threadIdx.x % all, way = threadIdx.x / all, r = r0 + x / WORDS, d = x % WORDS * 4;
            RowSum s = {-INFINITY, 0.f};
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (way < ways) {
                for (int p0 = first + way; p0 <= cut.last; p0 += 8 * ways) {     // eight pieces at a time
                    RowSum y[8];
                    float4 u[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int w = p0 + k * ways;
                        const size_t at = ((size_t)2 * w + (w == first ? 1 : 0)) * ROWS + r;
                        const float2 ml = w <= cut.last ? __ldcg(reinterpret_cast<const float2*>(left.rows + at)) : make_float2(-INFINITY, 0.f);
                        y[k] = {ml.x, ml.y};
                        u[k] = w <= cut.last ? __ldcg(reinterpret_cast<const float4*>(left.sums + at * D + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
                    }
                    add_pieces(s, v, y, u);
                }
            }
            if (ways > 1) {
                sums[threadIdx.x] = v;
                rows[threadIdx.x] = s;
                __syncthreads();
                if (way == 0)
                    for (int k = 1; k < ways; ++k) {
                        const RowSum y[1] = {rows[k * all + x]};
                        const float4 u[1] = {sums[k * all + x]};
                        add_pieces(s, v, y, u);
                    }
                __syncthreads();
            }
            const int head = r % heads_per_tile;
            if (way == 0 && head < cut.heads) {
                Sum total = {s.total, 0};
                if (s.total < 0.f) {      // again, with the powers
                    double all = 0.;
#pragma unroll 1
                    for (int w = first; w <= cut.last; ++w) {
                        const size_t at = ((size_t)2 * w + (w == first ? 1 : 0)) * ROWS + r;
                        const float2 ml = __ldcg(reinterpret_cast<const float2*>(left.rows + at));
                        const int k = ml.y < 0.f ? __ldcg(left.powers + at) : 0;
                        all += whole_of({fabsf(ml.y), k + (ml.x == s.m ? 0 : (int)fmaxf(ml.x - s.m, -2000.f))});
                    }
                    total = sum_of(all);
                }
                const Power unit = final_unit(total, cut.base_exp);
                const float f = 1.f / total.f * unit.a;
                float4 z = make_float4(v.x * f * unit.b, v.y * f * unit.b, v.z * f * unit.b, v.w * f * unit.b);
                if (total.f == 0.f) z = make_float4(0.f, 0.f, 0.f, 0.f);
                store4(out + ((size_t)(cut.token + r / heads_per_tile) * H + cut.head + head) * D + d, z);
            }
        }
    }
}
static_assert(JOIN_ROWS * D / 4 <= JOIN_THREADS, "a thread for every entry of the rows that a block takes");

// A pool of pages seen as boxes of `piece` keys x PW bytes of one KV head.
bool make_map(CUtensorMap* map, const void* base, const Kv8Args& a, int piece) {
    OxrEncodeTiledFn fn = oxr_encode_tiled();
    if (fn == nullptr) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)a.KV * D, (cuuint64_t)a.page_size, (cuuint64_t)a.num_pages};
    const cuuint64_t strides[2] = {(cuuint64_t)a.KV * D, (cuuint64_t)a.page_stride};
    const cuuint32_t box[3] = {(cuuint32_t)PW, (cuuint32_t)piece, 1u};
    const cuuint32_t elem[3] = {1, 1, 1};
    const CUtensorMapSwizzle swizzle = !SWIZZLED ? CU_TENSOR_MAP_SWIZZLE_NONE : PW == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : PW == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B;
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
              CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, bool TMA, int NQ>
int allow() {   // once per device and thread: the shared memory of the kernel
    static thread_local int ready = -1;
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return oxr_launch_status();
    if (ready == device) return 0;
    if (cudaFuncSetAttribute(attn_kv8_kernel<T, TMA, NQ>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Shape<T, NQ>::SMEM) != cudaSuccess) return oxr_launch_status();
    ready = device;
    return 0;
}

template <typename T, int NQ>
int launch(void* out, const void* q, const Kv8Args& a, int blocks, float* scratch, cudaStream_t stream) {
    int piece_shift = 0;
    while (piece_shift < 5 && a.page_size % (2 << piece_shift) == 0) ++piece_shift;
    CUtensorMap map_k = {}, map_v = {};
    const bool tma = piece_shift >= 3 && a.num_pages > 0 && make_map(&map_k, a.k_cache, a, 1 << piece_shift) && make_map(&map_v, a.v_cache, a, 1 << piece_shift);
    const int code = tma ? allow<T, true, NQ>() : allow<T, false, NQ>();
    if (code != 0) return code;
    const int warps = blocks * WARPS;
    RowSum* rows = reinterpret_cast<RowSum*>(scratch + (size_t)2 * warps * 8 * NQ * D);
    int* powers = reinterpret_cast<int*>(rows + (size_t)2 * warps * 8 * NQ);
    const Pieces left = {scratch, rows, powers, reinterpret_cast<Cut*>(powers + (size_t)2 * warps * 8 * NQ)};
    const dim3 grid(blocks), threads(THREADS);
    if (tma) oxr_launch(attn_kv8_kernel<T, true, NQ>, grid, threads, Shape<T, NQ>::SMEM, stream, true, (T*)out, (const T*)q, map_k, map_v, piece_shift, a, left);
    else oxr_launch(attn_kv8_kernel<T, false, NQ>, grid, threads, Shape<T, NQ>::SMEM, stream, true, (T*)out, (const T*)q, map_k, map_v, piece_shift, a, left);
    const dim3 join(warps < JOIN_BLOCKS ? warps : JOIN_BLOCKS, 8 * NQ / JOIN_ROWS);
    oxr_launch(attn_kv8_join_kernel<T, NQ>, join, dim3(JOIN_THREADS), 0, stream, true, (T*)out, left, warps, a.H, a.heads_per_tile);
    return oxr_launch_status();
}
}  // namespace

OXR_API void oxr_set_chain(int on) { oxr_chain_kernels = on; }
OXR_API int oxr_kv8_head_dim() { return D; }
// Blocks (of four warps) of the split-key kernel that an SM holds.
OXR_API int oxr_kv8_blocks_per_sm(int dtype, int tile_rows) {
    return tile_rows == 8 ? (dtype == 0 ? Shape<float, 1>::BLOCKS : Shape<__nv_bfloat16, 1>::BLOCKS) : (dtype == 0 ? Shape<float, 2>::BLOCKS : Shape<__nv_bfloat16, 2>::BLOCKS);
}

OXR_API int oxr_kv8_attention(const Kv8Call* c) {
    if (!kv8_call_ok(*c) || c->blocks < 1 || c->blocks > 65536 || c->scratch == nullptr || (c->tile_rows != 8 && c->tile_rows != 16)) return OXR_BAD_ARGUMENT;
    if (c->n == 0 || c->n_tokens == 0) return 0;
    const Kv8Args a = kv8_args(*c, c->tile_rows);
    if (c->tile_rows == 8)
        return c->dtype == 0 ? launch<float, 1>(c->out, c->q, a, c->blocks, c->scratch, c->stream) : launch<__nv_bfloat16, 1>(c->out, c->q, a, c->blocks, c->scratch, c->stream);
    return c->dtype == 0 ? launch<float, 2>(c->out, c->q, a, c->blocks, c->scratch, c->stream) : launch<__nv_bfloat16, 2>(c->out, c->q, a, c->blocks, c->scratch, c->stream);
}
