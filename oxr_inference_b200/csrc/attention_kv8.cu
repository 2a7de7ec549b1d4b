// Paged grouped-query attention over a cache of 8-bit floating-point numbers (e4m3) with one scale for each page and KV head. Compiled once
// per head size: -DHEAD_DIM=<multiple of 16, at most 256>.
//
// A cached key is ks * K and a cached value vs * V, with e4m3 codes K, V and the fp32 scales of the page that holds them. A query q at position p
// of its request sees the keys j <= p (j > p - window behind a window):
//     s_j = scale * ks_j * (q . K_j),     o = sum_j exp(s_j) vs_j V_j / sum_j exp(s_j).
//
// Every e4m3 number is an fp16 number, so the codes go through the tensor cores as they are (mma.sync m16n8k16, fp16 operands, fp32 sums; a
// pair of codes costs one conversion, 64 lanes a clock) and both scales stay outside the products: ks multiplies the fp32 score, vs the weight.
// A bf16 query is an fp16 number too once its row is multiplied by a power of two that brings its largest entry to 2^14 (entries 2^-39
// below that are lost); an fp32 query is the sum of two fp16 numbers to 22 bits. The weights are rounded to fp16 (11 bits) against the row's
// running maximum, times 2^15 so that they keep their bits down to 2^-29 of it; with fp32 queries they too are two numbers.
//
// The weights of a block of keys are taken against the maximum of s_j + log2(vs) instead of s_j: weights times scales then never exceed one
// however much the scales of pages differ, and a rescaled sum needs nothing but the usual factor. (log2(vs) stands for the integer 2^lv >= the
// block's largest scale, relative to the scale of the last page, so that neither sums nor weights leave the fp32 range.)
//
// Each warp walks over blocks of 32 keys of its own: a ring of three stages filled with cp.async, one online softmax per warp, no block-wide barrier
// until the end, where the warps' results are joined in shared memory and those of the blocks of a cluster (which share one request's keys when
// there are few requests) through distributed shared memory. What bounds it is reading the cache: 2 D bytes per key and KV head.
#include <cuda_fp16.h>

#include "tma.cuh"

#ifndef HEAD_DIM
#error "compile with -DHEAD_DIM=<head size>"
#endif
static_assert(HEAD_DIM % 16 == 0 && HEAD_DIM >= 16 && HEAD_DIM <= 256, "head size: a multiple of 16 up to 256");

#include "attention_kv8.cuh"

namespace {
constexpr int ROWS = 16;                       // rows of a tile: (token, query head) pairs of one KV head
constexpr int WARPS = 4;
constexpr int THREADS = WARPS * 32;
constexpr int KEYS = 32;                       // keys of a block: one per lane while addresses are worked out
constexpr int STAGES = D <= 64 ? 4 : 3;
constexpr int PITCH = (D / 16) % 2 ? D : D + 16;   // bytes from key to key: an odd number of 16-byte words, so that eight rows lie on different banks
constexpr int STAGE_BYTES = 2 * KEYS * PITCH + 2 * KEYS * 4;
constexpr int KSTEPS = D / 16;
constexpr int RING_BYTES = WARPS * STAGES * STAGE_BYTES;
constexpr int PART_BYTES = ROWS * D * 4;       // a warp's sums when they are joined: they take the place of its ring
static_assert(PART_BYTES <= STAGES * STAGE_BYTES, "the sums of a warp fit into its ring");
constexpr float P_FACTOR = 32768.f;            // weights are kept as 2^15 w

template <int PIECES> __host__ __device__ constexpr bool q_in_regs() { return PIECES * D <= 256; }
template <int PIECES> constexpr size_t smem_bytes() {
    return RING_BYTES + WARPS * ROWS * 8 + ROWS * 8 + (q_in_regs<PIECES>() ? 0 : PIECES * KSTEPS * 512);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool take) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
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
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t map_to_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float2 ld_cluster_f2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
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
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// What rounding a pair to fp16 left over, as fp16 again.
__device__ __forceinline__ uint32_t pack_rest(float lo, float hi, uint32_t packed) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&packed));
    return pack_f16(lo - f.x, hi - f.y);
}

// One tile of ROWS rows. The walk over the keys is cut between the blocks of a cluster (`splits` of them) and their warps.
template <typename T>
__global__ void __launch_bounds__(THREADS, D <= 128 ? 2 : 1)
attn_kv8_kernel(T* __restrict__ out, const T* __restrict__ q, const Kv8Args a, const int splits) {
    constexpr int PIECES = sizeof(T) == 4 ? 2 : 1;
    constexpr bool QREG = q_in_regs<PIECES>();
    extern __shared__ __align__(16) unsigned char smem[];
    float2* warp_ml = reinterpret_cast<float2*>(smem + RING_BYTES);            // [WARPS][ROWS] running maximum and sum
    float2* block_ml = warp_ml + WARPS * ROWS;                                // [ROWS]
    [[maybe_unused]] uint4* q_smem = reinterpret_cast<uint4*>(block_ml + ROWS);   // [PIECES][KSTEPS][32 lanes]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, quad = lane & 3;
    pdl_wait();
    pdl_trigger();

    // ---- which rows
    const int unit = (int)(blockIdx.x / (unsigned)splits), rank = splits > 1 ? (int)cluster_rank() : 0;
    const int per_tile = a.KV * a.head_groups;
    const int y = unit % per_tile, kvh = y / a.head_groups, hg = y % a.head_groups;
    const Kv8Tile t = kv8_find_tile(a, unit / per_tile, a.tokens_per_tile, unit == 0);
    if (t.req < 0) return;                    // the same for every block of a cluster
    const int q_len = t.q_len, tok0 = t.tok0;
    const int tokens = min(a.tokens_per_tile, q_len - tok0);
    const int ctx = __ldg(a.ctx_lens + t.req), pos0 = ctx - q_len;   // position of the request's first new token
    const int rows = tokens * a.heads_per_tile;
    const int G = a.H / a.KV;
    const int first_pos = pos0 + tok0, last_pos = first_pos + tokens - 1;
    int hi = last_pos + 1;
    const int lo = a.window > 0 ? max(0, first_pos - a.window + 1) : 0;
    if (hi > (long long)a.table_width * a.page_size) {
        if (threadIdx.x == 0) oxr_report(a.status, OXR_BAD_PAGE, t.req);
        hi = a.table_width * a.page_size;
    }
    const int block0 = max(lo, 0) / KEYS, blocks = hi > lo ? (hi + KEYS - 1) / KEYS - block0 : 0;
    const int* table_row = a.block_table + (size_t)t.req * a.table_width;
    const int walkers = splits * WARPS, me = rank * WARPS + warp;

    // the scale that scales are relative to: the last visible page's
    int base_exp = 0;
    if (blocks > 0) {
        const int page = __ldg(table_row + a.page_of(hi - 1));
        if (page >= 0 && page < a.num_pages) {
            const float s = __ldg(a.v_scale + (size_t)page * a.KV + kvh);
            if (s > 0.f && s < INFINITY) base_exp = scale_exponent(s);
        }
    }

    // ---- the keys' way into the ring
    const uint32_t ring = smem_addr(smem) + warp * STAGES * STAGE_BYTES;
    auto page_for = [&](int i) -> int {       // of this lane's key of the warp's i-th block; -1: nothing to fetch
        const int key = (block0 + me + i * walkers) * KEYS + lane;
        if (me + i * walkers >= blocks || key < lo || key >= hi) return -1;
        return __ldg(table_row + a.page_of(key));
    };
    auto fetch = [&](int i, int page) {
        if (me + i * walkers < blocks) {
            const int key = (block0 + me + i * walkers) * KEYS + lane;
            const bool wanted = key >= lo && key < hi, good = wanted && page >= 0 && page < a.num_pages;
            if (wanted && !good) oxr_report(a.status, OXR_BAD_PAGE, t.req);
            const long long row = good ? (long long)page * a.page_stride + ((long long)a.in_page(key) * a.KV + kvh) * D : -1;
            const uint32_t st = ring + (i % STAGES) * STAGE_BYTES;
#pragma unroll
            for (int c = 0; c < KSTEPS; ++c) {
                const int chunk = c * 32 + lane, r = chunk / KSTEPS, col = chunk % KSTEPS;
                const long long at = __shfl_sync(0xffffffffu, row, r);
                const bool take = at >= 0;
                const long long off = (take ? at : 0) + col * 16;
                cp_async16(st + r * PITCH + col * 16, a.k_cache + off, take);
                cp_async16(st + (KEYS + r) * PITCH + col * 16, a.v_cache + off, take);
            }
            const size_t sc = good ? (size_t)page * a.KV + kvh : 0;
            cp_async4(st + 2 * KEYS * PITCH + lane * 4, a.k_scale + sc, good);
            cp_async4(st + 2 * KEYS * PITCH + (KEYS + lane) * 4, a.v_scale + sc, good);
        }
        cp_async_commit();
    };
    int next_page = page_for(0);
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) {
        const int page = next_page;
        next_page = page_for(i + 1);
        fetch(i, page);
    }

    // ---- the queries: rows g and g + 8 of the tile, entries 16 kk + 4 quad .. + 3
    bool row_ok[2];
    int row_pos[2];
    float row_factor[2];
    uint32_t qa[QREG ? PIECES : 1][QREG ? KSTEPS : 1][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = g + 8 * h, tok = r / a.heads_per_tile, head = hg * a.heads_per_tile + r % a.heads_per_tile;
        row_ok[h] = r < rows && head < G;
        row_pos[h] = first_pos + tok;
        const T* src = q + (size_t)(t.q_begin + tok0 + tok) * a.q_stride + (size_t)(kvh * G + head) * D + 4 * quad;
        float4 v[KSTEPS];
        float most = 0.f;
#pragma unroll
        for (int kk = 0; kk < KSTEPS; ++kk) {
            v[kk] = row_ok[h] ? load4(src + 16 * kk) : make_float4(0.f, 0.f, 0.f, 0.f);
            most = fmaxf(fmaxf(most, fmaxf(fabsf(v[kk].x), fabsf(v[kk].y))), fmaxf(fabsf(v[kk].z), fabsf(v[kk].w)));
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        // a power of two: the largest entry of the row goes to [2^14, 2^15)
        const int shift = (most > 0.f && most < INFINITY) ? min(14 - (int)((__float_as_uint(most) >> 23) & 255) + 127, 126) : 0;
        const float f = __uint_as_float((uint32_t)(shift + 127) << 23);
        row_factor[h] = a.scale * LOG2E * __uint_as_float((uint32_t)(127 - shift) << 23);
#pragma unroll
        for (int kk = 0; kk < KSTEPS; ++kk) {
            const uint32_t x = pack_f16(v[kk].x * f, v[kk].y * f), z = pack_f16(v[kk].z * f, v[kk].w * f);
            uint32_t* q0 = QREG ? qa[0][QREG ? kk : 0] : reinterpret_cast<uint32_t*>(q_smem + kk * 32 + lane);
            if (QREG || warp == 0) { q0[h] = x; q0[h + 2] = z; }
            if constexpr (PIECES == 2) {
                uint32_t* q1 = QREG ? qa[PIECES - 1 < (QREG ? PIECES : 1) ? PIECES - 1 : 0][QREG ? kk : 0] : reinterpret_cast<uint32_t*>(q_smem + (KSTEPS + kk) * 32 + lane);
                if (QREG || warp == 0) { q1[h] = pack_rest(v[kk].x * f, v[kk].y * f, x); q1[h + 2] = pack_rest(v[kk].z * f, v[kk].w * f, z); }
            }
        }
    }
    if constexpr (!QREG) __syncthreads();
    const int row_lo0 = a.window > 0 ? row_pos[0] - a.window + 1 : 0, row_lo1 = a.window > 0 ? row_pos[1] - a.window + 1 : 0;
    const int last_lo = a.window > 0 ? last_pos - a.window + 1 : 0;   // the latest start of a row's window
    // (rows of the tile without a token or head hold zeros; what they compute goes nowhere)

    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    // ---- the walk
    const int mine = blocks > me ? (blocks - me + walkers - 1) / walkers : 0;
    for (int i = 0; i < mine; ++i) {
        cp_async_wait<STAGES - 2>();
        __syncwarp();
        {   // the stage that the block before this one has left
            const int page = next_page;
            next_page = page_for(i + STAGES);
            fetch(i + STAGES - 1, page);
        }
        const uint32_t st = ring + (i % STAGES) * STAGE_BYTES;
        const float* scales = reinterpret_cast<const float*>(smem + (st - smem_addr(smem)) + 2 * KEYS * PITCH);
        const int key0 = (block0 + me + i * walkers) * KEYS;

        // scores: four tiles of 8 keys
        float c[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) c[j][e] = 0.f;
        const uint32_t k_addr = st + lane * PITCH;
#pragma unroll
        for (int kk = 0; kk < KSTEPS; ++kk) {
            uint32_t w[4];
            ldsm4(w, k_addr + kk * 16);
            uint32_t b[4][2];
#pragma unroll
            for (int j = 0; j < 4; ++j) { b[j][0] = codes_to_f16(w[j]); b[j][1] = codes_to_f16(w[j] >> 16); }
#pragma unroll
            for (int pc = 0; pc < PIECES; ++pc) {
                uint32_t qf[4];
                if constexpr (QREG) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) qf[e] = qa[pc][kk][e];
                } else {
                    const uint4 v = q_smem[(pc * KSTEPS + kk) * 32 + lane];
                    qf[0] = v.x; qf[1] = v.y; qf[2] = v.z; qf[3] = v.w;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) mma_f16(c[j], qf, b[j][0], b[j][1]);
            }
        }
        // the largest value scale of the block as a power of two, relative to the last page's
        const float my_vs = scales[KEYS + lane];
        const uint32_t most_vs = __reduce_max_sync(0xffffffffu, (my_vs > 0.f && my_vs < INFINITY) ? __float_as_uint(my_vs) : 0u);
        const int lv = most_vs ? scale_exponent(__uint_as_float(most_vs)) - base_exp : 0;
        const float lvf = (float)lv;
        const float v_inverse = exp2_of(-(float)(lv + base_exp));
        // (c0, c1) row g, (c2, c3) row g + 8; keys 8 j + 2 quad, + 1
        float mx0 = -INFINITY, mx1 = -INFINITY;
        const bool whole = key0 >= last_lo && key0 + KEYS - 1 <= min(first_pos, hi - 1);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 ks = *reinterpret_cast<const float2*>(scales + 8 * j + 2 * quad);
            c[j][0] *= row_factor[0] * ks.x; c[j][1] *= row_factor[0] * ks.y;
            c[j][2] *= row_factor[1] * ks.x; c[j][3] *= row_factor[1] * ks.y;
            if (!whole) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int key = key0 + 8 * j + 2 * quad + e;
                    if (key > row_pos[0] || key < row_lo0 || key >= hi) c[j][e] = -INFINITY;
                    if (key > row_pos[1] || key < row_lo1 || key >= hi) c[j][2 + e] = -INFINITY;
                }
            }
            mx0 = fmaxf(mx0, fmaxf(c[j][0], c[j][1]));
            mx1 = fmaxf(mx1, fmaxf(c[j][2], c[j][3]));
        }
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
        const float n0 = fmaxf(m[0], mx0 + lvf), n1 = fmaxf(m[1], mx1 + lvf);
        if (__any_sync(0xffffffffu, n0 > m[0] || n1 > m[1])) {
            const float a0 = n0 > m[0] ? exp2_of(m[0] - n0) : 1.f, a1 = n1 > m[1] ? exp2_of(m[1] - n1) : 1.f;
            l[0] *= a0; l[1] *= a1;
#pragma unroll
            for (int x = 0; x < D / 8; ++x) { o[x][0] *= a0; o[x][1] *= a0; o[x][2] *= a1; o[x][3] *= a1; }
            m[0] = n0; m[1] = n1;
        }
        // weights: exp2(s - m) carries 2^lv into the products and none of it into the sum
        const float off0 = m[0] == -INFINITY ? 0.f : lvf - m[0], off1 = m[1] == -INFINITY ? 0.f : lvf - m[1];
        float sum0 = 0.f, sum1 = 0.f;
        uint32_t p[PIECES][2][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 vs = *reinterpret_cast<const float2*>(scales + KEYS + 8 * j + 2 * quad);
            const float f0 = vs.x * v_inverse * P_FACTOR, f1 = vs.y * v_inverse * P_FACTOR;   // at most 2^15
            float w0 = exp2_of(c[j][0] + off0), w1 = exp2_of(c[j][1] + off0), w2 = exp2_of(c[j][2] + off1), w3 = exp2_of(c[j][3] + off1);
            sum0 += w0 + w1;
            sum1 += w2 + w3;
            w0 *= f0; w1 *= f1; w2 *= f0; w3 *= f1;
            if (!whole) {   // a hidden key's scale may be anything
                if (c[j][0] == -INFINITY) w0 = 0.f;
                if (c[j][1] == -INFINITY) w1 = 0.f;
                if (c[j][2] == -INFINITY) w2 = 0.f;
                if (c[j][3] == -INFINITY) w3 = 0.f;
            }
            p[0][j >> 1][(j & 1) * 2] = pack_f16(w0, w1);
            p[0][j >> 1][(j & 1) * 2 + 1] = pack_f16(w2, w3);
            if constexpr (PIECES == 2) {
                p[PIECES - 1][j >> 1][(j & 1) * 2] = pack_rest(w0, w1, p[0][j >> 1][(j & 1) * 2]);
                p[PIECES - 1][j >> 1][(j & 1) * 2 + 1] = pack_rest(w2, w3, p[0][j >> 1][(j & 1) * 2 + 1]);
            }
        }
        const float down = exp2_of(-lvf);
        l[0] += sum0 * down;
        l[1] += sum1 * down;

        // o += weights V. Lanes 0-7 / 8-15 of an ldmatrix name keys 16 s .. + 7 / 8 .. 15 at entries 16 n, lanes 16-31 the same keys 16 entries on
        // (or, for an odd number of 16-entry columns, at the last one again).
        const uint32_t v_addr = st + (KEYS + (lane & 15)) * PITCH;
        bool apart = false;
        if (!whole && tokens > 1) {   // a NaN among the values must not reach the rows that do not see it
            bool nan = false;
            for (int x = lane; x < KEYS * D / 4; x += 32) {
                const uint32_t w = *reinterpret_cast<const uint32_t*>(smem + (st - smem_addr(smem)) + (KEYS + x / (D / 4)) * PITCH + x % (D / 4) * 4);
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
                    ldsm4_trans(w, v_addr + s * 16 * PITCH + (n + 1 < KSTEPS ? n + (lane >> 4) : n) * 16);
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        if (n + half >= KSTEPS) break;
                        const uint32_t x = __byte_perm(w[2 * half], 0, 0x3120), z = __byte_perm(w[2 * half + 1], 0, 0x3120);
#pragma unroll
                        for (int pc = 0; pc < PIECES; ++pc) {
                            mma_f16(o[2 * (n + half)], p[pc][s], codes_to_f16(x), codes_to_f16(z));
                            mma_f16(o[2 * (n + half) + 1], p[pc][s], codes_to_f16(x >> 16), codes_to_f16(z >> 16));
                        }
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
                const bool take0 = row_pos[0] == pos, take1 = row_pos[1] == pos;
#pragma unroll
                for (int n = 0; n < KSTEPS; ++n) {
                    float even[4] = {0.f, 0.f, 0.f, 0.f}, odd[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        uint32_t w[4];
                        ldsm4_trans(w, v_addr + s * 16 * PITCH + n * 16);
                        const uint32_t x = __byte_perm(w[0], 0, 0x3120) & keep[s][0], z = __byte_perm(w[1], 0, 0x3120) & keep[s][1];
#pragma unroll
                        for (int pc = 0; pc < PIECES; ++pc) {
                            mma_f16(even, p[pc][s], codes_to_f16(x), codes_to_f16(z));
                            mma_f16(odd, p[pc][s], codes_to_f16(x >> 16), codes_to_f16(z >> 16));
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (e < 2 ? take0 : take1) { o[2 * n][e] += even[e]; o[2 * n + 1][e] += odd[e]; }
                }
            }
        }
        __syncwarp();   // every lane has read the stage before the next turn fills it
    }
    cp_async_wait<0>();

    // ---- join: warps in shared memory, then blocks of the cluster
    l[0] += __shfl_xor_sync(0xffffffffu, l[0], 1);
    l[1] += __shfl_xor_sync(0xffffffffu, l[1], 1);
    l[0] += __shfl_xor_sync(0xffffffffu, l[0], 2);
    l[1] += __shfl_xor_sync(0xffffffffu, l[1], 2);
    __syncwarp();
    float* part = reinterpret_cast<float*>(smem + (size_t)warp * STAGES * STAGE_BYTES);   // [ROWS][D]
#pragma unroll
    for (int n = 0; n < KSTEPS; ++n) {
        if (g < rows) *reinterpret_cast<float4*>(part + g * D + 16 * n + 4 * quad) = make_float4(o[2 * n][0], o[2 * n + 1][0], o[2 * n][1], o[2 * n + 1][1]);
        if (g + 8 < rows) *reinterpret_cast<float4*>(part + (g + 8) * D + 16 * n + 4 * quad) = make_float4(o[2 * n][2], o[2 * n + 1][2], o[2 * n][3], o[2 * n + 1][3]);
    }
    if (quad == 0) {
        warp_ml[warp * ROWS + g] = make_float2(m[0], l[0]);
        warp_ml[warp * ROWS + g + 8] = make_float2(m[1], l[1]);
    }
    __syncthreads();
    const float unscale = exp2_of((float)base_exp);
    auto put = [&](int r, int d, float4 v, float total) {
        const int tok = r / a.heads_per_tile, head = hg * a.heads_per_tile + r % a.heads_per_tile;
        if (head >= G) return;
        const float f = (1.f / P_FACTOR) / total;
        v.x = v.x * f * unscale; v.y = v.y * f * unscale; v.z = v.z * f * unscale; v.w = v.w * f * unscale;
        if (total == 0.f) v = make_float4(0.f, 0.f, 0.f, 0.f);
        store4(out + ((size_t)(t.q_begin + tok0 + tok) * a.H + (size_t)kvh * G + head) * D + d, v);
    };
    for (int x = threadIdx.x; x < rows * (D / 4); x += THREADS) {
        const int r = x / (D / 4), d = x % (D / 4) * 4;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top = fmaxf(top, warp_ml[w * ROWS + r].x);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        float total = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float2 ml = warp_ml[w * ROWS + r];
            const float f = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : exp2_of(ml.x - top);   // (a NaN sum without a maximum is kept)
            const float4 u = *reinterpret_cast<const float4*>(smem + (size_t)w * STAGES * STAGE_BYTES + (size_t)(r * D + d) * 4);
            if (f != 0.f) { v.x += u.x * f; v.y += u.y * f; v.z += u.z * f; v.w += u.w * f; total += ml.y * f; }
        }
        if (splits == 1) {
            put(r, d, v, total);
        } else {   // over the first warp's part: this thread alone has read these entries of it
            *reinterpret_cast<float4*>(smem + (size_t)(r * D + d) * 4) = v;
            if (d == 0) block_ml[r] = make_float2(top, total);
        }
    }
    if (splits == 1) return;
    cluster_barrier();
    const int pieces = rows * (D / 4);
    for (int x = rank * THREADS + threadIdx.x; x < pieces; x += splits * THREADS) {
        const int r = x / (D / 4), d = x % (D / 4) * 4;
        const uint32_t ml_at = smem_addr(block_ml + r), v_at = smem_addr(smem) + (uint32_t)(r * D + d) * 4;
        float top = -INFINITY;
        for (int s = 0; s < splits; ++s) top = fmaxf(top, ld_cluster_f2(map_to_rank(ml_at, s)).x);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        float total = 0.f;
        for (int s = 0; s < splits; ++s) {
            const float2 ml = ld_cluster_f2(map_to_rank(ml_at, s));
            const float4 u = ld_cluster_f4(map_to_rank(v_at, s));
            const float f = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : exp2_of(ml.x - top);
            if (f != 0.f) { v.x += u.x * f; v.y += u.y * f; v.z += u.z * f; v.w += u.w * f; total += ml.y * f; }
        }
        put(r, d, v, total);
    }
    cluster_barrier();   // no block leaves while another may still read its shared memory
}

template <typename T>
int launch(void* out, const void* q, const Kv8Args& a, int tiles, int splits, cudaStream_t stream) {
    constexpr size_t smem = smem_bytes<sizeof(T) == 4 ? 2 : 1>();
    static_assert(smem <= 227 * 1024, "shared memory of a block");
    auto kernel = attn_kv8_kernel<T>;
    const long long grid = (long long)tiles * a.KV * a.head_groups * splits;
    if (grid > 0x7fffffffll) return OXR_BAD_ARGUMENT;
    static thread_local int ready = -1;
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return oxr_launch_status();
    if (ready != device) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) return oxr_launch_status();
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) return oxr_launch_status();
        ready = device;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attrs[2];
    int n = 0;
    if (splits > 1) {
        attrs[n].id = cudaLaunchAttributeClusterDimension;
        attrs[n].val.clusterDim.x = (unsigned)splits;
        attrs[n].val.clusterDim.y = 1;
        attrs[n].val.clusterDim.z = 1;
        ++n;
    }
    if (oxr_chain_kernels) {
        attrs[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attrs[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = attrs;
    cfg.numAttrs = n;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, (T*)out, (const T*)q, a, splits);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return 1000 + (int)e;
    }
    return 0;
}

template <typename T>
int clusters_of(int splits) {
    constexpr size_t smem = smem_bytes<sizeof(T) == 4 ? 2 : 1>();
    auto kernel = attn_kv8_kernel<T>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess ||
        cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)splits);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)splits;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    return n;
}
}  // namespace

OXR_API void oxr_set_chain(int on) { oxr_chain_kernels = on; }
OXR_API int oxr_kv8_head_dim() { return D; }
// How many clusters of `splits` blocks the current device holds at a time (0: none can be launched).
OXR_API int oxr_kv8_clusters(int dtype, int splits) { return dtype == 0 ? clusters_of<float>(splits) : clusters_of<__nv_bfloat16>(splits); }

// q [n_tokens, H, D] (tokens q_stride entries apart), out [n_tokens, H, D]; K and V pools of e4m3 codes with pages page_stride bytes apart and each
// page [page_size, KV, D]; scales [num_pages, KV]; cu_q [n + 1], ctx_lens [n], block_table [n, table_width]. Requests of min_q .. max_q new
// tokens are worked on; `any_q` is the most that any request may bring. dtype 0: fp32, 1: bf16.
OXR_API int oxr_kv8_attention(void* out, const void* q, const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale, const int* cu_q,
                              const int* ctx_lens, const int* block_table, int n, int n_tokens, int table_width, int page_size, long long page_stride,
                              int num_pages, int H, int KV, long long q_stride, float scale, int window, int min_q, int max_q, int any_q, int tiles, int splits,
                              int dtype, int* status, cudaStream_t stream) {
    if (n < 0 || n_tokens < 0 || KV <= 0 || H <= 0 || H % KV || page_size <= 0 || table_width < 0 || num_pages < 0 || window < 0 || tiles < 0) return OXR_BAD_ARGUMENT;
    if (splits < 1 || splits > 16 || (splits & (splits - 1)) || (dtype != 0 && dtype != 1) || any_q < 1 || min_q < 1) return OXR_BAD_ARGUMENT;
    if (tiles == 0 || n == 0 || n_tokens == 0) return 0;
    Kv8Args a = kv8_args(k_cache, v_cache, k_scale, v_scale, cu_q, ctx_lens, block_table, n, n_tokens, table_width, page_size, page_stride, num_pages, H, KV,
                         q_stride, scale, window, min_q, max_q, any_q, ROWS, status);
    return dtype == 0 ? launch<float>(out, q, a, tiles, splits, stream) : launch<__nv_bfloat16>(out, q, a, tiles, splits, stream);
}
