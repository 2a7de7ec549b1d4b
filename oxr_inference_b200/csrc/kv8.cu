// What stands around attention over the 8-bit cache: the store that rounds new keys and values into it, and the page tables of a step worked out
// on the GPU.
#include <cuda_fp8.h>

#include "common.cuh"

namespace {
// ---- the store
// A page of a KV head holds e4m3 codes c of entries s * c with one fp32 scale s. New tokens bring entries x with a largest magnitude a: the page
// then needs s >= 2^e, the smallest power of two with a <= 448 * 2^e. The scale starts at that when the page's first slot is stored and only grows
// after that; when it grows, the codes that are there already become round(c * s_old / s_new), which for powers of two changes none but those that
// fall below e4m3's normal range. Powers of two cost e4m3 nothing (its precision does not depend on where in its range a number lies) and make
// the result independent of how a request's tokens were cut into calls, but for those entries.
//
// One block works on a page: the block of the first token in the call that names it. (A token whose predecessor names the same page is not the
// first; the others look through all slots before their own, then gather the page's tokens from those behind.) So any order of slots is taken, nothing
// is shared between blocks, and of two tokens with one slot the later one stays. What bounds it: reading x and writing the codes; in a decode step
// the launch.
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(u[i] << 16); v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
}
__device__ __forceinline__ uint2 codes_of(const float (&v)[8]) {
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * i], v[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
    return make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
}
__device__ __forceinline__ void values_of(uint2 w, float (&v)[8]) {
    const uint32_t h[4] = {w.x & 0xffffu, w.x >> 16, w.y & 0xffffu, w.y >> 16};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)h[i], __NV_E4M3);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
// The smallest power of two that brings `most` to 448 or below; 0 for 0.
__device__ __forceinline__ float scale_for(float most) {
    if (!(most > 0.f)) return 0.f;
    const uint32_t b = __float_as_uint(most);
    const int e = max((int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u), -118);   // 448 = 1.75 * 2^8
    return __uint_as_float((uint32_t)(e + 127) << 23);
}

struct Kv8Pool {
    unsigned char* cache;   // pages of [page_size, KV, D] codes
    float* scale;           // [num_pages, KV]
    const void* x;          // [n, KV, D]
    long long x_stride;     // entries from token to token
};

template <typename T>
__global__ void store_kv8_kernel(const Kv8Pool kp, const Kv8Pool vp, const int* __restrict__ slots, int n, long long page_stride, int num_pages, int page_size,
                                 int KV, int D, int heads_per_block, int* status) {
    extern __shared__ int winner[];   // [page_size] the token that is stored at each place of the page, or -1
    pdl_wait();
    pdl_trigger();
    const int i = blockIdx.x;
    const int slot = __ldg(slots + i);
    if (slot < 0) return;
    const int page = slot / page_size;
    if (page >= num_pages) {
        if (threadIdx.x == 0 && blockIdx.y == 0) oxr_report(status, OXR_BAD_SLOT, i);
        return;
    }
    const int first = page * page_size;   // below 2^31: `slot` is
    auto here = [&](int s) { return (unsigned)(s - first) < (unsigned)page_size; };   // (negative slots wrap far above)
    if (i > 0 && here(__ldg(slots + i - 1))) return;
    bool earlier = false;
#pragma unroll 8
    for (int j = threadIdx.x; j < i - 1; j += blockDim.x) earlier |= here(__ldg(slots + j));
    for (int j = threadIdx.x; j < page_size; j += blockDim.x) winner[j] = -1;
    if (__syncthreads_or(earlier)) return;
#pragma unroll 8
    for (int j = i + threadIdx.x; j < n; j += blockDim.x) {
        const int s = __ldg(slots + j);
        if (here(s)) atomicMax(winner + (s - first), j);
    }
    __syncthreads();
    const bool begun = winner[0] >= 0;

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int eights = D / 8, items = page_size * eights;
    const int h0 = blockIdx.y * heads_per_block, h1 = min(KV, h0 + heads_per_block);
    for (int u = 2 * h0 + warp; u < 2 * h1; u += warps) {
        const int h = u >> 1;
        const Kv8Pool& pool = (u & 1) ? vp : kp;
        const T* x = reinterpret_cast<const T*>(pool.x) + (size_t)h * D;
        unsigned char* cache = pool.cache + (long long)page * page_stride + (size_t)h * D;
        float most = 0.f;
#pragma unroll 4
        for (int e = lane; e < items; e += 32) {
            const int t = winner[e / eights];
            if (t < 0) continue;
            float v[8];
            load8(x + t * pool.x_stride + e % eights * 8, v);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float f = fabsf(v[k]);
                if (f < INFINITY) most = fmaxf(most, f);   // neither infinities nor NaN have a say
            }
        }
        most = warp_max(most);
        float* where = pool.scale + (size_t)page * KV + h;
        const float old = begun ? 0.f : *where;
        const float scale = fmaxf(old, scale_for(most));
        const bool again = !begun && scale > old;
        const float ratio = again ? old / scale : 1.f, inverse = scale > 0.f ? 1.f / scale : 0.f;
#pragma unroll 4
        for (int e = lane; e < items; e += 32) {
            const int off = e / eights, t = winner[off];
            uint2* at = reinterpret_cast<uint2*>(cache + (size_t)off * KV * D + e % eights * 8);
            float v[8];
            if (t >= 0) {
                load8(x + t * pool.x_stride + e % eights * 8, v);
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = fabsf(v[k]) < INFINITY ? v[k] * inverse : __uint_as_float(0x7fffffffu);   // e4m3 has no infinity
            } else if (again) {
                values_of(*at, v);
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] *= ratio;
            } else {
                continue;
            }
            *at = codes_of(v);
        }
        __syncwarp();
        if (lane == 0) *where = scale;
    }
}

// ---- the page tables of a step
// Row r of the tables is a request with `lengths[r]` cached tokens on `held[r]` pages. Its step brings `q_lens[r]` more; a row marked fresh begins
// anew: its pages go back and it starts at length 0. The free pages are a stack: what is given back goes on top, row after row and page after page,
// then rows take what they need from the top in the same order. If the step cannot be had whole (too few pages, a row too long, too many tokens)
// nothing moves and all its arrays say so.
//
// Three prefix sums over the rows (new tokens, pages given, pages taken) settle everything; every block of the cluster has all of them in its
// shared memory and works on its share of rows and tokens. The blocks meet once, between giving back and taking: until then nobody changes what
// others read. What bounds it: the launch and a handful of dependent reads; three words a token are written.
constexpr int PAGE_THREADS = 1024, PAGE_ROWS = 8192;
__device__ __forceinline__ uint32_t block_in_cluster() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

struct StepPages {
    int *lengths, *held, *table, *free_list, *free_count;
    const int *q_lens, *fresh;
    int rows, width, page_size, pool, tokens;
    int *slots, *positions, *req_of_token, *cu_q, *ctx_lens;
    int advance, blocks;
    int* status;
};

__global__ void __launch_bounds__(PAGE_THREADS) step_pages_kernel(const StepPages a) {
    extern __shared__ int rows_smem[];
    int* cu = rows_smem;                  // [rows + 1] first token
    int* given = cu + a.rows + 1;         // [rows + 1] pages given back by the rows before
    int* taken = given + a.rows + 1;      // [rows + 1] pages taken by the rows before
    int* begin = taken + a.rows + 1;      // [rows] length before the step
    int* keeps = begin + a.rows;          // [rows] pages that stay
    __shared__ long long warp_sum3[3][32];
    __shared__ long long totals[3];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_wait();
    pdl_trigger();
    const int rank = a.blocks > 1 ? (int)block_in_cluster() : 0;
    const int top0 = *a.free_count;

    // each thread adds up its own stretch of rows, then the block adds the stretches
    const int each = (a.rows + PAGE_THREADS - 1) / PAGE_THREADS, r0 = min(tid * each, a.rows), r1 = min(r0 + each, a.rows);
    long long mine[3] = {0, 0, 0};
    int bad = 0;
    for (int r = r0; r < r1; ++r) {
        const bool anew = a.fresh != nullptr && a.fresh[r] != 0;
        const int len = a.lengths[r], h = a.held[r], q = a.q_lens[r];
        const int b = anew ? 0 : len, k = anew ? 0 : h;
        const long long after = (long long)b + q, want = (after + a.page_size - 1) / a.page_size;
        if (len < 0 || h < 0 || h > a.width || q < 0 || want > a.width) bad = 1;
        begin[r] = b;
        keeps[r] = k;
        cu[r] = q;
        given[r] = anew ? h : 0;
        taken[r] = want > k && want <= a.width ? (int)want - k : 0;
        mine[0] += q; mine[1] += given[r]; mine[2] += taken[r];
    }
    long long upto[3];
#pragma unroll
    for (int s = 0; s < 3; ++s) {
        long long v = mine[s];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long w = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += w;
        }
        upto[s] = v - mine[s];
        if (lane == 31) warp_sum3[s][warp] = v;
    }
    bad = __syncthreads_or(bad);
    if (warp < 3) {
        const long long own = warp_sum3[warp][lane];
        long long v = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long w = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += w;
        }
        warp_sum3[warp][lane] = v - own;
        if (lane == 31) totals[warp] = v;
    }
    __syncthreads();
    const long long new_tokens = totals[0], gives = totals[1], takes = totals[2];
    const int code = bad ? OXR_LONG_REQUEST : new_tokens > a.tokens ? OXR_MANY_TOKENS
                   : top0 < 0 || top0 + gives > a.pool || takes > top0 + gives ? OXR_NO_PAGES : 0;
    const int threads = a.blocks * PAGE_THREADS, at = rank * PAGE_THREADS + tid;
    if (code) {
        if (at == 0) oxr_report(a.status, code, 0);
        for (int t = at; t < a.tokens; t += threads) { a.slots[t] = -1; a.positions[t] = 0; a.req_of_token[t] = -1; }
        for (int r = at; r <= a.rows; r += threads) {
            a.cu_q[r] = 0;
            if (r < a.rows) a.ctx_lens[r] = 0;
        }
        return;   // every block of the cluster comes to the same end: none waits
    }
    int run[3];
#pragma unroll
    for (int s = 0; s < 3; ++s) run[s] = (int)(upto[s] + warp_sum3[s][warp]);
    for (int r = r0; r < r1; ++r) {
        const int q = cu[r], g = given[r], t = taken[r];
        cu[r] = run[0]; given[r] = run[1]; taken[r] = run[2];
        run[0] += q; run[1] += g; run[2] += t;
    }
    if (tid == 0) { cu[a.rows] = (int)new_tokens; given[a.rows] = (int)gives; taken[a.rows] = (int)takes; }
    __syncthreads();

    // pages given back, a warp per row
    const int top = top0 + (int)gives;
    for (int r = rank * 32 + warp; r < a.rows; r += a.blocks * 32) {
        const int g = given[r + 1] - given[r];
        for (int j = lane; j < g; j += 32) a.free_list[top0 + given[r] + j] = a.table[(size_t)r * a.width + j];
    }
    if (a.blocks > 1) {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    } else {
        __syncthreads();
    }
    // pages taken, and what is said of each row
    for (int r = rank * 32 + warp; r < a.rows; r += a.blocks * 32) {
        const int n = taken[r + 1] - taken[r], k = keeps[r];
        for (int j = lane; j < n; j += 32) a.table[(size_t)r * a.width + k + j] = a.free_list[top - 1 - (taken[r] + j)];
        if (lane == 0) {
            const int after = begin[r] + cu[r + 1] - cu[r];
            a.cu_q[r] = cu[r];
            a.ctx_lens[r] = after;
            a.held[r] = k + n;
            if (a.advance) a.lengths[r] = after;
        }
    }
    if (at == 0) {
        a.cu_q[a.rows] = (int)new_tokens;
        *a.free_count = top - (int)takes;
    }
    // tokens: the request by bisection, its page from the part of its row that stays or from the stack
    for (int t = at; t < a.tokens; t += threads) {
        if (t >= (int)new_tokens) {   // behind the last request
            a.slots[t] = -1; a.positions[t] = 0; a.req_of_token[t] = -1;
            continue;
        }
        int low = 0, high = a.rows;       // the last row with cu[row] <= t (rows without tokens share their start with the next)
        while (high - low > 1) {
            const int mid = (low + high) >> 1;
            if (cu[mid] <= t) low = mid; else high = mid;
        }
        const int pos = begin[low] + t - cu[low], j = pos / a.page_size, k = keeps[low];
        const int page = j < k ? a.table[(size_t)low * a.width + j] : a.free_list[top - 1 - (taken[low] + j - k)];
        a.slots[t] = page < 0 ? -1 : page * a.page_size + pos % a.page_size;
        a.positions[t] = pos;
        a.req_of_token[t] = low;
    }
}
}  // namespace

// k, v [n, KV, D] (tokens k_stride / v_stride entries apart, rows 16-byte aligned) -> slots of the pools. dtype 0: fp32, 1: bf16.
OXR_API int oxr_store_kv8(void* k_cache, void* v_cache, float* k_scale, float* v_scale, const void* k, const void* v, long long k_stride, long long v_stride,
                          const int* slots, int n, long long page_stride, int num_pages, int page_size, int KV, int D, int dtype, int* status, cudaStream_t stream) {
    if (n < 0 || num_pages < 0 || page_size <= 0 || page_size > 8192 || KV <= 0 || D <= 0 || D % 16 || (dtype != 0 && dtype != 1)) return OXR_BAD_ARGUMENT;
    if (n == 0) return 0;
    const Kv8Pool kp = {(unsigned char*)k_cache, k_scale, k, k_stride}, vp = {(unsigned char*)v_cache, v_scale, v, v_stride};
    // Few tokens, most of them alone on their pages: a block per two KV heads (64 tokens of 8 heads of 128 are then 256 blocks). Many tokens fill the
    // GPU with their pages alone, and one block saves the others the search for the page's tokens.
    const bool few = n <= 1024;
    const int heads = few ? (KV < 2 ? KV : 2) : KV, threads = few ? 128 : 256;
    const dim3 grid(n, (KV + heads - 1) / heads);
    const size_t smem = (size_t)page_size * sizeof(int);
    if (dtype == 0)
        oxr_launch(store_kv8_kernel<float>, grid, dim3(threads), smem, stream, true, kp, vp, slots, n, page_stride, num_pages, page_size, KV, D, heads, status);
    else
        oxr_launch(store_kv8_kernel<__nv_bfloat16>, grid, dim3(threads), smem, stream, true, kp, vp, slots, n, page_stride, num_pages, page_size, KV, D, heads, status);
    return oxr_launch_status();
}

OXR_API int oxr_step_pages(int* lengths, int* held, int* table, int* free_list, int* free_count, const int* q_lens, const int* fresh, int rows, int width,
                           int page_size, int pool, int tokens, int* slots, int* positions, int* req_of_token, int* cu_q, int* ctx_lens, int advance, int* status,
                           cudaStream_t stream) {
    if (rows < 0 || rows > PAGE_ROWS || width < 0 || page_size <= 0 || pool < 0 || tokens < 0) return OXR_BAD_ARGUMENT;
    // one block while its threads have a token each, else the eight of a cluster (the most that any GPU with clusters takes)
    const int blocks = tokens <= PAGE_THREADS && rows <= PAGE_THREADS ? 1 : 8;
    const StepPages a = {lengths, held, table, free_list, free_count, q_lens, fresh, rows, width, page_size, pool, tokens,
                         slots, positions, req_of_token, cu_q, ctx_lens, advance, blocks, status};
    const size_t smem = (size_t)(5 * rows + 3) * sizeof(int);
    if (smem > 40 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(step_pages_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (5 * PAGE_ROWS + 3) * (int)sizeof(int));
        if (e != cudaSuccess) return oxr_launch_status();
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(PAGE_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attrs[2];
    int n = 0;
    if (blocks > 1) {
        attrs[n].id = cudaLaunchAttributeClusterDimension;
        attrs[n].val.clusterDim.x = (unsigned)blocks;
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
    const cudaError_t e = cudaLaunchKernelEx(&cfg, step_pages_kernel, a);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return 1000 + (int)e;
    }
    return 0;
}
