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
// One block works on a page (of two KV heads): that of the first token in the call that names it. (A token whose predecessor names the same page is not
// the first; for the others the block looks through all slots before, then gathers the page's tokens from those behind, or, where the tokens are
// many, another kernel has found the first and the last token of each page.) So any order of slots is taken, nothing is shared between blocks,
// and of two tokens with one slot the later one stays. A warp has one head's keys or values of the page: their
// largest magnitude, then the codes, from registers where they fit. What bounds it: reading x and writing the codes; in a decode step the launch.
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

// Eight entries as they come.
template <typename T> struct Raw;
template <> struct Raw<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) { a = __ldg(reinterpret_cast<const float4*>(p)); b = __ldg(reinterpret_cast<const float4*>(p) + 1); }
    __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
    // the largest of `bits` and the magnitudes, compared as integers (infinities and NaN then lie above all numbers)
    __device__ __forceinline__ uint32_t most(uint32_t bits) const {
        float v[8];
        get(v);
#pragma unroll
        for (int i = 0; i < 8; ++i) bits = max(bits, __float_as_uint(v[i]) & 0x7fffffffu);
        return bits;
    }
    static __device__ __forceinline__ uint32_t as_float(uint32_t bits) { return bits; }
    __device__ __forceinline__ void get(float (&v)[8]) const { v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w; }
};
template <> struct Raw<__nv_bfloat16> {
    uint4 w;
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { w = __ldg(reinterpret_cast<const uint4*>(p)); }
    __device__ __forceinline__ void zero() { w = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ uint32_t most(uint32_t bits) const {      // two 16-bit numbers
        constexpr uint32_t M = 0x7fff7fffu;
        return __vmaxu2(__vmaxu2(__vmaxu2(bits, w.x & M), __vmaxu2(w.y & M, w.z & M)), w.w & M);
    }
    static __device__ __forceinline__ uint32_t as_float(uint32_t bits) { return max(bits << 16, bits & 0xffff0000u); }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(u[i] << 16); v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
    }
};

// Which tokens of the call name a page, for calls of many tokens: the first and the last of them. `ends` [num_pages][2] comes as -1.
__global__ void store_kv8_ends_kernel(int* __restrict__ ends, const int* __restrict__ slots, int n, int page_size, int num_pages) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    const int s = i < n ? __ldg(slots + i) : -1;
    if (s < 0 || s / page_size >= num_pages) return;
    const int page = s / page_size, before = i > 0 ? __ldg(slots + i - 1) : -1, after = i + 1 < n ? __ldg(slots + i + 1) : -1;
    if (before < 0 || before / page_size != page) atomicMin(reinterpret_cast<unsigned*>(ends) + 2ll * page, (unsigned)i);
    if (after < 0 || after / page_size != page) atomicMax(ends + 2ll * page + 1, i);
}

constexpr int FEW_TOKENS = 1024;
constexpr int HELD = 8;   // groups of eight entries that a lane keeps between the two looks at them: pages of up to 2,048 entries a head

// EIGHTS: D / 8 where that divides a warp, else 0 (taken from D). Blocks an SM: the held groups want 80 registers of 16-bit entries; at 72 (seven blocks)
// 10,300 tokens of 8 heads of 128 take 22 us, at 80 (six) 23.3.
template <typename T, int EIGHTS>
__global__ void __launch_bounds__(128, sizeof(T) == 4 ? 4 : 7) store_kv8_kernel(const Kv8Pool kp, const Kv8Pool vp, const int* __restrict__ slots, const int* __restrict__ ends, int n,
                                                           long long page_stride, int num_pages, int page_size, int KV, int D, int tokens_per_block, int* status) {
    extern __shared__ int winner[];   // [page_size] the token that is stored at each place of the page, or -1
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int eights = EIGHTS ? EIGHTS : D / 8;
    // which of the block's tokens (32 at most) begin a run of tokens of one page
    const int i0 = blockIdx.x * tokens_per_block;
    bool begins = false;
    if (lane < tokens_per_block && i0 + lane < n) {
        const int s = __ldg(slots + i0 + lane), before = i0 + lane > 0 ? __ldg(slots + i0 + lane - 1) : -1;
        if (s >= 0) {
            const int page = s / page_size;
            if (page >= num_pages) {
                if (warp == 0 && blockIdx.y == 0) oxr_report(status, OXR_BAD_SLOT, i0 + lane);
            } else {
                begins = (before < 0 || before / page_size != page) && (ends == nullptr || __ldg(ends + 2ll * page) == i0 + lane);
            }
        }
    }
    for (unsigned runs = __ballot_sync(0xffffffffu, begins); runs; runs &= runs - 1) {     // the same in every warp
        const int i = i0 + __ffs(runs) - 1;
        const int page = __ldg(slots + i) / page_size, first = page * page_size;   // below 2^31, as the slot is
        auto here = [&](int s) { return (unsigned)s - (unsigned)first < (unsigned)page_size; };   // (negative slots wrap above it: `first` is 8,192 and more below 2^31)
        const int u = 2 * blockIdx.y * 2 + warp, h = u >> 1;      // this warp's head and whether it has the keys or the values
        const Kv8Pool& pool = (u & 1) ? vp : kp;
        const unsigned x_stride = (unsigned)pool.x_stride;
        float* where = pool.scale + (size_t)page * KV + h;
        const float before = h < KV ? *where : 0.f;
        const int last = ends != nullptr ? __ldg(ends + 2ll * page + 1) : n - 1;
        for (int j = threadIdx.x; j < page_size; j += blockDim.x) winner[j] = -1;
        if (ends == nullptr) {
            bool earlier = false;
#pragma unroll 8
            for (int j = threadIdx.x; j < i - 1; j += blockDim.x) earlier |= here(__ldg(slots + j));
            if (__syncthreads_or(earlier)) continue;      // the page is another block's
        } else {
            __syncthreads();
        }
#pragma unroll 8
        for (int j = i + threadIdx.x; j <= last; j += blockDim.x) {
            const int s = __ldg(slots + j);
            if (here(s)) atomicMax(winner + (s - first), j);
        }
        __syncthreads();
        const bool begun = winner[0] >= 0;
        const int items = page_size * eights;
        if (h < KV) {
            const T* x = reinterpret_cast<const T*>(pool.x) + (size_t)h * D;
            unsigned char* cache = pool.cache + (long long)page * page_stride + (size_t)h * D;
            const float old = begun ? 0.f : before;
            const bool hold = items <= 32 * HELD;
            auto from = [&](int e, int t) { return x + (size_t)(unsigned)t * x_stride + e % eights * 8; };
            auto to = [&](int e) { return reinterpret_cast<uint2*>(cache + (unsigned)(e / eights * KV * D + e % eights * 8)); };
            Raw<T> held[HELD];
            int token[HELD];
            uint32_t bits = 0u;
            if (hold) {
#pragma unroll
                for (int c = 0; c < HELD; ++c) token[c] = c * 32 + lane < items ? winner[(c * 32 + lane) / eights] : -1;
#pragma unroll
                for (int c = 0; c < HELD; ++c) {
                    held[c].zero();
                    if (token[c] >= 0) held[c].load(from(c * 32 + lane, token[c]));
                }
#pragma unroll
                for (int c = 0; c < HELD; ++c) bits = held[c].most(bits);
            } else {
#pragma unroll 4
                for (int e = lane; e < items; e += 32) {
                    const int t = winner[e / eights];
                    if (t < 0) continue;
                    Raw<T> r;
                    r.load(from(e, t));
                    bits = r.most(bits);
                }
            }
            bits = __reduce_max_sync(0xffffffffu, Raw<T>::as_float(bits));
            const bool odd = bits >= 0x7f800000u;      // infinities or NaN, which have no say
            float most = __uint_as_float(bits);
            if (odd) {
                most = 0.f;
                for (int e = lane; e < items; e += 32) {
                    const int t = winner[e / eights];
                    if (t < 0) continue;
                    Raw<T> r;
                    float w[8];
                    r.load(from(e, t));
                    r.get(w);
                    for (int k = 0; k < 8; ++k)
                        if (fabsf(w[k]) < INFINITY) most = fmaxf(most, fabsf(w[k]));
                }
                most = warp_max(most);
            }
            const float scale = fmaxf(old, scale_for(most));
            const bool again = !begun && scale > old;
            const float inverse = scale > 0.f ? 1.f / scale : 0.f;
            if (hold && !odd) {
#pragma unroll
                for (int c = 0; c < HELD; ++c)
                    if (token[c] >= 0) {
                        float w[8];
                        held[c].get(w);
#pragma unroll
                        for (int k = 0; k < 8; ++k) w[k] *= inverse;
                        *to(c * 32 + lane) = codes_of(w);
                    }
            } else {
                for (int e = lane; e < items; e += 32) {
                    const int t = winner[e / eights];
                    if (t < 0) continue;
                    Raw<T> r;
                    float w[8];
                    r.load(from(e, t));
                    r.get(w);
#pragma unroll
                    for (int k = 0; k < 8; ++k) w[k] = fabsf(w[k]) < INFINITY ? w[k] * inverse : __uint_as_float(0x7fffffffu);   // e4m3 has no infinity
                    *to(e) = codes_of(w);
                }
            }
            if (again) {       // what the page holds already, to the new scale
                const float ratio = old / scale;
                for (int e = lane; e < items; e += 32) {
                    if (winner[e / eights] >= 0) continue;
                    float w[8];
                    values_of(*to(e), w);
#pragma unroll
                    for (int k = 0; k < 8; ++k) w[k] *= ratio;
                    *to(e) = codes_of(w);
                }
            }
            __syncwarp();
            if (lane == 0) *where = scale;
        }
        __syncthreads();      // `winner` is read
    }
}

template <typename T>
void launch_store(dim3 grid, size_t smem, cudaStream_t stream, const Kv8Pool& kp, const Kv8Pool& vp, const int* slots, const int* ends, int n, long long page_stride,
                  int num_pages, int page_size, int KV, int D, int tokens, int* status) {
    auto go = [&](auto kernel) { oxr_launch(kernel, grid, dim3(128), smem, stream, true, kp, vp, slots, ends, n, page_stride, num_pages, page_size, KV, D, tokens, status); };
    switch (D) {
        case 16: go(store_kv8_kernel<T, 2>); break;
        case 32: go(store_kv8_kernel<T, 4>); break;
        case 64: go(store_kv8_kernel<T, 8>); break;
        case 128: go(store_kv8_kernel<T, 16>); break;
        case 256: go(store_kv8_kernel<T, 32>); break;
        default: go(store_kv8_kernel<T, 0>);
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
        const long long slot = (long long)page * a.page_size + pos % a.page_size;
        a.slots[t] = page < 0 ? -1 : (int)min(slot, 0x7fffffffll);      // a number that no page has stays one that no pool has, and the store reports it
        a.positions[t] = pos;
        a.req_of_token[t] = low;
    }
}
}  // namespace

// Calls as the host lays them out in one block of memory each.
struct StoreCall {
    void *k_cache, *v_cache;
    float *k_scale, *v_scale;
    const void *k, *v;              // [n, KV, D], tokens k_stride / v_stride entries apart, rows 16-byte aligned
    const int* slots;
    int* ends;                      // scratch of [num_pages][2] words, needed for more than FEW_TOKENS tokens
    int* status;
    cudaStream_t stream;
    long long k_stride, v_stride, page_stride;
    int n, num_pages, page_size, KV, D, dtype;      // dtype 0: fp32, 1: bf16
};
OXR_API int oxr_store_kv8(const StoreCall* c) {
    const int n = c->n, num_pages = c->num_pages, page_size = c->page_size, KV = c->KV, D = c->D, dtype = c->dtype;
    const long long k_stride = c->k_stride, v_stride = c->v_stride, page_stride = c->page_stride;
    const int* slots = c->slots;
    int *ends = c->ends, *status = c->status;
    cudaStream_t stream = c->stream;
    if (n < 0 || num_pages < 0 || page_size <= 0 || page_size > 8192 || KV <= 0 || D <= 0 || D % 16 || (dtype != 0 && dtype != 1)) return OXR_BAD_ARGUMENT;
    if (k_stride < 0 || v_stride < 0 || k_stride > 0x7fffffffll || v_stride > 0x7fffffffll || (long long)page_size * KV * D > 0x7fffffffll
        || (long long)num_pages * page_size > 0x80000000ll - 8192) return OXR_BAD_ARGUMENT;
    if (n == 0) return 0;
    const Kv8Pool kp = {(unsigned char*)c->k_cache, c->k_scale, c->k, k_stride}, vp = {(unsigned char*)c->v_cache, c->v_scale, c->v, v_stride};
    // Few tokens, most of them alone on their pages: a block per token and two KV heads, which looks through all slots itself. Many tokens: a first
    // kernel finds each page's first and last token, and a block looks after 16 tokens, a page or two.
    const bool few = n <= FEW_TOKENS;
    if (!few) {
        if (ends == nullptr) return OXR_BAD_ARGUMENT;
        if (cudaMemsetAsync(ends, 0xff, (size_t)num_pages * 2 * sizeof(int), stream) != cudaSuccess) return oxr_launch_status();
        oxr_launch(store_kv8_ends_kernel, dim3((n + 255) / 256), dim3(256), 0, stream, false, ends, slots, n, page_size, num_pages);
    }
    const int tokens = few ? 1 : 16;
    const dim3 grid((n + tokens - 1) / tokens, (KV + 1) / 2);
    const size_t smem = (size_t)page_size * sizeof(int);
    if (dtype == 0) launch_store<float>(grid, smem, stream, kp, vp, slots, few ? nullptr : ends, n, page_stride, num_pages, page_size, KV, D, tokens, status);
    else launch_store<__nv_bfloat16>(grid, smem, stream, kp, vp, slots, few ? nullptr : ends, n, page_stride, num_pages, page_size, KV, D, tokens, status);
    return oxr_launch_status();
}
OXR_API int oxr_store_kv8_few() { return FEW_TOKENS; }

struct PagesCall {
    int *lengths, *held, *table, *free_list, *free_count;
    const int *q_lens, *fresh;
    int *slots, *positions, *req_of_token, *cu_q, *ctx_lens, *status;
    cudaStream_t stream;
    int rows, width, page_size, pool, tokens, advance;
};
OXR_API int oxr_step_pages(const PagesCall* c) {
    const int rows = c->rows, tokens = c->tokens;
    cudaStream_t stream = c->stream;
    if (rows < 0 || rows > PAGE_ROWS || c->width < 0 || c->page_size <= 0 || c->pool < 0 || tokens < 0) return OXR_BAD_ARGUMENT;
    // one block while its threads have a token each, else the eight of a cluster (the most that any GPU with clusters takes)
    const int blocks = tokens <= PAGE_THREADS && rows <= PAGE_THREADS ? 1 : 8;
    const StepPages a = {c->lengths, c->held, c->table, c->free_list, c->free_count, c->q_lens, c->fresh, rows, c->width, c->page_size, c->pool, tokens,
                         c->slots, c->positions, c->req_of_token, c->cu_q, c->ctx_lens, c->advance, blocks, c->status};
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
