// Page tables and slot maps of a paged key-value cache, built on the device
// from the requests' lengths, and the return of finished requests' pages.
//
// With P tokens a page, request b of length L_b that adds n_b tokens lacks
//   need_b = ceil((L_b + n_b) / P) - ceil(L_b / P)
// pages.  The exclusive scans of n_b (where its tokens start in the packed
// step) and of need_b (where its pages start in the ring of free pages) make
// every token independent of every other: token t finds its request by a
// binary search over the scan, and its page is either the request's last page
// or a fixed place of the ring.  The token that opens a page writes the table.
//
// What bounds it: latency.  The reads and writes of a step are a few hundred
// kilobytes at most.  So every CTA repeats the scan over all requests (two
// loads a request, kept in shared memory) instead of waiting for another
// launch, and takes kTokensPerCta tokens; a step of up to that many is one
// CTA.  Lengths and ring may be updated in place: with more than one CTA then
// by the one that finishes last (a ticket), when no other reads them any more.
// Measured: 64 requests of one token each 3.3 us (3.4 in place); 512 requests,
// half of them prompts of up to 1024 tokens (129 thousand slots), 5.2 us, and
// 7.2 in place, where 126 CTAs take a ticket.  Release: 5 of the 64 requests
// (781 pages) 3.3 us, 512 at once (182 thousand pages) 10.7.
#include <cstdio>

#include "common.cuh"
#include "ws_internal.h"

namespace ws {
namespace {

constexpr int kThreads = 1024;
constexpr int kTokensPerCta = 1024;
constexpr int kMaxRequests = 8192;   // 16 bytes of shared memory each

// Exclusive scans of two values per thread over the block; `carry` holds the
// totals of the earlier chunks and takes this chunk's.  All threads call it.
struct Two {
    long long a, b;
};
__device__ __forceinline__ Two operator+(Two x, Two y) { return {x.a + y.a, x.b + y.b}; }
__device__ __forceinline__ Two operator-(Two x, Two y) { return {x.a - y.a, x.b - y.b}; }
struct BlockScan {
    Two part[kThreads / 32];
    int taken[kThreads / 32];
};
__device__ __forceinline__ Two warp_scan(Two x) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const Two y = {__shfl_up_sync(0xffffffffu, x.a, o), __shfl_up_sync(0xffffffffu, x.b, o)};
        if ((threadIdx.x & 31) >= o) x = x + y;
    }
    return x;
}
__device__ __forceinline__ Two block_scan(Two v, BlockScan& sh, Two& carry) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    const Two x = warp_scan(v);
    __syncthreads();   // the previous call's reads are done
    if (lane == 31) sh.part[warp] = x;
    __syncthreads();
    // every warp sums the warps' totals for itself: one barrier less than asking one of them
    const Two p = warp_scan(lane < nw ? sh.part[lane] : Two{0, 0});
    const Two before = {__shfl_sync(0xffffffffu, p.a, (warp + 31) & 31), __shfl_sync(0xffffffffu, p.b, (warp + 31) & 31)};
    const Two ex = carry + (x - v) + (warp ? before : Two{0, 0});
    carry = carry + Two{__shfl_sync(0xffffffffu, p.a, 31), __shfl_sync(0xffffffffu, p.b, 31)};
    return ex;
}

// The CTA that writes the lengths and the ring.  In place, the one that gets
// here last, when no other reads them any more (the counter returns to 0);
// else the first.
__device__ __forceinline__ bool writes_state(bool in_place, int* counter) {
    if (!in_place || gridDim.x == 1) {
        __syncthreads();
        return blockIdx.x == 0;
    }
    __shared__ int last;
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        last = atomicAdd(counter, 1) == (int)gridDim.x - 1;
        if (last) *counter = 0;
        __threadfence();
    }
    __syncthreads();
    return last;
}

// Pages of P tokens that L tokens fill.
__device__ __forceinline__ uint32_t pages_of(uint32_t L, int P) {
    const uint32_t q = L / (uint32_t)P;
    return q + (q * (uint32_t)P != L);
}

// First b in [0, B) whose end[b] > t (ends ascend; t < end[B - 1]).
__device__ __forceinline__ int owner_of(const int* end, int B, int t) {
    int lo = 0, hi = B - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (end[mid] > t) hi = mid; else lo = mid + 1;
    }
    return lo;
}

__global__ void __launch_bounds__(kThreads)
paged_slots_kernel(const int32_t* seq_lens, const int32_t* new_lens, int B, int32_t* table,
                   int64_t table_stride, int max_pages, const int32_t* free_pages, int n_ring,
                   const int32_t* ring, int P, int64_t n_tokens, int64_t* __restrict__ slots,
                   int32_t* __restrict__ positions, int32_t* __restrict__ cu_new, int32_t* seq_lens_out,
                   int32_t* ring_out, int* counter) {
    extern __shared__ int sm[];
    __shared__ BlockScan sh;
    __shared__ int n_refused;
    int* end = sm;            // tokens of requests 0 .. b, clipped to n_tokens
    int* len = sm + B;        // tokens before the step, or -1: refused
    int* base = sm + 2 * B;   // first ring place (counted from the head) of b's new pages
    int* first = sm + 3 * B;  // first token of b in the packed step
    if (threadIdx.x == 0) n_refused = 0;
    pdl_wait_primary();
    pdl_launch_dependents();
    const int head = max(ring[0], 0), n_free = min(max(ring[1], 0), n_ring);
    Two sums;   // tokens, pages
    long long took;
    int refused;
    // Tokens and pages are scanned together.  Whether a request's tokens fit the step is known only afterwards, so a step
    // with less room than tokens scans once more, without the pages of those that do not fit.
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
        sums = {0, 0};
        took = refused = 0;
#pragma unroll 1
        for (int b0 = 0; b0 < B; b0 += blockDim.x) {
            const int b = b0 + threadIdx.x;
            const uint32_t L = b < B ? max(seq_lens[b], 0) : 0, n = b < B ? max(new_lens[b], 0) : 0;
            const uint32_t held = pages_of(L, P), want = pages_of(L + n, P);
            const bool fits = want <= (uint32_t)max_pages && L + n <= INT32_MAX &&
                              (pass == 0 || (b < B && first[b] + (long long)n <= n_tokens));
            const uint32_t need = fits ? want - held : 0;
            const Two at = block_scan({n, need}, sh, sums);
            if (b < B) {
                const bool served = fits && (need == 0 || at.b + need <= n_free);
                end[b] = (int)min(at.a + n, (long long)n_tokens);
                first[b] = (int)min(at.a, (long long)INT32_MAX);
                len[b] = served ? (int)L : -1;
                base[b] = (int)min(at.b, (long long)n_ring);
                refused += !served;
                if (served && need) took = max(took, at.b + need);
                if (blockIdx.x == 0) {
                    if (b == 0) cu_new[0] = 0;
                    cu_new[b + 1] = (int)min(at.a + n, (long long)INT32_MAX);
                }
            }
        }
        if (sums.a <= n_tokens) break;
    }
    if (B == 0 && blockIdx.x == 0 && threadIdx.x == 0) cu_new[0] = 0;
    __syncthreads();
    const int real = B > 0 ? end[B - 1] : 0;
    const int64_t t_end = min((int64_t)(blockIdx.x + 1) * kTokensPerCta, n_tokens);
    for (int64_t t = (int64_t)blockIdx.x * kTokensPerCta + threadIdx.x; t < t_end; t += blockDim.x) {
        int64_t slot = -1;
        int pos = 0;
        if (t < real) {
            const int b = owner_of(end, B, (int)t);
            if (len[b] >= 0) {
                const unsigned L = len[b];
                const unsigned p = L + (unsigned)((int)t - first[b]), col = p / (unsigned)P, off = p - col * P;
                const unsigned held = (L + P - 1) / (unsigned)P;
                int32_t* row = table + (int64_t)b * table_stride;
                int page;
                if (col < held) {
                    page = row[col];
                } else {
                    page = free_pages[(unsigned)((head + (long long)base[b] + (col - held)) % n_ring)];
                    if (off == 0) row[col] = page;
                }
                pos = (int)p;
                if (page >= 0) slot = (int64_t)page * P + off;
            }
        }
        slots[t] = slot;
        positions[t] = pos;
    }
    if (!writes_state(seq_lens_out == seq_lens || ring_out == ring, counter)) return;
    // served requests that took pages are a prefix of those that fit, so the largest end is what was taken
    refused = __reduce_add_sync(0xffffffffu, refused);
    if ((threadIdx.x & 31) == 0 && refused) atomicAdd(&n_refused, refused);
    const int taken = __reduce_max_sync(0xffffffffu, (int)took);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.taken[threadIdx.x >> 5] = taken;
    for (int b = threadIdx.x; b < B; b += blockDim.x) {
        const int n = max(new_lens[b], 0);
        const int L = max(seq_lens[b], 0);
        seq_lens_out[b] = len[b] >= 0 ? L + n : seq_lens[b];
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        int all = 0;
        for (int w = 0; w < (int)(blockDim.x >> 5); ++w) all = max(all, sh.taken[w]);
        ring_out[0] = (int)((head + (long long)all) % n_ring);
        ring_out[1] = n_free - all;
        ring_out[2] = n_refused;
    }
}

__global__ void __launch_bounds__(kThreads)
paged_release_kernel(const int32_t* seq_lens, const uint8_t* done, int B,
                     const int32_t* table, int64_t table_stride, int max_pages, int32_t* free_pages,
                     int n_ring, const int32_t* ring, int P, int32_t* seq_lens_out, int32_t* ring_out, int* counter,
                     int* status) {
    extern __shared__ int sm[];
    __shared__ BlockScan sh;
    int* end = sm;   // pages of requests 0 .. b that go back
    pdl_wait_primary();
    pdl_launch_dependents();
    const int head = max(ring[0], 0), n_free = min(max(ring[1], 0), n_ring);
    const int room = n_ring - n_free;
    Two pages = {0, 0};
    for (int b0 = 0; b0 < B; b0 += blockDim.x) {
        const int b = b0 + threadIdx.x;
        long long held = 0;
        if (b < B && done[b]) held = min(pages_of(max(seq_lens[b], 0), P), (uint32_t)max_pages);
        const long long start = block_scan({held, 0}, sh, pages).a;
        if (b < B) end[b] = (int)min(start + held, (long long)INT32_MAX);
    }
    __syncthreads();
    const int total = (int)min(pages.a, (long long)room);
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < total; i += gridDim.x * blockDim.x) {
        const int b = owner_of(end, B, i);
        const int j = i - (b ? end[b - 1] : 0);
        free_pages[(unsigned)((head + (long long)n_free + i) % n_ring)] = table[(int64_t)b * table_stride + j];
    }
    if (!writes_state(seq_lens_out == seq_lens || ring_out == ring, counter)) return;
    for (int b = threadIdx.x; b < B; b += blockDim.x) seq_lens_out[b] = done[b] ? 0 : seq_lens[b];
    if (threadIdx.x == 0) {
        ring_out[0] = head;
        ring_out[1] = n_free + total;
        ring_out[2] = 0;
        if (pages.a > room && status) atomicOr(status, kDevBadIndex);
    }
}

int checked(const char* what, int B, int max_pages, int64_t table_stride, int n_ring, int page_size, void* workspace,
            size_t workspace_bytes) {
    char buf[160];
    const char* why = nullptr;
    if (B < 0 || max_pages < 1 || n_ring < 1 || page_size < 1 || (B > 1 && table_stride < max_pages))
        why = "bad shape";
    else if (B > kMaxRequests) why = "more than 8192 requests";
    else if (!workspace || workspace_bytes < kCounterHeaderBytes || reinterpret_cast<uintptr_t>(workspace) % 16)
        why = "workspace missing, unaligned or too small";
    if (!why) return WS_OK;
    snprintf(buf, sizeof(buf), "%s: %s", what, why);
    return set_error(B > kMaxRequests ? WS_ERR_UNSUPPORTED : why[0] == 'w' ? WS_ERR_WORKSPACE : WS_ERR_INVALID_ARG, buf);
}

// CTAs of up to kThreads threads, as many as the requests or the CTA's tokens can use.
int block_threads(int64_t n) { return (int)std::min<int64_t>(kThreads, std::max<int64_t>(128, (n + 31) / 32 * 32)); }

int launch_status(cudaError_t e) {
    return e == cudaSuccess ? WS_OK : set_error(WS_ERR_CUDA, cudaGetErrorString(e));
}

}  // namespace
}  // namespace ws

using namespace ws;

extern "C" {

size_t ws_paged_slots_workspace_size(void) { return kCounterHeaderBytes; }

int ws_paged_slots(const int32_t* seq_lens, const int32_t* new_lens, int B, int32_t* page_table, int64_t table_stride,
                   int max_pages, const int32_t* free_pages, int n_ring, const int32_t* ring, int page_size,
                   int64_t n_tokens, int64_t* slots, int32_t* positions, int32_t* cu_new, int32_t* seq_lens_out,
                   int32_t* ring_out, void* workspace, size_t workspace_bytes, void* stream) {
    if (const int rc = checked("paged_slots", B, max_pages, table_stride, n_ring, page_size, workspace, workspace_bytes))
        return rc;
    if (n_tokens < 0 || n_tokens > INT32_MAX / 2) return set_error(WS_ERR_INVALID_ARG, "paged_slots: bad n_tokens");
    if (!ring || !ring_out || !cu_new || !free_pages || (B > 0 && (!seq_lens || !new_lens || !page_table || !seq_lens_out)) ||
        (n_tokens > 0 && (!slots || !positions)))
        return set_error(WS_ERR_INVALID_ARG, "paged_slots: null pointer");
    const size_t smem = (size_t)std::max(B, 1) * 16;
    static thread_local int set_for = -1;
    int dev = 0;
    cudaGetDevice(&dev);
    if (smem > 40 * 1024 && set_for != dev) {
        if (cudaFuncSetAttribute(paged_slots_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxRequests * 16) !=
            cudaSuccess)
            return set_error(WS_ERR_CUDA, "paged_slots: shared memory");
        set_for = dev;
    }
    const int64_t ctas = std::max<int64_t>(1, (n_tokens + kTokensPerCta - 1) / kTokensPerCta);
    const int threads = block_threads(std::max<int64_t>(B, std::min<int64_t>(n_tokens, kTokensPerCta)));
    return launch_status(launch_dependent(
        paged_slots_kernel, dim3((unsigned)ctas), threads, smem, static_cast<cudaStream_t>(stream),
        seq_lens, new_lens, B, page_table, table_stride, max_pages, free_pages, n_ring, ring, page_size, n_tokens, slots,
        positions, cu_new, seq_lens_out, ring_out, static_cast<int*>(workspace)));
}

int ws_paged_release(const int32_t* seq_lens, const uint8_t* done, int B, const int32_t* page_table,
                     int64_t table_stride, int max_pages, int32_t* free_pages, int n_ring, const int32_t* ring,
                     int page_size, int32_t* seq_lens_out, int32_t* ring_out, void* workspace, size_t workspace_bytes,
                     void* stream) {
    if (const int rc = checked("paged_release", B, max_pages, table_stride, n_ring, page_size, workspace, workspace_bytes))
        return rc;
    if (!ring || !ring_out || !free_pages || (B > 0 && (!seq_lens || !done || !page_table || !seq_lens_out)))
        return set_error(WS_ERR_INVALID_ARG, "paged_release: null pointer");
    // at most n_ring pages go back, and none of more than B rows
    const int64_t most = std::min<int64_t>(n_ring, (int64_t)B * max_pages);
    const int threads = block_threads(std::max<int64_t>(B, most));
    const int64_t ctas = std::max<int64_t>(1, std::min<int64_t>(device_sm_count(), most / (8 * kThreads)));
    const size_t smem = (size_t)std::max(B, 1) * 4;   // 32 KB at most
    return launch_status(launch_dependent(
        paged_release_kernel, dim3((unsigned)ctas), threads, smem, static_cast<cudaStream_t>(stream),
        seq_lens, done, B, page_table, table_stride, max_pages, free_pages, n_ring, ring, page_size, seq_lens_out,
        ring_out, static_cast<int*>(workspace), device_status_word()));
}

}  // extern "C"
