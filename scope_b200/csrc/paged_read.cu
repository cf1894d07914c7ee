// Reads a paged key-value cache back: requests' rows, packed one after the other, in 16 bits.
//
//   row cu[b] + i  =  token starts[b] + i of request b, its codes times their scale, rounded once.
//
// What bounds it: memory, each code read once and two bytes written for it.  A thread owns a unit of 16 dims of a head (16
// bytes of codes, 32 of output; 16-bit pools: 8 dims) and walks its CTA's tokens, two or four loads in flight.  The tokens'
// places are looked up once for a CTA.
// Measured: 16 requests of up to 32768 tokens from the first sixteenth on, 8 heads of 128 in e4m3, 168 us (1.04 GB, 6.2 TB/s,
// 0.94 of a copy's rate), from a bf16 pool 217 us (1.38 GB, 6.4 TB/s); 1000 tokens of 4 heads 2.8 us and 2.6.  Loads in flight: 1 took 182 us, 2 169, 4 178, 8 236 (registers,
// so fewer warps); but where all may lie in L2 (18 thousand tokens of 4 heads just written) 2 took 16.6 us and 4 14.0.  CTAs
// of 16 tokens took 163 us there, but 6.1 us for 4.1 where heads are few; of 64 tokens 183; of 128 threads 181, 512 194.
#include <cstdio>

#include "common.cuh"
#include "ws_internal.h"

#include <cuda_fp16.h>

#include <type_traits>

namespace ws {
namespace {

constexpr int kThreads = 256;
constexpr int kMostTok = 32;   // tokens of a CTA

struct Side {   // keys or values
    const uint8_t* src;                  // bytes
    int64_t page, tok, head;
    const float* scales;
    int64_t s_page, s_block, s_head;
    uint16_t* dst;                       // [n_tokens, Hkv, D]
    int D;
};
struct ReadArgs {
    Side side[2];
    const int32_t* table;
    int64_t table_stride;
    const int32_t* cu;
    const int32_t* starts;
    int64_t n_tokens;
    int B, Hkv, max_pages, page_size, n_pages, block;
    int tok;            // tokens of a CTA
    int units0, units;  // units of a token's keys; of keys and values
    int* status;
};

// 16 codes times a scale, as 16-bit floats.
template <bool F16, bool E4M3>
__device__ __forceinline__ void values16(const uint4& w, float s, uint32_t* y) {
    const uint32_t in[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t two = in[i >> 1] >> (16 * (i & 1));
        float lo, hi;
        if (E4M3) {
            uint32_t h;
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
            lo = f.x, hi = f.y;
        } else {
            lo = (float)(int8_t)two, hi = (float)(int8_t)(two >> 8);
        }
        lo = __fmul_rn(lo, s), hi = __fmul_rn(hi, s);
        if (F16) {
            const __half2 h = __floats2half2_rn(lo, hi);
            y[i] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
            y[i] = pack_bf16(lo, hi);
        }
    }
}

// KIND: 0 16-bit values, 1 int8, 2 e4m3.  AHEAD: loads in flight a thread.
template <bool F16, int KIND, int AHEAD>
__global__ void __launch_bounds__(kThreads) read_kernel(const __grid_constant__ ReadArgs a) {
    __shared__ int s_page[kMostTok], s_off[kMostTok];   // page < 0: -1 zeros, -2 nothing
    pdl_wait_primary();
    pdl_launch_dependents();
    const int tid = threadIdx.x;
    const int64_t row0 = (int64_t)blockIdx.x * a.tok;
    if (tid < a.tok) {
        const int64_t row = row0 + tid;
        int page = -2, off = 0;
        if (row < a.n_tokens) {
            int lo = 0, hi = a.B;   // the last request that begins at the row or before it
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (a.cu[mid] <= row) lo = mid;
                else hi = mid;
            }
            const int64_t from = a.cu[lo];
            if (from <= row && row < a.cu[lo + 1]) {
                const int64_t t = row - from + (a.starts ? a.starts[lo] : 0);
                const int64_t p = t >= 0 ? t / a.page_size : -1;
                page = -1;
                if (p >= 0 && p < a.max_pages) {
                    off = (int)(t - p * a.page_size);
                    const int entry = a.table[lo * a.table_stride + p];
                    if (entry >= 0 && entry < a.n_pages) page = entry;
                }
                if (page < 0 && blockIdx.y == 0 && a.status) atomicOr(a.status, kDevBadIndex);
            }
        }
        s_page[tid] = page, s_off[tid] = off;
    }
    __syncthreads();
    // this thread's unit, and the first of its tokens
    const int slice = min(a.units - (int)blockIdx.y * kThreads, kThreads), tok0 = tid / slice, step = kThreads / slice;
    if (tok0 >= step) return;
    const int at = blockIdx.y * kThreads + tid - tok0 * slice, kind = at >= a.units0, e = kind ? at - a.units0 : at;
    const Side& x = a.side[kind];
    constexpr int kDims = KIND ? 16 : 8;
    const int per = x.D / kDims, head = e / per, d = (e - head * per) * kDims;
    const uint8_t* const src = x.src + head * x.head + d * (KIND ? 1 : 2);
    const float* const scales = x.scales + head * x.s_head;
    uint16_t* const dst = x.dst + ((row0 * a.Hkv + head) * x.D + d);
    const int64_t row_elems = (int64_t)a.Hkv * x.D;
#pragma unroll 1
    for (int t = tok0; t < a.tok; t += step * AHEAD) {
        uint4 w[AHEAD];
        float s[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int tk = t + i * step;
            w[i] = make_uint4(0, 0, 0, 0), s[i] = 0.f;
            if (tk < a.tok && s_page[tk] >= 0) {
                const int64_t page = s_page[tk], off = s_off[tk];
                w[i] = *reinterpret_cast<const uint4*>(src + page * x.page + off * x.tok);
                if (KIND) s[i] = scales[page * x.s_page + (off / a.block) * x.s_block];
            }
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int tk = t + i * step;
            if (tk >= a.tok || s_page[tk] == -2) continue;
            uint4* const p = reinterpret_cast<uint4*>(dst + tk * row_elems);
            if (KIND) {
                uint32_t y[8];
                values16<F16, KIND == 2>(w[i], s[i], y);
                p[0] = make_uint4(y[0], y[1], y[2], y[3]), p[1] = make_uint4(y[4], y[5], y[6], y[7]);
            } else {
                p[0] = w[i];
            }
        }
    }
}

}  // namespace
}  // namespace ws

using namespace ws;

extern "C" int ws_paged_read(const ws_paged_kv* kv, const int32_t* page_table, int64_t table_stride, int max_pages, int B,
                             const int32_t* cu, const int32_t* starts, int64_t n_tokens, int out_dtype, void* k_out,
                             void* v_out, void* stream) {
    if (!kv || B < 0 || max_pages < 0 || table_stride < 0 || n_tokens < 0)
        return set_error(WS_ERR_INVALID_ARG, "paged_read: bad shape");
    if (const int rc = paged_kv_check("paged_read", kv)) return rc;
    if (out_dtype != WS_DTYPE_BF16 && out_dtype != WS_DTYPE_F16)
        return set_error(WS_ERR_INVALID_ARG, "paged_read: the output must be bf16 or fp16");
    const bool eight = kv->dtype == WS_DTYPE_I8 || kv->dtype == WS_DTYPE_E4M3;
    if (!eight && kv->dtype != out_dtype)
        return set_error(WS_ERR_INVALID_ARG, "paged_read: a 16-bit pool is read in its own type");
    if (B == 0 || n_tokens == 0) return WS_OK;
    if (!cu || !k_out || !v_out || (max_pages > 0 && !page_table))
        return set_error(WS_ERR_INVALID_ARG, "paged_read: null pointer");
    if (reinterpret_cast<uintptr_t>(k_out) % 16 || reinterpret_cast<uintptr_t>(v_out) % 16)
        return set_error(WS_ERR_INVALID_ARG, "paged_read: outputs must be 16-byte aligned");
    const int eb = eight ? 1 : 2, dims = eight ? 16 : 8;
    ReadArgs a;
    memset(&a, 0, sizeof(a));
    a.side[0] = {static_cast<const uint8_t*>(kv->k), kv->k_stride_page * eb, kv->k_stride_tok * eb, kv->k_stride_head * eb,
                 kv->k_scales, kv->ks_stride_page, kv->ks_stride_tok, kv->ks_stride_head, static_cast<uint16_t*>(k_out), kv->Dk};
    a.side[1] = {static_cast<const uint8_t*>(kv->v), kv->v_stride_page * eb, kv->v_stride_tok * eb, kv->v_stride_head * eb,
                 kv->v_scales, kv->vs_stride_page, kv->vs_stride_tok, kv->vs_stride_head, static_cast<uint16_t*>(v_out), kv->Dv};
    a.table = page_table, a.table_stride = table_stride, a.cu = cu, a.starts = starts, a.n_tokens = n_tokens;
    a.B = B, a.Hkv = kv->Hkv, a.max_pages = max_pages, a.page_size = kv->page_size, a.n_pages = (int)kv->n_pages;
    a.block = std::max(kv->scale_block, 1);
    const int64_t units = (int64_t)kv->Hkv * (kv->Dk + kv->Dv) / dims, slices = (units + kThreads - 1) / kThreads;
    if (slices > 65535) return set_error(WS_ERR_UNSUPPORTED, "paged_read: too many heads");
    a.units0 = kv->Hkv * kv->Dk / dims, a.units = (int)units;
    a.tok = kMostTok;
    // fewer tokens a CTA where there would not be two CTAs an SM
    while (a.tok > 4 && (n_tokens + a.tok - 1) / a.tok * slices < 2 * device_sm_count()) a.tok /= 2;
    const int64_t blocks = (n_tokens + a.tok - 1) / a.tok;
    if (blocks > INT32_MAX) return set_error(WS_ERR_UNSUPPORTED, "paged_read: too many tokens");
    a.status = device_status_word();
    const bool f16 = out_dtype == WS_DTYPE_F16, i8 = kv->dtype == WS_DTYPE_I8;
    // four loads in flight where what is read and written may lie in L2 and a thread has more than two tokens (31 requests
    // of one head, two tokens a thread: 5.4 us with four, 4.1 with two)
    const bool small = a.tok * std::min<int64_t>(units, kThreads) > 2 * kThreads && n_tokens * kv->Hkv * (kv->Dk + kv->Dv) <= 48 << 20;
    auto pick = [&](auto ahead) {
        constexpr int A = decltype(ahead)::value;
        return !eight ? read_kernel<false, 0, A>
               : f16  ? (i8 ? read_kernel<true, 1, A> : read_kernel<true, 2, A>)
                      : (i8 ? read_kernel<false, 1, A> : read_kernel<false, 2, A>);
    };
    auto fn = small ? pick(std::integral_constant<int, 4>{}) : pick(std::integral_constant<int, 2>{});
    const cudaError_t e = launch_dependent(fn, dim3((unsigned)blocks, (unsigned)slices), kThreads, 0,
                                           static_cast<cudaStream_t>(stream), a);
    return e == cudaSuccess ? WS_OK : set_error(WS_ERR_CUDA, cudaGetErrorString(e));
}
