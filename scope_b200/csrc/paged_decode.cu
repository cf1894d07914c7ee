// Decode attention over a paged key-value cache: one new token per request.
//
//   o = sum_t softmax_t(scale q.k_t) v_t,  lse = log sum_t exp(scale q.k_t),  t in [max(0, L - window), L)
//
// One CTA per (request, query head).  Its warps take every fourth token and
// keep a running maximum m, sum l and accumulator o; a token's score s moves
// them to m' = max(m, s), l' = l 2^(m-m') + 2^(s-m'), o' likewise; the warps'
// states are joined by the same rule.
#include "common.cuh"
#include "ws_internal.h"

#include <cuda_fp16.h>

namespace ws {
namespace {

constexpr int kWarps = 4;
constexpr int kMaxD = 256;

struct PagedDecodeArgs {
    const uint16_t* q;
    int64_t q_b, q_h;
    ws_paged_kv kv;
    const int32_t* table;
    int64_t table_stride;
    int max_pages;
    const int32_t* seq_lens;
    int G, window;
    float scale_log2;
    uint16_t* out;
    float* lse;
    int* status;
};

template <bool F16>
__device__ __forceinline__ float to_f32(uint16_t v) {
    if (F16) return __half2float(__ushort_as_half(v));
    return __bfloat162float(__ushort_as_bfloat16(v));
}

template <bool F16, bool I8>
__global__ void __launch_bounds__(32 * kWarps) paged_decode_kernel(const __grid_constant__ PagedDecodeArgs a) {
    __shared__ float so[kWarps][kMaxD], sml[kWarps][2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int b = blockIdx.y, h = blockIdx.x, kvh = h / a.G, H = gridDim.x;
    const ws_paged_kv& kv = a.kv;
    const int64_t L = min((int64_t)max(a.seq_lens[b], 0), (int64_t)a.max_pages * kv.page_size);
    const int64_t first = a.window > 0 ? max(L - a.window, (int64_t)0) : 0;
    const uint16_t* q = a.q + b * a.q_b + h * a.q_h;
    float qr[kMaxD / 32], o[kMaxD / 32], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < kMaxD / 32; ++i) {
        const int d = lane + 32 * i;
        qr[i] = d < kv.Dk ? to_f32<F16>(q[d]) : 0.f;
        o[i] = 0.f;
    }
    for (int64_t t = first + warp; t < L; t += kWarps) {
        const int page = a.table[b * a.table_stride + t / kv.page_size];
        if ((unsigned)page >= (uint64_t)kv.n_pages) {
            if (lane == 0 && a.status) atomicMax(a.status, kDevBadIndex);
            continue;
        }
        const int64_t off = t % kv.page_size;
        const int64_t ka = page * kv.k_stride_page + off * kv.k_stride_tok + kvh * kv.k_stride_head;
        const int64_t va = page * kv.v_stride_page + off * kv.v_stride_tok + kvh * kv.v_stride_head;
        const float ks = I8 ? kv.k_scales[page * kv.ks_stride_page + off * kv.ks_stride_tok + kvh * kv.ks_stride_head] : 1.f;
        const float vs = I8 ? kv.v_scales[page * kv.vs_stride_page + off * kv.vs_stride_tok + kvh * kv.vs_stride_head] : 1.f;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < kMaxD / 32; ++i) {
            const int d = lane + 32 * i;
            if (d < kv.Dk)
                s += qr[i] * (I8 ? (float)static_cast<const int8_t*>(kv.k)[ka + d]
                                 : to_f32<F16>(static_cast<const uint16_t*>(kv.k)[ka + d]));
        }
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        s *= ks * a.scale_log2;
        const float m2 = fmaxf(m, s);
        const float keep = m2 == -INFINITY ? 1.f : ex2(m - m2), p = m2 == -INFINITY ? 0.f : ex2(s - m2);
        l = l * keep + p;
#pragma unroll
        for (int i = 0; i < kMaxD / 32; ++i) {
            const int d = lane + 32 * i;
            if (d < kv.Dv)
                o[i] = o[i] * keep + p * vs * (I8 ? (float)static_cast<const int8_t*>(kv.v)[va + d]
                                                  : to_f32<F16>(static_cast<const uint16_t*>(kv.v)[va + d]));
        }
        m = m2;
    }
#pragma unroll
    for (int i = 0; i < kMaxD / 32; ++i) so[warp][lane + 32 * i] = o[i];
    if (lane == 0) sml[warp][0] = m, sml[warp][1] = l;
    __syncthreads();
    float M = -INFINITY, sum = 0.f;
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sml[w][0]);
    for (int w = 0; w < kWarps; ++w) sum += M == -INFINITY ? 0.f : sml[w][1] * ex2(sml[w][0] - M);
    for (int d = threadIdx.x; d < kv.Dv; d += blockDim.x) {
        float x = 0.f;
        for (int w = 0; w < kWarps; ++w) x += M == -INFINITY ? 0.f : so[w][d] * ex2(sml[w][0] - M);
        x = sum > 0.f ? x / sum : 0.f;
        uint16_t* p = a.out + ((int64_t)b * H + h) * kv.Dv + d;
        if (F16) *p = __half_as_ushort(__float2half_rn(x));
        else *p = __bfloat16_as_ushort(__float2bfloat16_rn(x));
    }
    if (threadIdx.x == 0 && a.lse) a.lse[(int64_t)b * H + h] = sum > 0.f ? M * kLn2 + logf(sum) : -INFINITY;
}

}  // namespace
}  // namespace ws

using namespace ws;

extern "C" {

size_t ws_paged_decode_workspace_size(int B, int Hkv, int G, int Dv) {
    (void)B, (void)Hkv, (void)G, (void)Dv;
    return kCounterHeaderBytes;
}

int ws_paged_decode(const void* q, int64_t q_stride_b, int64_t q_stride_h, int q_dtype, int B, int G,
                    const ws_paged_kv* kv, const int32_t* page_table, int64_t table_stride, int max_pages,
                    const int32_t* seq_lens, int window, float scale, void* out, float* out_lse, void* workspace,
                    size_t workspace_bytes, void* stream) {
    if (!kv || B < 0 || G < 1 || max_pages < 0 || window < 0 || table_stride < 0)
        return set_error(WS_ERR_INVALID_ARG, "paged_decode: bad shape");
    if (const int rc = paged_kv_check("paged_decode", kv)) return rc;
    if (q_dtype != WS_DTYPE_BF16 && q_dtype != WS_DTYPE_F16)
        return set_error(WS_ERR_INVALID_ARG, "paged_decode: q must be bf16 or fp16");
    if (kv->dtype != WS_DTYPE_I8 && kv->dtype != q_dtype)
        return set_error(WS_ERR_INVALID_ARG, "paged_decode: the pool must hold q's type or int8");
    if (B == 0) return WS_OK;
    if (!q || !out || !seq_lens || (max_pages > 0 && !page_table))
        return set_error(WS_ERR_INVALID_ARG, "paged_decode: null pointer");
    if (reinterpret_cast<uintptr_t>(q) % 16 || q_stride_b % 8 || q_stride_h % 8)
        return set_error(WS_ERR_INVALID_ARG, "paged_decode: q's rows must be 16-byte aligned");
    if (B > 65535) return set_error(WS_ERR_UNSUPPORTED, "paged_decode: more than 65535 requests");
    if (!workspace || workspace_bytes < ws_paged_decode_workspace_size(B, kv->Hkv, G, kv->Dv))
        return set_error(WS_ERR_WORKSPACE, "paged_decode: workspace missing or too small");
    PagedDecodeArgs a;
    a.q = static_cast<const uint16_t*>(q);
    a.q_b = q_stride_b, a.q_h = q_stride_h;
    a.kv = *kv;
    a.table = page_table, a.table_stride = table_stride, a.max_pages = max_pages;
    a.seq_lens = seq_lens;
    a.G = G, a.window = window;
    a.scale_log2 = scale * kLog2e;
    a.out = static_cast<uint16_t*>(out);
    a.lse = out_lse;
    a.status = device_status_word();
    const bool f16 = q_dtype == WS_DTYPE_F16, i8 = kv->dtype == WS_DTYPE_I8;
    auto fn = f16 ? (i8 ? paged_decode_kernel<true, true> : paged_decode_kernel<true, false>)
                  : (i8 ? paged_decode_kernel<false, true> : paged_decode_kernel<false, false>);
    fn<<<dim3(kv->Hkv * G, B), 32 * kWarps, 0, static_cast<cudaStream_t>(stream)>>>(a);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? WS_OK : set_error(WS_ERR_CUDA, cudaGetErrorString(e));
}

}  // extern "C"
