// Rotary positions with several axes, and the append of a step's keys and
// values into a paged cache, in one pass over q, k and v.
//
//   y1 = x1 cos - x2 sin,  y2 = x2 cos + x1 sin,   (cos, sin) = cos_sin[position[axis(i)], i]
//
// What bounds it: memory.  Each value is read once and written once, and the
// arithmetic is four operations a pair.  A thread owns a unit of 16 dims of a
// head -- eight pairs, so both halves of every pair are its own: 16 bytes at
// dim 8u and 16 at rope_dim/2 + 8u, or 32 contiguous bytes for adjacent pairs
// and for the dims that pass unrotated -- and walks the heads of its token, so
// the eight cosines and sines are loaded once for all of them (a warp for every
// step of heads would load them again and again: 94 us instead of 54).  The
// units of a head are padded to a power of two and lie in one warp, which the
// int8 form needs for the row's maximum.  Measured: 16384 x 32 heads of 128,
// three axes, 47.3 us (277 MB, 5.9 TB/s); append of 16384 tokens of 32 + 4 + 4
// heads 60.3 us (345 MB, 5.7 TB/s); 4097 tokens of 20 + 5 + 5 heads of 80 into
// int8 15.0 us; 17.9 thousand of 4 + 4 heads of 128 into e4m3 rows 24.  The
// first rows are asked for before the position is known, whose turns would else
// delay them by two latencies (47.9 and 61.9 us; 1202 tokens of 40 + 8 + 8
// heads 11.9 to 10.8; 64 tokens 2.65 to 2.47).
//
// Products and sums are rounded one by one (no fused multiply-add): the result
// is the elementwise formula's, bit for bit, so an int8 code never depends on
// which program computed it.
#include <cstdio>

#include "rope_append.cuh"

#include <type_traits>

namespace ws {
namespace {

constexpr int kWarps = 4;
constexpr int kGroup = 2;   // rows a thread loads before it turns the first, where it has several

template <bool F16, int CODE, bool VEC, int GROUP>
__global__ void __launch_bounds__(32 * kWarps) rope_append_kernel(const __grid_constant__ RopeAppendArgs a) {
    pdl_wait_primary();
    pdl_launch_dependents();
    rope_rows<F16, CODE, VEC, GROUP>(a, (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5));
}

}  // namespace

int paged_kv_check(const char* what, const ws_paged_kv* kv) {
    char buf[200];
    const char* why = nullptr;
    int code = WS_ERR_INVALID_ARG;
    const bool eight = kv->dtype == WS_DTYPE_I8 || kv->dtype == WS_DTYPE_E4M3;
    const int eb = eight ? 1 : 2;
    const int64_t st[6] = {kv->k_stride_page, kv->k_stride_tok, kv->k_stride_head,
                           kv->v_stride_page, kv->v_stride_tok, kv->v_stride_head};
    if (kv->dtype != WS_DTYPE_BF16 && kv->dtype != WS_DTYPE_F16 && !eight)
        why = "the pool's dtype must be bf16, fp16, int8 or e4m3";
    else if (kv->Hkv < 1 || kv->page_size < 1 || kv->n_pages < 0 || kv->Dk < 1 || kv->Dv < 1)
        why = "bad pool shape";
    else if (kv->Dk % 16 || kv->Dv % 16 || kv->Dk > 256 || kv->Dv > 256)
        why = "head dims must be multiples of 16, at most 256", code = WS_ERR_UNSUPPORTED;
    else if (eight && (kv->scale_block < 0 || kv->page_size % std::max(kv->scale_block, 1)))
        why = "a page must be whole blocks of a scale";
    else if (kv->n_pages > 0 && (!kv->k || !kv->v || (eight && (!kv->k_scales || !kv->v_scales))))
        why = "null pool pointer";
    else if (reinterpret_cast<uintptr_t>(kv->k) % 16 || reinterpret_cast<uintptr_t>(kv->v) % 16)
        why = "the pool must be 16-byte aligned";
    else if (kv->n_pages > INT32_MAX)
        why = "more than 2^31 - 1 pages", code = WS_ERR_UNSUPPORTED;
    else
        for (int i = 0; i < 6; ++i)
            if (st[i] < 0 || st[i] * eb % 16) why = "pool strides must be whole 16 bytes";
    if (!why) return WS_OK;
    snprintf(buf, sizeof(buf), "%s: %s", what, why);
    return set_error(code, buf);
}

}  // namespace ws

using namespace ws;

extern "C" int ws_rope_append(const ws_rope* rope, const void* q, int64_t q_stride_tok, int64_t q_stride_head, int H,
                              int D, void* q_out, int64_t qo_stride_tok, int64_t qo_stride_head, const void* k,
                              int64_t k_stride_tok, int64_t k_stride_head, const void* v, int64_t v_stride_tok,
                              int64_t v_stride_head, int dtype, int64_t N, const int64_t* slots, const ws_paged_kv* kv,
                              void* stream) {
    if (N < 0 || H < 0 || (!kv && D < 1)) return set_error(WS_ERR_INVALID_ARG, "rope_append: bad shape");
    if (dtype != WS_DTYPE_BF16 && dtype != WS_DTYPE_F16)
        return set_error(WS_ERR_INVALID_ARG, "rope_append: q, k, v must be bf16 or fp16");
    if (kv) {
        if (const int rc = paged_kv_check("rope_append", kv)) return rc;
        if (kv->dtype != WS_DTYPE_I8 && kv->dtype != WS_DTYPE_E4M3 && kv->dtype != dtype)
            return set_error(WS_ERR_INVALID_ARG, "rope_append: the pool must hold the inputs' type, int8 or e4m3");
        if (H > 0 && D != kv->Dk) return set_error(WS_ERR_INVALID_ARG, "rope_append: q and k differ in their head dim");
    }
    if (D % 16 || D > 256) return set_error(WS_ERR_UNSUPPORTED, "rope_append: head dims must be multiples of 16, at most 256");
    if (N == 0 || (H == 0 && !kv)) return WS_OK;
    if ((H > 0 && (!q || !q_out)) || (kv && (!k || !v || !slots)))
        return set_error(WS_ERR_INVALID_ARG, "rope_append: null pointer");
    if (kv && kv->n_pages == 0) return set_error(WS_ERR_INVALID_ARG, "rope_append: empty pool");
    RopeAppendArgs a;
    memset(&a, 0, sizeof(a));
    int Dmax = H > 0 ? D : 16;
    a.h[0].src = static_cast<const uint16_t*>(q);
    a.h[0].src_tok = q_stride_tok, a.h[0].src_head = q_stride_head;
    a.h[0].dst = static_cast<uint8_t*>(q_out);
    a.h[0].dst_tok = qo_stride_tok, a.h[0].dst_head = qo_stride_head;
    a.h[0].n = H, a.h[0].D = D;
    auto aligned = [](const void* p, int64_t s0, int64_t s1) {
        return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s0 % 8 == 0 && s1 % 8 == 0;
    };
    bool vec = H == 0 || (aligned(q, q_stride_tok, q_stride_head) && aligned(q_out, qo_stride_tok, qo_stride_head));
    if (kv) {
        a.h[1] = {static_cast<const uint16_t*>(k), k_stride_tok, k_stride_head, static_cast<uint8_t*>(kv->k),
                  kv->k_stride_tok, kv->k_stride_head, kv->k_stride_page, kv->k_scales, kv->ks_stride_page,
                  kv->ks_stride_tok, kv->ks_stride_head, kv->Hkv, kv->Dk};
        a.h[2] = {static_cast<const uint16_t*>(v), v_stride_tok, v_stride_head, static_cast<uint8_t*>(kv->v),
                  kv->v_stride_tok, kv->v_stride_head, kv->v_stride_page, kv->v_scales, kv->vs_stride_page,
                  kv->vs_stride_tok, kv->vs_stride_head, kv->Hkv, kv->Dv};
        a.slots = slots;
        a.n_slots = kv->n_pages * kv->page_size;
        a.page_size = kv->page_size;
        Dmax = std::max(Dmax, std::max(kv->Dk, kv->Dv));
        vec = vec && aligned(k, k_stride_tok, k_stride_head) && aligned(v, v_stride_tok, v_stride_head);
    }
    if (rope) {
        const int Dk = kv ? kv->Dk : D;
        if (rope->rope_dim < 16 || rope->rope_dim % 16 || rope->rope_dim > Dk)
            return set_error(WS_ERR_INVALID_ARG, "rope_append: rope_dim must be a multiple of 16 within the head dim");
        if (rope->n_axes < 1 || rope->n_axes > 4 || rope->max_pos < 1 || rope->max_pos > INT32_MAX || !rope->positions || !rope->cos_sin)
            return set_error(WS_ERR_INVALID_ARG, "rope_append: bad rope");
        for (int i = 0; i < rope->rope_dim / 2; ++i)
            if ((int)((rope->axis_map[i >> 4] >> (2 * (i & 15))) & 3) >= rope->n_axes)
                return set_error(WS_ERR_INVALID_ARG, "rope_append: a pair's axis has no positions");
        a.rope = *rope;
        a.turns_vec = reinterpret_cast<uintptr_t>(rope->cos_sin) % 16 == 0;
    }
    a.N = N;
    a.status = device_status_word();
    a.lanes = 1;
    while (a.lanes * 16 < Dmax) a.lanes *= 2;
    const int block = kv ? std::max(kv->scale_block, 1) : 1;
    const bool e4 = kv && kv->dtype == WS_DTYPE_E4M3, blocks8 = kv && block > 1 && (e4 || kv->dtype == WS_DTYPE_I8);
    if (blocks8 && H > 0 && !block_append_small(N, kv->Hkv)) {
        a.h[0].n = 0;
        if (const int rc = block_append_check(a, block)) return rc;   // before q_out, which may be q, is written
        if (const int rc = ws_rope_append(rope, q, q_stride_tok, q_stride_head, H, D, q_out, qo_stride_tok, qo_stride_head, nullptr, 0,
                                          0, nullptr, 0, 0, dtype, N, nullptr, nullptr, stream))
            return rc;
    }
    if (blocks8)
        return block_append_launch(a, dtype == WS_DTYPE_F16, kv->dtype == WS_DTYPE_E4M3, vec, block, static_cast<cudaStream_t>(stream));
    // One warp walks all heads of a token when there are tokens for every SM; with fewer, its rows are shared out.  Into
    // int8, where a row takes longer, that pays with half as many tokens only (4097 tokens of 20 + 5 + 5 heads, us with 16,
    // 32, 64 and 128 warps wanted an SM: 14.5, 15.5, 17.2, 20.4).
    const bool f16 = dtype == WS_DTYPE_F16, i8 = e4 || (kv && kv->dtype == WS_DTYPE_I8);
    const int rows = 32 / a.lanes, steps = (H + (kv ? 2 * kv->Hkv : 0) + rows - 1) / rows;
    const int64_t want = (int64_t)device_sm_count() * (i8 ? 16 : 32);
    a.parts = (int)std::max<int64_t>(1, std::min<int64_t>(steps, (want + N - 1) / N));
    const int64_t blocks = (N * a.parts + kWarps - 1) / kWarps;
    if (blocks > INT32_MAX) return set_error(WS_ERR_UNSUPPORTED, "rope_append: too many tokens");
    // Two rows in flight a thread where a warp walks many (16384 tokens of 32 heads, us a call with one and two: rotary
    // alone 51 and 48, append 67 and 62); with few rows, or int8 codes to compute, the registers cost more than that gives
    // (5212 tokens of 3 heads of 256: 15 and 18; 4097 tokens into int8: 38 and 41).
    const bool several = a.parts == 1 && steps >= 8 && !i8;
    auto pick = [&](auto half, auto codes) {
        constexpr bool F = decltype(half)::value;
        constexpr int C = decltype(codes)::value;
        if (!vec) return rope_append_kernel<F, C, false, 1>;
        if constexpr (C == kRows16)
            if (several) return rope_append_kernel<F, C, true, kGroup>;
        return rope_append_kernel<F, C, true, 1>;
    };
    auto by = [&](auto half) {
        if (e4) return pick(half, std::integral_constant<int, kRowsE4M3>{});
        return i8 ? pick(half, std::integral_constant<int, kRowsS8>{}) : pick(half, std::integral_constant<int, kRows16>{});
    };
    auto fn = f16 ? by(std::true_type{}) : by(std::false_type{});
    const cudaError_t e = launch_dependent(fn, dim3((unsigned)blocks), 32 * kWarps, 0, static_cast<cudaStream_t>(stream), a);
    return e == cudaSuccess ? WS_OK : set_error(WS_ERR_CUDA, cudaGetErrorString(e));
}
