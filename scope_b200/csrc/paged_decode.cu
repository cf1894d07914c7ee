// Entry of the decode attention over a paged key-value cache: checks, the choice of a variant, the launch.
// The kernel and its reasons: paged_decode.cuh.
#include <cstdio>

#include "paged_decode.cuh"

namespace ws {
namespace {

constexpr int kMaxWarps = 8;

// Heads a block: 8 (one tensor-core column tile) up to 8 query heads a kv head, 16 up to 16, and 32 beyond -- a
// block reads its keys and values once, so fewer blocks mean fewer bytes -- but at most 16 at head dims past 128,
// where the accumulators of 32 heads would not fit the registers.
int tiles_of(int G, int D) { return G <= 8 ? 1 : G <= 16 || D > 128 ? 2 : 4; }

}  // namespace
}  // namespace ws

using namespace ws;

extern "C" {

size_t ws_paged_decode_workspace_size(int B, int Hkv, int G, int Dv) {
    (void)B, (void)Hkv;
    return kCounterHeaderBytes +
           (size_t)device_sm_count() * (2 + kMaxWarps) * paged::piece_floats(tiles_of(G, 0), Dv) * sizeof(float);
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
    if (reinterpret_cast<uintptr_t>(out) % 16) return set_error(WS_ERR_INVALID_ARG, "paged_decode: out must be 16-byte aligned");
    if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 ||
        workspace_bytes < ws_paged_decode_workspace_size(B, kv->Hkv, G, kv->Dv))
        return set_error(WS_ERR_WORKSPACE, "paged_decode: workspace missing, unaligned or too small");
    const bool f16 = q_dtype == WS_DTYPE_F16, i8 = kv->dtype == WS_DTYPE_I8;
    const int64_t eb = i8 ? 1 : 2;
    const int D = std::max(kv->Dk, kv->Dv), DB = D <= 64 ? 64 : D <= 128 ? 128 : 256, NT = tiles_of(G, D);
    paged::Args a;
    memset(&a, 0, sizeof(a));
    a.q = static_cast<const uint16_t*>(q);
    a.q_b = q_stride_b, a.q_h = q_stride_h;
    a.k = static_cast<const uint8_t*>(kv->k), a.v = static_cast<const uint8_t*>(kv->v);
    a.kp = kv->k_stride_page * eb, a.kt = kv->k_stride_tok * eb, a.kh = kv->k_stride_head * eb;
    a.vp = kv->v_stride_page * eb, a.vt = kv->v_stride_tok * eb, a.vh = kv->v_stride_head * eb;
    a.ks = kv->k_scales, a.vs = kv->v_scales;
    a.ksp = kv->ks_stride_page, a.kst = kv->ks_stride_tok, a.ksh = kv->ks_stride_head;
    a.vsp = kv->vs_stride_page, a.vst = kv->vs_stride_tok, a.vsh = kv->vs_stride_head;
    a.table = page_table, a.table_stride = table_stride;
    a.seq_lens = seq_lens;
    a.cap = std::min<int64_t>((int64_t)max_pages * kv->page_size, INT32_MAX - 64);
    a.n_pages = (int)kv->n_pages, a.page_size = kv->page_size;
    // t / page_size for t < 2^31 as a multiply and a shift: shift = ceil(log2 P), mul = floor(2^32 (2^shift - P) / P) + 1
    while ((1ull << a.div_shift) < (uint64_t)kv->page_size) ++a.div_shift;
    a.div_mul = (uint32_t)((((1ull << a.div_shift) - kv->page_size) << 32) / kv->page_size + 1);
    a.B = B, a.Hkv = kv->Hkv, a.G = G, a.Dk = kv->Dk, a.Dv = kv->Dv, a.window = window;
    a.hb = (G + 8 * NT - 1) / (8 * NT);
    a.scale_log2 = scale * kLog2e;
    a.out = static_cast<uint16_t*>(out);
    a.lse = out_lse;
    a.counters = static_cast<int*>(workspace);
    a.pieces = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kCounterHeaderBytes);
    a.status = device_status_word();
    const int ctas = device_sm_count();
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (f16) return i8 ? paged::launch_f16_i8(a, DB, NT, ctas, st) : paged::launch_f16(a, DB, NT, ctas, st);
    return i8 ? paged::launch_bf16_i8(a, DB, NT, ctas, st) : paged::launch_bf16(a, DB, NT, ctas, st);
}

}  // extern "C"
