// Entry of the decode attention over a paged key-value cache: checks, the choice of a variant, the launch.
// The kernel and its reasons: paged_decode.cuh.
#include <cstdio>

#include "paged_decode.cuh"

namespace ws {
namespace {

// Heads a block: 8 (one tensor-core column tile) up to 8 query heads a kv head and at head dims past 128, else 16.  A
// block reads its keys and values once, so fewer blocks mean fewer bytes, but more accumulators do not fit the registers.
int tiles_of(int G, int DB) { return G <= 8 || DB > 128 ? 1 : 2; }
int bound_of(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : D <= 192 ? 192 : 256; }

}  // namespace
}  // namespace ws

using namespace ws;

extern "C" {

size_t ws_paged_decode_workspace_size(int B, int Hkv, int G, int Dv) {
    (void)B, (void)Hkv, (void)G, (void)Dv;
    // two row parts a CTA; the larger of the two forms that a key dim of up to 256 may choose
    const size_t piece = std::max(paged::piece_floats(256, 1), paged::piece_floats(128, 2));
    return kCounterHeaderBytes + (size_t)device_sm_count() * 2 * piece * sizeof(float);
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
    // the kernel keeps a kv head and its block of query heads in one word
    if (kv->Hkv > INT16_MAX || G > (1 << 18) || (int64_t)kv->Hkv * G > (1 << 24))
        return set_error(WS_ERR_UNSUPPORTED, "paged_decode: too many heads");
    const bool f16 = q_dtype == WS_DTYPE_F16, i8 = kv->dtype == WS_DTYPE_I8;
    const int64_t eb = i8 ? 1 : 2;
    const int D = std::max(kv->Dk, kv->Dv), DB = bound_of(D), NT = tiles_of(G, DB);
    paged::Args a;
    memset(&a, 0, sizeof(a));
    a.q = static_cast<const uint16_t*>(q);
    a.q_b = q_stride_b, a.q_h = q_stride_h;
    a.k = static_cast<const uint8_t*>(kv->k), a.v = static_cast<const uint8_t*>(kv->v);
    const int64_t strides[6] = {kv->k_stride_page, kv->k_stride_tok, kv->k_stride_head,
                                kv->v_stride_page, kv->v_stride_tok, kv->v_stride_head};
    uint32_t* const pieces[6] = {&a.kp, &a.kt, &a.kh, &a.vp, &a.vt, &a.vh};
    const int64_t scale_strides[6] = {kv->ks_stride_page, kv->ks_stride_tok, kv->ks_stride_head,
                                      kv->vs_stride_page, kv->vs_stride_tok, kv->vs_stride_head};
    uint32_t* const floats[6] = {&a.ksp, &a.kst, &a.ksh, &a.vsp, &a.vst, &a.vsh};
    for (int i = 0; i < 6; ++i) {
        if (strides[i] * eb / 16 > UINT32_MAX || (i8 && (scale_strides[i] > UINT32_MAX || scale_strides[i] < 0)))
            return set_error(WS_ERR_UNSUPPORTED, "paged_decode: a pool stride of 64 GB or more");
        *pieces[i] = (uint32_t)(strides[i] * eb / 16);
        *floats[i] = i8 ? (uint32_t)scale_strides[i] : 0;
    }
    a.ks = kv->k_scales, a.vs = kv->v_scales;
    a.table = page_table, a.table_stride = table_stride;
    a.seq_lens = seq_lens;
    a.cap = (int)std::min<int64_t>((int64_t)max_pages * kv->page_size, INT32_MAX - 64);
    a.whole = kv->page_size % 16 == 0;
    const int inner = paged::inner_of(DB * (int)eb);
    // Rows short by the table's width, or the window, are faster with cp.async, whose first bytes are there sooner and
    // whose last subtile costs less (us with TMA and with cp.async: 204 requests of up to 101 tokens 12.9 and 12.5, 64 of
    // up to 2 8.8 and 8.3; 1 of 4096 11.9 and 12.1, 16 of up to 32768 136 and 146).
    const bool whole_rows = kv->page_size % 16 == 0 && kv->Dk == DB && kv->Dv == DB && kv->n_pages > 0;
    a.tma = whole_rows && (window > 0 ? std::min(a.cap, window) : a.cap) > 512 &&
            make_page_map(&a.kmap, kv->k, DB * eb, kv->page_size, kv->Hkv, kv->n_pages, kv->k_stride_tok * eb,
                          kv->k_stride_head * eb, kv->k_stride_page * eb, inner, &a.k_head_dim2) &&
            make_page_map(&a.vmap, kv->v, DB * eb, kv->page_size, kv->Hkv, kv->n_pages, kv->v_stride_tok * eb,
                          kv->v_stride_head * eb, kv->v_stride_page * eb, inner, &a.v_head_dim2);
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
    // The kernel counts subtiles in 32 bits: more requests at once than that holds, were every row of the table full,
    // go in several launches.
    const int64_t most = (std::min<int64_t>(a.cap, window > 0 ? (int64_t)window + 32 : a.cap) / 16 + 1) *
                         kv->Hkv * a.hb;
    if (most > INT32_MAX / 2) return set_error(WS_ERR_UNSUPPORTED, "paged_decode: too many tokens times kv heads in one request");
    const int at_once = (int)std::min<int64_t>(B, INT32_MAX / 2 / most);
    for (int b = 0; b < B; b += at_once) {
        paged::Args c = a;
        c.B = std::min(at_once, B - b);
        c.q += b * q_stride_b, c.table += b * table_stride, c.seq_lens += b;
        c.out += (int64_t)b * kv->Hkv * G * kv->Dv;
        if (c.lse) c.lse += (int64_t)b * kv->Hkv * G;
        const int rc = f16 ? (i8 ? paged::launch_f16_i8(c, DB, NT, ctas, st) : paged::launch_f16(c, DB, NT, ctas, st))
                           : (i8 ? paged::launch_bf16_i8(c, DB, NT, ctas, st) : paged::launch_bf16(c, DB, NT, ctas, st));
        if (rc != WS_OK) return rc;
    }
    return WS_OK;
}

}  // extern "C"
