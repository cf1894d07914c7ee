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

// diff: null, or what differential attention takes more; G counts its maps then, two a head.
struct Diff {
    const float* lam;
    int lam_stride;
    const float* weight;
    float eps;
};
int decode(const char* what, const Diff* diff, const void* q, int64_t q_stride_b, int64_t q_stride_h, int q_dtype, int B, int G,
           const ws_paged_kv* kv, const int32_t* page_table, int64_t table_stride, int max_pages, const int32_t* seq_lens,
           int window, float scale, void* out, float* out_lse, void* workspace, size_t workspace_bytes, void* stream) {
    char msg[160];
    auto refuse = [&](int code, const char* why) {
        snprintf(msg, sizeof(msg), "%s: %s", what, why);
        return set_error(code, msg);
    };
    if (!kv || B < 0 || G < 1 || max_pages < 0 || window < 0 || table_stride < 0)
        return refuse(WS_ERR_INVALID_ARG, "bad shape");
    if (const int rc = paged_kv_check(what, kv)) return rc;
    if (q_dtype != WS_DTYPE_BF16 && q_dtype != WS_DTYPE_F16)
        return refuse(WS_ERR_INVALID_ARG, "q must be bf16 or fp16");
    const bool i8 = kv->dtype == WS_DTYPE_I8, e4 = kv->dtype == WS_DTYPE_E4M3, eight = i8 || e4;
    if (!eight && kv->dtype != q_dtype) return refuse(WS_ERR_INVALID_ARG, "the pool must hold q's type or int8 or e4m3");
    if (diff && (kv->Hkv % 2 || kv->Dk > 128 || kv->Dv > 128))
        return kv->Hkv % 2 ? refuse(WS_ERR_INVALID_ARG, "the pool's heads come in pairs")
                           : refuse(WS_ERR_UNSUPPORTED, "head dims of a map, and half a value, of at most 128");
    // a pair of heads is one of twice the dims
    const int maps = diff ? 2 : 1, Hkv = kv->Hkv / maps, Dk = maps * kv->Dk, Dv = maps * kv->Dv;
    if (B == 0) return WS_OK;
    if (!q || !out || !seq_lens || (diff && !diff->lam) || (max_pages > 0 && !page_table))
        return refuse(WS_ERR_INVALID_ARG, "null pointer");
    if (reinterpret_cast<uintptr_t>(q) % 16 || q_stride_b % 8 || q_stride_h % 8)
        return refuse(WS_ERR_INVALID_ARG, "q's rows must be 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(out) % 16) return refuse(WS_ERR_INVALID_ARG, "out must be 16-byte aligned");
    if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 ||
        workspace_bytes < ws_paged_decode_workspace_size(B, Hkv, G, Dv))
        return refuse(WS_ERR_WORKSPACE, "workspace missing, unaligned or too small");
    // the kernel keeps a kv head and its block of query heads in one word
    if (Hkv > INT16_MAX || G > (1 << 18) || (int64_t)Hkv * G > (1 << 24))
        return refuse(WS_ERR_UNSUPPORTED, "too many heads");
    const bool f16 = q_dtype == WS_DTYPE_F16;
    const int64_t eb = eight ? 1 : 2;
    const int D = std::max(Dk, Dv), DB = bound_of(D), NT = tiles_of(G, DB);
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
        const int64_t step = i % 3 == 2 ? maps * strides[i] : strides[i];   // from pair to pair
        if (step * eb / 16 > UINT32_MAX || (eight && (scale_strides[i] > UINT32_MAX || scale_strides[i] < 0)))
            return refuse(WS_ERR_UNSUPPORTED, "a pool stride of 64 GB or more");
        *pieces[i] = (uint32_t)(step * eb / 16);
        *floats[i] = eight ? (uint32_t)scale_strides[i] : 0;
    }
    if (diff) {
        a.kjump = (kv->k_stride_head - kv->Dk) * eb, a.vjump = (kv->v_stride_head - kv->Dv) * eb;
        a.lam = diff->lam, a.lam_stride = diff->lam_stride, a.weight = diff->weight, a.eps = diff->eps;
    }
    a.ks = kv->k_scales, a.vs = kv->v_scales;
    a.table = page_table, a.table_stride = table_stride;
    a.seq_lens = seq_lens;
    a.cap = (int)std::min<int64_t>((int64_t)max_pages * kv->page_size, INT32_MAX - 64);
    a.whole = kv->page_size % 16 == 0;
    const int head_bytes = DB / maps * (int)eb, inner = paged::inner_of(head_bytes);
    const int code = i8 ? paged::kS8 : e4 ? paged::kE4M3 : paged::k16, tok = paged::tok_of(code, diff != nullptr, DB);
    a.flat = eight && kv->page_size % tok == 0 && std::max(kv->scale_block, 1) % tok == 0;
    const int box = a.flat && paged::one_box(code, diff != nullptr, DB) ? 32 : 16;
    // Rows short by the table's width, or the window, are faster with cp.async, whose first bytes are there sooner and
    // whose last subtile costs less (us with TMA and with cp.async: 204 requests of up to 101 tokens 12.9 and 12.5, 64 of
    // up to 2 8.8 and 8.3; 1 of 4096 11.9 and 12.1, 16 of up to 32768 136 and 146).
    const bool whole_rows = kv->page_size % 16 == 0 && Dk == DB && Dv == DB && head_bytes % 64 == 0 && kv->n_pages > 0;
    a.tma = whole_rows && (window > 0 ? std::min(a.cap, window) : a.cap) > 512 &&
            make_page_map(&a.kmap, kv->k, head_bytes, kv->page_size, kv->Hkv, kv->n_pages, kv->k_stride_tok * eb,
                          kv->k_stride_head * eb, kv->k_stride_page * eb, inner, box, &a.k_head_dim2) &&
            make_page_map(&a.vmap, kv->v, head_bytes, kv->page_size, kv->Hkv, kv->n_pages, kv->v_stride_tok * eb,
                          kv->v_stride_head * eb, kv->v_stride_page * eb, inner, box, &a.v_head_dim2);
    a.n_pages = (int)kv->n_pages, a.page_size = kv->page_size;
    // t / P for t < 2^31 as a multiply and a shift: shift = ceil(log2 P), mul = floor(2^32 (2^shift - P) / P) + 1
    auto divide_by = [](int P, uint32_t& mul, uint32_t& shift) {
        while ((1ull << shift) < (uint64_t)P) ++shift;
        mul = (uint32_t)((((1ull << shift) - P) << 32) / P + 1);
    };
    divide_by(kv->page_size, a.div_mul, a.div_shift);
    divide_by(std::max(kv->scale_block, 1), a.blk_mul, a.blk_shift);
    a.B = B, a.Hkv = Hkv, a.G = G, a.Dk = Dk, a.Dv = Dv, a.window = window;
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
                         Hkv * a.hb;
    if (most > INT32_MAX / 2) return refuse(WS_ERR_UNSUPPORTED, "too many tokens times kv heads in one request");
    const int at_once = (int)std::min<int64_t>(B, INT32_MAX / 2 / most);
    for (int b = 0; b < B; b += at_once) {
        paged::Args c = a;
        c.B = std::min(at_once, B - b);
        c.q += b * q_stride_b, c.table += b * table_stride, c.seq_lens += b;
        c.out += (int64_t)b * Hkv * G / maps * Dv;
        if (c.lse) c.lse += (int64_t)b * Hkv * G;
        using namespace paged;
        auto fn = diff ? (f16 ? (i8 ? launch_diff_f16_i8 : e4 ? launch_diff_f16_e4 : launch_diff_f16)
                              : (i8 ? launch_diff_bf16_i8 : e4 ? launch_diff_bf16_e4 : launch_diff_bf16))
                       : (f16 ? (i8 ? launch_f16_i8 : e4 ? launch_f16_e4 : launch_f16)
                              : (i8 ? launch_bf16_i8 : e4 ? launch_bf16_e4 : launch_bf16));
        if (const int rc = fn(c, DB, NT, ctas, st)) return rc;
    }
    return WS_OK;
}

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
    return decode("paged_decode", nullptr, q, q_stride_b, q_stride_h, q_dtype, B, G, kv, page_table, table_stride, max_pages,
                  seq_lens, window, scale, out, out_lse, workspace, workspace_bytes, stream);
}

int ws_paged_diff_decode(const void* q, int64_t q_stride_b, int64_t q_stride_h, int q_dtype, int B, int G,
                         const ws_paged_kv* kv, const int32_t* page_table, int64_t table_stride, int max_pages,
                         const int32_t* seq_lens, int window, float scale, const float* lam, int lam_stride,
                         const float* norm_weight, float norm_eps, void* out, float* out_lse, void* workspace,
                         size_t workspace_bytes, void* stream) {
    if (G < 1 || G > (1 << 17)) return set_error(G < 1 ? WS_ERR_INVALID_ARG : WS_ERR_UNSUPPORTED, "paged_diff_decode: bad number of heads");
    const Diff diff = {lam, lam_stride, norm_weight, norm_eps};
    return decode("paged_diff_decode", &diff, q, q_stride_b, q_stride_h, q_dtype, B, 2 * G, kv, page_table, table_stride,
                  max_pages, seq_lens, window, scale, out, out_lse, workspace, workspace_bytes, stream);
}

}  // extern "C"
