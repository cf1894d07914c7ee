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
// int8 15.0 us.  The first rows are asked for before the position is known,
// whose turns would else delay them by two latencies (47.9 and 61.9 us; 1202
// tokens of 40 + 8 + 8 heads 11.9 to 10.8; 64 tokens 2.65 to 2.47).
//
// Products and sums are rounded one by one (no fused multiply-add): the result
// is the elementwise formula's, bit for bit, so an int8 code never depends on
// which program computed it.
#include <cstdio>

#include "common.cuh"
#include "ws_internal.h"

#include <cuda_fp16.h>

#include <type_traits>

namespace ws {
namespace {

constexpr int kWarps = 4;
constexpr int kGroup = 2;   // rows a thread loads before it turns the first, where it has several

struct Heads {          // one of q, k, v: rows of (token, head)
    const uint16_t* src;
    int64_t src_tok, src_head;
    uint8_t* dst;       // q: the output; k, v: the pool
    int64_t dst_tok;    // q: per token; k, v: per slot of a page  (elements)
    int64_t dst_head, dst_page;
    float* scales;      // int8 pool only
    int64_t s_page, s_tok, s_head;
    int n, D;
};

struct RopeAppendArgs {
    Heads h[3];
    ws_rope rope;
    const int64_t* slots;
    int64_t N, n_slots;
    int page_size, lanes;   // lanes: units of a head, padded to a power of two
    int parts;              // warps that share a token's heads
    int turns_vec;          // cos_sin is 16-byte aligned
    int* status;
};

template <bool F16>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
    if (F16) return __half22float2(*reinterpret_cast<const __half2*>(&v));
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if (F16) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    return pack_bf16(a, b);
}

// The larger of two, or NaN where either is.
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// Eight 16-bit values from p; without VEC the address need not be aligned.
template <bool VEC>
__device__ __forceinline__ uint4 load8(const uint16_t* p) {
    if (VEC) return *reinterpret_cast<const uint4*>(p);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (uint32_t)p[2 * i] | ((uint32_t)p[2 * i + 1] << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <bool VEC>
__device__ __forceinline__ void store8(uint16_t* p, const uint4& v) {
    if (VEC) {
        *reinterpret_cast<uint4*>(p) = v;
        return;
    }
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        p[2 * i] = (uint16_t)w[i];
        p[2 * i + 1] = (uint16_t)(w[i] >> 16);
    }
}

// F16: fp16 inputs (else bf16); I8: the pool holds int8 codes; VEC: q, k, v and q_out are 16-byte aligned throughout.
template <bool F16, bool I8, bool VEC, int GROUP>
__global__ void __launch_bounds__(32 * kWarps) rope_append_kernel(const __grid_constant__ RopeAppendArgs a) {
    pdl_wait_primary();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int64_t item = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
    const int64_t t = a.parts == 1 ? item : item / a.parts;
    if (t >= a.N) return;
    const int part = (int)(item - t * a.parts);
    const int u = lane & (a.lanes - 1), row0 = lane / a.lanes, rows = 32 / a.lanes;

    const ws_rope& r = a.rope;
    const bool turned = 16 * u < r.rope_dim;
    const int total = a.h[0].n + a.h[1].n + a.h[2].n;
    auto locate = [&](int at, int& h, int& kind) {   // row `at` of the token: a head of q, k or v
        h = at, kind = 0;
        if (h >= a.h[0].n) h -= a.h[0].n, kind = 1;
        if (kind == 1 && h >= a.h[1].n) h -= a.h[1].n, kind = 2;
        return at < total && 16 * u < a.h[kind].D;
    };
    auto halves = [&](int kind, int& d0, int& d1) {   // where the unit's two halves lie; true: rope_dim/2 apart
        const bool split = turned && kind < 2 && !r.adjacent;
        d0 = split ? 8 * u : 16 * u, d1 = split ? (r.rope_dim >> 1) + 8 * u : 16 * u + 8;
        return split;
    };
    // All loads of a group of rows.  The first group's are on their way before the turns, which wait for the position, and
    // before the slot.
    uint4 v0[GROUP], v1[GROUP];
    auto load = [&](int base) {
#pragma unroll
        for (int k = 0; k < GROUP; ++k) {
            int h, kind, d0, d1;
            if (locate(base + k * rows + row0, h, kind)) {
                halves(kind, d0, d1);
                const Heads& x = a.h[kind];
                const uint16_t* p = x.src + t * x.src_tok + h * x.src_head;
                v0[k] = load8<VEC>(p + d0), v1[k] = load8<VEC>(p + d1);
            }
        }
    };
    const int64_t slot = a.slots ? a.slots[t] : -1;
    int base0 = part * rows * GROUP;
    load(base0);

    // this unit's eight turns, shared by all of the token's q and k heads
    float c[8], s[8];
    if (turned) {
        const int n = r.rope_dim >> 1;
        auto position = [&](int axis) {
            const int64_t at = axis * r.axis_stride + t;
            int64_t p = r.positions_i64 ? static_cast<const int64_t*>(r.positions)[at]
                                        : static_cast<const int32_t*>(r.positions)[at];
            if ((uint64_t)p >= (uint64_t)r.max_pos) {
                if (a.status) atomicOr(a.status, kDevBadIndex);
                p = p < 0 ? 0 : r.max_pos - 1;
            }
            return p;
        };
        const uint32_t axes = r.axis_map[u >> 1] >> (16 * (u & 1)) & 0xffffu;   // of the eight pairs, two bits each
        if (a.turns_vec && axes == (axes & 3) * 0x5555u) {   // one axis: the eight lie together
            const float* row = r.cos_sin + position(axes & 3) * r.rope_dim + 8 * u;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float4 x = reinterpret_cast<const float4*>(row)[i], y = reinterpret_cast<const float4*>(row + n)[i];
                c[4 * i] = x.x, c[4 * i + 1] = x.y, c[4 * i + 2] = x.z, c[4 * i + 3] = x.w;
                s[4 * i] = y.x, s[4 * i + 1] = y.y, s[4 * i + 2] = y.z, s[4 * i + 3] = y.w;
            }
        } else {
            uint32_t at[4];   // each axis's position
#pragma unroll
            for (int x = 0; x < 4; ++x) at[x] = x < r.n_axes ? (uint32_t)position(x) : 0;
            const float* const unit = r.cos_sin + 8 * u;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int x = axes >> (2 * i) & 3;
                const float* p = unit + (x & 2 ? (x & 1 ? at[3] : at[2]) : (x & 1 ? at[1] : at[0])) * (uint64_t)(uint32_t)r.rope_dim;
                c[i] = p[i], s[i] = p[n + i];
            }
        }
        if (r.inverse) {
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] = -s[i];
        }
    }
    int64_t page = -1, off = 0;
    if (slot >= 0) {
        if (slot < a.n_slots) {
            if (slot >> 32 == 0) page = (uint32_t)slot / (uint32_t)a.page_size;
            else page = slot / a.page_size;
            off = slot - page * a.page_size;
        } else if (a.status) {
            atomicOr(a.status, kDevBadIndex);
        }
    }
#pragma unroll 1
    while (base0 < total) {
#pragma unroll
        for (int k = 0; k < GROUP; ++k) {
            int h, kind, d0, d1;
            const bool on = locate(base0 + k * rows + row0, h, kind) && (kind == 0 || page >= 0), split = halves(kind, d0, d1), turn = turned && kind < 2;
            const Heads& x = a.h[kind];
            float lo[8], hi[8];   // dims d0 .. d0+7 and d1 .. d1+7
            if (on) {
                const uint32_t w0[4] = {v0[k].x, v0[k].y, v0[k].z, v0[k].w}, w1[4] = {v1[k].x, v1[k].y, v1[k].z, v1[k].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 f = unpack2<F16>(w0[i]), g = unpack2<F16>(w1[i]);
                    lo[2 * i] = f.x, lo[2 * i + 1] = f.y, hi[2 * i] = g.x, hi[2 * i + 1] = g.y;
                }
                auto pair = [](float& x1, float& x2, float cs, float sn) {
                    const float y1 = __fsub_rn(__fmul_rn(x1, cs), __fmul_rn(x2, sn));
                    x2 = __fadd_rn(__fmul_rn(x2, cs), __fmul_rn(x1, sn));
                    x1 = y1;
                };
                if (split) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) pair(lo[i], hi[i], c[i], s[i]);
                } else if (turn) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        pair(lo[2 * i], lo[2 * i + 1], c[i], s[i]);
                        pair(hi[2 * i], hi[2 * i + 1], c[4 + i], s[4 + i]);
                    }
                }
            }
            if (I8) {
                float most = 0.f;   // a NaN in the row makes its scale one, and so all that is read back of it
                if (on && kind) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) most = max_nan(most, max_nan(fabsf(lo[i]), fabsf(hi[i])));
                }
                for (int o = a.lanes >> 1; o > 0; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
                if (on && kind) {
                    most = max_nan(most, 1e-6f);
                    const float inv = __fdiv_rn(127.f, most);
                    auto codes = [&](const float* f) {
                        uint32_t w[2] = {0, 0};
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const int q = max(-128, min(127, __float2int_rn(__fmul_rn(f[i], inv))));
                            w[i >> 2] |= (uint32_t)(q & 0xff) << (8 * (i & 3));
                        }
                        return make_uint2(w[0], w[1]);
                    };
                    uint8_t* p = x.dst + page * x.dst_page + off * x.dst_tok + h * x.dst_head;
                    *reinterpret_cast<uint2*>(p + d0) = codes(lo);
                    *reinterpret_cast<uint2*>(p + d1) = codes(hi);
                    if (u == 0) x.scales[page * x.s_page + off * x.s_tok + h * x.s_head] = __fmul_rn(most, 1.0f / 127.0f);
                }
            }
            if (on && (!I8 || kind == 0)) {
                uint32_t w0[4], w1[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    w0[i] = pack2<F16>(lo[2 * i], lo[2 * i + 1]);
                    w1[i] = pack2<F16>(hi[2 * i], hi[2 * i + 1]);
                }
                const int64_t at = (kind ? page * x.dst_page + off * x.dst_tok : t * x.dst_tok) + h * x.dst_head;
                uint16_t* p = reinterpret_cast<uint16_t*>(x.dst) + at;
                store8<VEC>(p + d0, make_uint4(w0[0], w0[1], w0[2], w0[3]));
                store8<VEC>(p + d1, make_uint4(w1[0], w1[1], w1[2], w1[3]));
            }
        }
        base0 += a.parts * rows * GROUP;
        if (base0 < total) load(base0);
    }
}

}  // namespace

int paged_kv_check(const char* what, const ws_paged_kv* kv) {
    char buf[200];
    const char* why = nullptr;
    int code = WS_ERR_INVALID_ARG;
    const int eb = kv->dtype == WS_DTYPE_I8 ? 1 : 2;
    const int64_t st[6] = {kv->k_stride_page, kv->k_stride_tok, kv->k_stride_head,
                           kv->v_stride_page, kv->v_stride_tok, kv->v_stride_head};
    if (kv->dtype != WS_DTYPE_BF16 && kv->dtype != WS_DTYPE_F16 && kv->dtype != WS_DTYPE_I8)
        why = "the pool's dtype must be bf16, fp16 or int8";
    else if (kv->Hkv < 1 || kv->page_size < 1 || kv->n_pages < 0 || kv->Dk < 1 || kv->Dv < 1)
        why = "bad pool shape";
    else if (kv->Dk % 16 || kv->Dv % 16 || kv->Dk > 256 || kv->Dv > 256)
        why = "head dims must be multiples of 16, at most 256", code = WS_ERR_UNSUPPORTED;
    else if (kv->n_pages > 0 && (!kv->k || !kv->v || (kv->dtype == WS_DTYPE_I8 && (!kv->k_scales || !kv->v_scales))))
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
        if (kv->dtype != WS_DTYPE_I8 && kv->dtype != dtype)
            return set_error(WS_ERR_INVALID_ARG, "rope_append: the pool must hold the inputs' type or int8");
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
    // One warp walks all heads of a token when there are tokens for every SM; with fewer, its rows are shared out.  Into
    // int8, where a row takes longer, that pays with half as many tokens only (4097 tokens of 20 + 5 + 5 heads, us with 16,
    // 32, 64 and 128 warps wanted an SM: 14.5, 15.5, 17.2, 20.4).
    const bool f16 = dtype == WS_DTYPE_F16, i8 = kv && kv->dtype == WS_DTYPE_I8;
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
        constexpr bool F = decltype(half)::value, I = decltype(codes)::value;
        if (!vec) return rope_append_kernel<F, I, false, 1>;
        if constexpr (!I)
            if (several) return rope_append_kernel<F, I, true, kGroup>;
        return rope_append_kernel<F, I, true, 1>;
    };
    using yes = std::true_type;
    using no = std::false_type;
    auto fn = f16 ? (i8 ? pick(yes{}, yes{}) : pick(yes{}, no{})) : (i8 ? pick(no{}, yes{}) : pick(no{}, no{}));
    const cudaError_t e = launch_dependent(fn, dim3((unsigned)blocks), 32 * kWarps, 0, static_cast<cudaStream_t>(stream), a);
    return e == cudaSuccess ? WS_OK : set_error(WS_ERR_CUDA, cudaGetErrorString(e));
}
