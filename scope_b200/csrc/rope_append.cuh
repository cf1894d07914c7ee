// Rows of queries, keys and values turned by their positions: what the two appends share (rope_append.cu: rows as they
// are, or a scale a row; block_append.cu: a scale a block of tokens).
#pragma once

#include "common.cuh"
#include "ws_internal.h"

#include <cuda_fp16.h>

namespace ws {

struct Heads {          // one of q, k, v: rows of (token, head)
    const uint16_t* src;
    int64_t src_tok, src_head;
    uint8_t* dst;       // q: the output; k, v: the pool
    int64_t dst_tok;    // q: per token; k, v: per slot of a page  (elements)
    int64_t dst_head, dst_page;
    float* scales;      // 8-bit pools only; s_tok: per slot, or per block of them
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

// Unit u's eight turns at token t: cosines and sines of its pairs.
__device__ __forceinline__ void unit_turns(const ws_rope& r, bool vec, int64_t t, int u, int* status, float* c, float* s) {
    const int n = r.rope_dim >> 1;
    auto position = [&](int axis) {
        const int64_t at = axis * r.axis_stride + t;
        int64_t p = r.positions_i64 ? static_cast<const int64_t*>(r.positions)[at]
                                    : static_cast<const int32_t*>(r.positions)[at];
        if ((uint64_t)p >= (uint64_t)r.max_pos) {
            if (status) atomicOr(status, kDevBadIndex);
            p = p < 0 ? 0 : r.max_pos - 1;
        }
        return p;
    };
    const uint32_t axes = r.axis_map[u >> 1] >> (16 * (u & 1)) & 0xffffu;   // of the eight pairs, two bits each
    if (vec && axes == (axes & 3) * 0x5555u) {   // one axis: the eight lie together
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

// One pair turned, each product and sum rounded by itself.
__device__ __forceinline__ void turn_pair(float& x1, float& x2, float c, float s) {
    const float y1 = __fsub_rn(__fmul_rn(x1, c), __fmul_rn(x2, s));
    x2 = __fadd_rn(__fmul_rn(x2, c), __fmul_rn(x1, s));
    x1 = y1;
}

// The scale that rows up to `most` ask for; NaN and infinity stay.
template <bool E4M3>
__device__ __forceinline__ float own_scale(float most) {
    most = max_nan(most, 1e-6f);
    if (!E4M3) return __fmul_rn(most, 1.0f / 127.0f);
    const uint32_t bits = __float_as_uint(most);
    if (!(most < INFINITY)) return most;
    // most = 1.m 2^e, 448 = 1.75 2^8
    return __uint_as_float(((bits >> 23) - 8 + ((bits & 0x7fffff) > 0x600000)) << 23);
}

// Four values times inv as codes.
template <bool E4M3>
__device__ __forceinline__ uint32_t codes4(float2 x, float2 y, float inv) {
    x = make_float2(__fmul_rn(x.x, inv), __fmul_rn(x.y, inv)), y = make_float2(__fmul_rn(y.x, inv), __fmul_rn(y.y, inv));
    uint32_t w;
    if (E4M3) {
        asm("{.reg .b16 l, h; cvt.rn.satfinite.e4m3x2.f32 l, %2, %1; cvt.rn.satfinite.e4m3x2.f32 h, %4, %3; mov.b32 %0, {l, h};}"
            : "=r"(w) : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y));
    } else {   // within 127 by clamping first: rounding keeps the order
        auto code = [](float f) { return (uint32_t)__float2int_rn(fminf(fmaxf(f, -127.f), 127.f)); };
        w = __byte_perm(__byte_perm(code(x.x), code(x.y), 0x0040), __byte_perm(code(y.x), code(y.y), 0x0040), 0x5410);
    }
    return w;
}
enum : int { kRows16 = 0, kRowsS8 = 1, kRowsE4M3 = 2 };   // how rows are held: as they are, or as codes with a scale a row

// A warp's rows: item = token * parts + part.  F16: fp16 inputs (else bf16); CODE: what the pool holds; VEC: q, k, v and
// q_out are 16-byte aligned throughout.
template <bool F16, int CODE, bool VEC, int GROUP>
__device__ __forceinline__ void rope_rows(const RopeAppendArgs& a, int64_t item) {
    constexpr bool I8 = CODE != kRows16;
    const int lane = threadIdx.x & 31;
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
    if (turned) unit_turns(r, a.turns_vec, t, u, a.status, c, s);
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
                if (split) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) turn_pair(lo[i], hi[i], c[i], s[i]);
                } else if (turn) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        turn_pair(lo[2 * i], lo[2 * i + 1], c[i], s[i]);
                        turn_pair(hi[2 * i], hi[2 * i + 1], c[4 + i], s[4 + i]);
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
                    const float scale = CODE == kRowsE4M3 ? own_scale<true>(most) : __fmul_rn(most, 1.0f / 127.0f);
                    const float inv = CODE == kRowsE4M3 ? (scale < INFINITY ? __fdiv_rn(1.f, scale) : 0.f) : __fdiv_rn(127.f, most);
                    auto codes = [&](const float* f) {
                        if (CODE == kRowsE4M3) {   // 0 where the scale is not finite
                            if (!(inv > 0.f)) return make_uint2(0, 0);
                            return make_uint2(codes4<true>(make_float2(f[0], f[1]), make_float2(f[2], f[3]), inv),
                                              codes4<true>(make_float2(f[4], f[5]), make_float2(f[6], f[7]), inv));
                        }
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
                    if (u == 0) x.scales[page * x.s_page + off * x.s_tok + h * x.s_head] = scale;
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

// The append into blocks of `block` tokens that share a scale (block_append.cu).  The queries go with it where the call is
// small, else by themselves, ahead of it and after its check.
bool block_append_small(int64_t N, int Hkv);
int block_append_check(const RopeAppendArgs& args, int block);
int block_append_launch(const RopeAppendArgs& args, bool f16, bool e4m3, bool vec, int block, cudaStream_t st);

}  // namespace ws
