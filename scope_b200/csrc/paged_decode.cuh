// Decode attention over a paged key-value cache: the kernel (see paged_decode.cu for the entry).
//
//   o = sum_t softmax_t(scale q.k_t) v_t,  lse = log sum_t exp(scale q.k_t),  t in [max(0, L - window), L)
//
// What bounds it: HBM.  Every key and value row is read once (the query heads that share it are one tensor-core
// tile), against G multiply-adds a byte, so the whole design is about keeping enough bytes in flight on every SM
// for any mix of lengths:
//
//   * Rows (request, kv head, block of 8*NT query heads) are cut into subtiles of 16 tokens, laid end to end, and the
//     line is split evenly over the CTAs (one a SM) and again over each CTA's warps.  Every warp runs alone over its
//     stretch with its own ring of S stages filled by 16-byte cp.async, so no warp ever waits for another and a short
//     row costs no barrier.  The lengths are read on the device; the host never needs them.
//   * A subtile is one stage.  Pages need not divide it: each lane looks up one token's page (an entry fetched one
//     subtile ahead) and the row addresses travel by shuffle.  Tokens past the length, before the window or on a page
//     that is none are not read: their shared-memory rows are zero and their scores -inf.
//   * Rows in shared memory are an odd number of 16-byte pieces apart, so ldmatrix reads are free of bank conflicts for
//     every head dim without a swizzle.
//   * S^T[16 tok x 8 heads] = K . Q^T and O^T[Dv x 8] += V^T . P^T by mma.sync with the heads as the narrow dimension:
//     at G <= 8 query heads a key there is no 128-row tile for tcgen05 to fill, and the tensor pipe is nearly idle.
//     Running maxima and sums are fp32; P enters the second product as the sum of two 16-bit values (the rounded one
//     and the rest), which keeps its error below the output's own rounding.
//   * int8 rows go from shared memory to bf16 (fp16) fragments by bit operations, exactly; the row's scale multiplies
//     the score, or the probability.
//   * A row that ends inside one warp's stretch is written at once.  The others leave a state (o, m, l) per warp,
//     which the CTA joins in shared memory; what crosses CTAs goes through the workspace and is joined by the CTA that
//     files the last part (a ticket), always in the same order, so results do not depend on timing.
#pragma once

#include "common.cuh"
#include "ws_internal.h"

#include <cuda_fp16.h>

namespace ws {
namespace paged {

constexpr int kTok = 16;   // tokens of a subtile

struct Args {
    const uint16_t* q;
    int64_t q_b, q_h;                    // elements
    const uint8_t* k;
    const uint8_t* v;
    int64_t kp, kt, kh, vp, vt, vh;      // bytes
    const float* ks;
    const float* vs;
    int64_t ksp, kst, ksh, vsp, vst, vsh;
    const int32_t* table;
    int64_t table_stride;
    const int32_t* seq_lens;
    int64_t cap;                         // max_pages * page_size
    int n_pages, page_size;
    uint32_t div_mul, div_shift;         // t / page_size = (umulhi(t, div_mul) + t) >> div_shift
    int B, Hkv, G, hb, Dk, Dv, window;   // hb: head blocks of a kv head
    float scale_log2;
    uint16_t* out;
    float* lse;
    int* counters;
    float* pieces;                       // [cta][2 + warps][piece floats]
    int* status;
};

// The variant for head dims up to DB, 8*NT query heads a block.
template <bool F16, bool I8, int DB, int NT>
struct Cfg {
    static constexpr int kWarps = DB <= 128 ? 8 : 4;
    static constexpr int kRow = I8 ? ((DB / 16) | 1) * 16 : DB * 2 + 16;
    static constexpr int kStage = 2 * kTok * kRow + (I8 ? 128 : 0) + 32;
    static constexpr int kFit = (220 << 10) / (kWarps * kStage);
    static constexpr int kStages = kFit > 6 ? 6 : kFit;
    static constexpr int kUnits = NT * (DB / 16);   // 16 x 8 fragments of an accumulator
    static_assert(kStages >= 3, "ring");
};
__host__ __device__ inline int row_bytes(bool i8, int D) { return i8 ? ((D / 16) | 1) * 16 : D * 2 + 16; }
// shared memory of one warp: its ring, or its last part when that is larger
__host__ __device__ inline size_t warp_bytes(bool i8, int stages, int NT, int Dk, int Dv) {
    const size_t ring = stages * ((size_t)kTok * (row_bytes(i8, Dk) + row_bytes(i8, Dv)) + (i8 ? 128 : 0) + 32);
    const size_t part = ((size_t)NT * 8 * Dv + 16 * NT) * 4;
    return ring > part ? ring : part;
}
// floats of one row part: the accumulator's fragments, then m and l of its 8*NT heads
__host__ __device__ inline int piece_floats(int NT, int Dv) { return NT * 8 * Dv + 16 * NT; }

// What the filler of a stage leaves for its reader.
struct __align__(16) Meta {
    uint32_t mask;      // bit i: token i counts; bit 16: the row starts here; bit 17: the row ends here
    int b, hr, n;       // request, kv head * hb + head block, the row's subtiles
    long long start;    // the row's first place on the line
    long long pad;
};
static_assert(sizeof(Meta) == 32, "meta");

// A row part, as the CTA's last step sees it.
struct Part {
    long long start;   // < 0: none
    int b, hr, n;
};

__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(valid ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void mma_f16_16816(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                              uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
        "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <bool F16>
__device__ __forceinline__ void mma16(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
    if (F16) mma_f16_16816(d, a0, a1, a2, a3, b0, b1);
    else mma_bf16_16816(d, a0, a1, a2, a3, b0, b1);
}
template <bool F16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
    if (F16) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    return pack_bf16(lo, hi);
}
template <bool F16>
__device__ __forceinline__ float2 unpack16(uint32_t v) {
    if (F16) return __half22float2(*reinterpret_cast<const __half2*>(&v));
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}

// Bytes 0 and 2 of r, signed, as a pair of 16-bit floats (exact).  bf16: 0x4300 is 128 and holds 7 bits below it, so
// (128 + low 7 bits) - (128 or, with the sign bit set, 256) is the value.  fp16: 0x6400 is 1024 and holds all 8 bits:
// 1024 + (value + 128) - 1152.
template <bool F16>
__device__ __forceinline__ uint32_t s8_pair(uint32_t r) {
    uint32_t d;
    if (F16) {
        const uint32_t x = (r & 0x00ff00ffu) ^ 0x64806480u;
        asm("sub.f16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(0x64806480u));
    } else {
        const uint32_t x = (r & 0x007f007fu) | 0x43004300u, y = (r & 0x00800080u) | 0x43004300u;
        asm("sub.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(y));
    }
    return d;
}

// Where request b's attended tokens lie: subtiles [first/16, first/16 + n), tokens [lo, L).
struct Span {
    int lo, L, n;
};
__device__ __forceinline__ Span span_of(const Args& a, int b) {
    Span s;
    s.L = (int)min((long long)max(__ldg(a.seq_lens + b), 0), (long long)a.cap);
    s.lo = a.window > 0 ? max(s.L - a.window, 0) : 0;
    s.n = s.L > 0 ? (s.L - (s.lo & ~(kTok - 1)) + kTok - 1) / kTok : 0;
    return s;
}

// The running joint state of row parts for one lane's fragment unit (two heads, two dims each).
struct Join {
    float m[2], l[2], o[4];
    __device__ __forceinline__ void reset() {
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
        o[0] = o[1] = o[2] = o[3] = 0.f;
    }
    __device__ __forceinline__ void add(const float2& pm, const float2& pl, const float4& po) {
        const float nm[2] = {pm.x, pm.y}, nl[2] = {pl.x, pl.y}, no[4] = {po.x, po.y, po.z, po.w};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float top = fmaxf(m[j], nm[j]), ref = top == -INFINITY ? 0.f : top;
            const float x = ex2(m[j] - ref), y = ex2(nm[j] - ref);
            l[j] = l[j] * x + nl[j] * y;
            o[j] = o[j] * x + no[j] * y;
            o[j + 2] = o[j + 2] * x + no[j + 2] * y;
            m[j] = top;
        }
    }
};

// Write one fragment unit of a finished row: O^T[dims x heads] of m-tile mt, heads nt*8 + 2t, +1 of the block.
// 16-bit pools: this lane's o[0..1] are dim 16mt + g, o[2..3] dim 16mt + g + 8; int8 pools: dims 16mt + 2g and + 1.
template <bool F16, bool I8>
__device__ __forceinline__ void store_unit(const Args& a, int b, int hr, int heads0, int nt, int mt, const float* o,
                                           const float* inv) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int kvh = hr / a.hb, left = a.G - heads0;
    uint16_t* base = a.out + ((int64_t)b * a.Hkv * a.G + (int64_t)kvh * a.G + heads0) * a.Dv + 16 * mt;
    if (I8) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int h = nt * 8 + 2 * t + j;
            if (h < left)
                *reinterpret_cast<uint32_t*>(base + (int64_t)h * a.Dv + 2 * g) = pack16<F16>(o[j] * inv[j], o[j + 2] * inv[j]);
        }
    } else {
        // transposed: lane (g, t) gets head g, dims 2t, 2t+1 (and +8)
        const uint32_t lo = movmatrix_t(pack16<F16>(o[0] * inv[0], o[1] * inv[1]));
        const uint32_t hi = movmatrix_t(pack16<F16>(o[2] * inv[0], o[3] * inv[1]));
        const int h = nt * 8 + g;
        if (h < left) {
            *reinterpret_cast<uint32_t*>(base + (int64_t)h * a.Dv + 2 * t) = lo;
            *reinterpret_cast<uint32_t*>(base + (int64_t)h * a.Dv + 8 + 2 * t) = hi;
        }
    }
}
// m, l of the lane's two heads -> 1/l; lanes with g == 0 write the lse when asked.
__device__ __forceinline__ void finish(const Args& a, int b, int hr, int heads0, int nt, const float* m, const float* l,
                                       bool write_lse, float* inv) {
    const int lane = threadIdx.x & 31, t = lane & 3;
    const int kvh = hr / a.hb;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        inv[j] = l[j] > 0.f ? 1.f / l[j] : 0.f;
        const int h = nt * 8 + 2 * t + j;
        if (write_lse && a.lse && lane < 4 && heads0 + h < a.G)
            a.lse[(int64_t)b * a.Hkv * a.G + (int64_t)kvh * a.G + heads0 + h] =
                l[j] > 0.f ? m[j] * kLn2 + logf(l[j]) : -INFINITY;
    }
}

template <bool F16, bool I8, int DB, int NT>
__global__ void __launch_bounds__(32 * Cfg<F16, I8, DB, NT>::kWarps, 1) decode_kernel(const __grid_constant__ Args a) {
    using C = Cfg<F16, I8, DB, NT>;
    constexpr int kWarps = C::kWarps, S = C::kStages, kKs = DB / 16, kMt = DB / 16;
    constexpr bool kPF16 = F16 && !I8;   // the type of P and V in the second product (bf16's range for scaled P)
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ long long s_scan[kWarps], s_off[kWarps];
    __shared__ int s_b[kWarps], s_last[2];
    __shared__ Part s_part[2 * kWarps];

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t4 = lane & 3;
    const int R = a.Hkv * a.hb;          // rows of a request

    // ---- the line: total length, this CTA's stretch, and where each warp's begins
    long long N;
    const int per = (a.B + kWarps * 32 - 1) / (kWarps * 32), first_b = tid * per;
    long long mine = 0;
    for (int b = first_b; b < min(first_b + per, a.B); ++b) mine += span_of(a, b).n;
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
    }
    if (lane == 31) s_scan[warp] = upto;
    if (tid < 2 * kWarps) s_part[tid].start = -1;
    __syncthreads();
    long long before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += s_scan[w];
        total += s_scan[w];
    }
    N = total * R;
    const int nC = (int)min((long long)gridDim.x, N);
    const bool works = (int)blockIdx.x < nC;
    const long long x0 = works ? split_start(blockIdx.x, N, nC) : 0, x1 = works ? split_start(blockIdx.x + 1, N, nC) : 0;
    auto warp_start = [&](int w) { return x0 + (x1 - x0) * w / kWarps; };
    {
        long long off = (before + upto - mine) * R;
        for (int b = first_b; b < min(first_b + per, a.B); ++b) {
            const long long len = (long long)span_of(a, b).n * R;
            if (len > 0 && off < x1 && off + len > x0) {
                for (int w = 0; w < kWarps; ++w) {
                    const long long y = warp_start(w);
                    if (y >= off && y < off + len) s_b[w] = b, s_off[w] = off;
                }
            }
            off += len;
        }
    }
    __syncthreads();
    // requests without a token, dealt over the CTAs: zeros, -inf
    for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
        if (span_of(a, b).n) continue;
        const int64_t row = (int64_t)b * a.Hkv * a.G;
        for (int i = tid; i < a.Hkv * a.G * (a.Dv / 8); i += 32 * kWarps)
            reinterpret_cast<uint4*>(a.out + row * a.Dv)[i] = make_uint4(0, 0, 0, 0);
        for (int i = tid; a.lse && i < a.Hkv * a.G; i += 32 * kWarps) a.lse[row + i] = -INFINITY;
    }
    if (!works) return;

    // ---- this warp's stretch
    const long long w0 = warp_start(warp);
    const int count = (int)(warp_start(warp + 1) - w0);
    const int krow = row_bytes(I8, a.Dk), vrow = row_bytes(I8, a.Dv);
    const uint32_t stage_sz = kTok * (krow + vrow) + (I8 ? 128 : 0) + 32;
    const size_t warp_sz = warp_bytes(I8, S, NT, a.Dk, a.Dv);
    uint8_t* const ring = smem + warp * warp_sz;
    const uint32_t ring_u = smem_u32(ring);
    const uint32_t v_at = kTok * krow, s_at = v_at + kTok * vrow, m_at = s_at + (I8 ? 128 : 0);
    const int pf = piece_floats(NT, a.Dv);
    float* const cta_pieces = a.pieces + (int64_t)blockIdx.x * (2 + kWarps) * pf;

    // filler state: the row being filled and the next subtile's page entry
    int fb = 0, fhr = 0, fsub = 0;
    long long fstart = 0;
    Span fs = {0, 0, 0};
    int f_entry = 0, f_off = 0;   // this lane's token: page entry and place in the page
    bool f_ok = false;
    int left = count;
    const int tok = lane & 15;

    auto look_up = [&]() {   // the page of this lane's token of subtile fsub
        const uint32_t t = (uint32_t)(fs.lo & ~(kTok - 1)) + (uint32_t)fsub * kTok + tok;
        f_ok = (int)t >= fs.lo && (int)t < fs.L;
        const uint32_t page = (__umulhi(t, a.div_mul) + t) >> a.div_shift;
        f_off = (int)(t - page * (uint32_t)a.page_size);
        f_entry = f_ok ? __ldg(a.table + (int64_t)fb * a.table_stride + page) : 0;
    };
    if (count > 0) {
        fb = s_b[warp];
        fs = span_of(a, fb);
        const long long rel = w0 - s_off[warp];
        fhr = (int)(rel / fs.n);
        fsub = (int)(rel - (long long)fhr * fs.n);
        fstart = w0 - fsub;
        look_up();
    }
    const int l8 = lane & 7, r4 = lane >> 3;
    const int kchunks = I8 ? a.Dk >> 4 : a.Dk >> 3, vchunks = I8 ? a.Dv >> 4 : a.Dv >> 3;
    constexpr int kCols = (I8 ? DB / 16 : DB / 8) / 8 > 0 ? (I8 ? DB / 16 : DB / 8) / 8 : 1;

    auto fill = [&](int slot) {
        if (left > 0) {
            --left;
            const uint32_t st = ring_u + slot * stage_sz;
            bool ok = f_ok;
            if (ok && (uint32_t)f_entry >= (uint32_t)a.n_pages) {
                ok = false;
                if (a.status) atomicMax(a.status, kDevBadIndex);
            }
            const int kvh = fhr / a.hb;
            const long long page = ok ? f_entry : 0, off = ok ? f_off : 0;
            const long long ka = page * a.kp + off * a.kt + kvh * a.kh, va = page * a.vp + off * a.vt + kvh * a.vh;
            const uint32_t mask = __ballot_sync(0xffffffffu, ok) & 0xffffu;
            if (I8) {
                const float* src = lane < 16 ? a.ks + (page * a.ksp + off * a.kst + kvh * a.ksh)
                                             : a.vs + (page * a.vsp + off * a.vst + kvh * a.vsh);
                cp_async4(st + s_at + lane * 4, src, ok);
            }
            if (lane == 0) {
                Meta m;
                m.mask = mask | (fsub == 0 ? 1u << 16 : 0u) | (fsub == fs.n - 1 ? 1u << 17 : 0u);
                m.b = fb, m.hr = fhr, m.n = fs.n, m.start = fstart, m.pad = 0;
                *reinterpret_cast<Meta*>(ring + slot * stage_sz + m_at) = m;
            }
            // 8 lanes a row, 4 rows at a time
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = 4 * i + r4;
                const long long kr = __shfl_sync(0xffffffffu, ka, row), vr = __shfl_sync(0xffffffffu, va, row);
                const bool on = (mask >> row) & 1;
                const uint8_t* kp = a.k + kr + l8 * 16;
                const uint8_t* vp = a.v + vr + l8 * 16;
                const uint32_t kd = st + row * krow + l8 * 16, vd = st + v_at + row * vrow + l8 * 16;
#pragma unroll
                for (int j = 0; j < kCols; ++j) {
                    if (l8 + 8 * j < kchunks) cp_async16(kd + j * 128, kp + j * 128, on);
                    if (l8 + 8 * j < vchunks) cp_async16(vd + j * 128, vp + j * 128, on);
                }
            }
            // the next subtile
            if (++fsub == fs.n) {
                fsub = 0;
                fstart += fs.n;
                if (++fhr == R && left > 0) {
                    fhr = 0;
                    do fs = span_of(a, ++fb);
                    while (fs.n == 0);
                }
            }
            if (left > 0) look_up();
        }
        cp_async_commit();
    };

    // ---- reader state
    float m_run[NT][2], l_run[NT][2], acc[NT][kMt][4];
    uint32_t bq[NT][kKs][2];
    bool began = false;
    const int nks = a.Dk >> 4, nmt = a.Dv >> 4;

    auto load_q = [&](int b, int hr) {
        const int kvh = hr / a.hb, h0 = (hr - kvh * a.hb) * 8 * NT;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int h = h0 + nt * 8 + g;
            const uint16_t* q = a.q + b * a.q_b + ((int64_t)kvh * a.G + h) * a.q_h;
#pragma unroll
            for (int ks = 0; ks < kKs; ++ks) {
                uint32_t x = 0, y = 0;
                if (ks < nks && h < a.G) {
                    if (I8) {   // the order in which s8_pair gives the dims: (0, 2), (1, 3) of each four
                        const uint2 w = __ldg(reinterpret_cast<const uint2*>(q + 16 * ks + 4 * t4));
                        x = __byte_perm(w.x, w.y, 0x5410);
                        y = __byte_perm(w.x, w.y, 0x7632);
                    } else {
                        x = __ldg(reinterpret_cast<const uint32_t*>(q + 16 * ks + 2 * t4));
                        y = __ldg(reinterpret_cast<const uint32_t*>(q + 16 * ks + 2 * t4 + 8));
                    }
                }
                bq[nt][ks][0] = x, bq[nt][ks][1] = y;
            }
            m_run[nt][0] = m_run[nt][1] = -INFINITY;
            l_run[nt][0] = l_run[nt][1] = 0.f;
#pragma unroll
            for (int mt = 0; mt < kMt; ++mt) acc[nt][mt][0] = acc[nt][mt][1] = acc[nt][mt][2] = acc[nt][mt][3] = 0.f;
        }
    };

    // this lane's part of the row into piece memory (shared or global)
    auto file_piece = [&](float* p) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int mt = 0; mt < kMt; ++mt)
                if (mt < nmt)
                    *reinterpret_cast<float4*>(p + ((nt * nmt + mt) * 32 + lane) * 4) =
                        make_float4(acc[nt][mt][0], acc[nt][mt][1], acc[nt][mt][2], acc[nt][mt][3]);
            if (lane < 4) {
                float* ml = p + NT * 8 * a.Dv + nt * 16;
                *reinterpret_cast<float2*>(ml + 2 * t4) = make_float2(m_run[nt][0], m_run[nt][1]);
                *reinterpret_cast<float2*>(ml + 8 + 2 * t4) = make_float2(l_run[nt][0], l_run[nt][1]);
            }
        }
    };

#pragma unroll
    for (int s = 0; s < S - 1; ++s) fill(s);
    int slot = 0;
    for (int it = 0; it < count; ++it) {
        cp_async_wait<S - 2>();
        __syncwarp();
        fill(slot == 0 ? S - 1 : slot - 1);
        const uint32_t st = ring_u + slot * stage_sz;
        const Meta* meta = reinterpret_cast<const Meta*>(ring + slot * stage_sz + m_at);
        const uint32_t mask = meta->mask;
        if (it == 0 || (mask & (1u << 16))) {
            load_q(meta->b, meta->hr);
            began = mask & (1u << 16);
        }
        // scores
        float c[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) c[nt][0] = c[nt][1] = c[nt][2] = c[nt][3] = 0.f;
        const uint32_t k_ld = st + (lane & 15) * krow + (lane >> 4) * 16;
        if (I8) {
#pragma unroll
            for (int ks = 0; ks < kKs; ks += 2) {
                if (ks < nks) {
                    uint32_t r[4];
                    ldsm_x4(k_ld + ks * 16, r[0], r[1], r[2], r[3]);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        if (u == 0 || ks + 1 < nks) {
                            const uint32_t a0 = s8_pair<F16>(r[2 * u]), a1 = s8_pair<F16>(r[2 * u + 1]);
                            const uint32_t a2 = s8_pair<F16>(r[2 * u] >> 8), a3 = s8_pair<F16>(r[2 * u + 1] >> 8);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
                                mma16<F16>(c[nt], a0, a1, a2, a3, bq[nt][ks + u][0], bq[nt][ks + u][1]);
                        }
                    }
                }
            }
        } else {
#pragma unroll
            for (int ks = 0; ks < kKs; ++ks) {
                if (ks < nks) {
                    uint32_t a0, a1, a2, a3;
                    ldsm_x4(k_ld + ks * 32, a0, a1, a2, a3);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma16<F16>(c[nt], a0, a1, a2, a3, bq[nt][ks][0], bq[nt][ks][1]);
                }
            }
        }
        float f0 = a.scale_log2, f1 = a.scale_log2, v0 = 1.f, v1 = 1.f;
        if (I8) {
            const float* sc = reinterpret_cast<const float*>(ring + slot * stage_sz + s_at);
            f0 *= sc[g], f1 *= sc[g + 8], v0 = sc[16 + g], v1 = sc[24 + g];
        }
        const bool on0 = (mask >> g) & 1, on1 = (mask >> (g + 8)) & 1;
        uint32_t ph[NT][2], pl[NT][2];
        bool moved = false;
        float keep[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                c[nt][j] = on0 ? c[nt][j] * f0 : -INFINITY;
                c[nt][j + 2] = on1 ? c[nt][j + 2] * f1 : -INFINITY;
                float top = fmaxf(c[nt][j], c[nt][j + 2]);
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                const float m2 = fmaxf(m_run[nt][j], top), ref = m2 == -INFINITY ? 0.f : m2;
                moved |= m2 > m_run[nt][j];
                keep[nt][j] = ex2(m_run[nt][j] - ref);
                m_run[nt][j] = m2;
                const float p0 = ex2(c[nt][j] - ref), p1 = ex2(c[nt][j + 2] - ref);
                l_run[nt][j] = l_run[nt][j] * keep[nt][j] + (p0 + p1);
                c[nt][j] = I8 ? p0 * v0 : p0;
                c[nt][j + 2] = I8 ? p1 * v1 : p1;
            }
            const uint32_t h0 = pack16<kPF16>(c[nt][0], c[nt][1]), h1 = pack16<kPF16>(c[nt][2], c[nt][3]);
            const float2 e0 = unpack16<kPF16>(h0), e1 = unpack16<kPF16>(h1);
            ph[nt][0] = movmatrix_t(h0), ph[nt][1] = movmatrix_t(h1);
            pl[nt][0] = movmatrix_t(pack16<kPF16>(c[nt][0] - e0.x, c[nt][1] - e0.y));
            pl[nt][1] = movmatrix_t(pack16<kPF16>(c[nt][2] - e1.x, c[nt][3] - e1.y));
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int mt = 0; mt < kMt; ++mt) {
                    acc[nt][mt][0] *= keep[nt][0], acc[nt][mt][1] *= keep[nt][1];
                    acc[nt][mt][2] *= keep[nt][0], acc[nt][mt][3] *= keep[nt][1];
                }
        }
        // values
        if (I8) {
            const uint32_t v_ld = st + v_at + (lane & 15) * vrow + (lane >> 4) * 16;
#pragma unroll
            for (int mt = 0; mt < kMt; mt += 2) {
                if (mt < nmt) {
                    uint32_t r[4];
                    ldsm_x4_t(v_ld + mt * 16, r[0], r[1], r[2], r[3]);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        if (u == 0 || mt + 1 < nmt) {
                            const uint32_t a0 = s8_pair<kPF16>(r[2 * u]), a1 = s8_pair<kPF16>(r[2 * u] >> 8);
                            const uint32_t a2 = s8_pair<kPF16>(r[2 * u + 1]), a3 = s8_pair<kPF16>(r[2 * u + 1] >> 8);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                mma16<kPF16>(acc[nt][mt + u], a0, a1, a2, a3, ph[nt][0], ph[nt][1]);
                                mma16<kPF16>(acc[nt][mt + u], a0, a1, a2, a3, pl[nt][0], pl[nt][1]);
                            }
                        }
                    }
                }
            }
        } else {
            const uint32_t v_ld = st + v_at + ((lane & 7) + ((lane >> 4) << 3)) * vrow + ((lane >> 3) & 1) * 16;
#pragma unroll
            for (int mt = 0; mt < kMt; ++mt) {
                if (mt < nmt) {
                    uint32_t a0, a1, a2, a3;
                    ldsm_x4_t(v_ld + mt * 32, a0, a1, a2, a3);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma16<kPF16>(acc[nt][mt], a0, a1, a2, a3, ph[nt][0], ph[nt][1]);
                        mma16<kPF16>(acc[nt][mt], a0, a1, a2, a3, pl[nt][0], pl[nt][1]);
                    }
                }
            }
        }
        // the row, or this warp's stretch, ends
        const bool ends = mask & (1u << 17), last = it == count - 1;
        if (ends || last) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    l_run[nt][j] += __shfl_xor_sync(0xffffffffu, l_run[nt][j], 4);
                    l_run[nt][j] += __shfl_xor_sync(0xffffffffu, l_run[nt][j], 8);
                    l_run[nt][j] += __shfl_xor_sync(0xffffffffu, l_run[nt][j], 16);
                }
            const Meta mm = *meta;
            const int kvh = mm.hr / a.hb, h0 = (mm.hr - kvh * a.hb) * 8 * NT;
            if (ends && began) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float inv[2];
                    finish(a, mm.b, mm.hr, h0, nt, m_run[nt], l_run[nt], true, inv);
#pragma unroll
                    for (int mt = 0; mt < kMt; ++mt)
                        if (mt < nmt) store_unit<F16, I8>(a, mm.b, mm.hr, h0, nt, mt, acc[nt][mt], inv);
                }
            } else {
                // the stretch's last part stays in this warp's own ring (nothing is in flight into it any more), an
                // earlier one goes through L2
                __syncwarp();
                file_piece(last ? reinterpret_cast<float*>(ring) : cta_pieces + (2 + warp) * pf);
                if (lane == 0) {
                    Part p;
                    p.start = mm.start, p.b = mm.b, p.hr = mm.hr, p.n = mm.n;
                    s_part[2 * warp + (last ? 1 : 0)] = p;
                }
            }
        }
        slot = slot == S - 1 ? 0 : slot + 1;
    }
    __syncthreads();

    // ---- join the CTA's parts row by row; a row that leaves the CTA is filed for the last of its CTAs
    const int units = NT * nmt;
    auto part_at = [&](int i) -> const float* {
        return (i & 1) ? reinterpret_cast<const float*>(smem + (i >> 1) * warp_sz)
                       : cta_pieces + (2 + (i >> 1)) * pf;
    };
    Part cross[2];
    cross[0].start = cross[1].start = -1;
    int i0 = 0;
    while (i0 < 2 * kWarps) {
        const Part p = s_part[i0];
        if (p.start < 0) {
            ++i0;
            continue;
        }
        int i1 = i0 + 1;
        while (i1 < 2 * kWarps && (s_part[i1].start < 0 || s_part[i1].start == p.start)) ++i1;
        const bool inside = p.start >= x0 && p.start + p.n <= x1;
        const int which = p.start >= x0 ? 1 : 0;
        const int kvh = p.hr / a.hb, h0 = (p.hr - kvh * a.hb) * 8 * NT;
        float* const to = cta_pieces + which * pf;
        for (int u = warp; u < units; u += kWarps) {
            const int nt = u / nmt, mt = u - nt * nmt;
            Join z;
            z.reset();
            for (int i = i0; i < i1; ++i) {
                if (s_part[i].start < 0) continue;
                const float* src = part_at(i);
                const float* ml = src + NT * 8 * a.Dv + nt * 16;
                z.add(*reinterpret_cast<const float2*>(ml + 2 * t4), *reinterpret_cast<const float2*>(ml + 8 + 2 * t4),
                      *reinterpret_cast<const float4*>(src + (u * 32 + lane) * 4));
            }
            if (inside) {
                float inv[2];
                finish(a, p.b, p.hr, h0, nt, z.m, z.l, mt == 0, inv);
                store_unit<F16, I8>(a, p.b, p.hr, h0, nt, mt, z.o, inv);
            } else {
                *reinterpret_cast<float4*>(to + (u * 32 + lane) * 4) = make_float4(z.o[0], z.o[1], z.o[2], z.o[3]);
                if (mt == 0 && lane < 4) {
                    float* ml = to + NT * 8 * a.Dv + nt * 16;
                    *reinterpret_cast<float2*>(ml + 2 * t4) = make_float2(z.m[0], z.m[1]);
                    *reinterpret_cast<float2*>(ml + 8 + 2 * t4) = make_float2(z.l[0], z.l[1]);
                }
            }
        }
        if (!inside) cross[which] = p;
        i0 = i1;
    }
    if (cross[0].start < 0 && cross[1].start < 0) return;   // the same in every thread
    __threadfence();
    __syncthreads();
    if (tid < 2) {
        const Part p = tid ? cross[1] : cross[0];
        int last = 0;
        if (p.start >= 0) {
            // the row's first CTA keeps its counter: a CTA is the first of one crossing row at most
            const int c0 = (int)split_owner(p.start, N, nC), c1 = (int)split_owner(p.start + p.n - 1, N, nC);
            last = atomicAdd(a.counters + c0, 1) == c1 - c0;
            if (last) a.counters[c0] = 0;
        }
        s_last[tid] = last;
        __threadfence();
    }
    __syncthreads();
    for (int e = 0; e < 2; ++e) {
        if (!s_last[e]) continue;
        const Part p = e ? cross[1] : cross[0];
        const int c0 = (int)split_owner(p.start, N, nC), c1 = (int)split_owner(p.start + p.n - 1, N, nC);
        const int kvh = p.hr / a.hb, h0 = (p.hr - kvh * a.hb) * 8 * NT;
        for (int u = warp; u < units; u += kWarps) {
            const int nt = u / nmt, mt = u - nt * nmt;
            Join z;
            z.reset();
            constexpr int kDeep = 8;
            for (int c = c0; c <= c1; c += kDeep) {
                float2 pm[kDeep], pl[kDeep];
                float4 po[kDeep];
#pragma unroll
                for (int i = 0; i < kDeep; ++i) {
                    if (c + i <= c1) {
                        // the first CTA filed the row's start as its slot 1, the others as their slot 0
                        const float* src = a.pieces + ((int64_t)(c + i) * (2 + kWarps) + (c + i == c0 ? 1 : 0)) * pf;
                        const float* ml = src + NT * 8 * a.Dv + nt * 16;
                        pm[i] = __ldcg(reinterpret_cast<const float2*>(ml + 2 * t4));
                        pl[i] = __ldcg(reinterpret_cast<const float2*>(ml + 8 + 2 * t4));
                        po[i] = __ldcg(reinterpret_cast<const float4*>(src + (u * 32 + lane) * 4));
                    }
                }
#pragma unroll
                for (int i = 0; i < kDeep; ++i)
                    if (c + i <= c1) z.add(pm[i], pl[i], po[i]);
            }
            float inv[2];
            finish(a, p.b, p.hr, h0, nt, z.m, z.l, mt == 0, inv);
            store_unit<F16, I8>(a, p.b, p.hr, h0, nt, mt, z.o, inv);
        }
    }
}

// Host: the variants of one pair of types, by head-dim bound and heads a block (paged_decode_*.cu).
int launch_bf16(const Args& a, int DB, int NT, int ctas, cudaStream_t st);
int launch_f16(const Args& a, int DB, int NT, int ctas, cudaStream_t st);
int launch_bf16_i8(const Args& a, int DB, int NT, int ctas, cudaStream_t st);
int launch_f16_i8(const Args& a, int DB, int NT, int ctas, cudaStream_t st);

// Launch the variant for these args (grid: one CTA a SM, capped by `ctas`).
template <bool F16, bool I8, int DB, int NT>
int launch(const Args& a, int ctas, cudaStream_t st) {
    using C = Cfg<F16, I8, DB, NT>;
    const size_t smem = C::kWarps * warp_bytes(I8, C::kStages, NT, a.Dk, a.Dv);
    static thread_local int set_for = -1;
    int dev = 0;
    cudaGetDevice(&dev);
    if (set_for != dev) {
        const size_t most = C::kWarps * warp_bytes(I8, C::kStages, NT, DB, DB);
        if (cudaFuncSetAttribute(decode_kernel<F16, I8, DB, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most) !=
            cudaSuccess)
            return set_error(WS_ERR_CUDA, "paged_decode: shared memory");
        set_for = dev;
    }
    decode_kernel<F16, I8, DB, NT><<<ctas, 32 * C::kWarps, smem, st>>>(a);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? WS_OK : set_error(WS_ERR_CUDA, cudaGetErrorString(e));
}

template <bool F16, bool I8>
int launch_any(const Args& a, int DB, int NT, int ctas, cudaStream_t st) {
    if (DB == 64) return NT == 1 ? launch<F16, I8, 64, 1>(a, ctas, st) : NT == 2 ? launch<F16, I8, 64, 2>(a, ctas, st)
                                                                                 : launch<F16, I8, 64, 4>(a, ctas, st);
    if (DB == 128) return NT == 1 ? launch<F16, I8, 128, 1>(a, ctas, st) : NT == 2 ? launch<F16, I8, 128, 2>(a, ctas, st)
                                                                                   : launch<F16, I8, 128, 4>(a, ctas, st);
    return NT == 1 ? launch<F16, I8, 256, 1>(a, ctas, st) : launch<F16, I8, 256, 2>(a, ctas, st);
}

}  // namespace paged
}  // namespace ws
