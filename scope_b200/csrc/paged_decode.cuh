// Decode attention over a paged key-value cache: the kernel (see paged_decode.cu for the entry).
//
//   o = sum_t softmax_t(scale q.k_t) v_t,  lse = log sum_t exp(scale q.k_t),  t in [max(0, L - window), L)
//
// What bounds it: HBM.  Every key and value row is read once (the query heads that share it are one tensor-core
// tile), against G multiply-adds a byte, so the design keeps enough bytes in flight on every SM for any mix of lengths,
// at few instructions a byte:
//
//   * Rows (request, kv head, block of 8*NT query heads) are cut into subtiles of 16 or 32 tokens, laid end to end, and the
//     line is split evenly over the CTAs (one a SM) and again over each CTA's warps.  Every warp runs alone over its
//     stretch with its own ring of S stages, so no warp ever waits for another and a short row costs no barrier.  The
//     lengths are read on the device; the host never needs them.
//   * A stage is filled by TMA where the pages are whole 16-token tiles, Dk = Dv is the variant's bound and the pool's
//     strides are what a tensor map takes; else by 16-byte cp.async (any page size, any head dims).  The memory gives more
//     to the fewer and larger requests: loads alone run at 7.3 TB/s in blocks of 4 KB by TMA, 6.7 in 16-byte pieces, 6.7
//     in rows of 256 bytes by bulk copies.  Measured under lasting load: 32 requests of 131072 tokens 1365 us with
//     cp.async, 1274 with TMA; 16 ragged 146 and 136; 8 in int8 87 and 84; 1 request of 4096 tokens 12.1 and 11.9.
//   * A subtile is one stage.  With pages of whole 16-token tiles a tile has one page, and its rows lie at one stride; else
//     each lane looks up one token's page and the row addresses travel by shuffle.  Entries are fetched a subtile ahead.
//     Of tokens past the length, before the window or on a page that is none, the scores are -inf, and the values in
//     shared memory zero, whatever the pool holds there.
//   * ldmatrix reads are free of bank conflicts: TMA swizzles; cp.async puts rows an odd number of 16-byte pieces apart.
//   * S^T[16 tok x 8 heads] = K . Q^T and O^T[Dv x 8] += V^T . P^T by mma.sync with the heads as the narrow dimension:
//     at G <= 8 query heads a key there is no 128-row tile for tcgen05 to fill, and the tensor pipe is nearly idle.
//   * The softmax's reference moves only when a score passes it by 2^kSlack: then, and not every subtile, the lanes
//     agree on a new maximum and the accumulators are rescaled.  Sums are fp32, and only a subtile's own is left to the
//     tensor cores, which cut partial sums off instead of rounding them (over 11 thousand tokens a warp that came to
//     2^-14 of the sum, always the same way; the additions cost nothing to 2 %).  A probability enters the second
//     product exactly, as the sum of three bf16 values, or to 2^-22 as two in fp16.  (As two bf16 values: 0.15 to 0.3 %
//     of the 16-bit outputs not the nearest ones; so 0.02 to 0.05 %, the plain form in fp32 0.07 to 0.3 %; 1 request of
//     4096 tokens 11.7 us and 11.9, the others within 1 %.)  No part is 0 where values may be infinite, so an infinite
//     value gives an infinite output.
//   * int8 rows go from shared memory to bf16 (fp16) fragments by bit operations, exactly; the row's scale multiplies
//     the score, or the probability, which then enters as two fp16 values (three bf16 values: 85 us to 78).
//   * A row that ends inside one warp's stretch is written at once.  The others leave a state (o, m, l) per warp,
//     which the CTA joins in shared memory; what crosses CTAs goes through the workspace and is joined by the CTA that
//     files the last part (a ticket), always in the same order, so results do not depend on timing.
//
// Measured on a B200 (device time, a few replays on a cool card): 32 requests of 131072 tokens, 32 query and 4 kv heads of
// 128, bf16: 1207 us (8.59 GB, 7.1 TB/s; a copy reaches 6.55); 16 ragged to 32768 tokens, 32 and 8 heads: 131.7 us
// (852 MB, 6.5 TB/s); 8 of 16384 to 65536 tokens in int8: 78 us (393 MB, 5.0 TB/s).  What is left at those is some 4 us
// before the first rows arrive (the lengths, the table and the rows come one after the other) and 8 us after the last
// (join, ticket, join).  Small calls are those latencies alone: 1 request of 4096 tokens 12.0 us, of 100 9.8.
//
// Why an even split suffices: with 128 KB of copies in flight an SM, 16 of the 148 SMs ended 10% after the others, which
// the memory serves first; with 80 KB all end within 3% of one another, and the whole sooner.  Built and measured slower:
// rows straight from global memory into fragment registers, no shared memory in the loop (half the instructions, but
// each warp waits for its own loads: 224 us on the 16 ragged requests, when this design took 160); TMA for head dims not
// known when compiling (182 requests with keys of 128 and values of 64: 832 us, with cp.async 661; 13 of 112: 88 and 80).
#pragma once

#include "common.cuh"
#include "ws_internal.h"

#include <cuda_fp16.h>

namespace ws {
namespace paged {

// Shared memory for the rings: a CTA's 227 KB without what the kernel declares itself.
constexpr int most_smem(int warps) { return ((227 << 10) - 464 * warps - 128) & ~15; }
constexpr int kMinTok = 32;     // tokens a warp takes before another CTA joins in
// Rows up to so many tokens are not cut by a border between two CTAs, or two warps: the border moves to the nearer end
// of the row, which unbalances the stretches by half a row at most and saves the joining (about 5 us; measured with
// 640, 320, 160 and 0 tokens: 78 requests of 26 to 377 tokens 14.0, 15.1, 15.8, 16.6 us; 128 of up to 700, 26.8, 29.2,
// 27.9, 27.9 us; longer rows the same.  The price is balance: 116 subtiles in the longest CTA of the latter's like, 96 on
// average).
constexpr int kSnapCta = 640;
constexpr int kSnapWarp = 64;
constexpr float kSlack = 6.f;   // log2 of how far a probability may pass its bound before the reference moves

// Bytes of a row that one TMA box takes, and one span of its swizzle.
constexpr int inner_of(int row_bytes) { return row_bytes % 128 ? 64 : 128; }

struct Args {
    CUtensorMap kmap, vmap;              // where tma: boxes of 16 tokens of one head and page
    int tma, k_head_dim2, v_head_dim2;   // the map's order: dims, tokens, heads, pages; else dims, heads, tokens, pages
    const uint16_t* q;
    int64_t q_b, q_h;                    // elements
    const uint8_t* k;
    const uint8_t* v;
    uint32_t kp, kt, kh, vp, vt, vh;     // strides in 16-byte pieces
    const float* ks;
    const float* vs;
    uint32_t ksp, kst, ksh, vsp, vst, vsh;   // floats
    const int32_t* table;
    int64_t table_stride;
    const int32_t* seq_lens;
    int cap;                             // max_pages * page_size, or less than 2^31
    int whole;                           // page_size is a multiple of 16
    int n_pages, page_size;
    uint32_t div_mul, div_shift;         // t / page_size = (umulhi(t, div_mul) + t) >> div_shift
    int B, Hkv, G, hb, Dk, Dv, window;   // hb: head blocks of a kv head
    float scale_log2;
    uint16_t* out;
    float* lse;
    int* counters;
    float* pieces;                       // [cta][2][piece floats]
    int* status;
    int krow, vrow, stages, warp_smem;   // where Dk, Dv are not known when compiling: the ring's geometry (launch)
};

// The variant for head dims up to DB, 8*NT query heads a block.  A subtile is 16 tokens, or 32 where 16 would be 4 KB or
// less (int8, head dims up to 64): what a subtile costs beside its bytes then counts half (measured with int8 rows of 128,
// 8 requests to 65536: 82 us to 78; 127 requests to 13489 with rows of 64: 167 us to 132).  As many warps, each with two
// stages, as shared memory and the registers allow
// (measured at D = 128 in 16 bits, 16 ragged requests to 32768: 8 warps 160 us, 10 warps 152, 12 warps 157; three stages
// put more in flight than the memory takes, and the SMs it serves last fall behind).  These figures are of when the choice
// was made, with cp.async and each probability in two parts.
template <bool I8, int DB, int NT>
struct Cfg {
    static constexpr int kMt = DB / 16;                                   // accumulator fragments of a head tile
    static constexpr int kTok = I8 || DB == 64 ? 32 : 16;                 // tokens of a subtile
    static constexpr int kWarps = DB == 256 ? 5 : DB == 192 ? (I8 ? 6 : 7) : DB == 128 ? (I8 || NT == 2 ? 8 : 10) : I8 ? (NT == 1 ? 16 : 12) : 10;
    static constexpr int kPiece = NT * (8 * DB + 16);                     // floats: fragments, then m and l of the heads
    static constexpr int kUnits = NT * kMt;
    // kExact: stages of rows an odd number of 16-byte pieces apart, each with its scales and meta, then the first part (a
    // stretch's last part takes the ring's place)
    static constexpr int kGapRow = I8 ? ((DB / 16) | 1) * 16 : DB * 2 + 16;
    static constexpr int kGapStage = 2 * kTok * kGapRow + (I8 ? 8 * kTok : 0) + 16;
    static constexpr int kGapFit = (most_smem(kWarps) / kWarps - kPiece * 4) / kGapStage;
    static constexpr int kGapStages = kGapFit > 4 ? 4 : kGapFit;
    static constexpr int kGapWarpSmem = kGapStages * kGapStage + kPiece * 4;
    static_assert(kGapStages >= 2 && kGapStages * kGapStage >= kPiece * 4 && kGapStage % 16 == 0, "ring");
    // kTma: the stages' rows, swizzled and so without gaps, then their scales and meta, then the first part
    static constexpr int kRowB = DB * (I8 ? 1 : 2);
    static constexpr int kInner = inner_of(kRowB), kParts = kRowB / kInner;
    static constexpr int kTile = 16 * kRowB;                              // 16 tokens' keys, or values
    static constexpr int kRows = 2 * kTok * kRowB, kMore = (I8 ? 8 * kTok : 0) + 16;
    static constexpr int kFit = (((most_smem(kWarps) - 1024) / kWarps & ~1023) - kPiece * 4) / (kRows + kMore);
    static constexpr int kStages = kFit > 4 ? 4 : kFit;
    static constexpr int kWarpSmem = (kStages * (kRows + kMore) + kPiece * 4 + 1023) & ~1023;
    static_assert(kStages >= 2 && kStages * kRows >= kPiece * 4 && kRows % 1024 == 0, "ring");
};
inline int piece_floats(int DB, int NT) { return NT * (8 * DB + 16); }

// What the filler of a stage leaves for its reader.
struct __align__(16) Meta {
    uint32_t mask;       // bit i: token i counts
    int b, row;          // request; kv head << 16 | head block
    int sub;             // place in the row; the sign bit: the row ends here
};

__device__ __forceinline__ void cp_async16_all(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
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
// d = A B, or d + A B.
template <bool F16, bool FIRST>
__device__ __forceinline__ void mma16_part(float* d, const uint32_t* a, const uint32_t* b) {
    if (!FIRST) {
        mma16<F16>(d, a[0], a[1], a[2], a[3], b[0], b[1]);
    } else if (F16) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "f"(0.f));
    } else {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "f"(0.f));
    }
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

// Two sums in one instruction: x += a, y += b.
__device__ __forceinline__ void add2(float& x, float& y, float a, float b) {
    uint64_t v, w;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
    asm("mov.b64 %0, {%1, %2};" : "=l"(w) : "f"(a), "f"(b));
    asm("add.rn.f32x2 %0, %0, %1;" : "+l"(v) : "l"(w));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v));
}
// Two floats' leading bits as a pair of 16-bit floats, towards zero: what is left has the sign of the whole.
template <bool F16>
__device__ __forceinline__ uint32_t top16(float lo, float hi) {
    uint32_t d;
    if (F16) asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    else d = __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632);
    return d;
}
template <bool F16>
__device__ __forceinline__ uint32_t max16(uint32_t a, uint32_t b) {
    uint32_t d;
    if (F16) asm("max.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    else asm("max.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
template <bool F16>
__device__ __forceinline__ uint32_t min16(uint32_t a, uint32_t b) {
    uint32_t d;
    if (F16) asm("min.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    else asm("min.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
// Two probabilities as PARTS pairs of 16-bit floats that sum to them: in bf16 three, exactly; in fp16 two, to 2^-22 of the
// larger ones.  Where values may be infinite (not I8), no part of a probability above 0 is 0, else 0 * inf would make a NaN
// of what is infinite: it is the type's least number at least (2^-133; 2^-24 of probabilities kept 2^8 larger).
template <bool F16, bool I8, int PARTS>
__device__ __forceinline__ void split16(float x, float y, uint32_t* part) {
    const uint32_t least = F16 ? __byte_perm(x > 0.f, y > 0.f, 0x5410) : min16<F16>(top16<F16>(x, y), 0x00010001u);
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
        part[i] = F16 && i + 1 == PARTS ? pack16<F16>(x, y) : top16<F16>(x, y);
        const float2 e = unpack16<F16>(part[i]);
        add2(x, y, -e.x, -e.y);
        if (!I8 && (F16 || i)) part[i] = max16<F16>(part[i], least);
    }
}

// (r & m) ^ x in one instruction.
__device__ __forceinline__ uint32_t and_xor(uint32_t r, uint32_t m, uint32_t x) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(d) : "r"(r), "r"(m), "r"(x));
    return d;
}

// Bytes 0 and 2 of r, signed, as a pair of 16-bit floats, exactly, times s8_unit.  With the sign bit turned the byte is
// u = value + 128.  fp16: 0x6400 is 1024 and holds all 8 bits below it, so 1024 + u - 1152 is the value.  bf16 holds 7
// bits below a leading one, but the pattern 0x00uu is u 2^-133 over the whole byte, where subnormal numbers run on into
// normal ones: u 2^-133 2^120 - 2^-6 is value 2^-13.
template <bool F16>
__device__ __forceinline__ uint32_t s8_pair(uint32_t r) {
    uint32_t d;
    if (F16) {
        const uint32_t x = and_xor(r, 0x00ff00ffu, 0x64806480u);
        asm("sub.f16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(0x64806480u));
    } else {
        const uint32_t x = and_xor(r, 0x00ff00ffu, 0x00800080u);
        asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(x), "r"(0x7b807b80u), "r"(0xbc80bc80u));
    }
    return d;
}
template <bool F16>
constexpr float s8_unit = F16 ? 1.f : 8192.f;   // the factor that s8_pair leaves out

// Where request b's attended tokens lie: tokens [lo, L), n subtiles from lo rounded down to one.
struct Span {
    int lo, L, n;
};
template <int kTok>
__device__ __forceinline__ Span span_of(const Args& a, int b) {
    Span s;
    s.L = min(max(a.seq_lens[b], 0), a.cap);
    s.lo = a.window > 0 ? max(s.L - a.window, 0) : 0;
    s.n = (s.L - (s.lo & ~(kTok - 1)) + kTok - 1) / kTok;   // lo = 0 without a token
    return s;
}

// An even split of a line of N places over n CTAs: the first `more` take one place more than `each`.
struct Split {
    int each, more;
    float inv;
    __device__ __forceinline__ Split(int N, int n) {
        each = (uint32_t)N / (uint32_t)n;
        more = N - each * n;
        inv = __fdividef(n, (float)N);
    }
    __device__ __forceinline__ int start(int c) const { return c * each + min(c, more); }
    // The CTA that holds place t: a guess in fp32, which is off by one at most, and the starts beside it.
    __device__ __forceinline__ int owner(int t) const {
        int c = (int)((float)t * inv);
        while (c > 0 && start(c) > t) --c;
        while (start(c + 1) <= t) ++c;
        return c;
    }
};
// Adds to a counter, after everything that this CTA wrote before its last barrier and before everything it reads next.
__device__ __forceinline__ int take_ticket(int* counter) {
    int old;
    asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(old) : "l"(counter) : "memory");
    return old;
}

// Two heads' 1/l; with `write`, lanes of the first row write their lse.
__device__ __forceinline__ void finish(const Args& a, int64_t head0, int left, int nt, const float* m, const float* l,
                                       bool write, float* inv) {
    const int lane = threadIdx.x & 31, t = lane & 3;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        inv[j] = l[j] != 0.f ? 1.f / l[j] : 0.f;   // a NaN stays one
        const int h = nt * 8 + 2 * t + j;
        if (write && a.lse && lane < 4 && h < left) a.lse[head0 + h] = l[j] != 0.f ? m[j] * kLn2 + logf(l[j]) : -INFINITY;
    }
}

// How rows come, and what is known of them when compiling.
enum : int {
    kAny = 0,     // 16-byte cp.async; head dims up to DB
    kExact = 1,   // 16-byte cp.async; Dk = Dv = DB, so a row's pieces need no bounds (8 requests to 65536
                  // tokens in int8 99 us to 87, 204 of up to 101 tokens 14.5 to 12.5, 2 of 100 in pages of 8 11.5 to 10.2)
    kTma = 2,     // TMA; Dk = Dv = DB, pages of whole 16-token tiles
};
template <bool F16, bool I8, int DB, int NT, int MODE>
__global__ void __launch_bounds__(32 * Cfg<I8, DB, NT>::kWarps, 1) decode_kernel(const __grid_constant__ Args a) {
    using C = Cfg<I8, DB, NT>;
    constexpr bool EXACT = MODE != kAny, TMA = MODE == kTma;
    constexpr int kWarps = C::kWarps, kMt = C::kMt, kUnits = C::kUnits, kPiece = C::kPiece;
    constexpr int kTok = C::kTok, H = kTok / 16;   // H: 16-token tiles of a subtile
    constexpr int kMinSub = kMinTok / kTok, kSnapC = kSnapCta / kTok, kSnapW = kSnapWarp / kTok;
    constexpr bool kPF16 = F16 || I8;        // the type of P and V in the second product
    constexpr int kParts = kPF16 ? 2 : 3;    // the 16-bit floats that a probability enters it as
    // fp16 probabilities are kept 2^8 larger, so that the sum of many small ones is not lost below fp16's least value
    constexpr float kUp = kPF16 ? 8.f : 0.f;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    uint8_t* const smem = TMA ? smem_raw + (-smem_u32(smem_raw) & 1023) : smem_raw;   // [kWarps][warp_smem]
    __shared__ uint64_t s_bar[TMA ? kWarps * 4 : 1];
    __shared__ int s_border[kWarps], s_scan[kWarps], s_from[32 * kWarps], s_start[2 * kWarps];   // s_start < 0: no part
    __shared__ int s_list[kWarps][32], s_cnt[32 * kWarps], s_req[2 * kWarps], s_row[2 * kWarps], s_n[2 * kWarps], s_first[2], s_ctas[2];

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t4 = lane & 3;
    const int R = a.Hkv * a.hb;          // rows of a request
    const int Dk = EXACT ? DB : a.Dk, Dv = EXACT ? DB : a.Dv;
    const int S = TMA ? C::kStages : EXACT ? C::kGapStages : a.stages;
    const uint32_t bars = smem_u32(s_bar) + warp * 32;
    if (TMA) {
        if (lane < S) mbar_init(bars + 8 * lane, 1);
        if (lane < 2) tma_prefetch_desc(lane ? &a.vmap : &a.kmap);
        fence_mbar_init();
        __syncwarp();
    }

    // A programmatic dependent launch: everything before this overlaps the kernel before; its writes are seen after.
    pdl_wait_primary();
    pdl_launch_dependents();

    // ---- the line (shorter than 2^31 places): its length, this CTA's stretch and this warp's
    if (lane < 2) s_start[2 * warp + lane] = -1;
    int N;
    const int per = a.B <= 32 ? 1 : (a.B + kWarps * 32 - 1) / (kWarps * 32);   // requests a lane, or a thread, looks at
    int my_from = 0, my_to = 0;   // up to 32 requests: where this lane's request lies
    int my_n = 0;                 // (with one request each) its subtiles a row
    if (a.B <= 32) {              // every warp for itself
        my_n = lane < a.B ? span_of<kTok>(a, lane).n : 0;
        my_to = my_n;
    } else {
        const int first = tid * per;
#pragma unroll 1
        for (int b = first; b < min(first + per, a.B); ++b) my_n = span_of<kTok>(a, b).n, my_to += my_n;
    }
    my_from = my_to;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, my_to, o);
        if (lane >= o) my_to += y;
    }
    my_from = (my_to - my_from) * R, my_to *= R;
    if (a.B <= 32) {
        N = __shfl_sync(0xffffffffu, my_to, 31);
    } else {
        if (lane == 31) s_scan[warp] = my_to;
        __syncthreads();
        int before = 0;
        N = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w == warp) before = N;
            N += s_scan[w];
        }
        s_from[tid] = before + my_from;
        s_cnt[tid] = my_n;
        __syncthreads();
    }
    // A border at place y: where it goes, and the row that begins or goes on there.  In a short row (of up to `most`
    // subtiles) it moves to the row's nearer end.
    struct Border {
        int y, b, row, sub;   // row: R at the request's end
    };
    auto border = [&](int y, int most) {
        if (y >= N) return Border{y, 0, 0, 0};   // the line's end
        int b = 0, from = my_from, n = my_n;
        if (a.B <= 32) {
            b = lane;   // the lane whose request holds y knows best
        } else {
            // the last thread whose requests begin at or before y: its group of kWarps threads, then itself
            const int group = (__popc(__ballot_sync(0xffffffffu, s_from[lane * kWarps] <= y)) - 1) * kWarps;
            const int c = group + __popc(__ballot_sync(0xffffffffu, lane < kWarps && s_from[group + lane % kWarps] <= y)) - 1;
            b = c * per, from = s_from[c], n = s_cnt[c];
            while (per > 1) {   // and the one of them that holds it, 32 at a time
                const int i = b + lane, k = i < min((c + 1) * per, a.B) ? span_of<kTok>(a, i).n : 0;
                int to = k;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int x = __shfl_up_sync(0xffffffffu, to, o);
                    if (lane >= o) to += x;
                }
                to = from + to * R;
                const uint32_t here = __ballot_sync(0xffffffffu, y < to && k > 0);
                if (here || b + 32 >= (c + 1) * per) {
                    const int src = here ? __ffs(here) - 1 : 0;
                    b += src;
                    n = __shfl_sync(0xffffffffu, k, src);
                    from = __shfl_sync(0xffffffffu, to - k * R, src);
                    break;
                }
                b += 32, from = __shfl_sync(0xffffffffu, to, 31);
            }
        }
        Border r = {y, b, 0, 0};
        if (n > 0) {
            const int rel = y - from;
            r.row = (int)__fdividef((float)rel, (float)n);   // off by one at most
            r.sub = rel - r.row * n;
            if (r.sub < 0) --r.row, r.sub += n;
            if (r.sub >= n) ++r.row, r.sub -= n;
            if (n <= most && r.sub > 0) {
                if (2 * r.sub < n) r.y -= r.sub;
                else r.y += n - r.sub, ++r.row;
                r.sub = 0;
            }
        }
        if (a.B <= 32) {
            const uint32_t here = __ballot_sync(0xffffffffu, y >= my_from && y < my_to);
            const int src = __ffs(here) - 1;
            r.y = __shfl_sync(0xffffffffu, r.y, src), r.row = __shfl_sync(0xffffffffu, r.row, src);
            r.sub = __shfl_sync(0xffffffffu, r.sub, src), r.b = src;
        }
        return r;
    };
    // CTAs that work: all, or as many as get kMinSub subtiles a warp
    const int nC = min((int)gridDim.x, (int)((uint32_t)(N + kWarps * kMinSub - 1) / (kWarps * kMinSub)));
    int x0 = 0, x1 = 0, w0 = 0, w1 = 0;
    Border first = {0, 0, 0, 0};
    if ((int)blockIdx.x < nC) {
        const Split split(N, nC);
        if (a.B <= 32) {
            x0 = border(split.start(blockIdx.x), kSnapC).y, x1 = border(split.start(blockIdx.x + 1), kSnapC).y;
            const int len = x1 - x0, each = (uint32_t)len / kWarps, more = len - each * kWarps;
            first = border(x0 + each * warp + min(warp, more), kSnapW);
            w0 = first.y, w1 = border(x0 + each * (warp + 1) + min(warp + 1, more), kSnapW).y;
        } else {   // where finding a border takes longer: each by one warp
            if (warp < 2) {
                const int y = border(split.start(blockIdx.x + warp), kSnapC).y;
                if (lane == 0) s_scan[warp] = y;
            }
            __syncthreads();
            x0 = s_scan[0], x1 = s_scan[1];
            const int len = x1 - x0, each = (uint32_t)len / kWarps, more = len - each * kWarps;
            first = border(x0 + each * warp + min(warp, more), kSnapW);
            w0 = first.y;
            if (lane == 0) s_border[warp] = w0;
            __syncthreads();
            w1 = warp == kWarps - 1 ? x1 : s_border[warp + 1];
        }
    }
    // requests without a token, dealt over the CTAs: zeros, -inf
#pragma unroll 1
    for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
        if (span_of<kTok>(a, b).n) continue;
        const int64_t head0 = (int64_t)b * a.Hkv * a.G;
        for (int i = tid; i < a.Hkv * a.G * (Dv / 8); i += 32 * kWarps)
            reinterpret_cast<uint4*>(a.out + head0 * Dv)[i] = make_uint4(0, 0, 0, 0);
        for (int i = tid; a.lse && i < a.Hkv * a.G; i += 32 * kWarps) a.lse[head0 + i] = -INFINITY;
    }
    if (x0 == x1) return;

    // ---- this warp's stretch
    const int count = w1 - w0;
    const int warp_smem = TMA ? C::kWarpSmem : EXACT ? C::kGapWarpSmem : a.warp_smem;
    uint8_t* const ring = smem + warp * warp_smem;
    float* const first_part = reinterpret_cast<float*>(ring + warp_smem) - kPiece;
    const uint32_t ring_u = smem_u32(ring);
    // a stage: key rows, value rows; int8 scales (the keys', the values'), meta
    const int krow = TMA ? C::kRowB : EXACT ? C::kGapRow : a.krow, vrow = TMA ? C::kRowB : EXACT ? C::kGapRow : a.vrow;
    const int kV = kTok * krow, rows = kV + kTok * vrow, stage = TMA ? rows : rows + C::kMore;
    auto scales_at = [&](int slot) { return TMA ? S * C::kRows + slot * C::kMore : slot * stage + rows; };
    auto meta_at = [&](int slot) { return scales_at(slot) + C::kMore - 16; };
    float* const cta_pieces = a.pieces + (int64_t)blockIdx.x * 2 * kPiece;

    // filler: the row being filled, and the next subtile's page entry (of this lane's 16 tokens, or of its token where
    // pages are not whole tiles)
    bool dead = false;   // a copy did not come within its limit: no more are asked for
    Span fs = {0, 0, 0};
    int f_b = 0, f_kvh = 0, f_blk = 0, f_sub = 0, f_entry = -1, f_left = count;
    uint32_t f_off = 0;
    const int tok = lane & (kTok - 1);
    const int l8 = lane & 7, r4 = lane >> 3;   // copies: eight lanes a row, four rows at a time
    const int kchunks = I8 ? Dk >> 4 : Dk >> 3, vchunks = I8 ? Dv >> 4 : Dv >> 3;
    constexpr int kCols = ((I8 ? DB / 16 : DB / 8) + 7) / 8;
    const uint64_t k_lane = (uint64_t)r4 * a.kt + l8, v_lane = (uint64_t)r4 * a.vt + l8;

    auto look_up = [&]() {
        uint32_t t = (uint32_t)(fs.lo & ~(kTok - 1)) + (uint32_t)f_sub * kTok;
        // within the tokens that count: the entry of any other place may be of no page
        t = a.whole ? min(max(t + (tok & 16), (uint32_t)fs.lo & ~15u), (uint32_t)fs.L - 1) & ~15u
                    : min(max(t + tok, (uint32_t)fs.lo), (uint32_t)fs.L - 1);
        const uint32_t page = (__umulhi(t, a.div_mul) + t) >> a.div_shift;
        f_off = t - page * (uint32_t)a.page_size;
        f_entry = a.table[(int64_t)f_b * a.table_stride + page];
    };
    auto fill = [&](int slot) {
        if (f_left > 0) {
            const uint32_t st = ring_u + slot * stage;
            const int t0 = (fs.lo & ~(kTok - 1)) + f_sub * kTok;
            constexpr uint32_t kAll = kTok == 32 ? 0xffffffffu : 0xffffu;
            uint32_t mask = (kAll >> max(t0 + kTok - fs.L, 0)) & (kAll << max(fs.lo - t0, 0));
            const bool page_ok = (uint32_t)f_entry < (uint32_t)a.n_pages;
            const uint32_t pages_ok = __ballot_sync(0xffffffffu, page_ok);
            if (pages_ok != 0xffffffffu) {
                if (a.status) atomicOr(a.status, kDevBadIndex);
                mask &= pages_ok;   // whole pages: 16 lanes looked at the same one
            }
            const uint32_t page = page_ok ? f_entry : 0;
            const uint64_t ka = (uint64_t)page * a.kp + (uint64_t)f_off * a.kt + (uint64_t)f_kvh * a.kh;
            const uint64_t va = (uint64_t)page * a.vp + (uint64_t)f_off * a.vt + (uint64_t)f_kvh * a.vh;
            if (I8) {
                const uint32_t off = a.whole ? f_off + (lane & 15) : f_off;
                const uint64_t ks = page * (uint64_t)a.ksp + off * (uint64_t)a.kst + f_kvh * (uint64_t)a.ksh;
                const uint64_t vs = page * (uint64_t)a.vsp + off * (uint64_t)a.vst + f_kvh * (uint64_t)a.vsh;
                const bool on = (mask >> tok) & 1;
                cp_async4(ring_u + scales_at(slot) + tok * 4, a.ks + ks, on);
                cp_async4(ring_u + scales_at(slot) + 4 * kTok + tok * 4, a.vs + vs, on);
            }
            if (lane == 0) {
                Meta m;
                m.mask = mask;
                m.b = f_b, m.row = f_kvh << 16 | f_blk, m.sub = f_sub | (f_sub == fs.n - 1 ? INT32_MIN : 0);
                *reinterpret_cast<Meta*>(ring + meta_at(slot)) = m;
            }
            if (TMA) {   // a box of each 16-token tile with a token that counts, for keys and values
                const uint32_t bar = bars + 8 * slot;
                const int page1 = H == 2 ? __shfl_sync(0xffffffffu, (int)page, 16) : 0;
                const int off1 = H == 2 ? __shfl_sync(0xffffffffu, (int)f_off, 16) : 0;
                if (lane == 0 && !dead) {
                    const int tiles = ((mask & 0xffff) != 0) + (H == 2 && (mask >> 16) != 0);
                    mbar_arrive_expect_tx(bar, tiles * 2 * C::kTile);
#pragma unroll
                    for (int h = 0; h < H; ++h) {
                        if ((mask >> (16 * h) & 0xffff) == 0) continue;
                        const int at = h ? off1 : (int)f_off, pg = h ? page1 : (int)page;
#pragma unroll
                        for (int p = 0; p < C::kParts; ++p) {
                            const uint32_t to = st + h * C::kTile + p * 16 * C::kInner;
                            tma_load_4d(to, &a.kmap, bar, p * C::kInner, a.k_head_dim2 ? at : f_kvh, a.k_head_dim2 ? f_kvh : at, pg);
                            tma_load_4d(to + kV, &a.vmap, bar, p * C::kInner, a.v_head_dim2 ? at : f_kvh, a.v_head_dim2 ? f_kvh : at, pg);
                        }
                    }
                }
            } else {
                const uint32_t kd = st + r4 * krow + l8 * 16, vd = st + kV + r4 * vrow + l8 * 16;
                if (a.whole && mask == kAll) {
    #pragma unroll
                    for (int h = 0; h < H; ++h) {
                        const uint64_t kb = H == 1 ? ka : __shfl_sync(0xffffffffu, ka, 16 * h);
                        const uint64_t vb = H == 1 ? va : __shfl_sync(0xffffffffu, va, 16 * h);
                        const uint8_t *kp = a.k + ((kb + k_lane) << 4), *vp = a.v + ((vb + v_lane) << 4);
    #pragma unroll
                        for (int i = 4 * h; i < 4 * h + 4; ++i) {
    #pragma unroll
                            for (int j = 0; j < kCols; ++j) {
                                if (l8 + 8 * j < kchunks) cp_async16_all(kd + 4 * i * krow + j * 128, kp + j * 128);
                                if (l8 + 8 * j < vchunks) cp_async16_all(vd + 4 * i * vrow + j * 128, vp + j * 128);
                            }
                            kp += (uint64_t)a.kt << 6, vp += (uint64_t)a.vt << 6;
                        }
                    }
                } else {
    #pragma unroll
                    for (int i = 0; i < kTok / 4; ++i) {
                        const int row = 4 * i + r4;
                        const bool on = (mask >> row) & 1;
                        const int in_page = a.whole && on ? row & 15 : 0, src = a.whole ? row & 16 : row;
                        const uint64_t kr = __shfl_sync(0xffffffffu, ka, src) + in_page * (uint64_t)a.kt;
                        const uint64_t vr = __shfl_sync(0xffffffffu, va, src) + in_page * (uint64_t)a.vt;
                        const uint8_t *kp = a.k + ((kr + l8) << 4), *vp = a.v + ((vr + l8) << 4);
    #pragma unroll
                        for (int j = 0; j < kCols; ++j) {
                            if (l8 + 8 * j < kchunks) cp_async16(kd + 4 * i * krow + j * 128, kp + j * 128, on);
                            if (l8 + 8 * j < vchunks) cp_async16(vd + 4 * i * vrow + j * 128, vp + j * 128, on);
                        }
                    }
                }
            }
            // on to the next subtile
            if (--f_left > 0) {
                if (++f_sub == fs.n) {
                    f_sub = 0;
                    if (++f_blk == a.hb) {
                        f_blk = 0;
                        if (++f_kvh == a.Hkv) {
                            f_kvh = 0;
                            do fs = span_of<kTok>(a, ++f_b);
                            while (fs.n == 0);
                        }
                    }
                }
                look_up();
            }
        }
        cp_async_commit();
    };

    float m_ref[NT][2], l_run[NT][2], acc[NT][kMt][4];
    uint32_t bq[NT][DB / 16][2];
    bool began = false;                // the row's first subtile was this warp's

    const int nks = Dk >> 4, nmt = Dv >> 4;

    // A row's first head of the block in the output, and how many of the kv head's heads are left from it.
    auto head_of = [&](int b, int row) { return ((int64_t)b * a.Hkv + (row >> 16)) * a.G + (row & 0xffff) * 8 * NT; };
    auto left_of = [&](int row) { return a.G - (row & 0xffff) * 8 * NT; };

    // A row's queries as they lie, 16 (int8 pools: 8) bytes a lane; order_q makes fragments of them once they are here.
    auto load_q = [&](int b, int row) {
        const int kvh = row >> 16, h0 = (row & 0xffff) * 8 * NT;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int h = h0 + nt * 8 + g;
            const uint16_t* q = a.q + b * a.q_b + ((int64_t)kvh * a.G + h) * a.q_h + (I8 ? 4 : 8) * t4;
            if (I8) {
#pragma unroll
                for (int ks = 0; ks < DB / 16; ++ks) {   // dims 16ks + 4t .. 4t + 3
                    uint2 w = make_uint2(0, 0);
                    if (ks < nks && h < a.G) w = *reinterpret_cast<const uint2*>(q + 16 * ks);
                    bq[nt][ks][0] = w.x, bq[nt][ks][1] = w.y;
                }
            } else {
#pragma unroll
                for (int i = 0; i < DB / 32; ++i) {      // dims 32i + 8t .. 8t + 7
                    uint4 w = make_uint4(0, 0, 0, 0);
                    if (32 * i + 8 * t4 < Dk && h < a.G) w = *reinterpret_cast<const uint4*>(q + 32 * i);
                    bq[nt][2 * i][0] = w.x, bq[nt][2 * i][1] = w.y, bq[nt][2 * i + 1][0] = w.z, bq[nt][2 * i + 1][1] = w.w;
                }
            }
        }
    };
    auto order_q = [&]() {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if (I8) {   // the order in which s8_pair gives the dims: (0, 2), (1, 3) of each four
#pragma unroll
                for (int ks = 0; ks < DB / 16; ++ks) {
                    const uint32_t x = bq[nt][ks][0], y = bq[nt][ks][1];
                    bq[nt][ks][0] = __byte_perm(x, y, 0x5410), bq[nt][ks][1] = __byte_perm(x, y, 0x7632);
                }
            } else {    // word i of lane t to word t of lane i, within each four lanes: what ldmatrix gives of the keys
#pragma unroll
                for (int i = 0; i < DB / 16; i += 2) {
                    uint32_t w[4] = {bq[nt][i][0], bq[nt][i][1], bq[nt][i + 1][0], bq[nt][i + 1][1]};
#pragma unroll
                    for (int o = 1; o <= 2; o <<= 1) {
                        const bool up = t4 & o;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            if (k & o) continue;
                            const uint32_t mine = up ? w[k] : w[k + o];
                            const uint32_t other = __shfl_xor_sync(0xffffffffu, mine, o);
                            if (up) w[k] = other;
                            else w[k + o] = other;
                        }
                    }
                    bq[nt][i][0] = w[0], bq[nt][i][1] = w[1], bq[nt][i + 1][0] = w[2], bq[nt][i + 1][1] = w[3];
                }
            }
            m_ref[nt][0] = m_ref[nt][1] = -INFINITY;
            l_run[nt][0] = l_run[nt][1] = 0.f;
#pragma unroll
            for (int mt = 0; mt < kMt; ++mt) acc[nt][mt][0] = acc[nt][mt][1] = acc[nt][mt][2] = acc[nt][mt][3] = 0.f;
        }
    };
    auto file_piece = [&](float* p) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int mt = 0; mt < kMt; ++mt)
                *reinterpret_cast<float4*>(p + ((nt * kMt + mt) * 32 + lane) * 4) =
                    make_float4(acc[nt][mt][0], acc[nt][mt][1], acc[nt][mt][2], acc[nt][mt][3]);
            if (lane < 4) {
                float* ml = p + NT * 8 * DB + nt * 16;
                *reinterpret_cast<float2*>(ml + 2 * t4) = make_float2(m_ref[nt][0], m_ref[nt][1]);
                *reinterpret_cast<float2*>(ml + 8 + 2 * t4) = make_float2(l_run[nt][0], l_run[nt][1]);
            }
        }
    };
    // One fragment of a finished row: O^T[16 dims x 8 heads], dims from 16mt.
    auto store_unit = [&](int64_t head0, int left, int nt, int mt, const float* o, const float* inv) {
        uint16_t* base = a.out + head0 * Dv + 16 * mt;
        if (I8) {   // dims 2g and 2g + 1 of heads 2t, 2t + 1
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int h = nt * 8 + 2 * t4 + j;
                if (h < left)
                    *reinterpret_cast<uint32_t*>(base + (int64_t)h * Dv + 2 * g) = pack16<F16>(o[j] * inv[j], o[j + 2] * inv[j]);
            }
        } else {    // dims g and g + 8; transposed, lane (g, t) gets head g, dims 2t, 2t + 1 and + 8
            const uint32_t lo = movmatrix_t(pack16<F16>(o[0] * inv[0], o[1] * inv[1]));
            const uint32_t hi = movmatrix_t(pack16<F16>(o[2] * inv[0], o[3] * inv[1]));
            const int h = nt * 8 + g;
            if (h < left) {
                *reinterpret_cast<uint32_t*>(base + (int64_t)h * Dv + 2 * t4) = lo;
                *reinterpret_cast<uint32_t*>(base + (int64_t)h * Dv + 8 + 2 * t4) = hi;
            }
        }
    };

    if (count > 0) {
        f_b = first.b, f_sub = first.sub;
        fs = span_of<kTok>(a, f_b);
        int row = first.row;
        if (row == R) {
            row = 0;
            do fs = span_of<kTok>(a, ++f_b);
            while (fs.n == 0);
        }
        f_kvh = a.hb == 1 ? row : row / a.hb;
        f_blk = row - f_kvh * a.hb;
        look_up();
    }
    const int first_b = f_b, first_row = f_kvh << 16 | f_blk;
    int slot = 0;   // the stage that iteration `it` reads; the one before it is filled
    uint32_t phase = 0;
#pragma unroll 1
    for (int it = 1 - S; it < count; ++it) {
        if (it >= 0) {
            if (TMA) {
                if (I8) cp_async_wait<C::kStages - 2>();   // the scales
                if (!dead && !mbar_wait_bounded(bars + 8 * slot, phase)) {
                    if (a.status) atomicOr(a.status, kDevTimeout);
                    // whatever is in flight lands before the ring is used for anything else, or the kernel ends
                    for (int i = 0; i < S - 1 && it + i < count; ++i)
                        mbar_wait_bounded(bars + 8 * ((slot + i) % S), phase ^ (slot + i >= S));
                    dead = true;
                }
                dead = __any_sync(0xffffffffu, dead);
            } else if (EXACT) {
                cp_async_wait<C::kGapStages - 2>();
            } else {
                if (S == 2) cp_async_wait<0>();
                else if (S == 3) cp_async_wait<1>();
                else cp_async_wait<2>();
            }
            __syncwarp();
        }
        const uint32_t st = ring_u + slot * stage;
        Meta meta;
        if (it < 0) meta.b = first_b, meta.row = first_row, meta.sub = it == 1 - S ? 0 : 1;
        else meta = *reinterpret_cast<const Meta*>(ring + meta_at(slot));
        const bool ends = meta.sub < 0;
        meta.sub &= INT32_MAX;
        // a row's queries (the first row's before anything else is asked for)
        if (meta.sub == 0 && it != 0 && count > 0) load_q(meta.b, meta.row);
        fill(it < 0 ? it + S - 1 : slot == 0 ? S - 1 : slot - 1);
        if (it < 0) continue;
        if (it == 0 || meta.sub == 0) {
            order_q();
            began = meta.sub == 0;
        }
        // scores of each 16-token tile; a single tile's in two chains
        constexpr int kChains = H == 1 ? 2 : 1;
        float c[H][NT][4], e[kChains == 2 ? NT : 1][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int h = 0; h < H; ++h) c[h][nt][i] = 0.f;
                if (kChains == 2) e[nt][i] = 0.f;
            }
        // values of tokens that do not count, which TMA brought with the others: zero (int8 codes are finite)
        if (TMA && !I8 && meta.mask != (kTok == 32 ? 0xffffffffu : 0xffffu)) {
            constexpr int kLine = C::kInner / 16;
            const uint32_t off = ~meta.mask >> lane / kLine;
#pragma unroll
            for (int i = 0; i < kTok * C::kRowB / 512; ++i) {   // 32 / kLine tokens at a time
                constexpr int kStep = 32 / kLine;
                const int tile = i * 32 / (C::kTile / 16), tok_in = i * kStep & 15;
                if (off >> (16 * tile + tok_in) & 1)
                    *reinterpret_cast<uint4*>(ring + slot * stage + kV + (i * 32 + lane) * 16) = make_uint4(0, 0, 0, 0);
            }
            if (f_left > 0) fence_proxy_async_smem();   // before TMA writes there again
            __syncwarp();
        }
        // with TMA: 16-byte piece `c` (even) of a lane's row lies where the swizzle puts it
        constexpr int kLine = C::kInner / 16;
        const uint32_t turn_of = C::kInner == 128 ? (lane & 7) << 4 : (lane >> 1 & 3) << 4;
        auto piece = [&](uint32_t base, int row, int hi, int c) {
            return base + row * C::kInner + ((hi << 4 ^ turn_of) ^ (c % kLine << 4)) + c / kLine * 16 * C::kInner;
        };
        const uint32_t k_ld = st + (lane & 15) * krow + (lane >> 4) * 16;
        if (I8) {
#pragma unroll
            for (int ks = 0; ks < DB / 16; ks += 2) {
                if (ks >= nks) break;
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    uint32_t r[4];
                    ldsm_x4(TMA ? piece(st + h * C::kTile, lane & 15, lane >> 4, ks) : k_ld + h * 16 * krow + ks * 16, r[0], r[1], r[2], r[3]);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {   // past an odd nks the queries are zero and what was read is finite
                        const uint32_t a0 = s8_pair<F16>(r[2 * u]), a1 = s8_pair<F16>(r[2 * u + 1]);
                        const uint32_t a2 = s8_pair<F16>(r[2 * u] >> 8), a3 = s8_pair<F16>(r[2 * u + 1] >> 8);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
                            mma16<F16>(kChains == 2 && u ? e[nt] : c[h][nt], a0, a1, a2, a3, bq[nt][ks + u][0], bq[nt][ks + u][1]);
                    }
                }
            }
        } else {
#pragma unroll
            for (int ks = 0; ks < DB / 16; ++ks) {
                if (ks >= nks) break;
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    uint32_t a0, a1, a2, a3;
                    ldsm_x4(TMA ? piece(st + h * C::kTile, lane & 15, lane >> 4, 2 * ks) : k_ld + h * 16 * krow + ks * 32, a0, a1, a2, a3);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        mma16<F16>(kChains == 2 && (ks & 1) ? e[nt] : c[h][nt], a0, a1, a2, a3, bq[nt][ks][0], bq[nt][ks][1]);
                }
            }
        }
        const float* sc = reinterpret_cast<const float*>(ring + scales_at(slot));
#pragma unroll
        for (int h = 0; h < H; ++h) {
            const float f0 = I8 ? sc[16 * h + g] * (s8_unit<F16> * a.scale_log2) : a.scale_log2;
            const float f1 = I8 ? sc[16 * h + g + 8] * (s8_unit<F16> * a.scale_log2) : a.scale_log2;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    c[h][nt][i] = (kChains == 2 ? c[h][nt][i] + e[nt][i] : c[h][nt][i]) * (i < 2 ? f0 : f1);
        }
        if (meta.mask != (kTok == 32 ? 0xffffffffu : 0xffffu)) {   // tokens that do not count (their values and scales are zero)
#pragma unroll
            for (int h = 0; h < H; ++h) {
                const bool on0 = (meta.mask >> (16 * h + g)) & 1, on1 = (meta.mask >> (16 * h + g + 8)) & 1;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) c[h][nt][i] = (i < 2 ? on0 : on1) ? c[h][nt][i] : -INFINITY;
            }
        }
        float tops[NT][2];
        bool past = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                tops[nt][j] = fmaxf(c[0][nt][j], c[0][nt][j + 2]);
                if (H == 2) tops[nt][j] = fmaxf(tops[nt][j], fmaxf(c[H - 1][nt][j], c[H - 1][nt][j + 2]));
                past |= tops[nt][j] > m_ref[nt][j] + (kUp + kSlack);
            }
        if (__any_sync(0xffffffffu, past)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float keep[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float top = tops[nt][j];
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                    top = fmaxf(top - kUp, m_ref[nt][j]);
                    keep[j] = top == -INFINITY ? 1.f : ex2(m_ref[nt][j] - top);
                    m_ref[nt][j] = top;
                    l_run[nt][j] *= keep[j];
                }
#pragma unroll
                for (int mt = 0; mt < kMt; ++mt) {
                    acc[nt][mt][0] *= keep[0], acc[nt][mt][1] *= keep[1];
                    acc[nt][mt][2] *= keep[0], acc[nt][mt][3] *= keep[1];
                }
            }
        }
        uint32_t ps[H][NT][2][kParts];
        // int8: the values' scales over the power of two below the subtile's largest, so that fp16 holds their products with
        // probabilities; what is left out of them is 2^-32 of the largest scale at most
        float down = 1.f, back = 1.f;
        if (I8) {
            static_assert(!I8 || kTok == 32, "a scale a lane");
            const uint32_t e = min(max(__reduce_max_sync(0xffffffffu, __float_as_uint(sc[kTok + lane]) & INT32_MAX) >> 23, 1u), 253u);
            down = __uint_as_float((254 - e) << 23), back = __uint_as_float(e << 23);
        }
#pragma unroll
        for (int h = 0; h < H; ++h) {
            const float v0 = I8 ? sc[kTok + 16 * h + g] * down : 1.f;
            const float v1 = I8 ? sc[kTok + 16 * h + g + 8] * down : 1.f;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float(&p)[4] = c[h][nt];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    // while every score so far is -inf the reference is too: any finite one in its place gives 0
                    const float ref = fmaxf(m_ref[nt][j], -3.0e38f);
                    p[j] = ex2(p[j] - ref), p[j + 2] = ex2(p[j + 2] - ref);
                    l_run[nt][j] += p[j] + p[j + 2];
                    if (I8) p[j] *= v0, p[j + 2] *= v1;
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    split16<kPF16, I8, kParts>(p[2 * j], p[2 * j + 1], ps[h][nt][j]);
#pragma unroll
                    for (int i = 0; i < kParts; ++i) ps[h][nt][j][i] = movmatrix_t(ps[h][nt][j][i]);
                }
            }
        }
        // values, two fragments at a time: the subtile's own sum on the tensor cores, added to the row's in fp32
        const uint32_t v_ld = st + kV + (I8 ? (lane & 15) * vrow + (lane >> 4) * 16 : ((lane & 7) + ((lane >> 4) << 3)) * vrow + ((lane >> 3) & 1) * 16);
#pragma unroll
        for (int mt = 0; mt < kMt; mt += 2) {
            if (mt >= nmt) break;
            float sum[2][NT][4];
#pragma unroll
            for (int h = 0; h < H; ++h) {
                uint32_t v[2][4];   // past an odd nmt: sums that nobody reads
                if (I8) {
                    uint32_t r[4];
                    ldsm_x4_t(TMA ? piece(st + kV + h * C::kTile, lane & 15, lane >> 4, mt) : v_ld + h * 16 * vrow + mt * 16, r[0], r[1], r[2], r[3]);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        v[u][0] = s8_pair<kPF16>(r[2 * u]), v[u][1] = s8_pair<kPF16>(r[2 * u] >> 8);
                        v[u][2] = s8_pair<kPF16>(r[2 * u + 1]), v[u][3] = s8_pair<kPF16>(r[2 * u + 1] >> 8);
                    }
                } else {
#pragma unroll
                    for (int u = 0; u < 2; ++u)
                        ldsm_x4_t(TMA ? piece(st + kV + h * C::kTile, (lane & 7) + (lane >> 4 << 3), lane >> 3 & 1, 2 * (mt + u)) : v_ld + h * 16 * vrow + (mt + u) * 32, v[u][0], v[u][1], v[u][2], v[u][3]);
                }
#pragma unroll
                for (int i = 0; i < kParts; ++i)
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const uint32_t p[2] = {ps[h][nt][0][i], ps[h][nt][1][i]};
                            if (h == 0 && i == 0) mma16_part<kPF16, true>(sum[u][nt], v[u], p);
                            else mma16_part<kPF16, false>(sum[u][nt], v[u], p);
                        }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; i += 2) {
                        float* const o = acc[nt][mt + u] + i;
                        if (I8) o[0] = fmaf(sum[u][nt][i], back, o[0]), o[1] = fmaf(sum[u][nt][i + 1], back, o[1]);
                        else add2(o[0], o[1], sum[u][nt][i], sum[u][nt][i + 1]);
                    }
        }
        // the row, or this warp's stretch, ends
        const bool more = it + 1 < count;
        if (ends || !more) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    l_run[nt][j] += __shfl_xor_sync(0xffffffffu, l_run[nt][j], 4);
                    l_run[nt][j] += __shfl_xor_sync(0xffffffffu, l_run[nt][j], 8);
                    l_run[nt][j] += __shfl_xor_sync(0xffffffffu, l_run[nt][j], 16);
                }
            if (ends && began) {
                const int left = left_of(meta.row);
                const int64_t head0 = head_of(meta.b, meta.row);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float inv[2];
                    finish(a, head0, left, nt, m_ref[nt], l_run[nt], true, inv);
#pragma unroll
                    for (int mt = 0; mt < kMt; ++mt)
                        if (mt < nmt) store_unit(head0, left, nt, mt, acc[nt][mt], inv);
                }
            } else {
                // the stretch's last part takes the ring's place (nothing is in flight into it any more)
                const int part = 2 * warp + (more ? 0 : 1);
                __syncwarp();
                file_piece(more ? first_part : reinterpret_cast<float*>(ring));
                if (lane == 0) {
                    s_start[part] = w0 + it - meta.sub;
                    s_req[part] = meta.b;
                    s_row[part] = meta.row;
                    s_n[part] = span_of<kTok>(a, meta.b).n;
                }
            }
        }
        if (++slot == S) slot = 0, phase ^= 1;
    }
    __syncthreads();

    // ---- join parts.  First the CTA's, row by row; lane i looks at part i: warp i/2's first (even) or last (odd).  Then,
    // if this CTA is the last of a row's to file its part, the row's, copied to shared memory.  A job is kJob units (16 x 8
    // fragments) of a row; the jobs are dealt over the warps.
    constexpr int kJob = 2, kJobs = kUnits / kJob;
    static_assert(kMt % kJob == 0, "a job's units have the same heads");
    const int my_start = lane < 2 * kWarps ? s_start[lane] : -1;
    uint32_t todo = __ballot_sync(0xffffffffu, my_start >= 0);
    int cross0 = -1, cross1 = -1;   // the row that came from an earlier CTA, the one that goes on into the next
    int id0 = 0, id1 = 0, turn = warp, ended = -1, done = 0, ahead = 0;
    const int room = min(kWarps * warp_smem / (kPiece * 4), 32) - 2;
#pragma unroll 1
    while (true) {
        int id, n;              // one of the row's parts here; how many parts to join: s_list[warp][0 .. n-1], bytes
        float* to = nullptr;    // a piece in the workspace or in shared memory, or the output
        __syncwarp();
        if (todo) {
            id = __ffs(todo) - 1;
            const int start = __shfl_sync(0xffffffffu, my_start, id);
            const uint32_t parts = __ballot_sync(0xffffffffu, my_start == start);
            todo &= ~parts;
            n = __popc(parts);
            if ((parts >> lane) & 1)
                s_list[warp][__popc(parts & ((1u << lane) - 1))] =
                    (lane >> 1) * warp_smem + (lane & 1 ? 0 : warp_smem - kPiece * 4);
            if (start < x0) cross0 = start, id0 = id, to = cta_pieces;
            else if (start + s_n[id] > x1) cross1 = start, id1 = id, to = cta_pieces + kPiece;
        } else {
            if (ended < 0) {
                if (cross0 < 0 && cross1 < 0) return;   // the same in every thread
                __syncthreads();
                if (tid < 2) {
                    const int start = tid ? cross1 : cross0;
                    int ctas = 0;
                    if (start >= 0) {
                        // the row's first CTA keeps its counter: a CTA is the first of one crossing row at most
                        const Split split(N, nC);
                        const int c = tid ? blockIdx.x : split.owner(start);
                        ctas = split.owner(start + s_n[tid ? id1 : id0] - 1) - c + 1;
                        if (take_ticket(a.counters + c) == ctas - 1) a.counters[c] = 0;
                        else ctas = 0;
                        s_first[tid] = c;
                    }
                    s_ctas[tid] = ctas;
                }
                __syncthreads();
                ended = 0;
            }
            if (ended < 2 && done == s_ctas[ended]) {
                ++ended, done = 0;
                if (ended < 2 && s_ctas[ended] == 0) ++ended;
            }
            if (ended == 2) return;
            const int ctas = s_ctas[ended], carry = done > 0;
            id = ended ? id1 : id0;
            if (ended && ahead) {   // came with the other row's
                n = done = ctas;
                if (lane < n) s_list[warp][lane] = (2 + ahead + lane) * kPiece * 4;
            } else {
                // `room` parts at a time, with what came of the earlier ones (in place 0 or 1 by turns) as the first; and
                // the other row's too if they fit
                const int take = min(ctas - done, room), first0 = s_first[ended], first1 = s_first[1];
                const int extra = ended == 0 && ctas + s_ctas[1] <= room ? s_ctas[1] : 0;
                ahead = extra ? take : 0;
                __syncthreads();
#pragma unroll 1
                for (int p = warp; p < take + extra; p += kWarps) {
                    // the first CTA filed the row as its slot 1, the others as their slot 0
                    const int c = p < take ? done + p : p - take;
                    const float* src = a.pieces + ((int64_t)((p < take ? first0 : first1) + c) * 2 + (c == 0 ? 1 : 0)) * kPiece + lane * 4;
                    const uint32_t dst = smem_u32(smem) + ((p + 2) * kPiece + lane * 4) * 4;
#pragma unroll
                    for (int r = 0; r < kPiece / 4; r += 32)
                        if (r + 32 <= kPiece / 4 || r + lane < kPiece / 4) cp_async16_all(dst + r * 16, src + r * 4);
                }
                const int round = done / room;
                done += take;
                n = take + carry;
                if (lane < n) s_list[warp][lane] = (carry && lane == 0 ? (round & 1) : lane - carry + 2) * kPiece * 4;
                if (done < ctas) to = reinterpret_cast<float*>(smem + ((round + 1) & 1) * kPiece * 4);
                turn = warp;
                cp_async_commit();
                cp_async_wait<0>();
                __syncthreads();
            }
        }
        __syncwarp();
        const int row = s_row[id], left = left_of(row);
        const int64_t head0 = head_of(s_req[id], row);
#pragma unroll 1
        for (; turn < kJobs; turn += kWarps) {
            const int nt = turn * kJob / kMt, mt0 = turn * kJob - nt * kMt, ml = NT * 8 * DB + nt * 16 + 2 * t4;
            const int at = (turn * kJob * 32 + lane) * 16;
            float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[kJob][4];
#pragma unroll
            for (int q = 0; q < kJob; ++q) o[q][0] = o[q][1] = o[q][2] = o[q][3] = 0.f;
#pragma unroll 1
            for (int i = 0; i < n; i += 8) {   // eight parts: lane (g, t) looks at part g's m and l of its two heads
                const bool in = i + g < n;
                const int mine = s_list[warp][in ? i + g : 0];
                const float* src = reinterpret_cast<const float*>(smem + mine);
                const float2 x = in ? *reinterpret_cast<const float2*>(src + ml) : make_float2(-INFINITY, -INFINITY);
                const float2 y = in ? *reinterpret_cast<const float2*>(src + ml + 8) : make_float2(0.f, 0.f);
                const float px[2] = {x.x, x.y}, py[2] = {y.x, y.y};
                float w[2], keep[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float top = fmaxf(px[j], __shfl_xor_sync(0xffffffffu, px[j], 4));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                    top = fmaxf(fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16)), m[j]);
                    const float ref = fmaxf(top, -3.0e38f);
                    keep[j] = ex2(m[j] - ref);
                    m[j] = top;
                    w[j] = ex2(px[j] - ref);
                    float sum = py[j] * w[j];
                    sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                    l[j] = l[j] * keep[j] + sum;
                }
                if (i) {
#pragma unroll
                    for (int q = 0; q < kJob; ++q) o[q][0] *= keep[0], o[q][1] *= keep[1], o[q][2] *= keep[0], o[q][3] *= keep[1];
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    if (i + k >= n) break;
                    const uint8_t* z = smem + __shfl_sync(0xffffffffu, mine, 4 * k) + at;
                    const float w0 = __shfl_sync(0xffffffffu, w[0], 4 * k + t4), w1 = __shfl_sync(0xffffffffu, w[1], 4 * k + t4);
#pragma unroll
                    for (int q = 0; q < kJob; ++q) {
                        const float4 v = *reinterpret_cast<const float4*>(z + q * 512);
                        o[q][0] += v.x * w0, o[q][1] += v.y * w1, o[q][2] += v.z * w0, o[q][3] += v.w * w1;
                    }
                }
            }
            if (to) {
#pragma unroll
                for (int q = 0; q < kJob; ++q)
                    *reinterpret_cast<float4*>(reinterpret_cast<uint8_t*>(to) + at + q * 512) = make_float4(o[q][0], o[q][1], o[q][2], o[q][3]);
                if (mt0 == 0 && lane < 4) {
                    *reinterpret_cast<float2*>(to + ml) = make_float2(m[0], m[1]);
                    *reinterpret_cast<float2*>(to + ml + 8) = make_float2(l[0], l[1]);
                }
            } else {
                float inv[2];
                finish(a, head0, left, nt, m, l, mt0 == 0, inv);
#pragma unroll
                for (int q = 0; q < kJob; ++q)
                    if (mt0 + q < nmt) store_unit(head0, left, nt, mt0 + q, o[q], inv);
            }
        }
        turn = (turn - kJobs) % kWarps;
    }
}

// Host: the variants of one pair of types, by head-dim bound and heads a block (paged_decode_*.cu).
int launch_bf16(const Args& a, int DB, int NT, int ctas, cudaStream_t st);
int launch_f16(const Args& a, int DB, int NT, int ctas, cudaStream_t st);
int launch_bf16_i8(const Args& a, int DB, int NT, int ctas, cudaStream_t st);
int launch_f16_i8(const Args& a, int DB, int NT, int ctas, cudaStream_t st);

template <bool F16, bool I8, int DB, int NT, int MODE>
int launch(Args a, int ctas, cudaStream_t st) {
    using C = Cfg<I8, DB, NT>;
    int smem = MODE == kTma ? C::kWarps * C::kWarpSmem + 1024 : C::kWarps * C::kGapWarpSmem;
    if (MODE == kAny) {
        // rows as long as they are; stages until the copies in flight are 72 KB an SM (what two stages of 128-dim rows in
        // 16 bits give)
        a.krow = I8 ? ((a.Dk / 16) | 1) * 16 : a.Dk * 2 + 16, a.vrow = I8 ? ((a.Dv / 16) | 1) * 16 : a.Dv * 2 + 16;
        const int bytes = C::kTok * (a.Dk + a.Dv) * (I8 ? 1 : 2);
        const int stage = C::kTok * (a.krow + a.vrow) + (I8 ? 8 * C::kTok : 0) + 16;
        auto warp_smem = [&](int stages) { return std::max(stages * stage, C::kPiece * 4) + C::kPiece * 4; };
        a.stages = 2;
        while (a.stages < 4 && (a.stages - 1) * bytes * C::kWarps < 72 << 10 && C::kWarps * warp_smem(a.stages + 1) <= most_smem(C::kWarps))
            ++a.stages;
        a.warp_smem = warp_smem(a.stages);
        smem = C::kWarps * a.warp_smem;
    }
    static thread_local int set_for = -1;
    int dev = 0;
    cudaGetDevice(&dev);
    if (set_for != dev) {
        if (cudaFuncSetAttribute(decode_kernel<F16, I8, DB, NT, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 MODE != kAny ? smem : most_smem(C::kWarps)) != cudaSuccess)
            return set_error(WS_ERR_CUDA, "paged_decode: shared memory");
        set_for = dev;
    }
    const cudaError_t e = launch_dependent(decode_kernel<F16, I8, DB, NT, MODE>, dim3(ctas), 32 * C::kWarps, smem, st, a);
    return e == cudaSuccess ? WS_OK : set_error(WS_ERR_CUDA, cudaGetErrorString(e));
}

template <bool F16, bool I8, int DB, int NT>
int launch_dims(const Args& a, int ctas, cudaStream_t st) {
    if (a.tma) return launch<F16, I8, DB, NT, kTma>(a, ctas, st);
    return a.Dk == DB && a.Dv == DB ? launch<F16, I8, DB, NT, kExact>(a, ctas, st) : launch<F16, I8, DB, NT, kAny>(a, ctas, st);
}

template <bool F16, bool I8>
int launch_any(const Args& a, int DB, int NT, int ctas, cudaStream_t st) {
    if (DB == 64) return NT == 1 ? launch_dims<F16, I8, 64, 1>(a, ctas, st) : launch_dims<F16, I8, 64, 2>(a, ctas, st);
    if (DB == 128) return NT == 1 ? launch_dims<F16, I8, 128, 1>(a, ctas, st) : launch_dims<F16, I8, 128, 2>(a, ctas, st);
    if (DB == 192) return launch_dims<F16, I8, 192, 1>(a, ctas, st);
    return launch_dims<F16, I8, 256, 1>(a, ctas, st);
}

}  // namespace paged
}  // namespace ws
