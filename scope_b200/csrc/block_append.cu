// The append into pages of 8 bits with one scale for each block of tokens and head: keys turned, blocks quantised as they
// are written.  (Rows as they are, and a scale a row: rope_append.cu.)
//
// A block's rows of this call, from offset o on, and the codes it held before, with scale s_old where o > 0:
//   s_new = max(max|x|, 1e-6) / 127 (int8), the least power of two with max(max|x|, 1e-6) <= 448 s_new (e4m3),
//   s = max(s_old, s_new),  code = rne(x / s);  where s > s_old the earlier rows' codes become rne(code s_old / s).
// With powers of two an e4m3 code is requantised without loss as long as it stays normal; an int8 code moves by half a
// step of the new scale at most, each time its block grows.
//
// What bounds it: long appends, memory (q, k, v in, q and codes out); a decode step, latency.  A CTA takes one head's keys
// or values of a stretch of tokens and, one after the other, the blocks that begin there: its threads hold a block's rows
// (16 dims each, turned, in fp32), agree on the largest, and write codes, so every row is read once.  Only an open block
// that grows is read and written again.  The queries are turned by further CTAs of the same launch.
#include <cstdio>

#include "rope_append.cuh"

#include <type_traits>

namespace ws {
namespace {

constexpr int kMostThreads = 512;
constexpr int kHeld = 4;    // rows of a block that a thread keeps; those behind them are read twice

struct BlockAppendArgs {
    RopeAppendArgs q;       // the queries' rows; positions, slots
    Heads kv[2];
    int block, nb, chunk;   // tokens of a block, blocks of a page, tokens of a CTA
    uint32_t jobs;          // CTAs for keys and values
};

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
__device__ __forceinline__ uint32_t codes4(const float* x, float inv) {
    if (E4M3) {
        uint16_t lo, hi;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(__fmul_rn(x[1], inv)), "f"(__fmul_rn(x[0], inv)));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(__fmul_rn(x[3], inv)), "f"(__fmul_rn(x[2], inv)));
        return (uint32_t)lo | (uint32_t)hi << 16;
    }
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= (uint32_t)(max(-127, min(127, __float2int_rn(__fmul_rn(x[i], inv)))) & 0xff) << (8 * i);
    return w;
}
// Four codes times `ratio` as codes again.
template <bool E4M3>
__device__ __forceinline__ uint32_t again4(uint32_t w, float ratio) {
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        if (E4M3) {
            uint32_t h;
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)(w >> (8 * i))));
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
            x[i] = f.x, x[i + 1] = f.y;
        } else {
            x[i] = (float)(int8_t)(w >> (8 * i)), x[i + 1] = (float)(int8_t)(w >> (8 * i + 8));
        }
    }
    return codes4<E4M3>(x, ratio);
}

// F16: fp16 inputs (else bf16); VEC: q, k, v and q_out are 16-byte aligned throughout; HELD: rows a thread keeps.
template <bool F16, bool E4M3, bool VEC, int HELD>
__global__ void __launch_bounds__(kMostThreads) block_append_kernel(const __grid_constant__ BlockAppendArgs a) {
    __shared__ float s_most[2][kMostThreads / 32];
    __shared__ int s_first[2][kMostThreads / 32];
    pdl_wait_primary();
    pdl_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    if (blockIdx.x >= a.jobs) {
        rope_rows<F16, false, VEC, 2>(a.q, (int64_t)(blockIdx.x - a.jobs) * warps + warp);
        return;
    }
    const int Hkv = a.kv[0].n, part = blockIdx.x / (2 * Hkv), job = blockIdx.x - part * 2 * Hkv;
    const int kind = job >= Hkv, head = kind ? job - Hkv : job;
    const Heads& x = a.kv[kind];
    const ws_rope& r = a.q.rope;
    const int lanes = a.q.lanes, u = tid & (lanes - 1), row = tid / lanes, rows = blockDim.x / lanes;
    const bool in = 16 * u < x.D, turn = kind == 0 && 16 * u < r.rope_dim, split = turn && !r.adjacent;
    const int d0 = split ? 8 * u : 16 * u, d1 = split ? (r.rope_dim >> 1) + 8 * u : 16 * u + 8;
    const int64_t N = a.q.N;

    auto slot_of = [&](int64_t t) -> int64_t {   // -1: dropped, or none
        const int64_t s = t >= 0 && t < N ? a.q.slots[t] : -1;
        return s < a.q.n_slots ? max(s, (int64_t)-1) : -1;
    };
    auto block_of = [&](int64_t s) -> int64_t {   // blocks are counted through the pool
        if (s < 0) return -1;
        return s >> 32 == 0 ? (int64_t)((uint32_t)s / (uint32_t)a.block) : s / a.block;
    };
    // The first token at or after t that is not dropped, or N; the last before t, or -1.  (Past many dropped ones: 256 at a time.)
    auto next_kept = [&](int64_t t) {
        for (; t < N; t += 256) {
            uint32_t any[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) any[i] = slot_of(t + 32 * i + lane) >= 0;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (const uint32_t b = __ballot_sync(0xffffffffu, any[i])) return t + 32 * i + __ffs(b) - 1;
        }
        return N;
    };
    auto last_kept = [&](int64_t t) {
        for (; t > 0; t -= 256) {
            uint32_t any[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) any[i] = slot_of(t - 32 * (i + 1) + lane) >= 0;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (const uint32_t b = __ballot_sync(0xffffffffu, any[i])) return t - 32 * (i + 1) + 31 - __clz(b);
        }
        return (int64_t)-1;
    };
    int turns = 0;   // blocks done

    // The block whose tokens of this call begin at i.
    auto run = [&](const int64_t i, const int64_t key) {
        int64_t end = i + 1, from = end;   // end: one past the block's last token here
        while (from < N) {
            const int64_t s = slot_of(from + lane), k = block_of(s);
            uint32_t same = __ballot_sync(0xffffffffu, k == key);
            const uint32_t other = __ballot_sync(0xffffffffu, k >= 0 && k != key);
            if (other) same &= (other & -other) - 1;
            if (same) end = from + 32 - __clz(same);
            if (other) break;
            if (same) {
                // the block's last slot: nothing of it follows
                if (__shfl_sync(0xffffffffu, s, 31 - __clz(same)) == key * a.block + a.block - 1) break;
                from = end;
            } else {
                from = next_kept(from + 32);
            }
        }
        const int64_t page = key / a.nb, j = key - page * a.nb, base = key * a.block;
        uint8_t* const dst = x.dst + page * x.dst_page + j * a.block * x.dst_tok + head * x.dst_head;
        float* const scale = x.scales + page * x.s_page + j * x.s_tok + head * x.s_head;

        float v[HELD][16];
        int off[HELD];
        float most = 0.f;
        int first = a.block;
        auto take = [&](int64_t t, float* y, int& o) {   // a token's row, turned
            o = -1;
            if (t >= end || !in) return;
            const uint16_t* p = x.src + t * x.src_tok + head * x.src_head;
            const uint4 w0 = load8<VEC>(p + d0), w1 = load8<VEC>(p + d1);
            const int64_t s = slot_of(t);
            float c[8], sn[8];
            if (turn) unit_turns(r, a.q.turns_vec, t, u, a.q.status, c, sn);
            if (block_of(s) != key) return;
            o = (int)(s - base);
            const uint32_t w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float2 f = unpack2<F16>(w[e]);
                y[2 * e] = f.x, y[2 * e + 1] = f.y;
            }
            if (split) {
#pragma unroll
                for (int e = 0; e < 8; ++e) turn_pair(y[e], y[8 + e], c[e], sn[e]);
            } else if (turn) {
#pragma unroll
                for (int e = 0; e < 8; ++e) turn_pair(y[2 * e], y[2 * e + 1], c[e], sn[e]);
            }
            first = min(first, o);
        };
        auto measure = [&](const float* y) {
#pragma unroll
            for (int e = 0; e < 16; ++e) most = max_nan(most, fabsf(y[e]));
        };
        auto put = [&](const float* y, int o, float inv, bool fine) {
            uint2 lo = make_uint2(codes4<E4M3>(y, inv), codes4<E4M3>(y + 4, inv));
            uint2 hi = make_uint2(codes4<E4M3>(y + 8, inv), codes4<E4M3>(y + 12, inv));
            if (!fine) lo = hi = make_uint2(0, 0);
            uint8_t* const p = dst + (int64_t)o * x.dst_tok;
            *reinterpret_cast<uint2*>(p + d0) = lo;
            *reinterpret_cast<uint2*>(p + d1) = hi;
        };
#pragma unroll
        for (int m = 0; m < HELD; ++m) {
            take(i + row + m * rows, v[m], off[m]);
            if (off[m] >= 0) measure(v[m]);
        }
        for (int64_t t = i + row + HELD * rows; t < end; t += rows) {
            float y[16];
            int o;
            take(t, y, o);
            if (o >= 0) measure(y);
        }
        const float held = *scale;   // whatever lies there, used only with rows before the first
        // all agree on the largest value and the first row
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
        first = __reduce_min_sync(0xffffffffu, first);
        const int buf = turns++ & 1;
        if (lane == 0) s_most[buf][warp] = most, s_first[buf][warp] = first;
        __syncthreads();
        for (int w = 0; w < warps; ++w) most = max_nan(most, s_most[buf][w]), first = min(first, s_first[buf][w]);

        const float need = own_scale<E4M3>(most), s = first > 0 ? max_nan(held, need) : need;
        const bool fine = s < INFINITY;   // a NaN is not
        const float inv = fine ? __fdiv_rn(1.f, s) : 0.f;
#pragma unroll
        for (int m = 0; m < HELD; ++m)
            if (off[m] >= 0) put(v[m], off[m], inv, fine);
        for (int64_t t = i + row + HELD * rows; t < end; t += rows) {
            float y[16];
            int o;
            take(t, y, o);
            if (o >= 0) put(y, o, inv, fine);
        }
        if (first > 0 && s != held && in) {   // the earlier rows
            const float ratio = __fmul_rn(held, inv);
            for (int o = row; o < first; o += rows) {
                uint4* const p = reinterpret_cast<uint4*>(dst + (int64_t)o * x.dst_tok + 16 * u);
                uint4 w = *p;
                w.x = fine ? again4<E4M3>(w.x, ratio) : 0, w.y = fine ? again4<E4M3>(w.y, ratio) : 0;
                w.z = fine ? again4<E4M3>(w.z, ratio) : 0, w.w = fine ? again4<E4M3>(w.w, ratio) : 0;
                *p = w;
            }
        }
        if (tid == 0) *scale = s;
    };

    const int64_t c0 = (int64_t)part * a.chunk, c1 = min(c0 + a.chunk, N);
#pragma unroll 1
    for (int64_t w = c0; w < c1; w += 32) {
        // of each token: does the one before it (dropped ones aside) lie in another block
        const int64_t t = w + lane, raw = t < c1 ? a.q.slots[t] : -1, slot = t < c1 ? slot_of(t) : -1;
        const int64_t mine = block_of(slot), prev = block_of(slot_of(w - 32 + lane));
        if (raw >= a.q.n_slots && job == 0 && warp == 0 && a.q.status) atomicOr(a.q.status, kDevBadIndex);
        const uint32_t kept = __ballot_sync(0xffffffffu, mine >= 0), behind = __ballot_sync(0xffffffffu, prev >= 0);
        if (!kept) continue;
        int64_t before = __shfl_sync(0xffffffffu, prev, behind ? 31 - __clz(behind) : 0);
        if (!behind) {   // many dropped ones: whom a token at its block's first slot need not look past
            before = -1;
            if (__shfl_sync(0xffffffffu, slot - mine * a.block, __ffs(kept) - 1) > 0) {
                const int64_t l = last_kept(w - 32);
                if (l >= 0) before = block_of(slot_of(l));
            }
        }
        const uint32_t below = kept & ((1u << lane) - 1);
        const int64_t near = __shfl_sync(0xffffffffu, mine, below ? 31 - __clz(below) : 0);
        uint32_t todo = __ballot_sync(0xffffffffu, mine >= 0 && mine != (below ? near : before));
#pragma unroll 1
        while (todo) {
            const int k = __ffs(todo) - 1;
            todo &= todo - 1;
            run(w + k, __shfl_sync(0xffffffffu, mine, k));
        }
    }
}

}  // namespace

int block_append_launch(const RopeAppendArgs& q, bool f16, bool e4m3, bool vec, int block, cudaStream_t st) {
    BlockAppendArgs a;
    memset(&a, 0, sizeof(a));
    a.q = q;
    a.kv[0] = q.h[1], a.kv[1] = q.h[2];
    a.q.h[1].n = a.q.h[2].n = 0;
    a.block = block, a.nb = q.page_size / block;
    const int64_t units = (int64_t)block * q.lanes;
    const int threads = (int)std::min<int64_t>(kMostThreads, (units + 31) / 32 * 32);
    const int held = units <= threads ? 1 : units <= 2 * threads ? 2 : kHeld;
    // A CTA takes one token's block where that gives two rounds of CTAs or fewer, else up to a block of tokens.
    const int Hkv = a.kv[0].n, sms = device_sm_count();
    const int64_t room = (int64_t)sms * (2048 / threads) * 2;
    a.chunk = (int)std::max<int64_t>(1, std::min<int64_t>(block, (q.N * 2 * Hkv + room - 1) / room));
    const int64_t jobs = (q.N + a.chunk - 1) / a.chunk * 2 * Hkv;
    // the queries: as in rope_append_kernel, two rows a turn
    const int rows = 32 / q.lanes, steps = (q.h[0].n + 2 * rows - 1) / (2 * rows), warps = threads / 32;
    a.q.parts = (int)std::max<int64_t>(1, std::min<int64_t>(steps, ((int64_t)sms * 32 + q.N - 1) / q.N));
    const int64_t blocks = jobs + (q.h[0].n ? (q.N * a.q.parts + warps - 1) / warps : 0);
    if (blocks > INT32_MAX) return set_error(WS_ERR_UNSUPPORTED, "rope_append: too many tokens");
    a.jobs = (uint32_t)jobs;
    auto pick = [&](auto half, auto eight, auto aligned) {
        constexpr bool F = decltype(half)::value, E = decltype(eight)::value, V = decltype(aligned)::value;
        return held == 1 ? block_append_kernel<F, E, V, 1> : held == 2 ? block_append_kernel<F, E, V, 2> : block_append_kernel<F, E, V, kHeld>;
    };
    using yes = std::true_type;
    using no = std::false_type;
    auto by_vec = [&](auto half, auto eight) { return vec ? pick(half, eight, yes{}) : pick(half, eight, no{}); };
    auto fn = f16 ? (e4m3 ? by_vec(yes{}, yes{}) : by_vec(yes{}, no{})) : (e4m3 ? by_vec(no{}, yes{}) : by_vec(no{}, no{}));
    const cudaError_t e = launch_dependent(fn, dim3((unsigned)blocks), threads, 0, st, a);
    return e == cudaSuccess ? WS_OK : set_error(WS_ERR_CUDA, cudaGetErrorString(e));
}

}  // namespace ws
