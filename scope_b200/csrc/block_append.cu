// The append into pages of 8 bits with one scale for each block of tokens and head: keys turned, blocks quantised as they
// are written.  (Rows as they are, and a scale a row: rope_append.cu.)
//
// A block's rows of this call, from offset o on, and the codes it held before, with scale s_old where o > 0:
//   s_new = max(max|x|, 1e-6) / 127 (int8), the least power of two with max(max|x|, 1e-6) <= 448 s_new (e4m3),
//   s = max(s_old, s_new),  code = rne(x / s);  where s > s_old the earlier rows' codes become rne(code s_old / s).
// With powers of two an e4m3 code is requantised without loss as long as it stays normal; an int8 code moves by half a
// step of the new scale at most, each time its block grows.
//
// What bounds it: a decode step, latency (slots, then the block's scale, rows and turns, then an agreement, then the codes);
// long appends, instructions: 480 a warp for 32 units of 16 dims, three fourths of them addresses, places and branches, at an
// issue rate of 0.47.  A job is one head's keys or values of the blocks that begin in a stretch of tokens; its threads look
// at as many tokens as a block has room for (their slots say which belong to it), keep the turned rows in shared memory,
// agree on the largest value and write codes, so every row is read once.  Only an open block that grows is read and written
// again.  The queries of a small call are turned by further CTAs of the same launch; those of a long one by a launch of
// their own, with fewer registers (4.6 thousand tokens of 20 + 5 + 5 heads of 80: 23.0 us, in one launch 24.3).
// Measured: 64 tokens of 32 + 8 + 8 heads of 128 into int8 4.7 us; 17.9 thousand of 32 + 4 + 4 into e4m3 78 (of which the
// queries 50); 4.6 thousand of 20 + 5 + 5 heads of 80 into int8 22.7 (7.8).  Built and measured slower: a CTA of up to 512
// threads with four heads a thread, which share a row's turns (35 us where this takes 29: an SM holds one, in one phase);
// products of two floats in one instruction (the moves into register pairs cost more).
#include <cstdio>

#include "rope_append.cuh"

#include <type_traits>

namespace ws {
namespace {

constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr int kHeld = 4;    // rows of a block that a thread keeps; those behind them are read twice

struct Side {           // keys or values: Heads with strides of tokens and blocks that fit 32 bits
    const uint16_t* src;
    uint8_t* dst;
    float* scales;
    int64_t dst_page, s_page, src_head, dst_head, s_head;
    uint32_t src_tok, dst_tok, s_tok;
    int n, D;
};
struct BlockAppendArgs {
    RopeAppendArgs q;       // the queries' rows; positions, slots
    Side kv[2];
    int block, chunk;       // tokens of a block, of a job
    uint32_t blk_mul, blk_shift;   // s / block = (umulhi(s, mul) + s) >> shift for s < 2^31
    int Hkv;
    int one_axis;           // all pairs turn by one axis, forward, their turns 16-byte aligned
    uint32_t jobs;          // stretches of tokens times keys and values times heads
    uint32_t job_rate;      // of 2^32 CTAs, how many are theirs
    int all_jobs;           // there are no others
};

// The largest magnitude of three, or NaN where one is.
__device__ __forceinline__ float most_of(float a, float b, float c) {
    float d;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// The largest of the warp's magnitudes: as bits they are in order, with NaN above infinity.
__device__ __forceinline__ float warp_most(float x) {
    return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(x) & INT32_MAX));
}

// Four codes times `ratio` as codes again.
template <bool E4M3>
__device__ __forceinline__ uint32_t again4(uint32_t w, float ratio) {
    float2 x[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (E4M3) {
            uint32_t h;
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)(w >> (16 * i))));
            x[i] = __half22float2(*reinterpret_cast<const __half2*>(&h));
        } else {
            x[i] = make_float2((float)(int8_t)(w >> (16 * i)), (float)(int8_t)(w >> (16 * i + 8)));
        }
    }
    return codes4<E4M3>(x[0], x[1], ratio);
}

// F16: fp16 inputs (else bf16); VEC: q, k, v and q_out are 16-byte aligned throughout.  A job, taken by
// a warp or by a CTA, is a head's keys or values of the blocks that begin in a stretch of tokens.
template <bool F16, bool E4M3, bool VEC, int WARPS>
__global__ void __launch_bounds__(kThreads, WARPS == 1 ? 4 : 5) block_append_kernel(const __grid_constant__ BlockAppendArgs a) {
    extern __shared__ float4 s_row[];   // [kHeld][4][kThreads]: turned rows; then int [kHeld][kThreads]: their places
    __shared__ float s_most[2][kWarps];
    __shared__ int2 s_more[2][kWarps];
    pdl_wait_primary();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // CTAs for keys and values are spread evenly among those for queries: the ones wait, the others stream
    const uint32_t nth = a.all_jobs ? blockIdx.x : __umulhi(blockIdx.x, a.job_rate);
    if (!a.all_jobs && nth == __umulhi(blockIdx.x + 1, a.job_rate)) {
        rope_rows<F16, kRows16, VEC, 2>(a.q, (int64_t)(blockIdx.x - nth) * kWarps + warp);
        return;
    }
    const uint32_t id = WARPS == 1 ? nth * kWarps + warp : nth;
    if (id >= a.jobs) return;
    const int part = id / (2 * a.Hkv), job = id - part * 2 * a.Hkv;
    const int kind = job >= a.Hkv, head = kind ? job - a.Hkv : job;
    const Side x = kind ? a.kv[1] : a.kv[0];
    const ws_rope& r = a.q.rope;
    const int lanes = a.q.lanes, tid = WARPS == 1 ? lane : threadIdx.x, u = tid & (lanes - 1), row = tid / lanes, rows = 32 * WARPS / lanes;
    const bool in = 16 * u < x.D, turn = kind == 0 && 16 * u < r.rope_dim, split = turn && !r.adjacent;
    const int d0 = split ? 8 * u : 16 * u, d1 = split ? (r.rope_dim >> 1) + 8 * u : 16 * u + 8;
    const int N = (int)a.q.N, block = a.block;
    const uint16_t* const src = x.src + head * x.src_head;
    int* const s_place = reinterpret_cast<int*>(s_row + kHeld * 4 * kThreads);

    auto slot_of = [&](int t) -> int64_t {   // -1: dropped, or none
        const int64_t s = t >= 0 && t < N ? a.q.slots[t] : -1;
        return s < a.q.n_slots ? max(s, (int64_t)-1) : -1;
    };
    auto offset_of = [&](int64_t s) {        // in its block
        if (s >> 31 == 0) return (int)((uint32_t)s - ((__umulhi((uint32_t)s, a.blk_mul) + (uint32_t)s) >> a.blk_shift) * (uint32_t)block);
        return (int)(s % block);
    };
    // The first token at or after t that is not dropped, or N; the last before t, or -1.  (Past many dropped ones: 256 at a time.)
    auto next_kept = [&](int t) {
#pragma unroll 1
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
    auto last_kept = [&](int t) {
#pragma unroll 1
        for (; t > 0; t -= 256) {
            uint32_t any[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) any[i] = slot_of(t - 32 * (i + 1) + lane) >= 0;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (const uint32_t b = __ballot_sync(0xffffffffu, any[i])) return t - 32 * (i + 1) + 31 - __clz(b);
        }
        return -1;
    };
    auto load = [&](const uint16_t* p, uint4* w) { w[0] = load8<VEC>(p + d0), w[1] = load8<VEC>(p + d1); };
    auto position = [&](int t) -> uint32_t {   // asked for ahead of the turns, where one axis is all; past the end: negative too
        if (!turn || !a.one_axis) return 0;
        if (!r.positions_i64) return static_cast<const uint32_t*>(r.positions)[t];
        const int64_t p = static_cast<const int64_t*>(r.positions)[t];
        return p < 0 ? UINT32_MAX : p > INT32_MAX ? INT32_MAX : (uint32_t)p;
    };
    const float* const turns_u = r.cos_sin + 8 * u;
    auto turns_at = [&](int t, uint32_t p, float* c, float* s) {   // of this thread's unit
        if (!a.one_axis) return unit_turns(r, a.q.turns_vec, t, u, a.q.status, c, s);
        if (p >= (uint32_t)r.max_pos) {
            if (a.q.status) atomicOr(a.q.status, kDevBadIndex);
            p = p > (uint32_t)INT32_MAX ? 0 : (uint32_t)r.max_pos - 1;
        }
        const float* const at = turns_u + (uint64_t)p * (uint32_t)r.rope_dim;
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
            const float4 x = *reinterpret_cast<const float4*>(at + i), y = *reinterpret_cast<const float4*>(at + (r.rope_dim >> 1) + i);
            c[i] = x.x, c[i + 1] = x.y, c[i + 2] = x.z, c[i + 3] = x.w;
            s[i] = y.x, s[i + 1] = y.y, s[i + 2] = y.z, s[i + 3] = y.w;
        }
    };
    // A row's 16 dims, turned: y[e] are dims d0 + 2e, d0 + 2e + 1, y[4 + e] the same from d1.
    auto turned = [&](int t, uint32_t p, const uint4* v, float2* y) {
        const uint32_t w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = unpack2<F16>(w[e]);
        if (!turn) return;
        float c[8], sn[8];
        turns_at(t, p, c, sn);
        if (split) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                turn_pair(y[e].x, y[4 + e].x, c[2 * e], sn[2 * e]), turn_pair(y[e].y, y[4 + e].y, c[2 * e + 1], sn[2 * e + 1]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) turn_pair(y[e].x, y[e].y, c[e], sn[e]);
        }
    };
    const int c0 = part * a.chunk, c1 = min(c0 + a.chunk, N);
    int turns = 0;    // agreements
    uint4 ahead[2];   // the row that is this thread's first, if a block begins at the first token
    if (in && c0 + row < N) load(src + (uint64_t)(uint32_t)(c0 + row) * x.src_tok, ahead);

    // The block whose tokens of this call begin at i, in slot s_i.
    auto run = [&](const int i, const int64_t s_i) {
        const int front = offset_of(s_i);
        const int64_t base = s_i - front, page = base >> 31 == 0 ? (int64_t)((uint32_t)base / (uint32_t)a.q.page_size) : base / a.q.page_size;
        const int at = (int)(base - page * a.q.page_size), j = (int)((__umulhi((uint32_t)at, a.blk_mul) + (uint32_t)at) >> a.blk_shift);
        uint8_t* const dst = x.dst + page * x.dst_page + (uint64_t)(uint32_t)at * x.dst_tok + head * x.dst_head;
        float* const scale = x.scales + page * x.s_page + (uint64_t)(uint32_t)j * x.s_tok + head * x.s_head;
        auto place_of = [&](int64_t s) { return (uint64_t)(s - base) < (uint64_t)block ? (int)(s - base) : -1; };
        // As many tokens as the block has room for are looked at: those of this block have their place by their slots.
        int end = (int)min((int64_t)i + block - front, (int64_t)N);
        const float held = *scale;   // what lies there, used only with rows before the first
        uint4 old = make_uint4(0, 0, 0, 0);   // the first of this thread's earlier rows, in case the scale grows
        if (in && row < front) old = *reinterpret_cast<const uint4*>(dst + (uint64_t)(uint32_t)row * x.dst_tok + 16 * u);
        float most = 0.f;
        int first = front;
        bool dropped = false;
        auto measure = [&](int t0) {   // the rows from t0 on
            int t = i + row, m = 0;
            while (t < t0) t += rows, ++m;
            const uint16_t* p = src + (uint64_t)(uint32_t)t * x.src_tok;
            const int64_t* slot = a.q.slots + t;
            const uint64_t step = (uint64_t)(uint32_t)rows * x.src_tok;
            uint4 next[2];
            next[0] = ahead[0], next[1] = ahead[1];
            int64_t next_slot = -1;
            uint32_t next_pos = 0;
            if (!in) return;   // a row's first unit is always there
            if (t < end) {
                if (t > i + row || i != c0) load(p, next);
                next_slot = *slot, next_pos = position(t);
            }
#pragma unroll 1
            for (; t < end; t += rows, ++m) {
                uint4 v[2];
                v[0] = next[0], v[1] = next[1];
                const int64_t s = next_slot;
                const uint32_t pos = next_pos;
                p += step, slot += rows;
                if (t + rows < end) {
                    load(p, next);
                    next_slot = *slot, next_pos = position(t + rows);
                }
                const int o = place_of(s);
                if (m < kHeld) s_place[m * kThreads + threadIdx.x] = o;
                if (o < 0) {
                    dropped |= (uint64_t)s >= (uint64_t)a.q.n_slots;
                    continue;
                }
                first = min(first, o);
                float2 y[8];
                turned(t, pos, v, y);
#pragma unroll
                for (int e = 0; e < 8; ++e) most = most_of(most, y[e].x, y[e].y);
                if (m < kHeld) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        s_row[(m * 4 + e) * kThreads + threadIdx.x] = make_float4(y[2 * e].x, y[2 * e].y, y[2 * e + 1].x, y[2 * e + 1].y);
                }
            }
        };
        // the largest of all the job's threads, the least of their firsts, whether one has seen a dropped token
        auto agree = [&]() {
            most = warp_most(most);
            first = __reduce_min_sync(0xffffffffu, first);
            dropped = __any_sync(0xffffffffu, dropped);
            if (WARPS == 1) return __syncwarp();   // all have read the scale that one is about to write
            const int buf = turns++ & 1;
            if (lane == 0) s_most[buf][warp] = most, s_more[buf][warp] = make_int2(first, dropped);
            __syncthreads();
            const int2 more = s_more[buf][lane % kWarps];
            most = warp_most(s_most[buf][lane % kWarps]);
            first = __reduce_min_sync(0xffffffffu, more.x);
            dropped = __any_sync(0xffffffffu, more.y);
        };
        measure(i);
        agree();
        if (dropped) {   // the same in every thread: the block may go on behind
            const int behind = end;
            for (int from = end; from < N;) {
                const int64_t z = slot_of(from + lane);
                const bool mine = z >= base && z < base + block;
                uint32_t same = __ballot_sync(0xffffffffu, mine);
                const uint32_t other = __ballot_sync(0xffffffffu, z >= 0 && !mine);
                if (other) same &= (other & -other) - 1;
                if (same) end = from + 32 - __clz(same);
                if (other) break;
                from = same ? end : next_kept(from + 32);
            }
            if (end > behind) {
                measure(behind);
                agree();
            }
        }
        const float need = own_scale<E4M3>(most), s = first > 0 ? max_nan(held, need) : need;
        const float inv = s < INFINITY ? __fdiv_rn(1.f, s) : 0.f;   // 0: not finite, codes of 0
        if (tid == 0) *scale = s;
#pragma unroll 1
        for (int t = i + row, m = 0; in && t < end; t += rows, ++m) {
            const int o = m < kHeld ? s_place[m * kThreads + threadIdx.x] : place_of(a.q.slots[t]);
            if (o < 0) continue;
            float2 y[8];
            if (m < kHeld) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float4 z = s_row[(m * 4 + e) * kThreads + threadIdx.x];
                    y[2 * e] = make_float2(z.x, z.y), y[2 * e + 1] = make_float2(z.z, z.w);
                }
            } else {
                uint4 v[2];
                load(src + (uint64_t)(uint32_t)t * x.src_tok, v);
                turned(t, position(t), v, y);
            }
            uint2 lo = make_uint2(0, 0), hi = lo;
            if (inv > 0.f) {
                lo = make_uint2(codes4<E4M3>(y[0], y[1], inv), codes4<E4M3>(y[2], y[3], inv));
                hi = make_uint2(codes4<E4M3>(y[4], y[5], inv), codes4<E4M3>(y[6], y[7], inv));
            }
            uint8_t* const to = dst + (uint64_t)(uint32_t)o * x.dst_tok;
            *reinterpret_cast<uint2*>(to + d0) = lo;
            *reinterpret_cast<uint2*>(to + d1) = hi;
        }
        if (first > 0 && s != held && in) {   // the earlier rows get the new scale
            const float ratio = __fmul_rn(held, inv);
#pragma unroll 1
            for (int o = row; o < first; o += rows) {
                uint4* const p = reinterpret_cast<uint4*>(dst + (uint64_t)(uint32_t)o * x.dst_tok + 16 * u);
                uint4 w = make_uint4(0, 0, 0, 0);
                if (inv > 0.f) {
                    w = o == row ? old : *p;
                    w.x = again4<E4M3>(w.x, ratio), w.y = again4<E4M3>(w.y, ratio);
                    w.z = again4<E4M3>(w.z, ratio), w.w = again4<E4M3>(w.w, ratio);
                }
                *p = w;
            }
        }
    };

#pragma unroll 1
    for (int w = c0; w < c1; w += 32) {
        // of each token: is it its block's first here?  The one before it (dropped ones aside) lies in another block then
        const int t = w + lane;
        const int64_t s = t < c1 ? slot_of(t) : -1;
        int64_t back = t < c1 ? slot_of(t - 1) : -1;
        if (t < c1 && job == 0 && a.q.slots[t] >= a.q.n_slots && a.q.status) atomicOr(a.q.status, kDevBadIndex);
        const int off = s >= 0 ? offset_of(s) : 0;
        uint32_t unsure = __ballot_sync(0xffffffffu, s >= 0 && off > 0 && back < 0 && t > 0);
        while (unsure) {   // dropped ones before it
            const int k = __ffs(unsure) - 1, l = last_kept(w + k);
            unsure &= unsure - 1;
            const int64_t z = l >= 0 ? slot_of(l) : -1;
            if (lane == k) back = z;
        }
        uint32_t todo = __ballot_sync(0xffffffffu, s >= 0 && (off == 0 || back < s - off || back >= s - off + block));
#pragma unroll 1
        while (todo) {
            const int k = __ffs(todo) - 1;
            todo &= todo - 1;
            run(w + k, __shfl_sync(0xffffffffu, s, k));
        }
    }
}

}  // namespace

bool block_append_small(int64_t N, int Hkv) { return N * 2 * Hkv <= (int64_t)device_sm_count() * 16; }

namespace {

// What a call refuses, and how it is cut: into `blocks` CTAs, a job taken by `warps` warps.
int plan(const RopeAppendArgs& q, int block, BlockAppendArgs& a, int& warps, int64_t& blocks) {
    memset(&a, 0, sizeof(a));
    a.q = q;
    for (int i = 0; i < 2; ++i) {
        const Heads& h = q.h[1 + i];
        for (const int64_t stride : {h.src_tok, h.dst_tok, h.s_tok})
            if (stride < 0 || stride > UINT32_MAX) return set_error(WS_ERR_UNSUPPORTED, "rope_append: a stride of tokens or blocks past 32 bits");
        a.kv[i] = {h.src, h.dst, h.scales, h.dst_page, h.s_page, h.src_head, h.dst_head, h.s_head,
                   (uint32_t)h.src_tok, (uint32_t)h.dst_tok, (uint32_t)h.s_tok, h.n, h.D};
    }
    a.q.h[1].n = a.q.h[2].n = 0;
    a.block = block;
    while ((1ull << a.blk_shift) < (uint64_t)block) ++a.blk_shift;
    a.blk_mul = (uint32_t)((((1ull << a.blk_shift) - block) << 32) / block + 1);
    a.one_axis = q.turns_vec && q.rope.n_axes == 1 && !q.rope.inverse;   // turning back is rare: unit_turns does it
    if (q.N > INT32_MAX - 4096) return set_error(WS_ERR_UNSUPPORTED, "rope_append: too many tokens");
    // A job is the block of one token where there are few, else those of up to a block of tokens, as long as every SM has 16
    // warps.  A warp takes it, or a CTA where blocks are large and tokens many (17 thousand tokens of 4 + 4 heads of 128 in
    // blocks of 64, us by warps and by CTAs: 59 and 29; 4.6 thousand of 5 + 5 heads of 80 in blocks of 8: 13 and 20).  Few
    // tokens are taken for a decode step's, one a block (8 requests, 2 kv heads of 128, blocks of 64, by warps and by CTAs: 3.4
    // and 3.6; 64 requests, 8 kv heads, blocks of 32: 4.8 and 6.3).  Where they are one request's instead, which the host cannot
    // see, large blocks pay for it: 64 tokens in blocks of 64 20.6 and 6.7, 512 of 2 kv heads in blocks of 256 89 and 24.
    const int Hkv = a.Hkv = a.kv[0].n, sms = device_sm_count();
    const int64_t each = q.N * 2 * Hkv, units = (int64_t)block * q.lanes;
    warps = units > kThreads && !block_append_small(q.N, Hkv) ? kWarps : 1;
    const int64_t room = (int64_t)sms * 16 / warps;
    a.chunk = (int)std::max<int64_t>(1, std::min<int64_t>(std::min(block, 4096), (each + room - 1) / room));
    const int64_t parts = (q.N + a.chunk - 1) / a.chunk;
    const int64_t jobs = parts * 2 * Hkv, job_ctas = warps == 1 ? (jobs + kWarps - 1) / kWarps : jobs;
    blocks = job_ctas;
    if (q.h[0].n) {   // the queries: as in rope_append_kernel, two rows a turn
        const int rows = 32 / q.lanes, steps = (q.h[0].n + 2 * rows - 1) / (2 * rows);
        a.q.parts = (int)std::max<int64_t>(1, std::min<int64_t>(steps, ((int64_t)sms * 32 + q.N - 1) / q.N));
        blocks += (q.N * a.q.parts + kWarps - 1) / kWarps;
    }
    if (blocks > INT32_MAX || jobs > INT32_MAX) return set_error(WS_ERR_UNSUPPORTED, "rope_append: too many tokens");
    a.jobs = (uint32_t)jobs;
    // CTA b is the n-th for jobs where n = floor(b rate / 2^32) is below floor((b + 1) rate / 2^32)
    a.all_jobs = job_ctas == blocks;
    a.job_rate = a.all_jobs ? 0 : (uint32_t)((((uint64_t)job_ctas << 32) + blocks - 1) / blocks);
    return WS_OK;
}

}  // namespace

int block_append_check(const RopeAppendArgs& q, int block) {
    BlockAppendArgs a;
    int warps;
    int64_t blocks;
    return plan(q, block, a, warps, blocks);
}

int block_append_launch(const RopeAppendArgs& q, bool f16, bool e4m3, bool vec, int block, cudaStream_t st) {
    BlockAppendArgs a;
    int warps;
    int64_t blocks;
    if (const int rc = plan(q, block, a, warps, blocks)) return rc;
    auto pick = [&](auto half, auto eight) {
        constexpr bool F = decltype(half)::value, E = decltype(eight)::value;
        if (warps == 1) return vec ? block_append_kernel<F, E, true, 1> : block_append_kernel<F, E, false, 1>;
        return vec ? block_append_kernel<F, E, true, kWarps> : block_append_kernel<F, E, false, kWarps>;
    };
    using yes = std::true_type;
    using no = std::false_type;
    auto fn = f16 ? (e4m3 ? pick(yes{}, yes{}) : pick(yes{}, no{})) : (e4m3 ? pick(no{}, yes{}) : pick(no{}, no{}));
    const cudaError_t e = launch_dependent(fn, dim3((unsigned)blocks), kThreads, kHeld * kThreads * (64 + 4), st, a);
    return e == cudaSuccess ? WS_OK : set_error(WS_ERR_CUDA, cudaGetErrorString(e));
}

}  // namespace ws
