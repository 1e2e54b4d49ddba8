// exl3c4_route.hip -- the routing around the routed-expert ops, on gfx950 (wave64): the router (softmax over all logits, top_k,
// renormalisation), moe_scatter (a stable counting sort of the flat (token, slot) pairs by expert) and moe_gather (each token's
// slots weighted and summed in f32, ascending slot order, cast to f16); and moe_route, the router by scores, with a bias and
// groups. The contract of the first three is radiance's (include/exl3_abi.h:90-158; the scatter as
// tests/ref/exl3_numpy.py:223-242 states it); the reference device library leaves these to its engine.
#include <hip/hip_runtime.h>

#include <float.h>
#include <math.h>
#include <stdint.h>

#include "exl3c4_dev.h"
#include "exl3c4_wave.h"

namespace {

// f32 -> f16 bits, round to nearest even; the register fence keeps the conversion a conversion (not folded into the
// instruction that produced v).
__device__ __forceinline__ uint16_t to_f16(float v) {
    asm volatile("" : "+v"(v));
    return __builtin_bit_cast(uint16_t, (_Float16)v);
}

// The router's ranking as one unsigned 64-bit key a (logit, id): a larger key ranks first. The high word orders the
// logits (the sign-magnitude bits turned into an unsigned order; -0 taken as +0; a NaN below every number), the low
// word the ids (a lower id ranks first among equal logits).
__device__ __forceinline__ uint64_t rank_key(float l, int e) {
    uint32_t k = 0u;                                           // NaN
    if (l == l) {
        const uint32_t u = __float_as_uint(l == 0.f ? 0.f : l);
        k = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    }
    return ((uint64_t)k << 32) | (uint64_t)(0xFFFFFFFFu - (uint32_t)e);
}
__device__ __forceinline__ float key_logit(uint64_t key) {
    const uint32_t k = (uint32_t)(key >> 32);
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

// The router for one token, by one wave: m = max logit; s = the sum of expf(l - m) (each lane over its ids e = lane +
// 64 j in ascending j, then a butterfly over the lanes); the top_k rank keys; p = expf(l - m) / s, renormalised by the
// sum of the top_k p (in rank order) when asked. The token's logits sit in registers (RPL a lane, ids e = lane + 64 j),
// all loaded at once. Lane r < top_k ends holding the r-th ranked id and its weight. cand: 64 keys of LDS.
struct Pick { int id; float w; };
__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int d) {
    return ((uint64_t)(uint32_t)__shfl_xor((int)(v >> 32), d) << 32) | (uint64_t)(uint32_t)__shfl_xor((int)(uint32_t)v, d);
}
// The value of lane l ^ J, without the LDS pipe's bpermute: DPP moves for J = 1, 2 (quad_perm) and 8 (row_ror 8), two
// for 4 (row_half_mirror is ^ 7, quad_perm ^ 3), gfx950's permlane swaps for 16 and 32 (each lane takes the half of
// the swapped pair that came from its partner). Every lane of the wave must be active.
template <int J> __device__ __forceinline__ uint32_t xor_lane(uint32_t v, int lane) {
    if constexpr (J == 1) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, false);
    else if constexpr (J == 2) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, false);
    else if constexpr (J == 4)
        return (uint32_t)__builtin_amdgcn_mov_dpp(__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, false), 0x1B, 0xF, 0xF, false);
    else if constexpr (J == 8) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x128, 0xF, 0xF, false);
    else if constexpr (J == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return (lane & 16) ? r[0] : r[1];
    } else {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return (lane & 32) ? r[0] : r[1];
    }
}
template <int J> __device__ __forceinline__ uint64_t xor_lane64(uint64_t v, int lane) {
    return ((uint64_t)xor_lane<J>((uint32_t)(v >> 32), lane) << 32) | (uint64_t)xor_lane<J>((uint32_t)v, lane);
}
template <int J> __device__ __forceinline__ float xor_lanef(float v, int lane) {
    return __uint_as_float(xor_lane<J>(__float_as_uint(v), lane));
}
__device__ __forceinline__ uint64_t readlane64(uint64_t v, int l) {
    return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32) |
           (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, l);
}
__device__ __forceinline__ uint32_t xor_lane_rt(uint32_t v, int j, int lane) {   // j a power of two <= 32
    switch (j) {
    case 1: return xor_lane<1>(v, lane);
    case 2: return xor_lane<2>(v, lane);
    case 4: return xor_lane<4>(v, lane);
    case 8: return xor_lane<8>(v, lane);
    case 16: return xor_lane<16>(v, lane);
    default: return xor_lane<32>(v, lane);
    }
}

// A bitonic sort of one u32 a lane across the wave, descending: lane 0 ends with the largest.
__device__ __forceinline__ uint32_t sort_desc32(uint32_t v, int lane) {
#pragma unroll
    for (int k = 2; k <= 64; k <<= 1)
#pragma unroll
        for (int j = k >> 1; j > 0; j >>= 1) {
            const uint32_t o = xor_lane_rt(v, j, lane);          // j is a constant once unrolled
            const bool take_max = ((lane & j) == 0) == ((lane & k) == 0);
            v = take_max ? max(o, v) : min(o, v);
        }
    return v;
}

template <int DT, int RPL>                                      // RPL logits a lane: n_expert <= 64 RPL
__device__ __forceinline__ Pick route_token(const void* logits, int64_t row, int32_t n_expert, int32_t top_k,
                                            int32_t renorm, int lane, uint64_t* cand) {
    float v[RPL];
    if (DT == EXL3C4_F32) {
        const float* p = (const float*)logits + row;
#pragma unroll
        for (int j = 0; j < RPL; ++j) v[j] = lane + 64 * j < n_expert ? p[lane + 64 * j] : -INFINITY;
    } else {
        const uint16_t* p = (const uint16_t*)logits + row;
        uint16_t b[RPL];
#pragma unroll
        for (int j = 0; j < RPL; ++j) b[j] = lane + 64 * j < n_expert ? p[lane + 64 * j] : (uint16_t)0xFC00u;
#pragma unroll
        for (int j = 0; j < RPL; ++j)
            v[j] = DT == EXL3C4_BF16 ? __uint_as_float((uint32_t)b[j] << 16) : (float)__builtin_bit_cast(_Float16, b[j]);
        if (DT == EXL3C4_BF16)
#pragma unroll
            for (int j = 0; j < RPL; ++j)
                if (lane + 64 * j >= n_expert) v[j] = -INFINITY;
    }
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < RPL; ++j) m = fmaxf(m, v[j]);              // a NaN never wins
    m = fmaxf(m, xor_lanef<32>(m, lane));
    m = fmaxf(m, xor_lanef<16>(m, lane));
    m = fmaxf(m, xor_lanef<8>(m, lane));
    m = fmaxf(m, xor_lanef<4>(m, lane));
    m = fmaxf(m, xor_lanef<2>(m, lane));
    m = fmaxf(m, xor_lanef<1>(m, lane));
    float s = 0.f;
    uint64_t key[RPL];
#pragma unroll
    for (int j = 0; j < RPL; ++j) {
        const bool in = lane + 64 * j < n_expert;
        s = s + (in ? expf(v[j] - m) : 0.f);
        key[j] = in ? rank_key(v[j], lane + 64 * j) : 0ull;     // 0: below every real key
    }
    s = s + xor_lanef<32>(s, lane);                               // the butterfly, partners 32, 16, .., 1
    s = s + xor_lanef<16>(s, lane);
    s = s + xor_lanef<8>(s, lane);
    s = s + xor_lanef<4>(s, lane);
    s = s + xor_lanef<2>(s, lane);
    s = s + xor_lanef<1>(s, lane);

    // The top_k keys all have a logit word of at least thr, the top_k-th largest logit word of the lanes' own largest
    // keys (top_k lanes hold a key that large; the logit word orders the keys, so a 32-bit sort finds it). Those
    // candidates -- at most 64 on this path -- are gathered one a lane and ranked; lane r then holds the r-th ranked
    // key. More than 64 (many equal logits in few lanes) take top_k rounds of a wave maximum.
    uint64_t lm = 0ull;
#pragma unroll
    for (int j = 0; j < RPL; ++j) lm = key[j] > lm ? key[j] : lm;
    const uint32_t thr = (uint32_t)__builtin_amdgcn_readlane((int)sort_desc32((uint32_t)(lm >> 32), lane), top_k - 1);
    int n = 0;
#pragma unroll
    for (int j = 0; j < RPL; ++j) {
        const bool c = key[j] != 0ull && (uint32_t)(key[j] >> 32) >= thr;
        const uint64_t bal = __ballot(c);
        const int at = n + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(bal >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)bal, 0));
        if (c && at < 64) cand[at] = key[j];
        n += __popcll(bal);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    uint64_t mykey = 0ull;
    if (n <= 64) {
        // the candidates ranked (keys are distinct: the id is in the low bits), then placed by rank: lane r ends with
        // the r-th largest. n rounds of independent compares instead of a 64-lane sort's 21 dependent stages.
        const uint64_t ck = lane < n ? cand[lane] : 0ull;
        int rank = 0;
        for (int c = 0; c < n; ++c) rank += readlane64(ck, c) > ck ? 1 : 0;
        if (lane < n) cand[rank] = ck;                            // this wave's row alone: its LDS ops run in order
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        mykey = lane < n ? cand[lane] : 0ull;
    } else {
        uint64_t prev = ~0ull;
        for (int r = 0; r < top_k; ++r) {
            uint64_t best = 0ull;
#pragma unroll
            for (int j = 0; j < RPL; ++j) best = (key[j] < prev && key[j] > best) ? key[j] : best;
#pragma unroll
            for (int d = 32; d >= 1; d >>= 1) {
                const uint64_t o = shfl_xor64(best, d);
                best = o > best ? o : best;
            }
            prev = best;
            if (lane == r) mykey = best;
        }
    }
    const float p = lane < top_k ? expf(key_logit(mykey) - m) / s : 0.f;
    float psum = 0.f;
    for (int r = 0; r < top_k; ++r) psum = psum + __builtin_bit_cast(float, __builtin_amdgcn_readlane(__float_as_int(p), r));   // rank order
    return Pick{ (int)(0xFFFFFFFFu - (uint32_t)mykey), renorm ? p / psum : p };
}

// The router, one wave a token (n_expert <= 1024).
template <int DT, int RPL>
__global__ __launch_bounds__(256) void k_router(const void* logits, int64_t n_tok, int32_t n_expert, int64_t pitch,
                                                int32_t top_k, int32_t renorm, int32_t* ids, float* w) {
    const int lane = threadIdx.x & 63;
    const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    __shared__ uint64_t cand[4][64];
    if (t >= n_tok) return;
    const Pick p = route_token<DT, RPL>(logits, t * pitch, n_expert, top_k, renorm, lane, cand[threadIdx.x >> 6]);
    if (lane < top_k) {
        ids[t * top_k + lane] = p.id;
        w[t * top_k + lane] = p.w;
    }
}

// moe_scatter over many workgroups without a workspace: each of them counts every pair's expert for itself, in LDS (the
// ids come from L2 after the first read), apart for the pairs before its segment and for the others; the totals'
// exclusive scan is expert_offset, and the offset plus the count before the segment is each expert's first row in it.
// The segment is then placed SC_SEG pairs at a time: a pair's rank is the number of earlier pairs of the same expert
// among them, counted by comparing ids held in LDS (wave w compares its 64 pairs with the 64 of quarter w / 4, those
// before its own whole). Stable by construction: no order depends on the atomics, which only count.
// What bounds it: a workgroup's chain -- three rounds of id loads, 40 LDS atomics a thread and two scans at 40,960
// pairs -- so the time is nearly one workgroup's, however many run: 800 us in one workgroup of 8 waves before (its ranks
// by readlane sweeps over every pair, twice), 14 us now, 401 -> 11 us at 20,480 pairs, 29 -> 6 at 1,280.
// LOADS: a thread's id loads in a round, no more than the pairs need (16 waves of which most load a copy of the last id
// issue for longer than the few pairs take), as waves without a pair rank none. 1 / 80 / 320 / 1,280 pairs over 512
// experts, us a launch of a chain of them: 4.76 / 4.90 / 4.87 / 5.28 with sixteen loads always, 2.50 / 3.69 / 4.31 / 4.69
// now; the single workgroup before took 3.28 / 4.83 / 9.11 / 27.8.
// A base that 32 bits hold (FAR: another one) lets a pair's expert be found in them: 81,920 pairs over 512 experts 18.1 -> 16 us; with
// their ids by 16-byte loads 13.2.
constexpr int SC_THREADS = 1024, SC_SEG = 256, SC_MAX_WG = 256;
template <bool FAR> __device__ __forceinline__ int expert_of(int32_t id, int64_t base, int n_expert) {
    if constexpr (FAR) {
        const int64_t g = (int64_t)id - base;
        return (g >= 0 && g < n_expert) ? (int)g : -1;
    } else {
        const uint32_t g = (uint32_t)id - (uint32_t)base;
        return id >= (int32_t)base && g < (uint32_t)n_expert ? (int)g : -1;
    }
}

template <int LOADS, bool FAR>
__global__ __launch_bounds__(SC_THREADS) void k_scatter(const int32_t* ids, uint32_t T, int64_t base, int32_t n_expert,
                                                        uint32_t seg, int32_t* sorted, int32_t* off, int32_t* count,
                                                        int32_t* row_of) {
    __shared__ int hist[2 * SC_THREADS];                          // counts before the segment; from it on
    __shared__ int wsum[SC_THREADS / 64];
    __shared__ __attribute__((aligned(16))) int eid[SC_SEG];
    __shared__ int rank_l[SC_SEG];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const uint32_t lo = blockIdx.x * seg, hi = T - lo < seg ? T : lo + seg;   // T < 2^31: nothing wraps
    const int mine = tid < SC_SEG && lo + tid < hi ? ids[lo + tid] : 0;   // the first SC_SEG pairs, loaded ahead
    hist[tid] = hist[SC_THREADS + tid] = 0;
    __syncthreads();
    uint32_t counted = 0;
    if constexpr (LOADS == 16) {
        // whole rounds of four ids a thread, four rounds' loads out together; a wave's 256 ids lie before the segment or not
        // (it starts at a multiple)
        struct __attribute__((packed, aligned(4))) Four { int32_t v[4]; };
        constexpr uint32_t ROUND = 4 * SC_THREADS;
        auto count = [&](const Four& q, uint32_t i0) {
            int* h = hist + (__builtin_amdgcn_readfirstlane(i0 + 256 * wv) < lo ? 0 : SC_THREADS);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int e = expert_of<FAR>(q.v[j], base, n_expert);
                if (e >= 0) atomicAdd(&h[e], 1);
            }
        };
        for (; counted + 4 * ROUND <= T; counted += 4 * ROUND) {
            Four q[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) q[r] = *(const Four*)(ids + counted + r * ROUND + 4 * tid);
#pragma unroll
            for (int r = 0; r < 4; ++r) count(q[r], counted + r * ROUND);
        }
    }
    for (uint32_t i0 = counted; i0 < T; i0 += SC_THREADS * LOADS) {
        int32_t f[LOADS];
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const uint32_t i = i0 + SC_THREADS * j + tid;
            f[j] = ids[i < T ? i : T - 1];
        }
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const uint32_t i = i0 + SC_THREADS * j + tid;
            const int e = i < T ? expert_of<FAR>(f[j], base, n_expert) : -1;
            if (e >= 0) atomicAdd(&hist[(i < lo ? 0 : SC_THREADS) + e], 1);
        }
    }
    __syncthreads();
    const int tot = hist[tid] + hist[SC_THREADS + tid];           // 0 past n_expert
    const int incl = wave_scan_incl(tot);
    if (lane == 63) wsum[wv] = incl;
    __syncthreads();
    const int pre = wave_scan_incl(lane < SC_THREADS / 64 ? wsum[lane] : 0);
    const int ex = (wv ? __builtin_amdgcn_readlane(pre, wv - 1) : 0) + incl - tot;
    const uint32_t live = (uint32_t)__builtin_amdgcn_readlane(pre, SC_THREADS / 64 - 1);
    hist[tid] += ex;                                              // expert tid's first row in this segment
    if (blockIdx.x == 0) {
        if (tid < n_expert) {
            off[tid] = ex;
            if (count) count[tid] = tot;
        }
        if (tid == 0) off[n_expert] = (int32_t)live;
    }
    for (uint32_t c0 = lo; c0 < hi; c0 += SC_SEG) {               // uniform
        const uint32_t i = c0 + tid;
        int e = -1;
        if (tid < SC_SEG) {
            if (i < hi) e = expert_of<FAR>(c0 == lo ? mine : ids[i], base, n_expert);
            eid[tid] = e;
            rank_l[tid] = 0;
        }
        __syncthreads();
        const int blk = wv & 3, part = wv >> 2;                   // SC_SEG / 64 of each
        if (part <= blk && c0 + blk * 64 < hi) {                  // uniform in the wave, like the loop's end
            const int own = eid[blk * 64 + lane];
            const int upto = part < blk ? 64 : lane;
            const int n = hi - c0 - part * 64 < 64 ? (int)(hi - c0) - part * 64 : 64;
            int r = 0;
#pragma unroll 4
            for (int j = 0; j < n; j += 4) {
                const int4 q = *(const int4*)&eid[part * 64 + j];
                r += (q.x == own && j < upto) + (q.y == own && j + 1 < upto) + (q.z == own && j + 2 < upto) +
                     (q.w == own && j + 3 < upto);
            }
            if (r) atomicAdd(&rank_l[blk * 64 + lane], r);
        }
        __syncthreads();
        int pos = -1;
        if (e >= 0) {
            pos = hist[e] + rank_l[tid];
            sorted[pos] = (int32_t)i;
        }
        if (row_of && tid < SC_SEG && i < hi) row_of[i] = pos;
        __syncthreads();                                          // every row read before the next pairs' counts
        if (e >= 0) atomicAdd(&hist[e], 1);
    }
    for (uint32_t i = live + blockIdx.x * SC_THREADS + tid; i < T; i += gridDim.x * SC_THREADS) sorted[i] = -1;
}

// moe_scatter by experts: a workgroup takes PO_EXPERTS or fewer neighbouring experts and reads every pair's id, each wave a
// part of the pairs. It counts the pairs of lower experts, whose sum is its first row, and lists its own in LDS in their order;
// what the waves before it found then places each. Three instructions an id (two comparisons and a count) in place of an LDS
// atomic, and no ranks among the pairs of a segment. What bounds it: every CU reads all ids, 3.8 us of L2's rate for 81,920
// pairs, and the same again goes into the pairs found.
// k_scatter / this, us a launch, pairs over experts evenly unless something is said:
//   512 experts     1 pair 2.8 / 3.2, 10 2.9 / 3.3, 80 3.9 / 3.5, 1,280 4.9 / 3.6, 6,130 6.3 / 4.2, 20,480 7.7 / 5.8, 81,920
//                   12.9 / 10.9, 200,000 28 / 22
//   8, 64 experts   32 pairs 3.2 / 3.3; 49,152 9.6 / 9.3
//   uneven          81,920 of 512: a fifth of them on one expert 21.6 / 19.4, all 75 / 54, Zipf in the order of the ids 21.4 /
//                   23.7, moe_route's choice of random tokens with a bias (0 to 2,468 an expert) 15.0 / 15.6; 200,000, a fifth
//                   on one 50 / 129: a list no longer holds a wave's own
//   no expert's     seven eighths of 81,920 of 64 12.5 / 13.1, of 65,536 of 32 9.4 / 11.7, of 131,072 of 8 31 / 93: few
//                   workgroups place, one fills the rest
constexpr uint32_t PO_LEAST = 33, PO_MOST = 1 << 17, PO_EACH = 1024;     // pairs that take it: from, up to, and how many an expert
constexpr int PO_THREADS = 1024, PO_WAVES = PO_THREADS / 64, PO_EXPERTS = 4, PO_LIST = 2048;
template <bool BASE>
__global__ __launch_bounds__(PO_THREADS) void k_pairs_by_expert(const int32_t* ids, uint32_t T, int32_t base, int32_t n_expert,
                                                                uint32_t per, uint32_t seg, int32_t* sorted, int32_t* off,
                                                                int32_t* count, int32_t* row_of) {
    __shared__ int tot[PO_WAVES][PO_EXPERTS + 1];                 // a wave's pairs of each own expert, and of lower ones
    __shared__ uint16_t list[PO_WAVES][PO_LIST];                  // its own pairs in order, from its part's first on: 4 pair + expert
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t first = blockIdx.x * per, n = min(per, (uint32_t)n_expert - first);
    // the pairs that no expert has, in the workgroup's segment
    if (row_of) {
        const uint32_t lo = blockIdx.x * seg, hi = lo >= T ? lo : T - lo < seg ? T : lo + seg;
        for (uint32_t i = lo + tid; i < hi; i += PO_THREADS)
            if ((uint32_t)ids[i] - (uint32_t)base >= (uint32_t)n_expert) row_of[i] = -1;
    }
    const uint32_t part = ((T + PO_WAVES - 1) / PO_WAVES + 255) / 256 * 256, from = min(T, wv * part), to = min(T, from + part);
    struct __attribute__((packed, aligned(4))) Four { uint32_t v[4]; };
    constexpr uint32_t NONE = 0x80000000u;                        // (no id less the base: both are far from 2^31)
    auto load = [&](uint32_t i) {
        Four q = { { NONE, NONE, NONE, NONE } };
        if (i + 4 <= to) {
            q = *(const Four*)(ids + i);
            if (BASE)
#pragma unroll
                for (int j = 0; j < 4; ++j) q.v[j] -= (uint32_t)base;
        } else {
#pragma unroll
            for (int j = 0; j < 3; ++j)
                if (i + j < to) q.v[j] = (uint32_t)ids[i + j] - (uint32_t)base;
        }
        return q;
    };
    int below = 0;
    uint32_t listed = 0;
    auto look = [&](const Four& q, uint32_t i) {
        uint64_t hit[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint64_t lower = __ballot(q.v[j] < first);
            hit[j] = __ballot(q.v[j] < first + n) & ~lower;
            below += q.v[j] < first ? 1 : 0;
        }
        if ((hit[0] | hit[1] | hit[2] | hit[3]) == 0) return;
        uint32_t at = listed;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            at = __builtin_amdgcn_mbcnt_hi((uint32_t)(hit[j] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)hit[j], at));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (hit[j] == 0) continue;                            // (uniform)
            if (q.v[j] - first < n) {
                if (at < PO_LIST) list[wv][at] = (uint16_t)(4 * (i - from + j) + q.v[j] - first);
                ++at;
            }
            listed += (uint32_t)__popcll(hit[j]);
        }
    };
    uint32_t i0 = from;
    for (; i0 + 1024 <= to; i0 += 1024) {                         // four rounds' loads out together
        Four q[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) q[r] = load(i0 + 256 * r + 4 * lane);
#pragma unroll
        for (int r = 0; r < 4; ++r) look(q[r], i0 + 256 * r + 4 * lane);
    }
    for (; i0 < to; i0 += 256) look(load(i0 + 4 * lane), i0 + 4 * lane);
    wave_sync();                                                  // the list is read by other lanes than wrote it
    below = wave_scan_incl(below);
    // f(x, pair) for 64 of the own pairs in order, one a lane (x: its expert of these, or PO_EXPERTS for none)
    auto each = [&](auto f) {
        if (listed <= PO_LIST) {
            for (uint32_t k = 0; k < listed; k += 64) {
                const uint32_t v = k + lane < listed ? list[wv][k + lane] : 0u;
                f(k + lane < listed ? v & 3 : PO_EXPERTS, from + (v >> 2));
            }
        } else {                                                  // too many: the ids again
            for (uint32_t i = from; i < to; i += 512) {
                uint32_t x[8];
#pragma unroll
                for (int r = 0; r < 8; ++r) x[r] = i + 64 * r + lane < to ? (uint32_t)ids[i + 64 * r + lane] - (uint32_t)base - first : NONE;
#pragma unroll 1
                for (int r = 0; r < 8; ++r) {
                    f(x[0] < n ? x[0] : PO_EXPERTS, i + 64 * r + lane);
#pragma unroll
                    for (int u = 0; u < 7; ++u) x[u] = x[u + 1];
                }
            }
        }
    };
    int own[PO_EXPERTS] = {};
    each([&](uint32_t x, uint32_t) {
#pragma unroll
        for (int e = 0; e < PO_EXPERTS; ++e)
            if (e < (int)n) own[e] += __popcll(__ballot(x == (uint32_t)e));
    });
    if (lane == 63) {
#pragma unroll
        for (int e = 0; e < PO_EXPERTS; ++e) tot[wv][e] = own[e];
        tot[wv][PO_EXPERTS] = below;
    }
    __syncthreads();
    // each expert's first row, and the wave's in it (lane w: wave w's counts)
    const int w16 = lane & (PO_WAVES - 1);
    int row = __builtin_amdgcn_readlane(wave_scan_incl(tot[w16][PO_EXPERTS]), PO_WAVES - 1), next[PO_EXPERTS];
#pragma unroll
    for (int e = 0; e < PO_EXPERTS; ++e) {
        const int c = tot[w16][e], incl = wave_scan_incl(c), all = __builtin_amdgcn_readlane(incl, PO_WAVES - 1);
        next[e] = row + __builtin_amdgcn_readlane(incl - c, wv);
        if (e < (int)n && tid == 0) {
            off[first + e] = row;
            if (count) count[first + e] = all;
        }
        row += all;
    }
    each([&](uint32_t x, uint32_t pair) {
        int pos = -1;
#pragma unroll
        for (int e = 0; e < PO_EXPERTS; ++e) {
            if (e >= (int)n) break;
            const uint64_t m = __ballot(x == (uint32_t)e);
            if (x == (uint32_t)e)
                pos = next[e] + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
            next[e] += __popcll(m);
        }
        if (pos >= 0) {
            sorted[pos] = (int32_t)pair;
            if (row_of) row_of[pair] = pos;
        }
    });
    if (first + n == (uint32_t)n_expert) {                        // the last workgroup: behind the last row
        if (tid == 0) off[n_expert] = row;
        for (uint32_t i = row + tid; i < T; i += PO_THREADS) sorted[i] = -1;
    }
}

// moe_scatter of the router's pairs (token t's top_k ids at t * top_k .., distinct experts, at most 32 tokens and
// blockDim.x pairs) for at most blockDim.x experts: each expert's set of tokens as a bit mask (LDS atomics), its count
// the mask's population; expert_offset the counts' exclusive scan (a DPP scan in each wave, then the waves' totals
// scanned the same way); pair (t, slot)'s row = offset of its expert + the number of earlier tokens holding that
// expert (the stable counting sort's row: a token holds an expert at most once, so the pairs of one expert are in
// token order). lds: n_expert + 1 + 16 ints, the first n_expert zeroed by the caller before a barrier.
__device__ __forceinline__ void scatter_small(const int32_t* ids_l, int T, int top_k, int n_expert, int32_t* sorted,
                                              int32_t* off, int32_t* count, int32_t* row_of, int* lds) {
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    int* cnt = lds;                                               // [n_expert]: token masks, then exclusive offsets
    int* wsum = lds + n_expert + 1;                               // [16]: the waves' totals
    int e = -1, w = 0;
    const int t = tid < T ? tid / top_k : 0;
    if (tid < T) {
        const int f = ids_l[tid];
        e = (f >= 0 && f < n_expert) ? f : -1;
        if (e >= 0) atomicOr((unsigned*)&cnt[e], 1u << t);
    }
    __syncthreads();
    const int c = tid < n_expert ? __popc((unsigned)cnt[tid]) : 0;
    if (e >= 0) w = __popc((unsigned)cnt[e] & ((1u << t) - 1u));  // read before any offset overwrites a mask
    const int incl = wave_scan_incl(c);                           // inclusive scan across the wave
    if (lane == 63) wsum[wv] = incl;
    __syncthreads();
    const int nw = (int)(blockDim.x >> 6);                        // the waves' totals, lane u holding wave u's,
    const int pre = wave_scan_incl(lane < nw ? wsum[lane] : 0);   // scanned across lanes (at most 16 waves)
    const int base = wv ? __builtin_amdgcn_readlane(pre, wv - 1) : 0, live = __builtin_amdgcn_readlane(pre, nw - 1);
    if (tid < n_expert) {
        const int ex = base + incl - c;
        off[tid] = ex;
        if (count) count[tid] = c;
        cnt[tid] = ex;                                            // every read of the masks lies before the barrier
    }
    if (tid == 0) off[n_expert] = live;
    __syncthreads();
    if (tid < T) {
        const int rank = e >= 0 ? cnt[e] + w : -1;
        if (e >= 0) sorted[rank] = tid;
        if (row_of) row_of[tid] = rank;
    }
    for (int i = live + tid; i < T; i += blockDim.x) sorted[i] = -1;
}

// router_topk_scatter (the two fused, as the contract names them, include/exl3_abi.h:96-98) for at most 16 tokens, in
// one workgroup of 16 waves: wave t routes token t, its ids go to LDS as well, then the scatter reads them there.
template <int DT, int RPL>
__global__ __launch_bounds__(1024) void k_route_scatter(const void* logits, int32_t n_tok, int32_t n_expert,
                                                        int64_t pitch, int32_t top_k, int32_t renorm, int32_t* ids,
                                                        float* w, int32_t* sorted, int32_t* off, int32_t* count,
                                                        int32_t* row_of) {
    extern __shared__ __attribute__((aligned(16))) int rs_lds[];   // ids first: 16-byte reads
    __shared__ uint64_t cand[16][64];
    int* ids_l = rs_lds;                                          // [16 * 64]
    int* cnt = rs_lds + 16 * 64;
    const int lane = threadIdx.x & 63, t = threadIdx.x >> 6;
    // 16 tokens of at most 64 slots and 1,024 experts at most (the entry's checks): scatter_small's bounds
    for (int i = threadIdx.x; i < n_expert; i += blockDim.x) cnt[i] = 0;   // zeroed while routing
    if (t < n_tok) {
        const Pick p = route_token<DT, RPL>(logits, (int64_t)t * pitch, n_expert, top_k, renorm, lane, cand[t]);
        if (lane < top_k) {
            ids[t * top_k + lane] = p.id;
            w[t * top_k + lane] = p.w;
            ids_l[t * top_k + lane] = p.id;
        }
    }
    __syncthreads();
    scatter_small(ids_l, n_tok * top_k, top_k, n_expert, sorted, off, count, row_of, cnt);
}

// ------------------------------------------------------------------------------------------ moe_route
// The order of experts and of groups is that of their values in 64 bits, for among thousands of tokens there are always experts
// whose values f32 would not tell apart. f32 finds who can be among the first (all within its error of them), f64 ranks those:
// one evaluation a lane. Groups whose place f32 leaves open, and more than 64 such experts, are evaluated in f64 as a whole.
// Weights come out of the f64 scores, rounded once.
// What bounds it: the VALU (86% busy), some 800 instructions a token of 512 experts: the scores 110, the order of the lanes'
// largest 110, the candidates' scores and ranks in f64 200. The groups' values are read from LDS with bank conflicts (lanes of
// all groups meet the same banks: 61% of LDS's cycles, which are 18% of all). 16 MiB of logits are 3.4 us.
// Alone, top-10 or top-8 with a bias, us:
//   8192 tokens      512 experts in 8 groups 13.3 (22 with f64 for every expert; 15.6 in the trace of a whole pass), 256
//                    experts in 8 10.4; 512 without groups, softmax 13.8
//   one token        4.9 with its scatter: latency
//   a group's place that f32 leaves open, in one token of some thousands: 613 tokens 5.4 without one, 7.4 with (13.3 with every
//   group in f64)
// e^x for x <= 0 (below -800: 0): x = n ln 2 + r with ln 2 in two parts (its first 37 bits, so that n times them is exact, and
// the rest), |r| <= ln 2 / 2, and the exponential series up to r^13, whose rest is below 2^-52 of e^r.
__device__ __forceinline__ double exp64(double x) {
    x = fmax(x, -800.0);
    constexpr double LN2_HI = 0x1.62e42fefap-1, LN2_LO = 0x1.cf79abc9e3b3ap-40;
    const double n = rint(x * 1.4426950408889634);
    double r = fma(n, -LN2_HI, x);
    r = fma(n, -LN2_LO, r);
    double p = 1.0 / 6227020800.0;
    p = fma(p, r, 1.0 / 479001600.0);
    p = fma(p, r, 1.0 / 39916800.0);
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return ldexp(p, (int)n);
}
// 1 / d for d in [2^-1000, 2^11]: the hardware's estimate (some 26 bits) and two steps of Newton's.
__device__ __forceinline__ double inverse64(double d) {
    double q = __builtin_amdgcn_rcp(d);
    q = fma(fma(-d, q, 1.0), q, q);
    return fma(fma(-d, q, 1.0), q, q);
}
__device__ __forceinline__ double sigmoid64(double l) {
    const double t = exp64(-fabs(l)), q = inverse64(1.0 + t);
    return l >= 0.0 ? q : t * q;
}
template <int J> __device__ __forceinline__ double xor_laned(double v, int lane) {
    return __builtin_bit_cast(double, xor_lane64<J>(__builtin_bit_cast(uint64_t, v), lane));
}
// The sum over a row of 16 lanes, and over all.
__device__ __forceinline__ double row_sum(double v, int lane) {
    v += xor_laned<8>(v, lane);
    v += xor_laned<4>(v, lane);
    v += xor_laned<2>(v, lane);
    return v + xor_laned<1>(v, lane);
}
__device__ __forceinline__ double wave_sum(double v, int lane) {
    v += xor_laned<32>(v, lane);
    return row_sum(v + xor_laned<16>(v, lane), lane);
}
// An order of doubles as unsigned numbers (-0 as +0); 0 stands for none.
__device__ __forceinline__ uint64_t order64(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v + 0.0);
    return u >> 63 ? ~u : u | (uint64_t)1 << 63;
}
__device__ __forceinline__ float logit(const Exl3c4DevRoute& a, int64_t at) {
    if (a.type == EXL3C4_F32) return ((const float*)a.logits)[at];
    const uint16_t b = ((const uint16_t*)a.logits)[at];
    return a.type == EXL3C4_BF16 ? __uint_as_float((uint32_t)b << 16) : (float)__builtin_bit_cast(_Float16, b);
}
__device__ __forceinline__ bool is_out(float v) { return !(v > -INFINITY); }       // -infinity or NaN

// What a token's experts are ranked by: softmax's largest logit and its sum's inverse.
struct Soft { float m; double inv; };
__device__ __forceinline__ double score64(const Exl3c4DevRoute& a, const Soft& sm, float l) {
    if (a.score == EXL3C4_SCORE_SIGMOID) return sigmoid64(l);
    return exp64(l == sm.m ? 0.0 : (double)l - (double)sm.m) * sm.inv;             // (infinity - infinity is none)
}
// An f32 score is within 2^-21 of its value: sigmoid's exponent, exponential, sum, reciprocal and product lose 5 steps of 2^-24
// together, softmax's (from f64 exponentials) 3. A choice is off by that and its own rounding; a sum of two by twice as much.
__device__ __forceinline__ float error_of(float c) { return 0x1p-21f + 0x1p-23f * fabsf(c); }
__device__ __forceinline__ float sigmoid32(float l) {
    const float t = __builtin_amdgcn_exp2f(fabsf(l) * -1.44269504088896340736f), q = __builtin_amdgcn_rcpf(1.f + t);
    return l >= 0.f ? q : t * q;
}
// The order of floats as unsigned numbers (-0 as +0); 0 stands for none, which a NaN is.
__device__ __forceinline__ uint32_t order32(float v) {
    const uint32_t u = __float_as_uint(v + 0.f);
    return v == v ? (u >> 31 ? ~u : u | 0x80000000u) : 0u;
}
__device__ __forceinline__ float value_of32(uint32_t k) { return __uint_as_float(k >> 31 ? k & 0x7FFFFFFFu : ~k); }

// An expert's choice in f64, its logit and bias read again (the rare paths: rolled, and without a hold on the registers of the others).
__device__ __forceinline__ double choice64(const Exl3c4DevRoute& a, const Soft& sm, int64_t row, int e, bool by_logit) {
    const float l = logit(a, row + e);
    return by_logit ? (double)l : score64(a, sm, l) + (a.bias ? (double)a.bias[e] : 0.0);
}
// Which `places` of the groups `of` stay, by f64 (bit g for group g).
__device__ __forceinline__ uint64_t groups64(const Exl3c4DevRoute& a, const Soft& sm, int64_t row, int lane, uint64_t of, int places) {
    uint64_t mine = 0;                                           // lane g: group g's value
#pragma unroll 1
    for (uint64_t left = of; left != 0; left &= left - 1) {
        const int g = __builtin_ctzll(left);
        double v1 = -INFINITY, v2 = -INFINITY;
#pragma unroll 1
        for (int i = lane; i < a.group; i += 64) {
            const int e = g * a.group + i;
            if (is_out(logit(a, row + e)) || (a.bias && is_out(a.bias[e]))) continue;
            const double v = choice64(a, sm, row, e, false);
            v2 = fmax(v2, fmin(v1, v));
            v1 = fmax(v1, v);
        }
#pragma unroll 1
        for (int d = 1; d < 64; d <<= 1) {
            const double o1 = __shfl_xor(v1, d), o2 = __shfl_xor(v2, d);
            v2 = fmax(fmax(v2, o2), fmin(v1, o1));
            v1 = fmax(v1, o1);
        }
        const double gv = a.group_score == EXL3C4_GROUP_TOP2 && v2 > -INFINITY ? v1 + v2 : v1;
        if (lane == g) mine = gv > -INFINITY ? order64(gv) : 0;
    }
    int ahead = 0;
#pragma unroll 1
    for (uint64_t left = of; left != 0; left &= left - 1) {
        const int q = __builtin_ctzll(left);
        const uint64_t o = readlane64(mine, q);
        ahead += o > mine || (o == mine && q < lane) ? 1 : 0;
    }
    return __ballot((of >> lane & 1) != 0 && ahead < places);
}

// A candidate's key, id, logit and bias; behind the ranking its id and score.
struct Cand { double s; float l, b; int id; };
// One token by one wave: the experts e = lane + 64 j in registers. Lane r < top_k ends with the r-th expert and its weight.
// cand: the wave's 64 places of LDS; value: its 64 RPL places (GROUPS).
template <int RPL, bool GROUPS>
__device__ __forceinline__ Pick score_token(const Exl3c4DevRoute& a, int64_t row, int lane, Cand* cand, float* value) {
    // (loads past the last expert repeat it: a mask for each load would cost as much as the score)
    float l[RPL], b[RPL];
    const int E = a.n_expert;
    int at[RPL];
#pragma unroll
    for (int j = 0; j < RPL; ++j) at[j] = j + 1 < RPL ? lane + 64 * j : min(lane + 64 * j, E - 1);
    if (RPL > 1 && E <= 64 * (RPL - 1))                          // more than the last of a lane's can be past it
#pragma unroll
        for (int j = 0; j < RPL; ++j) at[j] = min(lane + 64 * j, E - 1);
    if (a.type == EXL3C4_F32) {
        const float* p = (const float*)a.logits + row;
#pragma unroll
        for (int j = 0; j < RPL; ++j) l[j] = p[at[j]];
    } else {
        const uint16_t* p = (const uint16_t*)a.logits + row;
        uint16_t h[RPL];
#pragma unroll
        for (int j = 0; j < RPL; ++j) h[j] = p[at[j]];
#pragma unroll
        for (int j = 0; j < RPL; ++j)
            l[j] = a.type == EXL3C4_BF16 ? __uint_as_float((uint32_t)h[j] << 16) : (float)__builtin_bit_cast(_Float16, h[j]);
    }
    const bool biased = a.bias != nullptr, soft = a.score == EXL3C4_SCORE_SOFTMAX, top2 = GROUPS && a.group_score == EXL3C4_GROUP_TOP2;
#pragma unroll
    for (int j = 0; j < RPL; ++j) b[j] = 0.f;
    if (biased)
#pragma unroll
        for (int j = 0; j < RPL; ++j) b[j] = a.bias[at[j]];
    if (E < 64 * RPL)
#pragma unroll
        for (int j = 0; j < RPL; ++j)
            if (lane + 64 * j >= E) l[j] = -INFINITY;
    // s: the scores in f32, as far as something is ranked by them
    Soft sm = { 0.f, 1.0 };
    float s[RPL];
    if (soft) {
        sm.m = -INFINITY;
#pragma unroll
        for (int j = 0; j < RPL; ++j) sm.m = fmaxf(sm.m, l[j]);  // (a NaN never wins)
        sm.m = fmaxf(sm.m, xor_lanef<32>(sm.m, lane));
        sm.m = fmaxf(sm.m, xor_lanef<16>(sm.m, lane));
        sm.m = fmaxf(sm.m, xor_lanef<8>(sm.m, lane));
        sm.m = fmaxf(sm.m, xor_lanef<4>(sm.m, lane));
        sm.m = fmaxf(sm.m, xor_lanef<2>(sm.m, lane));
        sm.m = fmaxf(sm.m, xor_lanef<1>(sm.m, lane));
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < RPL; ++j) {
            const double e = is_out(l[j]) ? 0.0 : score64(a, sm, l[j]);
            s[j] = is_out(l[j]) ? __builtin_nanf("") : (float)e;
            sum += e;
        }
        sm.inv = inverse64(fmax(wave_sum(sum, lane), 1.0));        // (1 at least, but for a row that is out as a whole)
        const float inv = (float)sm.inv;
#pragma unroll
        for (int j = 0; j < RPL; ++j) s[j] *= inv;
    } else if (biased || top2) {
#pragma unroll
        for (int j = 0; j < RPL; ++j) s[j] = sigmoid32(l[j]);
    }
    // c: the choices, NaN for an expert that is out. Without a bias they are the logits, and f32 is exact.
    float c[RPL];
#pragma unroll
    for (int j = 0; j < RPL; ++j) {
        c[j] = biased ? s[j] + b[j] : l[j];                      // (NaN where l or b is, which fminf passes over)
        c[j] = fminf(l[j], b[j]) > -INFINITY ? c[j] : __builtin_nanf("");
    }
    if constexpr (GROUPS) {
        // the values by expert through LDS; then of 2^groups_log2 lanes, 64 >> groups_log2 times over, lane g finds group g's
        // two largest in a part of it
        const bool exact = !biased && !top2;
#pragma unroll
        for (int j = 0; j < RPL; ++j) value[lane + 64 * j] = c[j] != c[j] ? -INFINITY : biased || exact ? c[j] : s[j];
        wave_sync();
        const int g = lane & ((1 << a.groups_log2) - 1), parts = 64 >> a.groups_log2;
        float v1 = -INFINITY, v2 = -INFINITY;
        if (g < a.n_group)
            for (int i = lane >> a.groups_log2; i < a.group; i += parts) {
                const float v = value[g * a.group + i];
                v2 = fmaxf(v2, fminf(v1, v));
                v1 = fmaxf(v1, v);
            }
        wave_sync();                                             // read before the next token's values
        auto meet = [&](float o1, float o2) {
            v2 = fmaxf(fmaxf(v2, o2), fminf(v1, o1));
            v1 = fmaxf(v1, o1);
        };
        if (a.groups_log2 < 6) meet(xor_lanef<32>(v1, lane), xor_lanef<32>(v2, lane));
        if (a.groups_log2 < 5) meet(xor_lanef<16>(v1, lane), xor_lanef<16>(v2, lane));
        if (a.groups_log2 < 4) meet(xor_lanef<8>(v1, lane), xor_lanef<8>(v2, lane));
        if (a.groups_log2 < 3) meet(xor_lanef<4>(v1, lane), xor_lanef<4>(v2, lane));
        if (a.groups_log2 < 2) meet(xor_lanef<2>(v1, lane), xor_lanef<2>(v2, lane));
        // TOP2 by halves: two choices near f32's end, as masks by the type's lowest value are, leave f32 in their sum and not
        // in half of it. The value that is meant lies from lo to hi, by the group's own choices' errors (of a half sum: half of
        // both), the sum's rounding and these two's, so that a group of such choices leaves no other open (8192 tokens 34.6 ->
        // 13.2 us; of 64 groups, whose two ends each are read, 15.8 -> 17.0). A group without an expert is below all others,
        // whatever they are.
        const bool live = v1 > -INFINITY, two = top2 && v2 > -INFINITY;
        const float gv = top2 ? 0.5f * v1 + (two ? 0.5f * v2 : 0.f) : v1, err = error_of(v1) + (two ? 0x1p-23f * fabsf(v2) : 0.f);
        const float hi = live ? gv + err : -INFINITY, lo = !live || gv == INFINITY ? gv : fmaxf(gv - err, -FLT_MAX);
        int ahead = 0, beside = 0;                               // groups ahead for sure; ahead or too close to tell (its own among them)
        if (exact) {
            for (int q = 0; q < a.n_group; ++q) {
                const float o = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(gv), q));
                ahead += o > gv || (o == gv && q < g) ? 1 : 0;
            }
        } else {
            // (by twos: a lane past an odd last group is one without experts)
            for (int q = 0; q < a.n_group; q += 2)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    ahead += __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(lo), q + u)) > hi ? 1 : 0;
                    beside += __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(hi), q + u)) >= lo ? 1 : 0;
                }
            // those without an expert come last, by number; a single one that is certain has itself beside it
            if (!live) {
                for (int q = 0; q < g; ++q) ahead += __builtin_amdgcn_readlane(__float_as_uint(hi), q) == __float_as_uint(-INFINITY) ? 1 : 0;
                beside = ahead + 1;
            }
        }
        uint64_t stay = __ballot(lane < a.n_group && ahead < a.top_group);   // bit g: group g
        if (!exact) {                                            // (two groups or so, of one token in some thousands)
            const uint64_t open = __ballot(lane < a.n_group && ahead < a.top_group && beside > a.top_group);
            stay &= ~open;
            if (open != 0) stay |= groups64(a, sm, row, lane, open, a.top_group - __popcll(stay));
        }
#pragma unroll
        for (int j = 0; j < RPL; ++j) {
            const uint32_t of = (uint32_t)(lane + 64 * j) * a.group_inv >> 20;     // the expert's group (past the last expert: c is NaN)
            const uint32_t word = a.n_group > 32 && of > 31 ? (uint32_t)(stay >> 32) : (uint32_t)stay;
            if (!((word >> (of & 31)) & 1)) c[j] = __builtin_nanf("");
        }
    }
    // At least top_k experts have a choice of thr, the top_k-th largest of the lanes' own largest. Whoever is among the first
    // top_k is so by less than twice the error below it: those are gathered one a lane and ranked in f64, equal ones by id;
    // more than 64 of them by top_k rounds of a wave maximum.
    float most = c[0];
#pragma unroll
    for (int j = 1; j < RPL; ++j) most = fmaxf(most, c[j]);
    const uint32_t kth = (uint32_t)__builtin_amdgcn_readlane((int)sort_desc32(order32(most), lane), a.top_k - 1);
    float thr = kth ? value_of32(kth) : -INFINITY;
    if (biased && thr < INFINITY && kth) thr -= 2.f * error_of(thr) + 0x1p-22f * fabsf(thr);        // (and the subtraction's own rounding)
    int n = 0;
#pragma unroll
    for (int j = 0; j < RPL; ++j) {
        const bool in = c[j] >= thr;
        const uint64_t bal = __ballot(in);
        const int at = n + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(bal >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)bal, 0));
        if (in && at < 64) cand[at].l = l[j], cand[at].b = b[j], cand[at].id = lane + 64 * j;
        n += __popcll(bal);
    }
    wave_sync();
    int mine = -1;
    double w = 0.0;
    if (n <= 64) {
        Cand own = { 0.0, 0.f, 0.f, 0x7FFFFFFF };
        uint64_t ck = 0;
        if (lane < n) {
            own = cand[lane];
            own.s = score64(a, sm, own.l);
            ck = order64(biased ? own.s + (double)own.b : (double)own.l);
        }
        int rank = 0;
        for (int q = 0; q < n; ++q) rank += readlane64(ck, q) > ck ? 1 : 0;
        wave_sync();
        if (lane < n) cand[rank].s = own.s, cand[rank].id = own.id;
        wave_sync();
        if (__any(lane < n && cand[rank].id != own.id)) {        // equal keys wrote one place: in the candidates' order, which is the ids'
            for (int q = 0; q < n; ++q) rank += readlane64(ck, q) == ck && q < lane ? 1 : 0;
            wave_sync();
            if (lane < n) cand[rank].s = own.s, cand[rank].id = own.id;
            wave_sync();
        }
        if (lane < n && lane < a.top_k) mine = cand[lane].id, w = cand[lane].s;
    } else {
        uint32_t in = 0;                                         // which of the lane's experts can be chosen
#pragma unroll
        for (int j = 0; j < RPL; ++j) in |= (c[j] == c[j] ? 1u : 0u) << j;
        uint64_t last = ~(uint64_t)0;
        int last_id = -1;
#pragma unroll 1
        for (int r = 0; r < a.top_k; ++r) {
            uint64_t best = 0;
            int at = 0x7FFFFFFF;                                 // (ids ascend with j: the first of equal keys is the lowest)
#pragma unroll 1
            for (int j = 0; j < RPL; ++j) {
                const int e = lane + 64 * j;
                const uint64_t k = in >> j & 1 ? order64(choice64(a, sm, row, e, !biased)) : 0;
                if ((k < last || (k == last && e > last_id)) && k > best) best = k, at = e;
            }
#pragma unroll 1
            for (int d = 32; d >= 1; d >>= 1) {
                const uint64_t o = shfl_xor64(best, d);
                const int oe = __shfl_xor(at, d);
                if (o > best || (o == best && oe < at)) best = o, at = oe;
            }
            last = best;
            last_id = at;
            if (lane == r && best != 0) mine = at;
        }
        if (mine >= 0) w = score64(a, sm, logit(a, row + mine));
    }
    wave_sync();                                                 // read before the next token's
    if (a.renorm) {
        const double sum = a.top_k > 16 ? wave_sum(w, lane) : row_sum(w, lane);
        // (an f64 division is some 30 instructions; the reciprocal of a number below 2^-1000 may not be one)
        if (__any(lane < a.top_k && !(sum > 0x1p-1000))) w = sum > 0.0 ? w / sum : 0.0;
        else w *= inverse64(sum);
    }
    return Pick{ mine, (float)(w * (double)a.scale) };
}

// A wave a token.
template <int RPL, bool GROUPS>
__global__ __launch_bounds__(256) void k_score(Exl3c4DevRoute a) {
    __shared__ Cand cand[4][64];
    __shared__ float value[4][GROUPS ? 64 * RPL : 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t t = (int64_t)blockIdx.x * 4 + wave;
    if (t >= a.n_tok) return;
    const Pick p = score_token<RPL, GROUPS>(a, t * a.pitch, lane, cand[wave], value[wave]);
    if (lane < a.top_k) {
        a.ids[t * a.top_k + lane] = p.id;
        a.w[t * a.top_k + lane] = p.w;
    }
}

// With the scatter, for at most 16 tokens, in one workgroup (as k_route_scatter).
template <int RPL, bool GROUPS>
__global__ __launch_bounds__(1024) void k_score_scatter(Exl3c4DevRoute a) {
    __shared__ Cand cand[16][64];
    __shared__ float value[16][GROUPS ? 64 * RPL : 1];
    __shared__ int ids_l[16 * 64], cnt[64 * RPL + 17];
    const int lane = threadIdx.x & 63, t = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < a.n_expert; i += blockDim.x) cnt[i] = 0;
    if (t < a.n_tok) {
        const Pick p = score_token<RPL, GROUPS>(a, (int64_t)t * a.pitch, lane, cand[t], value[t]);
        if (lane < a.top_k) {
            a.ids[t * a.top_k + lane] = p.id;
            a.w[t * a.top_k + lane] = p.w;
            ids_l[t * a.top_k + lane] = p.id;
        }
    }
    __syncthreads();
    scatter_small(ids_l, (int)a.n_tok * a.top_k, a.top_k, a.n_expert, a.sorted, a.off, a.count, a.row_of, cnt);
}

// moe_gather: one thread a run of 8 columns of one token; the slots in ascending order, one f32 product and one add
// each, then f16. The rows and weights of 8 slots are read together, then their rows' values.
__global__ __launch_bounds__(256) void k_gather(const void* y, int32_t y_dtype, int64_t y_pitch, const float* w,
                                                const int32_t* row_of, int64_t n_tok, int32_t top_k, int64_t cols,
                                                uint16_t* out, int64_t out_pitch) {
    const int64_t t = blockIdx.x;
    const int64_t c = ((int64_t)blockIdx.y * 256 + threadIdx.x) * 8;
    if (t >= n_tok || c >= cols) return;
    float acc[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = 0.f;
    for (int s0 = 0; s0 < top_k; s0 += 8) {                      // (every load unconditional: no branches)
        int32_t r[8];
        float ws[8];
        uint4 q[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int sl = s0 + u < top_k ? s0 + u : top_k - 1;
            r[u] = row_of[t * top_k + sl];
            ws[u] = w[t * top_k + sl];
            if (s0 + u >= top_k) r[u] = -1;
        }
#pragma unroll
        for (int u = 0; u < 8; ++u)
            q[u] = *(const uint4*)((const uint16_t*)y + (int64_t)(r[u] < 0 ? 0 : r[u]) * y_pitch + c);
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const uint32_t h[4] = { q[u].x, q[u].y, q[u].z, q[u].w };
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint16_t b = (uint16_t)(h[j >> 1] >> (16 * (j & 1)));
                const float v = y_dtype == EXL3C4_BF16 ? __uint_as_float((uint32_t)b << 16)
                                                       : (float)__builtin_bit_cast(_Float16, b);
                const float prod = ws[u] * v;
                const float sum = acc[j] + prod;
                acc[j] = r[u] < 0 ? acc[j] : sum;                     // a pair without a row adds nothing
            }
        }
    }
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = (uint32_t)to_f16(acc[2 * j]) | ((uint32_t)to_f16(acc[2 * j + 1]) << 16);
    *(uint4*)(out + t * out_pitch + c) = uint4{ o[0], o[1], o[2], o[3] };
}

int launched() { return hipGetLastError() == hipSuccess ? 0 : EXL3C4_E_DEVICE; }

template <int DT, int RPL>
void launch_router(const void* logits, int64_t n_tok, int32_t n_expert, int64_t pitch, int32_t top_k, int32_t renorm,
                   int32_t* ids, float* w, hipStream_t st) {
    hipLaunchKernelGGL((k_router<DT, RPL>), dim3((unsigned)((n_tok + 3) / 4)), dim3(256), 0, st, logits, n_tok,
                       n_expert, pitch, top_k, renorm, ids, w);
}
template <int DT>
void launch_router_dt(const void* logits, int64_t n_tok, int32_t n_expert, int64_t pitch, int32_t top_k,
                      int32_t renorm, int32_t* ids, float* w, hipStream_t st) {
    if (n_expert <= 64) launch_router<DT, 1>(logits, n_tok, n_expert, pitch, top_k, renorm, ids, w, st);
    else if (n_expert <= 128) launch_router<DT, 2>(logits, n_tok, n_expert, pitch, top_k, renorm, ids, w, st);
    else if (n_expert <= 256) launch_router<DT, 4>(logits, n_tok, n_expert, pitch, top_k, renorm, ids, w, st);
    else if (n_expert <= 512) launch_router<DT, 8>(logits, n_tok, n_expert, pitch, top_k, renorm, ids, w, st);
    else launch_router<DT, 16>(logits, n_tok, n_expert, pitch, top_k, renorm, ids, w, st);
}

template <int DT, int RPL>
void launch_rs(const void* logits, int32_t n_tok, int32_t n_expert, int64_t pitch, int32_t top_k, int32_t renorm,
               int32_t* ids, float* w, int32_t* sorted, int32_t* off, int32_t* count, int32_t* row_of, uint32_t lds,
               hipStream_t st) {
    hipLaunchKernelGGL((k_route_scatter<DT, RPL>), dim3(1), dim3(1024), lds, st, logits, n_tok, n_expert, pitch, top_k,
                       renorm, ids, w, sorted, off, count, row_of);
}
template <int DT>
void launch_rs_dt(const void* logits, int32_t n_tok, int32_t n_expert, int64_t pitch, int32_t top_k, int32_t renorm,
                  int32_t* ids, float* w, int32_t* sorted, int32_t* off, int32_t* count, int32_t* row_of,
                  uint32_t lds, hipStream_t st) {
    if (n_expert <= 64) launch_rs<DT, 1>(logits, n_tok, n_expert, pitch, top_k, renorm, ids, w, sorted, off, count, row_of, lds, st);
    else if (n_expert <= 128) launch_rs<DT, 2>(logits, n_tok, n_expert, pitch, top_k, renorm, ids, w, sorted, off, count, row_of, lds, st);
    else if (n_expert <= 256) launch_rs<DT, 4>(logits, n_tok, n_expert, pitch, top_k, renorm, ids, w, sorted, off, count, row_of, lds, st);
    else if (n_expert <= 512) launch_rs<DT, 8>(logits, n_tok, n_expert, pitch, top_k, renorm, ids, w, sorted, off, count, row_of, lds, st);
    else launch_rs<DT, 16>(logits, n_tok, n_expert, pitch, top_k, renorm, ids, w, sorted, off, count, row_of, lds, st);
}

}  // namespace

extern "C" int exl3c4_dev_router(const void* logits, int32_t dtype, int64_t n_tok, int32_t n_expert, int64_t pitch,
                                 int32_t top_k, int32_t renorm, int32_t* ids, float* w, void* stream) {
    if (n_tok <= 0) return 0;
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == EXL3C4_F32) launch_router_dt<EXL3C4_F32>(logits, n_tok, n_expert, pitch, top_k, renorm, ids, w, st);
    else if (dtype == EXL3C4_BF16) launch_router_dt<EXL3C4_BF16>(logits, n_tok, n_expert, pitch, top_k, renorm, ids, w, st);
    else launch_router_dt<EXL3C4_F16>(logits, n_tok, n_expert, pitch, top_k, renorm, ids, w, st);
    return launched();
}

extern "C" int exl3c4_dev_scatter(const int32_t* ids, int64_t T, int64_t base, int32_t n_expert, int32_t* sorted,
                                  int32_t* off, int32_t* count, int32_t* row_of, void* stream) {
    // a workgroup each SC_SEG pairs, up to one a CU (a segment is then several SC_SEG); one when there is no pair, and one
    // when row_of is written over ids: it has counted every pair before it writes any, and reads a later segment's ids
    // before that segment's rows go out, while other workgroups would still be counting
    const int64_t segs = T > 0 ? (T + SC_SEG - 1) / SC_SEG : 1;
    const int64_t per = row_of == ids ? segs : (segs + SC_MAX_WG - 1) / SC_MAX_WG;
    const unsigned wgs = (unsigned)((segs + per - 1) / per);
    if (row_of != ids && T >= PO_LEAST && T <= PO_MOST && T <= (int64_t)PO_EACH * n_expert && base >= -(1 << 30) && base <= 1 << 30) {
        // (ids written over by row_of while other workgroups read them, and bases that 32 bits do not take from every id, are k_scatter's)
        const uint32_t by = ((uint32_t)n_expert + SC_MAX_WG - 1) / SC_MAX_WG, n = ((uint32_t)n_expert + by - 1) / by;
        hipLaunchKernelGGL(base == 0 ? k_pairs_by_expert<false> : k_pairs_by_expert<true>, dim3(n), dim3(PO_THREADS), 0,
                           (hipStream_t)stream, ids, (uint32_t)T, (int32_t)base, n_expert, by, ((uint32_t)T + n - 1) / n, sorted, off,
                           count, row_of);
        return launched();
    }
    const bool far = base < INT32_MIN || base > INT32_MAX;
    const auto f = T <= SC_THREADS       ? (far ? k_scatter<1, true> : k_scatter<1, false>)
                   : T <= 4 * SC_THREADS ? (far ? k_scatter<4, true> : k_scatter<4, false>)
                                         : (far ? k_scatter<16, true> : k_scatter<16, false>);
    hipLaunchKernelGGL(f, dim3(wgs), dim3(SC_THREADS), 0, (hipStream_t)stream, ids, (uint32_t)T, base, n_expert,
                       (uint32_t)(per * SC_SEG), sorted, off, count, row_of);
    return launched();
}

extern "C" int exl3c4_dev_route_scatter(const void* logits, int32_t dtype, int32_t n_tok, int32_t n_expert,
                                        int64_t pitch, int32_t top_k, int32_t renorm, int32_t* ids, float* w,
                                        int32_t* sorted, int32_t* off, int32_t* count, int32_t* row_of,
                                        void* stream) {
    const uint32_t lds = (uint32_t)((16 * 64 + n_expert + 17) * 4);   // ids, then scatter_small's
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == EXL3C4_F32)
        launch_rs_dt<EXL3C4_F32>(logits, n_tok, n_expert, pitch, top_k, renorm, ids, w, sorted, off, count, row_of, lds, st);
    else if (dtype == EXL3C4_BF16)
        launch_rs_dt<EXL3C4_BF16>(logits, n_tok, n_expert, pitch, top_k, renorm, ids, w, sorted, off, count, row_of, lds, st);
    else
        launch_rs_dt<EXL3C4_F16>(logits, n_tok, n_expert, pitch, top_k, renorm, ids, w, sorted, off, count, row_of, lds, st);
    return launched();
}

namespace {

template <int RPL, bool GROUPS>
void launch_score(const Exl3c4DevRoute& a, bool scatter, hipStream_t st) {
    if (scatter) hipLaunchKernelGGL((k_score_scatter<RPL, GROUPS>), dim3(1), dim3(1024), 0, st, a);
    else hipLaunchKernelGGL((k_score<RPL, GROUPS>), dim3((unsigned)((a.n_tok + 3) / 4)), dim3(256), 0, st, a);
}
template <int RPL>
void launch_score(const Exl3c4DevRoute& a, bool scatter, hipStream_t st) {
    if (a.n_group > 1 && a.top_group < a.n_group) launch_score<RPL, true>(a, scatter, st);
    else launch_score<RPL, false>(a, scatter, st);
}

}  // namespace

extern "C" int exl3c4_dev_score(const Exl3c4DevRoute* r, int scatter, void* stream) {
    const hipStream_t st = (hipStream_t)stream;
    if (r->n_tok <= 0 && !scatter) return 0;
    if (r->n_expert <= 64) launch_score<1>(*r, scatter, st);
    else if (r->n_expert <= 128) launch_score<2>(*r, scatter, st);
    else if (r->n_expert <= 256) launch_score<4>(*r, scatter, st);
    else if (r->n_expert <= 512) launch_score<8>(*r, scatter, st);
    else launch_score<16>(*r, scatter, st);
    return launched();
}

extern "C" int exl3c4_dev_gather(const void* y, int32_t y_dtype, int64_t y_pitch, const float* w,
                                 const int32_t* row_of, int64_t n_tok, int32_t top_k, int64_t cols, void* out,
                                 int64_t out_pitch, void* stream) {
    if (n_tok <= 0 || cols <= 0) return 0;
    hipLaunchKernelGGL(k_gather, dim3((unsigned)n_tok, (unsigned)((cols + 2047) / 2048)), dim3(256), 0,
                       (hipStream_t)stream, y, y_dtype, y_pitch, w, row_of, n_tok, top_k, cols, (uint16_t*)out,
                       out_pitch);
    return launched();
}
