// exl3c4_gemm_dev.h -- what the products of routed experts share (device code; exl3c4_gemm.hip has the 16-bit and MX4 kernels, exl3c4_gemm_f8.hip
// F8's): a workgroup's chunk of rows and its column tile, rows of x and of y, the activation, the 16-bit matrix step, loads to LDS, a launch's
// bounds.
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "exl3c4_dev.h"
#include "exl3c4_wave.h"

namespace {

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf8_t __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int F16 = EXL3C4_F16, BF16 = EXL3C4_BF16;

// Memory by addresses known to be global: a pointer out of a table is a flat one otherwise, whose loads also hold up LDS.
typedef const __attribute__((address_space(1))) char* gaddr;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint4 load16(gaddr p) {
    return __builtin_bit_cast(uint4, *(const __attribute__((address_space(1))) u32x4*)p);
}
typedef u32x4 u32x4_at4 __attribute__((aligned(4)));            // scale rows and offsets start at any word
__device__ __forceinline__ uint4 load_words(gaddr p) {
    return __builtin_bit_cast(uint4, (u32x4)*(const __attribute__((address_space(1))) u32x4_at4*)p);
}

// ------------------------------------------------------------------------------------------ the rows of a workgroup
// The largest v of lanes 0 .. lane - 1 (0 for lane 0; no v is below 0).
__device__ __forceinline__ int wave_max_before(int v, int lane) {
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false));
    const int up = __shfl_up(v, 1);
    return lane == 0 ? 0 : up;
}

struct Chunk { int expert, row0, rows, tile, alone; };          // expert -1: rows that no run holds (zeros); alone: its run has no other chunk

// 512 experts from `base` on, eight a lane: where each run starts, and the wave's inclusive sum of their chunks. The offsets are
// clamped to [0, T], and one below an earlier one counts as that one (`reach`: the largest so far). So whatever the table holds, the runs, the
// rows before the first and the rows behind the last are disjoint and make up [0, T): every row is written once.
template <int MT_LOG2> struct Runs {
    int v[9], own, incl;
    static __device__ __forceinline__ int chunks(int len) { return (len + (1 << MT_LOG2) - 1) >> MT_LOG2; }
    __device__ __forceinline__ void read(const Exl3c4DevGemm& a, int base, int lane, int& reach) {
        const int i = base + 8 * lane;
        if (i + 8 <= a.n_expert) {                               // (16-byte loads: a load a value costs nine times the requests)
            const uint4 p = load_words((gaddr)(a.off + i)), q = load_words((gaddr)(a.off + i + 4));
            v[0] = (int)p.x, v[1] = (int)p.y, v[2] = (int)p.z, v[3] = (int)p.w;
            v[4] = (int)q.x, v[5] = (int)q.y, v[6] = (int)q.z, v[7] = (int)q.w;
            v[8] = a.off[i + 8];
        } else {
#pragma unroll
            for (int j = 0; j < 9; ++j) v[j] = a.off[min(i + j, a.n_expert)];
        }
#pragma unroll
        for (int j = 0; j < 9; ++j) v[j] = min(max(v[j], 0), a.T);
        int fall = v[0] - reach;
#pragma unroll
        for (int j = 0; j < 8; ++j) fall |= v[j + 1] - v[j];
        if (__any(fall < 0)) {                                   // a table that is no routing
            v[0] = max(v[0], reach);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j + 1] = max(v[j + 1], v[j]);
            const int before = wave_max_before(v[8], lane);
#pragma unroll
            for (int j = 0; j < 9; ++j) v[j] = max(v[j], before);
        }
        reach = __builtin_amdgcn_readlane(v[8], 63);
        own = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) own += chunks(v[j + 1] - v[j]);
        incl = wave_scan_incl(own);
    }
    __device__ __forceinline__ int total() const { return __builtin_amdgcn_readlane(incl, 63); }
    // chunk c of these (c < total())
    __device__ __forceinline__ void find(int base, int lane, int c, Chunk& out) const {
        int r = c - (incl - own), e = 0, row0 = 0, rows = 0, alone = 0;
        const uint64_t hit = __ballot(r >= 0 && r < own);
        bool found = false;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int len = v[j + 1] - v[j], n = chunks(len);
            if (!found && r < n) {
                found = true;
                e = base + 8 * lane + j;
                row0 = v[j] + (r << MT_LOG2);
                rows = min(1 << MT_LOG2, len - (r << MT_LOG2));
                alone = n == 1;
            }
            r -= n;
        }
        const int from = __builtin_ctzll(hit);
        out.expert = __builtin_amdgcn_readlane(e, from);
        out.row0 = __builtin_amdgcn_readlane(row0, from);
        out.rows = __builtin_amdgcn_readlane(rows, from);
        out.alone = __builtin_amdgcn_readlane(alone, from);
    }
};

// The workgroup's chunk of at most 2^MT_LOG2 rows and its column tile, rows 0 if it has none. The launch's units are its chunks -- the
// experts', then those of the rows before the first run and behind the last one -- each with its column tiles in turn. One wave of the workgroup
// finds its unit from the offsets (one read and one scan for 512 experts), so a launch needs no plan before it.
// XCD: the units are cut into eight ranges, one an XCD (workgroups go to the XCDs in turn), whose L2 then holds a chunk's rows for all its
// tiles and an expert's weights for all its chunks (bf16, 400 tokens of top-10 over 512 experts: 437 us in plain order, 362 so). The rows
// kernel reads every weight once and its few rows of x from anywhere: the same either way, and plain.
template <int MT_LOG2, bool XCD>
__device__ __forceinline__ Chunk find_unit(const Exl3c4DevGemm& a, int lane) {
    typedef Runs<MT_LOG2> R;
    Chunk out = { -1, 0, 0, 0, 0 };
    R s;
    int live = 0, head = 0, tail = 0;
    for (int base = 0; base < a.n_expert; base += 512) {
        s.read(a, base, lane, tail);
        live += s.total();
        if (base == 0) head = __builtin_amdgcn_readlane(s.v[0], 0);
    }
    const int n_head = R::chunks(head), total = live + n_head + R::chunks(a.T - tail);
    const uint32_t units = (uint32_t)total * (uint32_t)a.tiles, x = blockIdx.x & 7u, i = blockIdx.x >> 3;
    uint32_t unit = blockIdx.x;
    if (XCD) {
        if (i >= (units >> 3) + (x < (units & 7u))) return out;
        unit = x * (units >> 3) + min(x, units & 7u) + i;
    } else if (unit >= units) {
        return out;
    }
    int c = (int)(unit / (uint32_t)a.tiles);
    out.tile = (int)(unit - (uint32_t)c * (uint32_t)a.tiles);
    if (c >= live) {
        c -= live;
        const int start = c < n_head ? 0 : tail, end = c < n_head ? head : a.T;
        out.row0 = start + ((c < n_head ? c : c - n_head) << MT_LOG2);
        out.rows = min(1 << MT_LOG2, end - out.row0);
    } else if (a.n_expert <= 512) {
        s.find(0, lane, c, out);
    } else {
        int reach = 0;
        for (int base = 0; base < a.n_expert; base += 512) {
            s.read(a, base, lane, reach);
            if (c < s.total()) {
                s.find(base, lane, c, out);
                break;
            }
            c -= s.total();
        }
    }
    return out;
}
// The same for the whole workgroup, by its first wave.
template <int MT_LOG2, bool XCD>
__device__ __forceinline__ Chunk my_unit(const Exl3c4DevGemm& a, int lane, int wave) {
    __shared__ Chunk unit;
    if (wave == 0) {
        const Chunk c = find_unit<MT_LOG2, XCD>(a, lane);
        if (lane == 0) unit = c;
    }
    __syncthreads();
    return { __builtin_amdgcn_readfirstlane(unit.expert), __builtin_amdgcn_readfirstlane(unit.row0),
             __builtin_amdgcn_readfirstlane(unit.rows), __builtin_amdgcn_readfirstlane(unit.tile), __builtin_amdgcn_readfirstlane(unit.alone) };
}

// The row of x that sorted row i reads, or -1: none (the row is zeros).
__device__ __forceinline__ int x_row(const Exl3c4DevGemm& a, int i) {
    int r = i;
    if (a.sorted) {
        const int t = a.sorted[i];
        r = t < 0 ? -1 : (int)((uint32_t)t / (uint32_t)a.top_k);
    }
    return r < a.x_rows ? r : -1;
}

// A weight's words and an expert's weights.
__device__ __forceinline__ uint32_t load4(gaddr p) { return *(const __attribute__((address_space(1))) uint32_t*)p; }
__device__ __forceinline__ gaddr entry(const void* base, int64_t stride, int e) {
    return stride ? (gaddr)base + (int64_t)e * stride : ((const gaddr*)base)[e];
}

// silu(g) u = g u / (1 + e^-g) in f32, by the hardware's exp2 and reciprocal. The exponent's argument is rounded once, an error of e^-g that grows
// with |g| and that a negative g meets in full: so from -8 up, where it is 9.8 steps of 2^-24 and the whole 16.8 at most. Below,
// e^g = 2^n e with the argument's fraction exact to a step, silu = g 2^n e / (1 + 2^n e), and u comes in between the two halves of 2^n: 9 steps,
// also where e^-g passes f32 (from -88.7 down) or silu is below it, and u brings the product back. Each value goes by its own g alone.
constexpr float SILU_NEAR = -8.f;
__device__ __forceinline__ float swiglu_near(float g, float u) {
    return g * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(g * -1.44269504088896340736f)) * u;
}
__device__ __forceinline__ float swiglu_far(float g, float u) {
    const float a = fmaxf(g, -1024.f);                           // (2^-1477: 0 beside any finite u)
    const float n = rintf(a * 1.44269502162933349609f);
    const float r = __builtin_fmaf(a, 1.92596299e-8f, __builtin_fmaf(a, 1.44269502162933349609f, -n));   // a log2 e - n, log2 e in two parts
    const float e = __builtin_amdgcn_exp2f(r);
    const int k = (int)n, half = k >> 1;
    const float v = g * e * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_ldexpf(e, k));
    const float y = __builtin_amdgcn_ldexpf(__builtin_amdgcn_ldexpf(v, half) * u, k - half);
    return g == -__builtin_inff() ? __builtin_nanf("") : y;      // -inf / inf
}
__device__ __forceinline__ float swiglu(float g, float u) {
    float y = swiglu_near(g, u);
    if (g < SILU_NEAR) y = swiglu_far(g, u);
    return y;
}
__device__ __forceinline__ f32x4 swiglu4(const f32x4& g, const f32x4& u) {
    f32x4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = swiglu_near(g[i], u[i]);
    if (__any(fminf(fminf(g[0], g[1]), fminf(g[2], g[3])) < SILU_NEAR)) {      // (rolled: four of them in line at each store of a tile
                                                                               // took MX4 2048 Zipf from 146 to 151 us, by the code's size)
        f32x4 a = g, b = u;
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
            const float v = a[0] < SILU_NEAR ? swiglu_far(a[0], b[0]) : y[0];
            a = { a[1], a[2], a[3], a[0] };
            b = { b[1], b[2], b[3], b[0] };
            y = { y[1], y[2], y[3], v };
        }
    }
    return y;
}

__device__ __forceinline__ void store(char* p, int type, float v) {
    if (type == EXL3C4_F32) *(float*)p = v;
    else if (type == BF16) *(__bf16*)p = (__bf16)v;
    else *(_Float16*)p = (_Float16)v;
}

// Four columns of a row, `left` of them inside y.
__device__ __forceinline__ void store4(char* p, int type, const f32x4& v, int left, bool whole) {
    if (left >= 4 && whole) {
        if (type == EXL3C4_F32) {
            *(f32x4*)p = v;
        } else if (type == BF16) {
            typedef __bf16 t4 __attribute__((ext_vector_type(4)));
            *(t4*)p = t4{ (__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3] };
        } else {
            typedef _Float16 t4 __attribute__((ext_vector_type(4)));
            *(t4*)p = t4{ (_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3] };
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < left) store(p + i * (type == EXL3C4_F32 ? 4 : 2), type, v[i]);
    }
}

// ------------------------------------------------------------------------------------------ the 16-bit matrix step
__device__ __forceinline__ f32x4 mma16(const uint4& a, const uint4& b, f32x4 c, half8_t*) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(const uint4& a, const uint4& b, f32x4 c, bf8_t*) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8_t, a), __builtin_bit_cast(bf8_t, b), c, 0, 0, 0);
}
template <int XT> struct Elem { typedef half8_t type; };
template <> struct Elem<BF16> { typedef bf8_t type; };
template <int XT> __device__ __forceinline__ f32x4 mma(const uint4& a, const uint4& b, f32x4 c) {
    return mma16(a, b, c, (typename Elem<XT>::type*)nullptr);
}

// ------------------------------------------------------------------------------------------ loads to LDS
__device__ const uint4 k_zero = { 0, 0, 0, 0 };                 // what loads read past the end of a row

// 16 or 4 bytes a lane from memory to LDS at `lds` (uniform; lane after lane). As asm, so that the compiler does not hold every
// later LDS read until it is done (it cannot tell one stage's buffer from another's): wait_loads and the barriers order
// them. No register is written; the address is read at issue, and s_nop keeps m0's wait state.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"                   // that m0 is reserved: nothing holds a value in it here
__device__ __forceinline__ void dma16(gaddr from, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void dma4(gaddr from, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(from), "s"(lds) : "memory", "m0");
}
// The same where `all` is -1, and nothing where it is 0 (uniform; the whole wave is active): no lane loads, without a branch.
__device__ __forceinline__ void dma16_of(gaddr from, uint32_t lds, int all) {
    asm volatile("s_mov_b32 m0, %1\n\ts_mov_b32 exec_lo, %2\n\ts_mov_b32 exec_hi, %2\n\tglobal_load_lds_dwordx4 %0, off\n\ts_mov_b64 exec, -1" ::"v"(from), "s"(lds), "s"(all) : "memory", "m0");
}
// And where `once` is not 0 (uniform), past the caches: bytes that no other workgroup reads. (The branch is in the asm, so that it divides nothing.)
__device__ __forceinline__ void dma16_of(gaddr from, uint32_t lds, int all, int once) {
    asm volatile("s_mov_b32 m0, %1\n\ts_mov_b32 exec_lo, %2\n\ts_mov_b32 exec_hi, %2\n\ts_cmp_lg_u32 %3, 0\n\ts_cbranch_scc1 .Lonce%=\n\t"
                 "global_load_lds_dwordx4 %0, off\n\ts_branch .Lthen%=\n.Lonce%=:\n\tglobal_load_lds_dwordx4 %0, off nt\n.Lthen%=:\n\ts_mov_b64 exec, -1"
                 ::"v"(from), "s"(lds), "s"(all), "s"(once) : "memory", "m0", "scc");
}
__device__ __forceinline__ void dma4_of(gaddr from, uint32_t lds, int all) {
    asm volatile("s_mov_b32 m0, %1\n\ts_mov_b32 exec_lo, %2\n\ts_mov_b32 exec_hi, %2\n\tglobal_load_lds_dword %0, off\n\ts_mov_b64 exec, -1" ::"v"(from), "s"(lds), "s"(all) : "memory", "m0");
}
#pragma clang diagnostic pop
// Until at most N of the wave's loads are out, and none of its LDS reads.
template <int N> __device__ __forceinline__ void wait_loads() {
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0070);
}

// ------------------------------------------------------------------------------------------ a launch
// Threads a launch may have in all: what it holds in 32 bits.
constexpr int64_t THREADS = UINT32_MAX;
int launched() { return hipGetLastError() == hipSuccess ? 0 : EXL3C4_E_DEVICE; }

// Chunks of at most `rows` that the segments of T rows (the runs of n_expert experts, and the rows before and behind them) can make.
int64_t chunk_bound(int64_t T, int64_t n_expert, int rows) {
    const int64_t seg = n_expert + 2;
    return T / rows + (seg < T ? seg : T);
}

}  // namespace
