// exl3c4_gemm.hip -- the products of routed experts whose weights are f16, bf16 or microscaled 4-bit floats (MX4), on
// gfx950 (wave64): y[i] = W_e x[row i] over the sorted rows of each expert's run, with SwiGLU where asked
// (include/exl3c4.h). No counterpart in the reference.
//
// THE MATRIX STEP. 64 bytes of a weight row feed one matrix instruction: 32 columns in 16 bits
// (v_mfma_f32_16x16x32) or 128 in MX4 (v_mfma_scale_f32_16x16x128_f8f6f4), lane l holding the 16 bytes g = l / 16 of
// row l % 16 -- in MX4 exactly one block, whose scale byte is the lane's own. x is the A operand (rows of D), W the B
// operand (columns of D): lane l ends with D[m = 4 g + r][n = l % 16], r = 0 .. 3.
//
// MX4 WEIGHTS AGAINST 16-BIT x. bf16 holds e2m1 x 2^s exactly, so with bf16 x a lane's block is converted with its scale
// (v_cvt_scalef32_pk_bf16_fp4) and multiplied as bf16. f16 does not hold the scales' range: with f16 x the codes alone are
// converted, the four lane groups' words are exchanged so that one instruction's 32 columns are one block, and its sums
// are scaled in f32 as they are added. Either way every product is exact.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include "exl3c4_dev.h"

namespace {

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf8_t __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int F16 = EXL3C4_F16, BF16 = EXL3C4_BF16, MX4 = EXL3C4_MX4;

// ------------------------------------------------------------------------------------------ the rows of a workgroup
// The inclusive sum of v over lanes 0 .. lane, by DPP (row shifts, then the rows' totals by row broadcasts).
__device__ __forceinline__ int wave_scan_incl(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return v;
}

struct Chunk { int expert, row0, rows; };                       // expert -1: rows that no run holds (zeros)

// Chunk c of the launch: the rows before the first run, the experts' runs and the rows behind the last one, each cut into
// chunks of at most 2^MT_LOG2 rows, numbered in this order. Every wave finds its own (the offsets come from L2; nine
// loads and one scan for 512 segments), so a launch needs no plan before it. The offsets are clamped to [0, T] and a run
// that ends before it starts is empty: whatever the table holds, every row is in [0, T). False past the last chunk.
// *total: the launch's chunks, when asked.
template <int MT_LOG2>
__device__ __forceinline__ bool find_chunk(const Exl3c4DevGemm& a, int c, int lane, Chunk& out) {
    const int n_seg = a.n_expert + 2;
    int before = 0;
    for (int base = 0; base < n_seg; base += 512) {
        int v[9], total = 0;
#pragma unroll
        for (int j = 0; j < 9; ++j) {                            // where segment i starts
            const int i = base + 8 * lane + j;
            const int o = a.off[min(max(i - 1, 0), a.n_expert)];
            v[j] = i <= 0 ? 0 : i > a.n_expert + 1 ? a.T : min(max(o, 0), a.T);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) total += (max(v[j + 1] - v[j], 0) + (1 << MT_LOG2) - 1) >> MT_LOG2;
        const int incl = wave_scan_incl(total);
        int r = c - before - (incl - total);                     // the chunk's number among this lane's
        const uint64_t hit = __ballot(r >= 0 && r < total);
        if (hit) {
            int seg = 0, row0 = 0, rows = 0;
            bool found = false;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int len = max(v[j + 1] - v[j], 0), n = (len + (1 << MT_LOG2) - 1) >> MT_LOG2;
                if (!found && r < n) {
                    found = true;
                    seg = base + 8 * lane + j;
                    row0 = v[j] + (r << MT_LOG2);
                    rows = min(1 << MT_LOG2, len - (r << MT_LOG2));
                }
                r -= n;
            }
            const int from = __builtin_ctzll(hit);
            seg = __builtin_amdgcn_readlane(seg, from);
            out.row0 = __builtin_amdgcn_readlane(row0, from);
            out.rows = __builtin_amdgcn_readlane(rows, from);
            out.expert = seg == 0 || seg == n_seg - 1 ? -1 : seg - 1;
            return true;
        }
        before += __builtin_amdgcn_readlane(incl, 63);
    }
    return false;
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

__device__ __forceinline__ const char* entry(const char* base, int64_t stride, int e) {
    return stride ? base + (int64_t)e * stride : ((const char* const*)base)[e];
}

// silu(g) u in f32: g / (1 + exp(-g)) by the hardware's exp2 and reciprocal (a few f32 steps from the exact value,
// below the rounding to 16 bits; 2^-22 or so beside an f32 output's own sums).
__device__ __forceinline__ float swiglu(float g, float u) {
    return g * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(g * -1.44269504088896340736f)) * u;
}

__device__ __forceinline__ void store(char* p, int type, float v) {
    if (type == EXL3C4_F32) *(float*)p = v;
    else if (type == BF16) *(__bf16*)p = (__bf16)v;
    else *(_Float16*)p = (_Float16)v;
}

// ------------------------------------------------------------------------------------------ the matrix step
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
__device__ __forceinline__ f32x4 mma_mx4(const uint4& a, int sa, const uint4& b, int sb, f32x4 c) {
    const i32x8 A = { (int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0 };
    const i32x8 B = { (int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0 };
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, c, 4, 4, 0, sa, 0, sb);
}

// 8 codes (a word) as 8 bf16 with their scale, or 8 f16 without.
__device__ __forceinline__ uint4 to_bf16(uint32_t q, float scale) {
    return { __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 0)),
             __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 1)),
             __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 2)),
             __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 3)) };
}
__device__ __forceinline__ uint4 to_f16(uint32_t q) {
    return { __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q, 1.f, 0)),
             __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q, 1.f, 1)),
             __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q, 1.f, 2)),
             __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q, 1.f, 3)) };
}
// A 4 x 4 transpose of words over the lane groups: group g's word j to group j's word g.
__device__ __forceinline__ uint4 exchange(const uint4& q) {
    const auto p = __builtin_amdgcn_permlane32_swap(q.x, q.z, false, false);
    const auto r = __builtin_amdgcn_permlane32_swap(q.y, q.w, false, false);
    const auto s = __builtin_amdgcn_permlane16_swap(p[0], r[0], false, false);
    const auto t = __builtin_amdgcn_permlane16_swap(p[1], r[1], false, false);
    return { s[0], s[1], t[0], t[1] };
}
// 2^(byte - 127) as an operand of the conversions (they read the exponent field), and as an f32 (255: NaN).
__device__ __forceinline__ float scale_arg(uint32_t byte) { return __uint_as_float(byte << 23); }
__device__ __forceinline__ float scale_f32(uint32_t byte) {
    const f32x2 v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(2u, scale_arg(byte), 0);      // code 2 is 1
    return v[0];
}

// ------------------------------------------------------------------------------------------ few rows an expert
// A workgroup: a chunk of up to 16 rows against 32 weight rows (with SwiGLU 16 gate rows and their 16 up rows), the four
// waves each a quarter of k; the weights go from memory straight to the matrix units' operands, each byte read once, and
// the quarters' sums meet in LDS in a fixed order.
constexpr int ROWS_LOG2 = 4;
constexpr int WAVES = 4;

// What one matrix step reads of the two weight strips and of x, and its products. FULL: every lane's bytes are inside
// the rows; else what lies past K reads as zeros (and their scales as 2^-127, never as a NaN).
template <int XT, int WT> struct Step {
    static constexpr int KB = WT == MX4 ? 128 : 32;             // columns of a weight row's 64 bytes
    static constexpr int NX = WT == MX4 && XT != MX4 ? 4 : 1;
    uint4 q[2], x[NX];
    uint32_t sc[2], xsc;

    template <bool FULL>
    __device__ __forceinline__ void load(int t, int K, int g, const char* xp, const uint8_t* xs, const char* const* w,
                                         const uint8_t* const* ws) {
        const int64_t k = (int64_t)t * KB;
        const uint4 none = { 0, 0, 0, 0 };
        const bool in = FULL || k + (KB / 4) * g < K;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            q[s] = in ? *(const uint4*)(w[s] + (int64_t)t * 64) : none;
            if constexpr (WT == MX4) sc[s] = *(const uint32_t*)(ws[s] + 4 * (int64_t)t);
            if constexpr (WT == MX4) if (!FULL) sc[s] &= live_bytes(K, k);
        }
        if constexpr (XT == MX4) {
            x[0] = in ? *(const uint4*)(xp + (int64_t)t * 64) : none;
            xsc = *(const uint32_t*)(xs + 4 * (int64_t)t);
            if (!FULL) xsc &= live_bytes(K, k);
        } else if constexpr (WT != MX4) {
            x[0] = in ? *(const uint4*)(xp + 2 * (k + 8 * g)) : none;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                // bf16: the lane's own block, word j; f16: block j, the lane group's word
                const int64_t c = k + (XT == BF16 ? 32 * g + 8 * j : 32 * j + 8 * g);
                x[j] = FULL || c < K ? *(const uint4*)(xp + 2 * c) : none;
            }
        }
    }
    // the scale bytes of the step's blocks before column K
    static __device__ __forceinline__ uint32_t live_bytes(int K, int64_t k) {
        const int n = (int)min((int64_t)(K - k) / 32, (int64_t)4);
        return n >= 4 ? 0xFFFFFFFFu : (1u << (8 * n)) - 1u;
    }
    __device__ __forceinline__ void multiply(int g, f32x4* acc) const {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            if constexpr (WT != MX4) {
                acc[s] = mma<XT>(x[0], q[s], acc[s]);
            } else if constexpr (XT == MX4) {
                acc[s] = mma_mx4(x[0], (xsc >> (8 * g)) & 255, q[s], (sc[s] >> (8 * g)) & 255, acc[s]);
            } else if constexpr (XT == BF16) {
                const float f = scale_arg((sc[s] >> (8 * g)) & 255);
                const uint32_t word[4] = { q[s].x, q[s].y, q[s].z, q[s].w };
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[s] = mma<BF16>(x[j], to_bf16(word[j], f), acc[s]);
            } else {
                const uint4 e = exchange(q[s]);
                const uint32_t word[4] = { e.x, e.y, e.z, e.w };
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float f = scale_f32((sc[s] >> (8 * j)) & 255);
                    const f32x4 p = mma<F16>(x[j], to_f16(word[j]), f32x4{ 0, 0, 0, 0 });
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[s][r] = __builtin_fmaf(p[r], f, acc[s][r]);
                }
            }
        }
    }
};

template <int XT, int WT, bool SW>
__global__ __launch_bounds__(64 * WAVES) void k_mg_rows(Exl3c4DevGemm a) {
    typedef Step<XT, WT> S;
    constexpr int AHEAD = S::NX == 4 ? 2 : 4;                   // steps whose loads are out together
    __shared__ f32x4 part[WAVES][2][64];
    __shared__ int alive[16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, g = lane >> 4;
    const int c = blockIdx.x / a.tiles, tile = blockIdx.x - c * a.tiles;
    Chunk ch;
    if (!find_chunk<ROWS_LOG2>(a, c, lane, ch)) return;
    const int n0 = tile * (SW ? 16 : 32);
    const int ysz = a.y_type == EXL3C4_F32 ? 4 : 2;
    if (ch.expert >= 0) {
        const int xr = l16 < ch.rows ? x_row(a, ch.row0 + l16) : -1;
        if (threadIdx.x < 16) alive[threadIdx.x] = xr >= 0;
        const char* x = a.x + (int64_t)max(xr, 0) * a.x_pitch + (XT == MX4 ? 16 * g : 0);
        const uint8_t* xs = XT == MX4 ? a.xs + (int64_t)max(xr, 0) * a.xs_pitch : nullptr;
        const char* we = entry(a.w, a.w_stride, ch.expert);
        const uint8_t* wse = WT == MX4 ? (const uint8_t*)entry((const char*)a.ws, a.ws_stride, ch.expert) : nullptr;
        const char* w[2];
        const uint8_t* ws[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {                            // rows past the last one repeat it and are not stored
            const int n = SW ? min(n0 + l16, a.n_out - 1) + s * a.n_out : min(n0 + 16 * s + l16, a.N - 1);
            w[s] = we + (int64_t)n * a.w_pitch + 16 * g;
            ws[s] = WT == MX4 ? wse + (int64_t)n * a.ws_pitch : nullptr;
        }
        const int steps = (a.K + S::KB - 1) / S::KB;
        const int to = (int)((int64_t)steps * (wave + 1) / WAVES), full = min(to, a.K / S::KB);
        int t = (int)((int64_t)steps * wave / WAVES);
        f32x4 acc[2] = {};
        for (; t + AHEAD <= full; t += AHEAD) {
            S st[AHEAD];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) st[u].template load<true>(t + u, a.K, g, x, xs, w, ws);
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) st[u].multiply(g, acc);
        }
        for (; t < to; ++t) {
            S st;
            st.template load<false>(t, a.K, g, x, xs, w, ws);
            st.multiply(g, acc);
        }
        part[wave][0][lane] = acc[0];
        part[wave][1][lane] = acc[1];
    }
    __syncthreads();
    // thread -> (row m, column j of the strip), and both strips: their sums at [strip][16 (m / 4) + j][m % 4]
    const int m = threadIdx.x >> 4, j = threadIdx.x & 15;
    if (m >= ch.rows) return;
    float v[2] = { 0.f, 0.f };
    if (ch.expert >= 0 && alive[m]) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int u = 0; u < WAVES; ++u) v[s] += part[u][s][16 * (m >> 2) + j][m & 3];
        if (SW) v[0] = swiglu(v[0], v[1]);
    }
    char* y = a.y + (int64_t)(ch.row0 + m) * a.y_pitch;
    if (n0 + j < a.n_out) store(y + (int64_t)(n0 + j) * ysz, a.y_type, v[0]);
    if (!SW && n0 + 16 + j < a.n_out) store(y + (int64_t)(n0 + 16 + j) * ysz, a.y_type, v[1]);
}

int launched() { return hipGetLastError() == hipSuccess ? 0 : EXL3C4_E_DEVICE; }

// Chunks of at most `rows` that the launch's segments (the runs, and the rows before and behind them) can make.
int64_t chunk_bound(const Exl3c4DevGemm& a, int rows) {
    const int64_t seg = (int64_t)a.n_expert + 2;
    return a.T / rows + (seg < a.T ? seg : a.T);
}

template <int XT, int WT, bool SW>
int launch(Exl3c4DevGemm& a, hipStream_t st) {
    a.tiles = (a.n_out + (SW ? 15 : 31)) / (SW ? 16 : 32);
    const int64_t grid = chunk_bound(a, 1 << ROWS_LOG2) * a.tiles;
    if (grid > INT32_MAX) return EXL3C4_E_SHAPE;
    hipLaunchKernelGGL((k_mg_rows<XT, WT, SW>), dim3((unsigned)grid), dim3(64 * WAVES), 0, st, a);
    return launched();
}

template <int XT, int WT>
int launch_act(Exl3c4DevGemm& a, int32_t act, hipStream_t st) {
    return act == EXL3C4_ACT_SWIGLU ? launch<XT, WT, true>(a, st) : launch<XT, WT, false>(a, st);
}

}  // namespace

extern "C" int exl3c4_dev_gemm(const Exl3c4DevGemm* g, int32_t x_type, int32_t w_type, int32_t act, void* stream) {
    Exl3c4DevGemm a = *g;
    const hipStream_t st = (hipStream_t)stream;
    if (w_type == F16) return launch_act<F16, F16>(a, act, st);
    if (w_type == BF16) return launch_act<BF16, BF16>(a, act, st);
    if (x_type == F16) return launch_act<F16, MX4>(a, act, st);
    if (x_type == BF16) return launch_act<BF16, MX4>(a, act, st);
    return launch_act<MX4, MX4>(a, act, st);
}
