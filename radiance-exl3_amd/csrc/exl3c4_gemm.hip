// exl3c4_gemm.hip -- the products of routed experts whose weights are f16, bf16 or microscaled 4-bit floats (MX4), on
// gfx950 (wave64): y[i] = W_e x[row i] over the sorted rows of each expert's run, with SwiGLU where asked
// (include/exl3c4.h). No counterpart in the reference.
//
// THE MATRIX STEP. 64 bytes of a weight row feed one matrix instruction: 32 columns in 16 bits
// (v_mfma_f32_16x16x32) or 128 in MX4 (v_mfma_scale_f32_16x16x128_f8f6f4), lane l holding the 16 bytes g = l / 16 of
// row l % 16 -- in MX4 exactly one block, whose scale byte is the lane's own. x is the A operand (rows of D), W the B
// operand (columns of D): lane l ends with D[m = 4 g + r][n = l % 16], r = 0 .. 3.
//
// MX4 WEIGHTS AGAINST 16-BIT x. bf16 holds e2m1 x 2^s exactly for all but the two largest scales, so with bf16 x a lane's block is
// converted with its scale (v_cvt_scalef32_pk_bf16_fp4) and multiplied as bf16; a wave (few rows) or a tile (many) that has met one of
// those two, whose larger elements pass 2^128, sums again, with a quarter of every weight, and takes four times that. f16 does not hold
// the scales' range: with f16 x a row's blocks are converted relative to the largest scale among some hundred columns (its level), where
// those within 2^-13 of it are exact in f16, and the sums are scaled in f32 as they are added; blocks further down, if any of them is not
// all zeros, have passes of their own. Either way every product is exact. (Scaling each block's sums by itself, one matrix instruction a
// block, took twice the time of levels when they were chosen, 125 us against 64. 32 tokens, top-10 of 512 experts, gate and up
// 2048 -> 2 x 512 now: f16 x 75, bf16 x 57.)
#include <hip/hip_runtime.h>

#include <stdint.h>

#include "exl3c4_dev.h"
#include "exl3c4_gemm_dev.h"

namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int MX4 = EXL3C4_MX4;

// ------------------------------------------------------------------------------------------ the matrix step
template <int BYTE = 0>
__device__ __forceinline__ f32x4 mma_mx4(const uint4& a, int sa, const uint4& b, int sb, f32x4 c) {
    const i32x8 A = { (int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0 };
    const i32x8 B = { (int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0 };
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, c, 4, 4, BYTE, sa, BYTE, sb);
}

// 8 codes (a word) times a scale as 8 bf16 or 8 f16.
template <int XT> __device__ __forceinline__ uint4 widen(uint32_t q, float scale) {
    if constexpr (XT == BF16)
        return { __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 0)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 1)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 2)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 3)) };
    else
        return { __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q, scale, 0)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q, scale, 1)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q, scale, 2)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q, scale, 3)) };
}
// 2^(byte - 127) as an operand of the conversions (they read the exponent field), and as an f32 (255: NaN).
constexpr uint32_t FAR = 253;                                   // scale bytes from here on: bf16 does not hold 4 or 6 times them
__device__ __forceinline__ float scale_arg(uint32_t byte) { return __uint_as_float(byte << 23); }
__device__ __forceinline__ float scale_f32(uint32_t byte) {
    const f32x2 v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(2u, scale_arg(byte), 0);      // code 2 is 1
    return v[0];
}

// 8 codes times a quarter of the scale `byte` as 8 bf16, exact whatever the scale: from 2^-130 to 6 x 2^125. (Through f32, which holds the least of
// them after the division; their low halves are zeros.)
__device__ __forceinline__ uint4 widen_quarter(uint32_t q, uint32_t byte) {
    const float scale = scale_arg(byte >= 2 && byte < 255 ? byte - 2 : byte), by = byte < 2 ? 0.25f : 1.f;
    uint32_t w[4];
#define PAIR(i) { const f32x2 v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, i); \
                  w[i] = __float_as_uint(v[0] * by) >> 16 | (__float_as_uint(v[1] * by) & 0xFFFF0000u); }
    PAIR(0) PAIR(1) PAIR(2) PAIR(3)
#undef PAIR
    return { w[0], w[1], w[2], w[3] };
}

// The levels of f16's passes: the largest scale byte of a word (of four), and the largest below `below` (-1: none).
__device__ __forceinline__ int top_byte(uint32_t w) {
    const uint32_t e = w & 0x00FF00FFu, o = (w >> 8) & 0x00FF00FFu;
    return (int)max(max(e & 0xFFFFu, o & 0xFFFFu), max(e >> 16, o >> 16));
}
__device__ __forceinline__ int top_byte_below(uint32_t w, int below) {
    int m = -1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int b = (int)((w >> (8 * i)) & 255u);
        m = b < below ? max(m, b) : m;
    }
    return m;
}
constexpr int LEVEL = 13;                                       // e2m1 x 2^-13 is a normal f16: 2^-14 at least
// A block's scale in a pass over the blocks within LEVEL of `level` and below `below`; the others as 2^-127, which f16 rounds to 0.
__device__ __forceinline__ float pass_scale(int byte, int level, int below) {
    return byte >= level - LEVEL && byte < below ? __uint_as_float((uint32_t)(byte - level + 127) << 23) : 0.f;
}
// The level of a word's pass k, and what it is below.
__device__ __forceinline__ int level_of(uint32_t w, int k, int& below) {
    int l = top_byte(w);
    for (int i = 0; i < k; ++i) {                                // (k is uniform)
        below = l < 0 ? -1 : l - LEVEL;
        l = top_byte_below(w, below);
    }
    return l;
}
__device__ __forceinline__ bool any_code(const uint4& q) { return ((q.x | q.y | q.z | q.w) & 0x77777777u) != 0; }

// ------------------------------------------------------------------------------------------ few rows an expert
// A workgroup: a chunk of up to 16 rows against NS strips of 16 weight rows (with SwiGLU half of them gate rows and half their up
// rows), each wave a part of k; the weights go from memory straight to the matrix units' operands, each byte read
// once, and the parts' sums meet in LDS in a fixed order. Bound by latency for one token (512 experts, bf16 1024 x 2048: 12.0 us, of
// which the 42 MB ask 6.7) and by memory beyond (f16 2048 x 512 at 8 tokens 32 us, 4.9 TB/s; MX4 w, bf16 x, 32 tokens 57 us, 4.7 TB/s, where the
// VALU is busy 30% of the SIMDs' cycles and the matrix units 12%). Four waves and two steps' loads out together, chosen at 13.2, 32 and
// 60 us for these: with four steps 14.4, 36.8 and 85, with eight waves 13.7, 42.5 and 92.
constexpr int ROWS_LOG2 = 4;
constexpr int WAVES = 4;

// What one matrix step reads of the NS weight strips and of x, and its products. FULL: every lane's bytes are inside
// the rows; else what lies past K reads as zeros (and their scales as 2^-127, never as a NaN).
template <int XT, int WT, int NS> struct Step {
    static constexpr int KB = WT == MX4 ? 128 : 32;             // columns of a weight row's 64 bytes
    static constexpr int NX = WT == MX4 && XT != MX4 ? 4 : 1;
    uint4 x[NX];
    uint32_t xsc;

    // w: the strips' first rows (uniform); at: the lane's row and bytes in a strip
    template <bool FULL>
    static __device__ __forceinline__ void load_w(uint4* q, int t, int K, int g, const gaddr* w, uint32_t at) {
        const bool in = FULL || (int64_t)t * KB + (KB / 4) * g < K;
#pragma unroll
        for (int s = 0; s < NS; ++s) q[s] = in ? load16(w[s] + (at + 64u * (uint32_t)t)) : uint4{ 0, 0, 0, 0 };
    }
    // has_x: the lane's row holds one (the others load nothing: what the products of their rows are is not used)
    template <bool FULL>
    __device__ __forceinline__ void load_x(int t, int K, int g, const char* xp, const uint8_t* xs, bool has_x) {
        const int64_t k = (int64_t)t * KB;
        const bool in = has_x && (FULL || k + (KB / 4) * g < K);
#pragma unroll
        for (int j = 0; j < NX; ++j) x[j] = uint4{ 0, 0, 0, 0 };
        xsc = 0;
        if constexpr (XT == MX4) {
            if (in) x[0] = *(const uint4*)(xp + (int64_t)t * 64);
            if (in) xsc = *(const uint32_t*)(xs + 4 * (int64_t)t);
            if (!FULL) xsc &= live_bytes(K, k);
        } else if constexpr (WT != MX4) {
            if (in) x[0] = *(const uint4*)(xp + 2 * (k + 8 * g));
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (in) x[j] = *(const uint4*)(xp + 2 * (k + 32 * g + 8 * j));   // of the lane's block, word j
            }
        }
    }
    // the scale bytes of a step's blocks before column K
    static __device__ __forceinline__ uint32_t live_bytes(int K, int64_t k) {
        const int n = (int)min((int64_t)(K - k) / 32, (int64_t)4);
        return n >= 4 ? 0xFFFFFFFFu : (1u << (8 * n)) - 1u;
    }
    // the products of a strip's 16 bytes: 16-bit weights, or MX4 with the word of their scales
    __device__ __forceinline__ f32x4 multiply(int g, const uint4& q, uint32_t sc, f32x4 acc) const {
        if constexpr (WT != MX4) return mma<XT>(x[0], q, acc);
        else return mma_mx4(x[0], (xsc >> (8 * g)) & 255, q, (sc >> (8 * g)) & 255, acc);
    }
    // MX4 against 16 bits: by a scale as the conversions take it, or by a quarter of a scale's byte
    __device__ __forceinline__ f32x4 multiply_quarter(const uint4& q, uint32_t byte, f32x4 acc) const {
        const uint32_t word[4] = { q.x, q.y, q.z, q.w };
#pragma unroll
        for (int j = 0; j < NX; ++j) acc = mma<XT>(x[j], widen_quarter(word[j], byte), acc);
        return acc;
    }
    __device__ __forceinline__ f32x4 multiply_by(const uint4& q, float f, f32x4 acc) const {
        const uint32_t word[4] = { q.x, q.y, q.z, q.w };
#pragma unroll
        for (int j = 0; j < NX; ++j) acc = mma<XT>(x[j], widen<XT>(word[j], f), acc);
        return acc;
    }
};

template <int XT, int WT, bool SW, int NS>
__global__ __launch_bounds__(64 * WAVES) void k_mg_rows(Exl3c4DevGemm a) {
    constexpr int WV = WAVES, AHEAD = 2;                         // steps whose loads are out together
    typedef Step<XT, WT, NS> S;
    constexpr int OUT = SW ? NS / 2 : NS;                        // strips of y
    __shared__ f32x4 part[WV][NS][64];
    __shared__ int alive[16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, g = lane >> 4;
    const Chunk ch = my_unit<ROWS_LOG2, false>(a, lane, wave);
    if (ch.rows == 0) return;
    const int n0 = ch.tile * (16 * OUT);
    // where strip s of y starts: at the last 16 columns if it would pass them (what it repeats is not stored)
    auto start_of = [&](int s) { return max(min(n0 + 16 * s, a.n_out - 16), 0); };
    const int ysz = a.y_type == EXL3C4_F32 ? 4 : 2;
    if (ch.expert >= 0) {
        const gaddr we = entry(a.w, a.w_stride, ch.expert);
        const gaddr wse = WT == MX4 ? entry(a.ws, a.ws_stride, ch.expert) : nullptr;
        gaddr w[NS], ws[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const int64_t n = start_of(s % OUT) + (s / OUT) * a.n_out;
            w[s] = we + n * a.w_pitch;
            ws[s] = WT == MX4 ? wse + n * a.ws_pitch : nullptr;
        }
        const uint32_t row = (uint32_t)min(l16, a.n_out - 1), at = row * (uint32_t)a.w_pitch + 16 * g;
        const uint32_t s_at = WT == MX4 ? row * (uint32_t)a.ws_pitch : 0;
        const int steps = (a.K + S::KB - 1) / S::KB;
        const int to = (int)((int64_t)steps * (wave + 1) / WV), full = min(to, a.K / S::KB);
        const int xr = l16 < ch.rows ? x_row(a, ch.row0 + l16) : -1;
        if (threadIdx.x < 16) alive[threadIdx.x] = xr >= 0;
        const char* x = a.x + (int64_t)max(xr, 0) * a.x_pitch + (XT == MX4 ? 16 * g : 0);
        const uint8_t* xs = XT == MX4 ? a.xs + (int64_t)max(xr, 0) * a.xs_pitch : nullptr;
        const bool has_x = xr >= 0;
        f32x4 acc[NS] = {};
        uint4 q[AHEAD][NS];
        const int from = (int)((int64_t)steps * wave / WV);
        int t = from;
        uint32_t top = 0;                                        // the largest scale that the lane has multiplied by
        constexpr bool LEVELS = XT == F16 && WT == MX4, QUARTERS = XT == BF16 && WT == MX4;
        // f16 x, MX4 weights: the passes behind the first over steps t .. t + n - 1, each strip's rows from their own level on
        auto more_passes = [&](int t, int n, int* level) {
            bool more;
            do {
                int below[NS], next[NS];
                f32x4 p[NS] = {};
                more = false;
#pragma unroll
                for (int s = 0; s < NS; ++s) {
                    below[s] = level[s] - LEVEL;
                    next[s] = -1;
                    for (int u = 0; u < n; ++u)
                        next[s] = max(next[s], top_byte_below(load4(ws[s] + (s_at + 4u * (uint32_t)(t + u))) &
                                                              S::live_bytes(a.K, (int64_t)(t + u) * S::KB), below[s]));
                }
                for (int u = 0; u < n; ++u) {
                    S st;
                    uint4 v[NS];
                    S::template load_w<false>(v, t + u, a.K, g, w, at);
                    st.template load_x<false>(t + u, a.K, g, x, xs, has_x);
#pragma unroll
                    for (int s = 0; s < NS; ++s) {
                        const int b = ((load4(ws[s] + (s_at + 4u * (uint32_t)(t + u))) &
                                        S::live_bytes(a.K, (int64_t)(t + u) * S::KB)) >> (8 * g)) & 255;
                        p[s] = st.multiply_by(v[s], next[s] < 0 ? 0.f : pass_scale(b, next[s], below[s]), p[s]);
                        more |= next[s] >= 0 && b < next[s] - LEVEL && any_code(v[s]);
                    }
                }
#pragma unroll
                for (int s = 0; s < NS; ++s) {
                    const float f = next[s] < 0 ? 0.f : scale_f32(next[s]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[s][r] = __builtin_fmaf(p[s][r], f, acc[s][r]);
                    level[s] = next[s] < 0 ? -1000 : next[s];
                }
            } while (__any(more));
        };
        for (; t + 4 <= full; t += 4) {                          // (the scale words of four steps are one load a strip)
            uint4 sc[NS];
            f32x4 p[NS] = {};
            int level[NS];
            bool more = false;
#pragma unroll
            for (int s = 0; s < NS; ++s)
                if constexpr (WT == MX4) sc[s] = load_words(ws[s] + (s_at + 4u * (uint32_t)t));
#pragma unroll
            for (int h = 0; h < 4; h += AHEAD) {
                S st[AHEAD];
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) S::template load_w<true>(q[u], t + h + u, a.K, g, w, at);
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) st[u].template load_x<true>(t + h + u, a.K, g, x, xs, has_x);
                if (LEVELS && h == 0)
#pragma unroll
                    for (int s = 0; s < NS; ++s)
                        level[s] = max(max(top_byte(sc[s].x), top_byte(sc[s].y)), max(top_byte(sc[s].z), top_byte(sc[s].w)));
#pragma unroll
                for (int u = 0; u < AHEAD; ++u)
#pragma unroll
                    for (int s = 0; s < NS; ++s) {
                        const uint32_t word = h + u == 0 ? sc[s].x : h + u == 1 ? sc[s].y : h + u == 2 ? sc[s].z : sc[s].w;
                        if constexpr (LEVELS) {
                            const int b = (word >> (8 * g)) & 255;
                            p[s] = st[u].multiply_by(q[u][s], pass_scale(b, level[s], 256), p[s]);
                            more |= b < level[s] - LEVEL && any_code(q[u][s]);
                        } else if constexpr (QUARTERS) {
                            const uint32_t byte = (word >> (8 * g)) & 255;
                            top = max(top, byte);
                            acc[s] = st[u].multiply_by(q[u][s], scale_arg(byte), acc[s]);
                        } else {
                            acc[s] = st[u].multiply(g, q[u][s], word, acc[s]);
                        }
                    }
            }
            if constexpr (LEVELS) {
#pragma unroll
                for (int s = 0; s < NS; ++s) {
                    const float f = scale_f32(level[s]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[s][r] = __builtin_fmaf(p[s][r], f, acc[s][r]);
                }
                if (__any(more)) more_passes(t, 4, level);
            }
        }
        for (; t < to; ++t) {
            if constexpr (LEVELS) {
                int level[NS];
#pragma unroll
                for (int s = 0; s < NS; ++s) level[s] = 256 + LEVEL;
                more_passes(t, 1, level);
            } else if constexpr (QUARTERS) {
                S st;
                S::template load_w<false>(q[0], t, a.K, g, w, at);
                st.template load_x<false>(t, a.K, g, x, xs, has_x);
                const uint32_t live = S::live_bytes(a.K, (int64_t)t * S::KB);
#pragma unroll
                for (int s = 0; s < NS; ++s) {
                    const uint32_t byte = ((load4(ws[s] + (s_at + 4u * (uint32_t)t)) & live) >> (8 * g)) & 255;
                    top = max(top, byte);
                    acc[s] = st.multiply_by(q[0][s], scale_arg(byte), acc[s]);
                }
            } else {
                S st;
                S::template load_w<false>(q[0], t, a.K, g, w, at);
                st.template load_x<false>(t, a.K, g, x, xs, has_x);
                const uint32_t live = WT == MX4 ? S::live_bytes(a.K, (int64_t)t * S::KB) : 0;
#pragma unroll
                for (int s = 0; s < NS; ++s) {
                    uint32_t word = 0;
                    if constexpr (WT == MX4) word = load4(ws[s] + (s_at + 4u * (uint32_t)t)) & live;
                    acc[s] = st.multiply(g, q[0][s], word, acc[s]);
                }
            }
        }
        if (QUARTERS && __any(top >= FAR)) {                     // the wave's sums again, a strip at a time (for registers)
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                f32x4 p = {};
#pragma unroll 1
                for (int u = from; u < to; ++u) {
                    S st;
                    st.template load_x<false>(u, a.K, g, x, xs, has_x);
                    const bool in = (int64_t)u * S::KB + (S::KB / 4) * g < a.K;
                    const uint4 v = in ? load16(w[s] + (at + 64u * (uint32_t)u)) : uint4{ 0, 0, 0, 0 };
                    const uint32_t word = load4(ws[s] + (s_at + 4u * (uint32_t)u)) & S::live_bytes(a.K, (int64_t)u * S::KB);
                    p = st.multiply_quarter(v, (word >> (8 * g)) & 255, p);
                }
                acc[s] = p * 4.f;
            }
        }
#pragma unroll
        for (int s = 0; s < NS; ++s) part[wave][s][lane] = acc[s];
    }
    __syncthreads();
    // thread -> row m, column j of each of its strips: the sums at [strip][16 (m / 4) + j][m % 4]
    const int j = threadIdx.x & 15, m = (threadIdx.x >> 4) & 15;
    if (m >= ch.rows) return;
    const bool live = ch.expert >= 0 && alive[m];
    char* y = a.y + (int64_t)(ch.row0 + m) * a.y_pitch;
    for (int s = threadIdx.x >> 8; s < OUT; s += WV / 4) {
        const int col = start_of(s) + j;
        if (col < n0 + 16 * s || col >= a.n_out) continue;
        float v[2] = { 0.f, 0.f };
        if (live) {
#pragma unroll
            for (int h = 0; h < (SW ? 2 : 1); ++h)
#pragma unroll
                for (int u = 0; u < WV; ++u) v[h] += part[u][s + h * OUT][16 * (m >> 2) + j][m & 3];
            if (SW) v[0] = swiglu(v[0], v[1]);
        }
        store(y + (int64_t)col * ysz, a.y_type, v[0]);
    }
}

// ------------------------------------------------------------------------------------------ many rows an expert
// A workgroup: a tile of MT rows of one expert against NT weight rows (with SwiGLU 16 gate rows and their 16 up rows in turn,
// so that a lane holds both), k in stages. A stage's rows go from memory to LDS without registers
// (global_load_lds_dwordx4), BUFS - 1 stages ahead of the products; a wave waits for its own loads by count, and one barrier
// a stage both publishes them and frees the buffer that the next ones fill.
//
// LDS. A row of a stage is 128 bytes (64 columns in 16 bits, 256 in MX4; x beside MX4 weights: two such halves, and the
// weights' rows 64 bytes). The loads write lane after lane, 16 bytes each, so the order within a row is chosen at the
// source: the chunk at place p of row r is number p ^ (r & 7) (of 64-byte rows p ^ ((r >> 1) & 3)), and the 16 rows and four lane
// groups that read a matrix operand fall on all the banks evenly.
//
// Weights are the A operand here (rows of D): a lane ends with 4 consecutive columns of one row of y.
//
// What bounds it, measured. Where experts have up to some 60 rows, memory: bf16, 200 and 400 tokens of top-10 over 512 experts 5.9 to 6.1 TB/s
// of weights, the card's reading rate. Beyond, the two sides of a stage, which only partly cover each other: bf16, 8192 tokens over 8
// experts (2816 x 2048) 192 us, 1.0 PFLOP/s; without its loads 149 (at the clock that the power then leaves, 1.27 PFLOP/s with starts and
// stores; a plain library product of 8192^3 reaches 1.44 in all), without its products 160: with 256 x 256 tiles two stages
// (128 KB) are all that LDS holds, so that one stage's loads are out at a time. MX4 (the same sizes) 88, 75 and 72.
// Tried without gain (us there): the waves in two halves that take turns with reads and products 211, products of 32 x 32 209, 128 x 256 tiles three stages deep 223, a line
// of each row of later stages asked for ahead 211, stages in another order by workgroup 197 to 202, the next step's operands read ahead
// into registers (188 -> 185, MX4 spilled), loads spread between the products (188 -> 198), four stages of half the columns (64-byte rows
// fetch each line twice: 188 -> 204), one workgroup a CU taking unit after unit with the next one's loads under the last one's
// stores (188 -> 199), weights asked for before the rows of x are known (the same), scales in 16-byte loads (MX4 4096 tokens
// 181 -> 172, but a workgroup less a CU: 2048 Zipf 153 -> 163). Neither the rows' pitch (K = 2048 against 2112) nor the order within
// a line changes the loads' rate.
template <bool B> struct Is { static constexpr bool value = B; };
// A lane holds columns 16 n + 4 g .. + 3 of row 16 (m0 + m) + l16 of the tile (SwiGLU: of gate tile 2 n and up tile 2 n + 1); col0: the wave's
// first column of y. 16 rows at a time cross LDS, in the wave's own part of it (`rows`, TILE_ROWS floats), so that a row's columns go out together, and what
// differs by type and edge is code for one store (stores straight from the lanes, 8 bytes a row each, took the same time and 30 times the code).
template <bool SW, int TN> constexpr int TILE_ROWS = 16 * (16 * (SW ? TN / 2 : TN) + 4);
template <bool SW, int TM, int TN>
__device__ __forceinline__ void store_tile(const Exl3c4DevGemm& a, const Chunk& ch, const int* rows_x, float* rows, const f32x4 (&acc)[TN][TM],
                                           int m0, int col0, int lane) {
    constexpr int TO = SW ? TN / 2 : TN, LANES = 4 * TO, PITCH = 16 * TO + 4;
    const int l16 = lane & 15, g = lane >> 4;
    const int ysz = a.y_type == EXL3C4_F32 ? 4 : 2;
    const bool whole = ((uintptr_t)a.y | (uintptr_t)a.y_pitch) % (4 * ysz) == 0;      // four columns are one aligned store
    const int col = col0 + 4 * (lane % LANES);
#pragma unroll
    for (int m = 0; m < TM; ++m) {
#pragma unroll
        for (int n = 0; n < TO; ++n) {
            f32x4 v = SW ? acc[2 * n][m] : acc[n][m];
            if (SW) v = swiglu4(v, acc[SW ? 2 * n + 1 : n][m]);
            *(f32x4*)(rows + l16 * PITCH + 16 * n + 4 * g) = v;
        }
        wave_sync();                                             // other lanes read what a lane has written
#pragma unroll 1
        for (int i = 0; i < TO; ++i) {
            const int q = i * (64 / LANES) + lane / LANES, r = (m0 + m) * 16 + q;
            f32x4 v = *(const f32x4*)(rows + q * PITCH + 4 * (lane % LANES));
            if (r >= ch.rows) continue;
            if (rows_x[r] < 0) v = f32x4{ 0, 0, 0, 0 };
            store4(a.y + (int64_t)(ch.row0 + r) * a.y_pitch + (int64_t)col * ysz, a.y_type, v, a.n_out - col, whole);
        }
        wave_sync();                                             // and are done before it is written again
    }
}

template <int XT, int WT, bool SW, int MT_LOG2, int NT, int WM, int WN, int BUFS> struct Tile {
    static constexpr int MT = 1 << MT_LOG2, WAVES_ = WM * WN;
    static constexpr bool MIXED = WT == MX4 && XT != MX4;
    static constexpr int KS = WT != MX4 ? 64 : MIXED ? 128 : 256;            // columns a stage
    static constexpr int XROW = MIXED ? 256 : 128, WROW = MIXED ? 64 : 128;  // bytes of a row a stage
    static constexpr int XG = MT * XROW / 1024, WG = NT * WROW / 1024;       // 1-KiB loads a stage
    static constexpr int XS = XT == MX4 ? MT * 8 / 256 : 0, WS = WT == MX4 ? NT * (KS / 32) / 256 : 0;   // of scales, 256 bytes
    static constexpr int XL = XG / WAVES_, WL = WG / WAVES_;
    static constexpr int XSL = (XS + WAVES_ - 1) / WAVES_, WSL = (WS + WAVES_ - 1) / WAVES_;
    static constexpr int LOADS = XL + WL + XSL + WSL;                        // a wave's, every stage
    static constexpr int AT_W = XG * 1024, AT_XS = AT_W + WG * 1024, AT_WS = AT_XS + XS * 256, STAGE = AT_WS + WS * 256;
    static constexpr int TM = MT / WM / 16, TN = NT / WN / 16;               // matrix tiles a wave
    // the chunk that place 4 h + g (before the rows' permutation) holds, for step h and lane group g: MX4 x's chunk 2 g + h, so that
    // a lane group's two blocks have neighbouring scale bytes
    static __device__ __forceinline__ int chunk(int place) { return XT == MX4 ? (place & 3) * 2 + (place >> 2) : place; }
    static_assert(XG % WAVES_ == 0 && WG % WAVES_ == 0 && LOADS * (BUFS - 1) < 64 && TN % 2 == 0, "tile");
};

template <int XT, int WT, bool SW, int MT_LOG2, int NT, int WM, int WN, int BUFS>
__global__ __launch_bounds__(64 * WM * WN) void k_mg_tile(Exl3c4DevGemm a) {
    typedef Tile<XT, WT, SW, MT_LOG2, NT, WM, WN, BUFS> G;
    constexpr int MT = G::MT, WV = WM * WN, KS = G::KS, TM = G::TM, TN = G::TN;
    __shared__ __align__(1024) char lds[BUFS * G::STAGE];
    __shared__ int rows_x[MT];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, g = lane >> 4;
    const int wm = wave / WN, wn = wave % WN;
    const Chunk ch = my_unit<MT_LOG2, true>(a, lane, wave);
    if (ch.rows == 0) return;
    const int n0 = ch.tile * (SW ? NT / 2 : NT);                    // the tile's first column of y
    // row r of the tile -> a row of the weight (past the last one: it again, not stored)
    auto w_row = [&](int r) {
        if (!SW) return min(n0 + r, a.N - 1);
        const int s = r >> 4;
        return min(n0 + 16 * (s >> 1) + (r & 15), a.n_out - 1) + (s & 1) * a.n_out;
    };
    f32x4 acc[TN][TM] = {};
    for (int r = threadIdx.x; r < MT; r += 64 * WV) rows_x[r] = ch.expert >= 0 && r < ch.rows ? x_row(a, ch.row0 + r) : -1;
    __syncthreads();
    if (ch.expert >= 0) {
        const gaddr we = entry(a.w, a.w_stride, ch.expert);
        const gaddr wse = WT == MX4 ? entry(a.ws, a.ws_stride, ch.expert) : nullptr;
        // where each of the wave's loads starts, for this lane: in 128-byte rows lane l takes place l % 8 of row l / 8
        const char* xp[G::XL];
        gaddr wp[G::WL];
        const char* xsp[G::XSL + 1];
        gaddr wsp[G::WSL + 1];
#pragma unroll
        for (int i = 0; i < G::XL; ++i) {
            const int q = wave + i * WV, r = 8 * (G::MIXED ? q >> 1 : q) + (lane >> 3);
            xp[i] = a.x + (int64_t)max(rows_x[r], 0) * a.x_pitch + 16 * G::chunk((lane & 7) ^ (r & 7)) + (G::MIXED ? 128 * (q & 1) : 0);
        }
#pragma unroll
        for (int i = 0; i < G::WL; ++i) {
            const int q = wave + i * WV;
            const int r = G::MIXED ? 16 * q + (lane >> 2) : 8 * q + (lane >> 3);
            wp[i] = we + (int64_t)w_row(r) * a.w_pitch +
                    16 * (G::MIXED ? (lane & 3) ^ ((r >> 1) & 3) : G::chunk((lane & 7) ^ (r & 7)));
        }
#pragma unroll
        for (int i = 0; i < G::XSL; ++i) {
            const int r = 32 * ((wave + i * WV) % max(G::XS, 1)) + (lane >> 1);
            xsp[i] = (const char*)a.xs + (int64_t)max(rows_x[r], 0) * a.xs_pitch + 4 * (lane & 1);
        }
#pragma unroll
        for (int i = 0; i < G::WSL; ++i) {
            const int q = (wave + i * WV) % max(G::WS, 1), r = G::MIXED ? 64 * q + lane : 32 * q + (lane >> 1);
            wsp[i] = wse + (int64_t)w_row(r) * a.ws_pitch + (G::MIXED ? 0 : 4 * (lane & 1));
        }
        const int stages = (a.K + KS - 1) / KS;
        const uint32_t at0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
        auto load = [&](int t, int buf) {
            const uint32_t to = at0 + buf * G::STAGE;
            const int64_t k = (int64_t)t * KS;
            const bool full = k + KS <= a.K;
#pragma unroll
            for (int i = 0; i < G::XL; ++i) {
                const int q = wave + i * WV, r = 8 * (G::MIXED ? q >> 1 : q) + (lane >> 3);
                const int col = (XT == MX4 ? 32 : 8) * G::chunk((lane & 7) ^ (r & 7)) + (G::MIXED ? 64 * (q & 1) : 0);
                const char* p = xp[i] + (int64_t)t * G::XROW;
                if (!full && k + col >= a.K) p = (const char*)&k_zero;
                dma16((gaddr)p, to + q * 1024);
            }
#pragma unroll
            for (int i = 0; i < G::WL; ++i) {
                const int q = wave + i * WV, r = G::MIXED ? 16 * q + (lane >> 2) : 8 * q + (lane >> 3);
                const int col = G::MIXED ? 32 * ((lane & 3) ^ ((r >> 1) & 3)) : (WT == MX4 ? 32 : 8) * G::chunk((lane & 7) ^ (r & 7));
                gaddr p = wp[i] + (int64_t)t * G::WROW;
                if (!full && k + col >= a.K) p = (gaddr)&k_zero;
                dma16(p, to + G::AT_W + q * 1024);
            }
#pragma unroll
            for (int i = 0; i < G::XSL; ++i) {
                const char* p = xsp[i] + (int64_t)t * 8;
                if (!full && k + 128 * (lane & 1) >= a.K) p = (const char*)&k_zero;
                dma4((gaddr)p, to + G::AT_XS + ((wave + i * WV) % max(G::XS, 1)) * 256);
            }
#pragma unroll
            for (int i = 0; i < G::WSL; ++i) {
                gaddr p = wsp[i] + (int64_t)t * (KS / 32);
                if (!full && k + (G::MIXED ? 0 : 128 * (lane & 1)) >= a.K) p = (gaddr)&k_zero;
                dma4(p, to + G::AT_WS + ((wave + i * WV) % max(G::WS, 1)) * 256);
            }
        };
        int top = 0;                                             // bf16 x, MX4 weights: the largest scale that the lane has multiplied by
        // the products of one stage, by quarters of the weights or as they are; last: scale bytes past K (in a word that begins before
        // it) count as 0
        auto multiply = [&](int t, int buf, bool last, auto quarters) {
            const char* X = lds + buf * G::STAGE;
            const char* W = X + G::AT_W;
            const int xr = wm * TM * 16 + l16, wr = wn * TN * 16 + l16;      // the lane's row in the first tile of each
            if constexpr (WT != MX4) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint4 xv[TM], wv[TN];
#pragma unroll
                    for (int i = 0; i < TN; ++i) wv[i] = *(const uint4*)(W + (wr + 16 * i) * 128 + 16 * ((4 * h + g) ^ (l16 & 7)));
#pragma unroll
                    for (int i = 0; i < TM; ++i) xv[i] = *(const uint4*)(X + (xr + 16 * i) * 128 + 16 * ((4 * h + g) ^ (l16 & 7)));
#pragma unroll
                    for (int n = 0; n < TN; ++n)
#pragma unroll
                        for (int m = 0; m < TM; ++m) acc[n][m] = mma<XT>(wv[n], xv[m], acc[n][m]);
                }
            } else if constexpr (XT == MX4) {
                // lane group g takes blocks 2 g and 2 g + 1: their scales are neighbours, and the instruction picks the byte
                const char* XS = X + G::AT_XS + 2 * g;
                const char* WS = X + G::AT_WS + 2 * g;
                int sx[TM], sw[TN], live = 0xFFFF;
                if (last) {
                    const int n = (a.K - t * KS) / 32 - 2 * g;
                    live = n >= 2 ? 0xFFFF : n == 1 ? 0xFF : 0;
                }
#pragma unroll
                for (int i = 0; i < TN; ++i) sw[i] = *(const uint16_t*)(WS + (wr + 16 * i) * 8) & live;
#pragma unroll
                for (int i = 0; i < TM; ++i) sx[i] = *(const uint16_t*)(XS + (xr + 16 * i) * 8) & live;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint4 xv[TM], wv[TN];
#pragma unroll
                    for (int i = 0; i < TN; ++i) wv[i] = *(const uint4*)(W + (wr + 16 * i) * 128 + 16 * ((4 * h + g) ^ (l16 & 7)));
#pragma unroll
                    for (int i = 0; i < TM; ++i) xv[i] = *(const uint4*)(X + (xr + 16 * i) * 128 + 16 * ((4 * h + g) ^ (l16 & 7)));
#pragma unroll
                    for (int n = 0; n < TN; ++n)
#pragma unroll
                        for (int m = 0; m < TM; ++m)
                            acc[n][m] = h == 0 ? mma_mx4<0>(wv[n], sw[n], xv[m], sx[m], acc[n][m])
                                               : mma_mx4<1>(wv[n], sw[n], xv[m], sx[m], acc[n][m]);
                }
            } else {
                const char* WS = X + G::AT_WS;
                uint32_t live = 0xFFFFFFFFu;
                if (last) {
                    const int n = (a.K - t * KS) / 32;
                    live = n >= 4 ? 0xFFFFFFFFu : (1u << (8 * n)) - 1u;
                }
                uint4 q[TN];
#pragma unroll
                for (int i = 0; i < TN; ++i) q[i] = *(const uint4*)(W + (wr + 16 * i) * 64 + 16 * (g ^ ((l16 >> 1) & 3)));
                // x's 16 bytes of columns 8 u .. 8 u + 7 of the stage
                auto x_at = [&](int m, int u) {
                    return *(const uint4*)(X + ((xr >> 3) + 2 * m) * 2048 + (u >> 3) * 1024 + (l16 & 7) * 128 + 16 * ((u & 7) ^ (l16 & 7)));
                };
                int byte[TN];
#pragma unroll
                for (int i = 0; i < TN; ++i) byte[i] = ((*(const uint32_t*)(WS + (wr + 16 * i) * 4) & live) >> (8 * g)) & 255;
                // the products with the weights' blocks scaled by f, added to `to`
                auto pass = [&](const float* f, f32x4 (*to)[TM]) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint4 xv[TM];
#pragma unroll
                        for (int m = 0; m < TM; ++m) xv[m] = x_at(m, 4 * g + j);
#pragma unroll
                        for (int n = 0; n < TN; ++n) {
                            const uint32_t word[4] = { q[n].x, q[n].y, q[n].z, q[n].w };
                            const uint4 wv = widen<XT>(word[j], f[n]);
#pragma unroll
                            for (int m = 0; m < TM; ++m) to[n][m] = mma<XT>(wv, xv[m], to[n][m]);
                        }
                    }
                };
                float f[TN];
                if constexpr (decltype(quarters)::value) {
#pragma unroll 1
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int n = 0; n < TN; ++n) {
                            const uint4 wv = widen_quarter(j == 0 ? q[n].x : j == 1 ? q[n].y : j == 2 ? q[n].z : q[n].w, byte[n]);
#pragma unroll
                            for (int m = 0; m < TM; ++m) acc[n][m] = mma<XT>(wv, x_at(m, 4 * g + j), acc[n][m]);
                        }
                } else if constexpr (XT == BF16) {
#pragma unroll
                    for (int n = 0; n < TN; ++n) f[n] = scale_arg(byte[n]), top = max(top, byte[n]);
                    pass(f, acc);
                } else {
                    // The rows of D are the weights': lane group g's are 4 g + r, whose scale words are 16 bytes in LDS. Each row's level
                    // follows from its word alone, so that the lanes that convert a row and those that hold its sums agree on it.
                    // (Everything but the sums is read again in the rare passes behind the first, for registers.)
                    bool more;
                    auto level_pass = [&](int k) {
                        f32x4 p[TN][TM] = {};
                        more = false;
#pragma unroll
                        for (int n = 0; n < TN; ++n) {
                            int below = 256;
                            const int l = level_of(*(const uint32_t*)(WS + (wr + 16 * n) * 4) & live, k, below);
                            f[n] = l < 0 ? 0.f : pass_scale(byte[n], l, below);
                            more |= byte[n] < l - LEVEL && any_code(q[n]);
                        }
                        pass(f, p);
#pragma unroll
                        for (int n = 0; n < TN; ++n) {
                            const uint4 w = *(const uint4*)(WS + (wr - l16 + 16 * n + 4 * g) * 4);
                            const uint32_t word[4] = { w.x, w.y, w.z, w.w };
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                int below = 256;
                                const int l = level_of(word[r] & live, k, below);
                                const float s = l < 0 ? 0.f : scale_f32(l);
#pragma unroll
                                for (int m = 0; m < TM; ++m) acc[n][m][r] = __builtin_fmaf(p[n][m][r], s, acc[n][m][r]);
                            }
                        }
                    };
                    level_pass(0);
                    for (int k = 1; __any(more); ++k) level_pass(k);
                }
            }
        };
        auto sum = [&](auto quarters) {
#pragma unroll
            for (int i = 0; i < BUFS - 1; ++i)
                if (i < stages) load(i, i);
            int buf = 0;
            for (int t = 0; t < stages; ++t) {
                if (BUFS == 2 || t + 1 >= stages) wait_loads<0>();
                else wait_loads<G::LOADS>();
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                const int next = buf == 0 ? BUFS - 1 : buf - 1;  // the buffer of stage t - 1, read by all before the barrier
                if (t + BUFS - 1 < stages) load(t + BUFS - 1, next);
                multiply(t, buf, t + 1 == stages, quarters);
                asm volatile("" ::: "memory");
                buf = buf + 1 == BUFS ? 0 : buf + 1;
            }
        };
        sum(Is<false>());
        if constexpr (XT == BF16 && WT == MX4) {
            if (__syncthreads_or(top >= (int)FAR)) {             // the tile's sums again
#pragma unroll
                for (int n = 0; n < TN; ++n)
#pragma unroll
                    for (int m = 0; m < TM; ++m) acc[n][m] = f32x4{ 0, 0, 0, 0 };
                sum(Is<true>());
#pragma unroll
                for (int n = 0; n < TN; ++n)
#pragma unroll
                    for (int m = 0; m < TM; ++m) acc[n][m] *= 4.f;
            }
        }
    }
    static_assert(WV * TILE_ROWS<SW, TN> * 4 <= (int)sizeof(lds), "the rows fit the stages' buffers");
    __syncthreads();
    store_tile<SW, TM, TN>(a, ch, rows_x, (float*)lds + wave * TILE_ROWS<SW, TN>, acc, wm * TM, n0 + wn * (SW ? TN / 2 : TN) * 16, lane);
}

template <int XT, int WT, bool SW, int NS>
int launch_rows(Exl3c4DevGemm& a, hipStream_t st) {
    constexpr int cols = 16 * (SW ? NS / 2 : NS);
    a.tiles = (a.n_out + cols - 1) / cols;
    const int64_t grid = chunk_bound(a.T, a.n_expert, 1 << ROWS_LOG2) * a.tiles;
    if (grid > THREADS / (64 * WAVES)) return EXL3C4_E_SHAPE;
    hipLaunchKernelGGL((k_mg_rows<XT, WT, SW, NS>), dim3((unsigned)grid), dim3(64 * WAVES), 0, st, a);
    return launched();
}

template <int XT, int WT, bool SW, int MT_LOG2, int NT, int WM, int WN, int BUFS>
int launch_tile(Exl3c4DevGemm& a, hipStream_t st) {
    constexpr int cols = SW ? NT / 2 : NT;
    a.tiles = (a.n_out + cols - 1) / cols;
    const int64_t grid = (chunk_bound(a.T, a.n_expert, 1 << MT_LOG2) * a.tiles + 7) / 8 * 8;
    if (grid > THREADS / (64 * WM * WN)) return EXL3C4_E_SHAPE;
    hipLaunchKernelGGL((k_mg_tile<XT, WT, SW, MT_LOG2, NT, WM, WN, BUFS>), dim3((unsigned)grid), dim3(64 * WM * WN), 0, st, a);
    return launched();
}

// Which kernel, and how large a tile: by the types, the sizes and the rows that an expert has at least on average, r = T / min(E, T)
// -- never by the routing, which is on the device. Larger tiles read weights and rows less often; smaller ones waste
// less of a chunk, make more workgroups and start sooner. Measured on one card, us with x's quantisation where x is MX4 (E / top-k, N x K, tokens; SwiGLU
// where E > 1; "down": 2048 columns of y, sorted rows in):
//   rows against tiles     bf16 512/10 1024x2048: 32 tokens 169 / 168, 64 256 / 248, 200 357 / 337. MX4 64: 84 / 78, 200 117 / 105.
//                          bf16 x, MX4 w 64: 83 / 97, 200 116 / 131; 64/6 at 400 49 / 22. One expert, 77 rows 512x2048: 8.5 / 15.8.
//   32 rows against 64     8/2 at 400 tokens: bf16 16.1 / 19.4, MX4 10.8 / 13.6; MX4 512/10 at 200 105 / 110, at 2048 Zipf 163 / 144; MX4 w at 4096:
//                          bf16 x 317 / 302, f16 x 425 / 444 (its 64-row tiles hold 236 registers, two waves a SIMD).
//   64 against 128         bf16 512/10 at 4096 518 / 412, 64/6 at 2000 107 / 94; MX4 184 / 167, 46 / 39; bf16 x, MX4 w 302 / 387 (not built).
//   128 against 256        bf16 64/6 at 2000 94 / 85, 8/2 2816x2048 at 8192 224 / 186; MX4 64/6 at 2000 39 / 31, 8/2 2816x2048 at 8192 94 / 82.
//                          MX4 by K, 8/2 at 8192: down 1024 60 / 63, 1408 72 / 77, 1792 80 / 83, 2048 91 / 91, 2560 99 / 105; 2816 with SwiGLU
//                          1024 63 / 54, 1408 78 / 68, 1792 83 / 75, 2560 112 / 95: less the stages of a tile than how full the last of
//                          the 256 CUs' two or three rounds is. The rule's K >= 2048 keeps a short K's down at 128 and gives up 8 to 10 us of its gate and up.
// Returns a tile's rows (32, 64, 128, 256), or for few rows an expert the strips of a workgroup (2, 4).
int choose(int x_type, int w_type, bool swiglu, int64_t T, int64_t n_expert, int64_t n_out, int64_t K) {
    const bool mixed = w_type == MX4 && x_type != MX4;
    const int64_t live = n_expert < T ? n_expert : T;
    // workgroups of tiles of `rows` x `cols` (SwiGLU: half as many columns of y)
    auto units = [&](int rows, int cols) {
        if (swiglu) cols /= 2;
        return chunk_bound(T, n_expert, rows) * ((n_out + cols - 1) / cols);
    };
    if (T <= (mixed ? 8 : 1) * live || units(32, 128) < 64 || (T <= 4 * live && units(32, 128) < 256))
        return units(16, 64) >= 1024 ? 4 : 2;
    if (mixed) return units(64, 128) < 256 ? 32 : 64;
    if (T > 160 * live && units(256, 256) >= 256 && (w_type != MX4 || K >= 2048)) return 256;
    if (T > 64 * live && units(128, 128) >= 256) return 128;
    if ((w_type == MX4 && T <= 16 * live) || units(64, 128) < 256) return 32;
    return 64;
}

template <int XT, int WT, bool SW>
int launch(Exl3c4DevGemm& a, hipStream_t st) {
    constexpr bool mixed = WT == MX4 && XT != MX4;
    const int path = choose(XT, WT, SW, a.T, a.n_expert, a.n_out, a.K);
    if (path == 2) return launch_rows<XT, WT, SW, 2>(a, st);
    if (path == 4) return launch_rows<XT, WT, SW, 4>(a, st);
    if (path == 32) return launch_tile<XT, WT, SW, 5, 128, 1, 4, 3>(a, st);
    if constexpr (!mixed) {
        if (path == 256) return launch_tile<XT, WT, SW, 8, 256, 2, 4, 2>(a, st);
        if (path == 128) return launch_tile<XT, WT, SW, 7, 128, 2, WT == MX4 ? 2 : 4, 2>(a, st);
    }
    return launch_tile<XT, WT, SW, 6, 128, 1, 4, WT == MX4 ? 2 : 3>(a, st);
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

extern "C" int exl3c4_dev_gemm_path(int32_t x_type, int32_t w_type, int32_t act, int64_t T, int64_t n_expert, int64_t N, int64_t K) {
    const bool swiglu = act == EXL3C4_ACT_SWIGLU;
    return choose(x_type, w_type, swiglu, T, n_expert, swiglu ? N / 2 : N, K);
}
