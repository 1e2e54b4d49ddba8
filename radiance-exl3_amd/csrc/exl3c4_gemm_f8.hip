// exl3c4_gemm_f8.hip -- the products of routed experts whose weights are F8 (e4m3 codes, an f32 scale each 128 x 128), against x in F8 (a
// scale each row and 128 columns), f16 or bf16, on gfx950 (wave64): y[i] = W_e x[row i] over the sorted rows of each expert's run, with SwiGLU
// where asked (include/exl3c4.h). No counterpart in the reference.
//
// THE MATRIX STEP. A block of 128 columns is one step: y += sw sx (sum over the block of w x). Scales are any f32 numbers, so they come in as a
// multiply-add of the sum, which begins at zero. It is taken in one of two ways:
//   widened   the codes become 16-bit floats, which hold every e4m3 (bf16 for bf16 x, else f16), and four v_mfma_f32_16x16x32 add their products, each
//             exact in f32.
//   as codes  one v_mfma_f32_16x16x128_f8f6f4, at some three times the rate. It adds eight neighbouring columns' products on a grid: each is cut
//             towards zero to a multiple of 2^(E - 13), E the largest of the eight sums of the two codes' exponents; the eights are then added in
//             f32 (found by giving it one product at a time beside a large one). A sum is off by less than 7 x 2^-13 of the largest product of
//             each eight; of normally distributed rows by 1.4e-5 of the products' norm.
// Few rows against many weights are bound by memory, and widen. Tiles take F8 x as codes where y has 16 bits, whose own rounding (2^-9 or 2^-12 of the
// value) and the codes' (2^-4) are far larger; where y is f32 they widen too.
// Lane l holds of row l % 16, with g = l / 16, the 16 columns from 16 g and those from 64 + 16 g of the block.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include "exl3c4_dev.h"
#include "exl3c4_gemm_dev.h"

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf2_t __attribute__((ext_vector_type(2)));

constexpr int F8 = EXL3C4_F8;

// A lane's 32 codes of a row's block.
struct Codes { uint4 h[2]; };

__device__ __forceinline__ f32x4 mma_f8(const Codes& a, const Codes& b, f32x4 c) {
    const i32x8 A = { (int)a.h[0].x, (int)a.h[0].y, (int)a.h[0].z, (int)a.h[0].w, (int)a.h[1].x, (int)a.h[1].y, (int)a.h[1].z, (int)a.h[1].w };
    const i32x8 B = { (int)b.h[0].x, (int)b.h[0].y, (int)b.h[0].z, (int)b.h[0].w, (int)b.h[1].x, (int)b.h[1].y, (int)b.h[1].z, (int)b.h[1].w };
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, c, 0, 0, 0, 127, 0, 127);      // (e8m0 127: times 1)
}

// 8 codes as 8 bf16 or f16 (e4m3 has four bits and exponents of -9 to 8: exact).
template <int XT> __device__ __forceinline__ uint4 widen8(uint32_t lo, uint32_t hi) {
    if constexpr (XT == BF16)
        return { __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true)) };
    else
        return { __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true)) };
}
// Eight codes of the lane's 32, j = 0 .. 3.
template <int XT> __device__ __forceinline__ uint4 widen_part(const Codes& q, int j) {
    const uint4& w = q.h[j >> 1];
    return j & 1 ? widen8<XT>(w.z, w.w) : widen8<XT>(w.x, w.y);
}

// The type that F8 codes widen to beside x of type XT.
template <int XT> constexpr int WIDER = XT == BF16 ? BF16 : F16;

__device__ __forceinline__ float load_f32(gaddr p) { return *(const __attribute__((address_space(1))) float*)p; }
__device__ __forceinline__ float word(const uint4& v, int i) { return __uint_as_float(i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w); }

// Rows of blocks of a weight, and the one that holds its row n (of a half with SwiGLU).
__device__ __forceinline__ int64_t scale_row(int n, int half, int n_out) { return (n >> 7) + (int64_t)half * ((n_out + 127) >> 7); }

// ------------------------------------------------------------------------------------------ few rows an expert
// A workgroup: a chunk of up to 16 rows against NS strips of 16 weight rows (with SwiGLU half of them gate rows and half their up rows), each wave
// a part of k; the weights go from memory straight to the matrix units' operands, each byte read once, and the parts' sums meet in LDS in a
// fixed order. x is the A operand (rows of D), W the B operand: lane l ends with D[m = 4 g + r][n = l % 16].
constexpr int ROWS_LOG2 = 4;
constexpr int WAVES = 4;

template <int XT, bool SW, int NS>
__global__ __launch_bounds__(64 * WAVES) void k_f8_rows(Exl3c4DevGemm a) {
    constexpr int WV = WAVES, AHEAD = 2;                         // steps whose loads are out together
    constexpr int OUT = SW ? NS / 2 : NS;                        // strips of y
    constexpr int NX = XT == F8 ? 2 : 4;                         // 16-byte loads of x a step
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
        const gaddr we = entry(a.w, a.w_stride, ch.expert), wse = entry(a.ws, a.ws_stride, ch.expert);
        gaddr w[NS], ws[NS];
        const int row = min(l16, a.n_out - 1);                   // the lane's row in a strip
        const uint32_t at = (uint32_t)row * (uint32_t)a.w_pitch + 16 * g;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const int n = start_of(s % OUT);
            w[s] = we + (n + (int64_t)(s / OUT) * a.n_out) * a.w_pitch;
            ws[s] = wse + scale_row(n + row, s / OUT, a.n_out) * a.ws_pitch;
        }
        const int steps = (a.K + 127) / 128;
        const int from = (int)((int64_t)steps * wave / WV), to = (int)((int64_t)steps * (wave + 1) / WV), full = min(to, a.K / 128);
        const int xr = l16 < ch.rows ? x_row(a, ch.row0 + l16) : -1;
        if (threadIdx.x < 16) alive[threadIdx.x] = xr >= 0;
        const char* x = a.x + (int64_t)max(xr, 0) * a.x_pitch + (XT == F8 ? 16 : 32) * g;
        const bool has_x = xr >= 0;
        gaddr xs[4] = {};                                        // the scales of rows 4 g + r
        if constexpr (XT == F8) {
#pragma unroll
            for (int r = 0; r < 4; ++r) xs[r] = (gaddr)a.xs + (int64_t)max(__shfl(xr, 4 * g + r), 0) * a.xs_pitch;
        }
        // a step's loads: codes of the NS strips and the lane's part of x; what lies past K reads as zeros
        auto load_w = [&](Codes* q, int t, bool whole) {
#pragma unroll
            for (int s = 0; s < NS; ++s)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    q[s].h[h] = whole || (int64_t)t * 128 + 64 * h + 16 * g < a.K ? load16(w[s] + at + ((int64_t)t * 128 + 64 * h)) : uint4{ 0, 0, 0, 0 };
        };
        auto load_x = [&](uint4* v, int t, bool whole) {
#pragma unroll
            for (int j = 0; j < NX; ++j) {
                // F8: the lane's 16 columns of half j; 16 bits: 8 columns, two to a half
                const int64_t k = (int64_t)t * 128 + (XT == F8 ? 64 * j : 64 * (j >> 1) + 8 * (j & 1));
                const bool in = has_x && (whole || k + 16 * g < a.K);
                v[j] = in ? *(const uint4*)(x + (XT == F8 ? k : 2 * k)) : uint4{ 0, 0, 0, 0 };
            }
        };
        f32x4 acc[NS] = {};
        // one step's products, scaled: sx of the lane's four rows of D
        auto step = [&](const Codes* q, const uint4* v, const float* sw, const float* sx) {
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                f32x4 p = { 0, 0, 0, 0 };
#pragma unroll
                for (int j = 0; j < 4; ++j) p = mma<WIDER<XT>>(XT == F8 ? widen_part<F16>(Codes{ v[0], v[1] }, j) : v[j], widen_part<WIDER<XT>>(q[s], j), p);
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[s][r] = __builtin_fmaf(p[r], XT == F8 ? sx[r] * sw[s] : sw[s], acc[s][r]);
            }
        };
        int t = from;
        for (; t + 4 <= full; t += 4) {                          // (the scales of four steps are one load a strip, and one a row of x)
            uint4 sw4[NS], sx4[4] = {};
#pragma unroll
            for (int s = 0; s < NS; ++s) sw4[s] = load_words(ws[s] + 4 * (int64_t)t);
            if constexpr (XT == F8)
#pragma unroll
                for (int r = 0; r < 4; ++r) sx4[r] = load_words(xs[r] + 4 * (int64_t)t);
#pragma unroll
            for (int h = 0; h < 4; h += AHEAD) {
                Codes q[AHEAD][NS];
                uint4 v[AHEAD][NX];
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) load_w(q[u], t + h + u, true);
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) load_x(v[u], t + h + u, true);
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) {
                    float sw[NS], sx[4];
#pragma unroll
                    for (int s = 0; s < NS; ++s) sw[s] = word(sw4[s], h + u);
#pragma unroll
                    for (int r = 0; r < 4; ++r) sx[r] = word(sx4[r], h + u);
                    step(q[u], v[u], sw, sx);
                }
            }
        }
        for (; t < to; ++t) {
            Codes q[NS];
            uint4 v[NX];
            float sw[NS], sx[4] = {};
            load_w(q, t, false);
            load_x(v, t, false);
#pragma unroll
            for (int s = 0; s < NS; ++s) sw[s] = load_f32(ws[s] + 4 * (int64_t)t);
            if constexpr (XT == F8)
#pragma unroll
                for (int r = 0; r < 4; ++r) sx[r] = load_f32(xs[r] + 4 * (int64_t)t);
            step(q, v, sw, sx);
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
// A workgroup: a tile of MT rows of one expert against NT weight rows (with SwiGLU 16 gate rows and their 16 up rows in turn, so that a lane holds
// both), k in stages of one block of 128 columns. A stage's rows and scales go from memory to LDS without registers, BUFS - 1 stages ahead of the
// products; a wave waits for its own loads by count, and one barrier a stage both publishes them and frees the buffer that the next ones fill.
//
// LDS. A row of a stage is 128 bytes (16-bit x: two such halves). The loads write lane after lane, 16 bytes each, so the order within a row is chosen
// at the source: place p of row r holds the chunk p ^ (r & 7), and the 16 rows and four lane groups that read a matrix operand fall on all the
// banks evenly. Behind them the scales: one of each row of x, and those of the tile's blocks of weight rows.
//
// Weights are the A operand here (rows of D): a lane ends with 4 consecutive columns of one row of y, so that a sum's scale is one number of the
// lane's row of x times one that the wave shares.
template <int XT, bool SW, int MT_LOG2, int NT, int WM, int WN, int BUFS> struct Tile {
    static constexpr int MT = 1 << MT_LOG2, WAVES_ = WM * WN;
    static constexpr int XROW = XT == F8 ? 128 : 256;                        // bytes of a row of x a stage
    static constexpr int XG = MT * XROW / 1024, WG = NT * 128 / 1024;        // 1-KiB loads a stage
    static constexpr int XS = XT == F8 ? (MT + 63) / 64 : 0;                 // of x's scales, 64 each
    static constexpr int XL = XG / WAVES_, WL = WG / WAVES_, XSL = (XS + WAVES_ - 1) / WAVES_;
    static constexpr int LOADS = XL + WL + XSL + 1;                          // a wave's, every stage
    static constexpr int AT_W = XG * 1024, AT_XS = AT_W + WG * 1024, AT_WS = AT_XS + XS * 256, STAGE = AT_WS + 256;
    static constexpr int TM = MT / WM / 16, TN = NT / WN / 16;               // matrix tiles a wave
    static_assert(XG % WAVES_ == 0 && WG % WAVES_ == 0 && LOADS * (BUFS - 1) < 64 && TN % 2 == 0, "tile");
    static_assert(NT == 128 || NT == 256, "one or two blocks of weight rows");
};

template <int XT, bool WIDE, bool SW, int MT_LOG2, int NT, int WM, int WN, int BUFS>
__global__ __launch_bounds__(64 * WM * WN) void k_f8_tile(Exl3c4DevGemm a) {
    typedef Tile<XT, SW, MT_LOG2, NT, WM, WN, BUFS> G;
    constexpr int MT = G::MT, WV = WM * WN, TM = G::TM, TN = G::TN;
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
        const gaddr we = entry(a.w, a.w_stride, ch.expert), wse = entry(a.ws, a.ws_stride, ch.expert);
        // where each of the wave's loads starts, for this lane: lane l takes place l % 8 of row l / 8
        const char* xp[G::XL];
        gaddr wp[G::WL];
        const char* xsp[G::XSL + 1];
#pragma unroll
        for (int i = 0; i < G::XL; ++i) {
            const int q = wave + i * WV, r = 8 * (XT == F8 ? q : q >> 1) + (lane >> 3);
            xp[i] = a.x + (int64_t)max(rows_x[r], 0) * a.x_pitch + 16 * ((lane & 7) ^ (r & 7)) + (XT == F8 ? 0 : 128 * (q & 1));
        }
#pragma unroll
        for (int i = 0; i < G::WL; ++i) {
            const int r = 8 * (wave + i * WV) + (lane >> 3);
            wp[i] = we + (int64_t)w_row(r) * a.w_pitch + 16 * ((lane & 7) ^ (r & 7));
        }
#pragma unroll
        for (int i = 0; i < G::XSL; ++i) {
            const int r = (64 * ((wave + i * WV) % max(G::XS, 1)) + lane) % MT;
            xsp[i] = (const char*)a.xs + (int64_t)max(rows_x[r], 0) * a.xs_pitch;
        }
        // the scales of the tile's weight rows: even lanes of its first block (SwiGLU: of the gate rows), odd lanes of the second (of the up rows)
        const gaddr wsp = wse + (SW ? scale_row(n0, lane & 1, a.n_out) : scale_row(min(n0 + (lane & 1) * 128, a.N - 1), 0, a.N)) * a.ws_pitch;
        const int stages = (a.K + 127) / 128;
        const uint32_t at0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
        auto load = [&](int t, int buf) {
            const uint32_t to = at0 + buf * G::STAGE;
            const int64_t k = (int64_t)t * 128;
            const bool full = k + 128 <= a.K;
#pragma unroll
            for (int i = 0; i < G::XL; ++i) {
                const int q = wave + i * WV, r = 8 * (XT == F8 ? q : q >> 1) + (lane >> 3);
                const int col = XT == F8 ? 16 * ((lane & 7) ^ (r & 7)) : 8 * ((lane & 7) ^ (r & 7)) + 64 * (q & 1);
                const char* p = xp[i] + (int64_t)t * G::XROW;
                if (!full && k + col >= a.K) p = (const char*)&k_zero;
                dma16((gaddr)p, to + q * 1024);
            }
#pragma unroll
            for (int i = 0; i < G::WL; ++i) {
                const int q = wave + i * WV, r = 8 * q + (lane >> 3);
                gaddr p = wp[i] + (int64_t)t * 128;
                if (!full && k + 16 * ((lane & 7) ^ (r & 7)) >= a.K) p = (gaddr)&k_zero;
                dma16(p, to + G::AT_W + q * 1024);
            }
#pragma unroll
            for (int i = 0; i < G::XSL; ++i)
                dma4((gaddr)(xsp[i] + 4 * (int64_t)t), to + G::AT_XS + ((wave + i * WV) % max(G::XS, 1)) * 256);
            dma4(wsp + 4 * (int64_t)t, to + G::AT_WS);           // (every wave the same ones: a wait counts alike in all)
        };
        const int xr = wm * TM * 16 + l16, wr = wn * TN * 16 + l16;      // the lane's row in the first tile of each
        auto multiply = [&](int buf) {
            const char* X = lds + buf * G::STAGE;
            const char* W = X + G::AT_W;
            const float* XS = (const float*)(X + G::AT_XS);
            const float* WS = (const float*)(X + G::AT_WS);
            auto codes = [&](const char* p, int row) {
                return Codes{ *(const uint4*)(p + row * 128 + 16 * (g ^ (l16 & 7))), *(const uint4*)(p + row * 128 + 16 * ((4 + g) ^ (l16 & 7))) };
            };
            // (a wave's weight rows lie in one block of 128; with SwiGLU its even tiles in the gate's, its odd ones in the up's)
            const float sw[2] = { WS[SW ? 0 : (wn * TN * 16) >> 7], WS[1] };
            if constexpr (!WIDE) {
                Codes wv[TN];
#pragma unroll
                for (int n = 0; n < TN; ++n) wv[n] = codes(W, wr + 16 * n);
#pragma unroll
                for (int m = 0; m < TM; ++m) {
                    const Codes xv = codes(X, xr + 16 * m);
                    const float sx = XS[xr + 16 * m], f[2] = { sx * sw[0], sx * sw[1] };
#pragma unroll
                    for (int n = 0; n < TN; ++n) {
                        const f32x4 p = mma_f8(wv[n], xv, f32x4{ 0, 0, 0, 0 });
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[n][m][r] = __builtin_fmaf(p[r], f[SW ? n & 1 : 0], acc[n][m][r]);
                    }
                }
            } else {
                // x's eights j of columns: 16 g + 8 j of the block's first half, then of its second
                uint4 xv[TM][4];
                float sx[TM];
#pragma unroll
                for (int m = 0; m < TM; ++m) {
                    if constexpr (XT == F8) {
                        const Codes c = codes(X, xr + 16 * m);
#pragma unroll
                        for (int j = 0; j < 4; ++j) xv[m][j] = widen_part<F16>(c, j);
                        sx[m] = XS[xr + 16 * m];
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            xv[m][j] = *(const uint4*)(X + ((xr >> 3) + 2 * m) * 2048 + (j >> 1) * 1024 + (l16 & 7) * 128 + 16 * ((2 * g + (j & 1)) ^ (l16 & 7)));
                    }
                }
#pragma unroll
                for (int n = 0; n < TN; ++n) {
                    const Codes q = codes(W, wr + 16 * n);
                    f32x4 p[TM] = {};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint4 w = widen_part<WIDER<XT>>(q, j);
#pragma unroll
                        for (int m = 0; m < TM; ++m) p[m] = mma<WIDER<XT>>(w, xv[m][j], p[m]);
                    }
#pragma unroll
                    for (int m = 0; m < TM; ++m) {
                        const float f = XT == F8 ? sx[m] * sw[SW ? n & 1 : 0] : sw[SW ? n & 1 : 0];
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[n][m][r] = __builtin_fmaf(p[m][r], f, acc[n][m][r]);
                    }
                }
            }
        };
#pragma unroll
        for (int i = 0; i < BUFS - 1; ++i)
            if (i < stages) load(i, i);
        int buf = 0;
        for (int t = 0; t < stages; ++t) {
            if (BUFS == 2 || t + 1 >= stages) wait_loads<0>();
            else wait_loads<G::LOADS>();
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            const int next = buf == 0 ? BUFS - 1 : buf - 1;      // the buffer of stage t - 1, read by all before the barrier
            if (t + BUFS - 1 < stages) load(t + BUFS - 1, next);
            multiply(buf);
            asm volatile("" ::: "memory");
            buf = buf + 1 == BUFS ? 0 : buf + 1;
        }
    }
    static_assert(WV * TILE_ROWS<SW, TN> * 4 <= (int)sizeof(lds), "the rows fit the stages' buffers");
    __syncthreads();
    store_tile<SW, TM, TN>(a, ch, rows_x, (float*)lds + wave * TILE_ROWS<SW, TN>, acc, wm * TM, n0 + wn * (SW ? TN / 2 : TN) * 16, lane);
}

template <int XT, bool SW, int NS>
int launch_rows(Exl3c4DevGemm& a, hipStream_t st) {
    constexpr int cols = 16 * (SW ? NS / 2 : NS);
    a.tiles = (a.n_out + cols - 1) / cols;
    const int64_t grid = chunk_bound(a.T, a.n_expert, 1 << ROWS_LOG2) * a.tiles;
    if (grid > THREADS / (64 * WAVES)) return EXL3C4_E_SHAPE;
    hipLaunchKernelGGL((k_f8_rows<XT, SW, NS>), dim3((unsigned)grid), dim3(64 * WAVES), 0, st, a);
    return launched();
}

template <int XT, bool WIDE, bool SW, int MT_LOG2, int NT, int WM, int WN, int BUFS>
int launch_tile(Exl3c4DevGemm& a, hipStream_t st) {
    constexpr int cols = SW ? NT / 2 : NT;
    a.tiles = (a.n_out + cols - 1) / cols;
    const int64_t grid = (chunk_bound(a.T, a.n_expert, 1 << MT_LOG2) * a.tiles + 7) / 8 * 8;
    if (grid > THREADS / (64 * WM * WN)) return EXL3C4_E_SHAPE;
    hipLaunchKernelGGL((k_f8_tile<XT, WIDE, SW, MT_LOG2, NT, WM, WN, BUFS>), dim3((unsigned)grid), dim3(64 * WM * WN), 0, st, a);
    return launched();
}

// Which kernel, and how large a tile: by the types, the sizes and the rows that an expert has at least on average, r = T / min(E, T) -- never by
// the routing, which is on the device. Returns a tile's rows (32, 64, 128, 256), or for few rows an expert the strips of a workgroup (2, 4).
int choose(bool wide, bool swiglu, int64_t T, int64_t n_expert, int64_t n_out, int64_t K) {
    const int64_t live = n_expert < T ? n_expert : T;
    // workgroups of tiles of `rows` x `cols` (SwiGLU: half as many columns of y)
    auto units = [&](int rows, int cols) {
        if (swiglu) cols /= 2;
        return chunk_bound(T, n_expert, rows) * ((n_out + cols - 1) / cols);
    };
    if (T <= (wide ? 8 : 1) * live || units(32, 128) < 64 || (T <= 4 * live && units(32, 128) < 256)) return units(16, 64) >= 1024 ? 4 : 2;
    if (wide) return units(64, 128) < 256 ? 32 : 64;
    if (T > 160 * live && units(256, 256) >= 256 && K >= 2048) return 256;
    if (T > 64 * live && units(128, 128) >= 256) return 128;
    if (T <= 16 * live || units(64, 128) < 256) return 32;
    return 64;
}

template <int XT, bool WIDE, bool SW>
int launch(Exl3c4DevGemm& a, hipStream_t st) {
    const int path = choose(WIDE, SW, a.T, a.n_expert, a.n_out, a.K);
    if (path == 2) return launch_rows<XT, SW, 2>(a, st);
    if (path == 4) return launch_rows<XT, SW, 4>(a, st);
    if (path == 32) return launch_tile<XT, WIDE, SW, 5, 128, 1, 4, 3>(a, st);
    if constexpr (!WIDE) {
        if (path == 256) return launch_tile<XT, WIDE, SW, 8, 256, 2, 4, 2>(a, st);
        if (path == 128) return launch_tile<XT, WIDE, SW, 7, 128, 2, 2, 2>(a, st);
    }
    return launch_tile<XT, WIDE, SW, 6, 128, 1, 4, 2>(a, st);
}

template <int XT, bool WIDE>
int launch_act(Exl3c4DevGemm& a, int32_t act, hipStream_t st) {
    return act == EXL3C4_ACT_SWIGLU ? launch<XT, WIDE, true>(a, st) : launch<XT, WIDE, false>(a, st);
}

// Whether the products are of widened codes (the file's head).
bool widens(int x_type, int y_type) { return x_type != F8 || y_type == EXL3C4_F32; }

}  // namespace

extern "C" int exl3c4_dev_gemm_f8(const Exl3c4DevGemm* g, int32_t x_type, int32_t act, void* stream) {
    Exl3c4DevGemm a = *g;
    const hipStream_t st = (hipStream_t)stream;
    if (x_type == F16) return launch_act<F16, true>(a, act, st);
    if (x_type == BF16) return launch_act<BF16, true>(a, act, st);
    return widens(x_type, a.y_type) ? launch_act<F8, true>(a, act, st) : launch_act<F8, false>(a, act, st);
}

extern "C" int exl3c4_dev_gemm_f8_path(int32_t x_type, int32_t y_type, int32_t act, int64_t T, int64_t n_expert, int64_t N, int64_t K) {
    const bool swiglu = act == EXL3C4_ACT_SWIGLU;
    return choose(widens(x_type, y_type), swiglu, T, n_expert, swiglu ? N / 2 : N, K);
}
