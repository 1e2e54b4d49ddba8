// exl3c4_gemm_f8.hip -- the products of routed experts whose weights are F8 (e4m3 codes, an f32 scale each 128 x 128), against
// x in F8 (a scale each row and 128 columns), f16 or bf16, on gfx950 (wave64): y[i] = W_e x[row i] over the sorted rows of each
// expert's run, with SwiGLU where asked (include/exl3c4.h). No counterpart in the reference.
//
// THE MATRIX STEP. A block of 128 columns is one step: y += sw sx (sum over the block of w x). Scales are any f32 numbers, so
// they come in as a multiply-add of the sum, which begins at zero. It is taken in one of two ways:
//   widened   the codes become 16-bit floats, which hold every e4m3 (f16 for f16 x, else bf16), and four v_mfma_f32_16x16x32
//             add their products, each exact in f32.
//   as codes  one v_mfma_f32_16x16x128_f8f6f4, at some three times the rate. It adds eight neighbouring columns' products on a
//             grid: each is cut towards zero to a multiple of 2^(E - 13), E the largest of the eight sums of the two codes'
//             exponents; the eights are then added in f32 (found by giving it one product at a time beside a large one). A
//             subnormal code's exponent is -6, however small it is: a sum is off by less than 7 x 2^-13 of each eight's largest
//             product of magnitudes that count as 2^-6 at least; of normally distributed rows by 1.4e-5 of the products' norm.
// Few rows against many weights are bound by memory, and widen. Tiles take F8 x as codes where y has 16 bits, whose own
// rounding (2^-9 or 2^-12 of the value) and the codes' (2^-4) are far larger: from 64 bits bf16 rows are as far either way
// (1.7e-3 of the norm). Codes / widened, us: 8192 tokens over 8 experts, 2816 x 2048 111 / 246; 4096 over 512 214 / 393; 1500
// 172 / 225; 800 over 8 16.5 / 20.8; 613 Zipf 147 / 153. Where y is f32 they widen.
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

// A weights' scale as f 2^(byte - 127), f of magnitude 1 to 2 and the byte as the matrix unit and the conversions take it. A
// sum of codes' products, with F8 x the product of the two scales as well, may be no f32 number, or one of few bits, though the
// other factors bring it back: so the power comes in before the sum, in the matrix unit or with the codes as they widen, and
// f32 multiplies by f (x's scale times f) behind it. With f16 x both stay in f32's range anyway. The power ends at 2^-108 and
// 2^102, between which f32 holds every sum of codes (f takes what is beyond, as it does zeros, infinities and NaN). (Splitting
// x's scale too, a row each: the tiles of codes 109 -> 114 us, 66 -> 69.)
struct Scale {
    float f;
    int byte;
    __device__ __forceinline__ explicit Scale(float s) {
        byte = min(max((int)(__float_as_uint(s) >> 23 & 255), 127 - 108), 127 + 102);
        f = __builtin_amdgcn_ldexpf(s, 127 - byte);
    }
    __device__ __forceinline__ float power() const { return __uint_as_float((uint32_t)byte << 23); }
};

// The products times 2^(by - 127).
__device__ __forceinline__ f32x4 mma_f8(const Codes& a, const Codes& b, int by, f32x4 c) {
    const i32x8 A = { (int)a.h[0].x, (int)a.h[0].y, (int)a.h[0].z, (int)a.h[0].w,
                      (int)a.h[1].x, (int)a.h[1].y, (int)a.h[1].z, (int)a.h[1].w };
    const i32x8 B = { (int)b.h[0].x, (int)b.h[0].y, (int)b.h[0].z, (int)b.h[0].w,
                      (int)b.h[1].x, (int)b.h[1].y, (int)b.h[1].z, (int)b.h[1].w };
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, c, 0, 0, 0, by, 0, 127);
}

// 8 codes, times a power of two, as 8 bf16 or f16 (e4m3 has four bits and exponents of -9 to 8: exact).
template <int XT> __device__ __forceinline__ uint4 widen8(uint32_t lo, uint32_t hi, float by) {
    if constexpr (XT == BF16)
        return { __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, by, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, by, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, by, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, by, true)) };
    else
        return { __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, by, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, by, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, by, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, by, true)) };
}
// Eight codes of the lane's 32, j = 0 .. 3.
template <int XT> __device__ __forceinline__ uint4 widen_part(const Codes& q, int j, float by = 1.f) {
    const uint4& w = q.h[j >> 1];
    return j & 1 ? widen8<XT>(w.z, w.w, by) : widen8<XT>(w.x, w.y, by);
}

// The type that F8 codes widen to beside x of type XT.
template <int XT> constexpr int WIDER = XT == F16 ? F16 : BF16;

__device__ __forceinline__ float load_f32(gaddr p) { return *(const __attribute__((address_space(1))) float*)p; }
__device__ __forceinline__ float word(const uint4& v, int i) { return __uint_as_float(i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w); }

// Rows of blocks of a weight, and the one that holds its row n (of a half with SwiGLU).
__device__ __forceinline__ int64_t scale_row(int n, int half, int n_out) { return (n >> 7) + (int64_t)half * ((n_out + 127) >> 7); }

// ------------------------------------------------------------------------------------------ few rows an expert
// A workgroup: a chunk of up to 16 rows against NS strips of 16 weight rows (with SwiGLU half of them gate rows and half their
// up rows), each wave a part of k; the weights go from memory straight to the matrix units' operands, each byte read once, and
// the parts' sums meet in LDS in a fixed order. x is the A operand (rows of D), W the B operand: lane l ends with D[m = 4 g +
// r][n = l % 16].
// What bounds it: for one token the start (offsets, rows, the first loads) and the last round trip, 8.6 us and 2.4 TB/s of 10
// experts' 1024 x 2048; then memory, one row against 8192 x 8192 16.4 us, 4.1 TB/s. Four steps ahead or loads past the caches:
// within 1%.
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
                    q[s].h[h] = whole || (int64_t)t * 128 + 64 * h + 16 * g < a.K ? load16(w[s] + at + ((int64_t)t * 128 + 64 * h))
                                                                                  : uint4{ 0, 0, 0, 0 };
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
                const Scale k(sw[s]);
                f32x4 p = { 0, 0, 0, 0 };
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    p = mma<WIDER<XT>>(XT == F8 ? widen_part<BF16>(Codes{ v[0], v[1] }, j) : v[j],
                                       widen_part<WIDER<XT>>(q[s], j, XT == F16 ? 1.f : k.power()), p);
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[s][r] = __builtin_fmaf(p[r], XT == F8 ? sx[r] * k.f : XT == BF16 ? k.f : sw[s], acc[s][r]);
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

// Two values in 16 bits each.
template <int T> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (T == BF16) return __builtin_bit_cast(uint32_t, bf2_t{ (__bf16)lo, (__bf16)hi });
    else return __builtin_bit_cast(uint32_t, half2_t{ (_Float16)lo, (_Float16)hi });
}

// ------------------------------------------------------------------------------------------ many rows an expert
// A workgroup: a tile of MT rows of one expert against NT weight rows (with SwiGLU 16 gate rows and their 16 up rows in turn,
// so that a lane holds both), k in stages of one block of 128 columns. A stage's rows and scales go from memory to LDS without
// registers. A wave reads its weight rows into registers at the start of a stage and then uses them for all its rows of x, so
// one place for weights is enough: once every wave has read them (a barrier among the products) the next stage's come in under
// the rest of the products. x has XB places, XB - 1 stages ahead. So a workgroup's LDS stays small and a CU holds several, one
// at its start or end under another's products.
//
// LDS. A row of a stage is 128 bytes (16-bit x: two such halves). The loads write lane after lane, 16 bytes each, so the order
// within a row is chosen at the source: place p of row r holds the chunk q = p ^ (r & 7), in a half of a 16-bit row the chunk
// whose number is q's with its highest bit moved to the end, so that lane groups g and g + 1 read places that differ in their
// lowest bit: the 16 rows and four lane groups that read a matrix operand then fall on all the banks evenly (16-bit rows by q
// itself: 39% of the LDS cycles were conflicts, 1% so; 4096 tokens over 8 experts 56.0 -> 54.4 us). Behind x's rows a scale for
// each; behind the weights' those of the tile's blocks of weight rows.
//
// Weights are the A operand here (rows of D): a lane ends with 4 consecutive columns of one row of y, so that a sum's scale is
// one number of the lane's row of x times one that the wave shares.
template <int XT, bool SW, int MT_LOG2, int NT, int WM, int WN, int XB> struct Tile {
    static constexpr int MT = 1 << MT_LOG2, WAVES_ = WM * WN;
    static constexpr int XROW = XT == F8 ? 128 : 256;                        // bytes of a row of x a stage
    static constexpr int XG = MT * XROW / 1024, WG = NT * 128 / 1024;        // 1-KiB loads a stage
    static constexpr int XS = XT == F8 ? (MT + 63) / 64 : 0;                 // of x's scales, 64 each
    static constexpr int XL = XG / WAVES_, WL = WG / WAVES_, XSL = (XS + WAVES_ - 1) / WAVES_;
    static constexpr int NX = XL + XSL, NW = WL + 1;                         // a wave's loads of x and of weights, every stage
    static constexpr int AT_XS = XG * 1024, XSLOT = AT_XS + XS * 256, AT_W = XB * XSLOT, AT_WS = AT_W + WG * 1024, LDS = AT_WS + 256;
    static constexpr int TM = MT / WM / 16, TN = NT / WN / 16;               // matrix tiles a wave
    // Rows of y go past the caches from tiles of more than 32 rows. Through them / past them, us:
    //   the product alone    512 experts, 1500 tokens 188 / 172, 2048 Zipf 222 / 213, 4096 216 / 210; 8 experts, 8192, 2048 x 1408 71 / 64
    //   whole layers         512 experts, 1500 tokens 350 / 329, 2048 371 / 345, 4096 460 / 450; 64 experts, 8192 686 / 684;
    //                        8 experts, 2000 99.6 / 97.0, 4096 163.5 / 163.0, 8192 267.1 / 267.8
    //   in tiles of 32 rows  400 tokens 162 / 165, a layer of 613 456 / 464: through them
    static constexpr bool LATER = MT_LOG2 > 5;
    // waves a SIMD, by the workgroups whose LDS a CU holds: what the compiler may use registers for
    static constexpr int GROUPS = 160 * 1024 / (LDS + 4 * MT + 1024), EU = GROUPS * WAVES_ / 4, WAVES_EU = EU > 8 ? 8 : EU;
    static_assert(XG % WAVES_ == 0 && WG % WAVES_ == 0 && (NX + NW) * 2 < 64 && TN % 2 == 0, "tile");
    static_assert((NT == 128 || NT == 256) && (XB == 2 || XB == 3), "one or two blocks of weight rows; places of x");
};

template <int XT, bool WIDE, bool SW, int MT_LOG2, int NT, int WM, int WN, int XB, bool ONCE,
          class G = Tile<XT, SW, MT_LOG2, NT, WM, WN, XB>>
__global__ __launch_bounds__(64 * WM * WN) __attribute__((amdgpu_waves_per_eu(G::WAVES_EU, G::WAVES_EU))) void k_f8_tile(Exl3c4DevGemm a) {
    constexpr int MT = G::MT, WV = WM * WN, TM = G::TM, TN = G::TN;
    __shared__ __align__(1024) char lds[G::LDS];
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
        // Each of the wave's loads of a stage: where it reads next, for this lane (lane l takes place l % 8 of row l / 8). A
        // stage is 128 columns on.
        gaddr xp[G::NX], wp[G::NW];
        auto x_chunk = [&](int) {
            const int q = (lane & 7) ^ (lane >> 3);
            return XT == F8 ? q : ((q & 3) << 1) | (q >> 2);
        };
        auto w_chunk = [&](int) { return (lane & 7) ^ (lane >> 3); };
#pragma unroll
        for (int i = 0; i < G::XL; ++i) {
            const int q = wave + i * WV, r = 8 * (XT == F8 ? q : q >> 1) + (lane >> 3);
            xp[i] = (gaddr)a.x + (int64_t)max(rows_x[r], 0) * a.x_pitch + 16 * x_chunk(i) + (XT == F8 ? 0 : 128 * (q & 1));
        }
#pragma unroll
        for (int i = 0; i < G::XSL; ++i)
            xp[G::XL + i] = (gaddr)a.xs + (int64_t)max(rows_x[(64 * ((wave + i * WV) % max(G::XS, 1)) + lane) % MT], 0) * a.xs_pitch;
#pragma unroll
        for (int i = 0; i < G::WL; ++i) wp[i] = we + (int64_t)w_row(8 * (wave + i * WV) + (lane >> 3)) * a.w_pitch + 16 * w_chunk(i);
        // the scales of the tile's weight rows: even lanes of its first block (SwiGLU: of the gate rows), odd lanes of the
        // second (of the up rows); every wave the same ones, so that a wait counts alike in all
        wp[G::WL] = wse + (SW ? scale_row(n0, lane & 1, a.n_out) : scale_row(min(n0 + (lane & 1) * 128, a.N - 1), 0, a.N)) * a.ws_pitch;
        const int stages = (a.K + 127) / 128, past = a.K - 128 * (stages - 1);          // columns of the last stage
        const uint32_t at0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
        // load i of x or of the weights (all 0: of no lane)
        auto load_x = [&](int i, uint32_t to, int all) {
            if (i < G::XL) dma16_of(xp[i], to + (wave + i * WV) * 1024, all);
            else dma4_of(xp[i], to + G::AT_XS + ((wave + (i - G::XL) * WV) % max(G::XS, 1)) * 256, all);
            xp[i] += i < G::XL ? G::XROW : 4;
        };
        auto load_w = [&](int i, int all) {
            const uint32_t to = at0 + G::AT_W + (wave + i * WV) * 1024;
            if (i < G::WL && ONCE) dma16_of(wp[i], to, all, ch.alone);
            else if (i < G::WL) dma16_of(wp[i], to, all);
            else dma4_of(wp[i], at0 + G::AT_WS, all);
            wp[i] += i < G::WL ? 128 : 4;
        };
        // before the last stage's loads: what lies past K reads as zeros
        auto end_x = [&]() {
#pragma unroll
            for (int i = 0; i < G::XL; ++i)
                if ((XT == F8 ? 16 * x_chunk(i) : 8 * x_chunk(i) + 64 * ((wave + i * WV) & 1)) >= past) xp[i] = (gaddr)&k_zero;
        };
        auto end_w = [&]() {
#pragma unroll
            for (int i = 0; i < G::WL; ++i)
                if (16 * w_chunk(i) >= past) wp[i] = (gaddr)&k_zero;
        };
        // -1 where stage t is one, else 0 (through a VGPR: the compiler else may leave the mask itself in one)
        auto there = [&](int t) {
            int v = (t - stages) >> 31;
            asm volatile("" : "+v"(v));
            return __builtin_amdgcn_readfirstlane(v);
        };
        const int xr = wm * TM * 16 + l16, wr = wn * TN * 16 + l16;      // the lane's row in the first tile of each
        // One stage's products. between(s) is called at s = 0 .. SLOTS - 1 among them, from s = 1 on with the weights in registers.
        constexpr int SLOTS = WIDE ? TN : TM;
        auto multiply = [&](int slot_x, auto between) {
            const char* X = lds + slot_x * G::XSLOT;
            const char* W = lds + G::AT_W;
            const float* XS = (const float*)(X + G::AT_XS);
            const float* WS = (const float*)(lds + G::AT_WS);
            auto codes = [&](const char* p, int row) {
                return Codes{ *(const uint4*)(p + row * 128 + 16 * (g ^ (l16 & 7))),
                              *(const uint4*)(p + row * 128 + 16 * ((4 + g) ^ (l16 & 7))) };
            };
            // (a wave's weight rows lie in one block of 128; with SwiGLU its even tiles in the gate's, its odd ones in the up's)
            const float sw[2] = { WS[SW ? 0 : (wn * TN * 16) >> 7], WS[1] };
            const Scale kw[2] = { Scale(sw[0]), Scale(sw[1]) };
            Codes wv[TN];
#pragma unroll
            for (int n = 0; n < TN; ++n) wv[n] = codes(W, wr + 16 * n);
            if constexpr (!WIDE) {
                // Row tile m + 1's operand is read while tile m's products run; a sum is scaled LAG products behind its own.
                constexpr int LAG = 3;
                Codes xv[2];
                float f[2][2];
                f32x4 p[LAG + 1];
                xv[0] = codes(X, xr);
                f[0][0] = f[0][1] = XS[xr];
                f[0][0] *= kw[0].f, f[0][1] *= kw[1].f;
#pragma unroll
                for (int i = 0; i < TM * TN + LAG; ++i) {
                    const int m = i / TN, n = i % TN;
                    if (i < TM * TN) {
                        if (n == 0) {
                            if (m + 1 < TM) xv[(m + 1) & 1] = codes(X, xr + 16 * (m + 1));
                            between(m);
                        }
                        p[i % (LAG + 1)] = mma_f8(wv[n], xv[m & 1], kw[SW ? n & 1 : 0].byte, f32x4{ 0, 0, 0, 0 });
                    }
                    if (i >= LAG) {
                        const int k = i - LAG, km = k / TN, kn = k % TN;
                        if (kn == 0 && km > 0) {
                            const float sx = XS[xr + 16 * km];
                            f[km & 1][0] = sx * kw[0].f, f[km & 1][1] = sx * kw[1].f;
                        }
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            acc[kn][km][r] = __builtin_fmaf(p[k % (LAG + 1)][r], f[km & 1][SW ? kn & 1 : 0], acc[kn][km][r]);
                    }
                }
            } else {
                // x's eights j of columns: 16 g + 8 j of the block's first half, then of its second. (The weights' power comes
                // in with x's codes where it is one for all: with the weights' a register more, and a spill's reload waits for
                // the loads ahead, 34.0 -> 36.2 us of 300 rows of 4096 x 4096.)
                uint4 xv[TM][4];
                float sx[TM];
#pragma unroll
                for (int m = 0; m < TM; ++m) {
                    if constexpr (XT == F8) {
                        const Codes c = codes(X, xr + 16 * m);
#pragma unroll
                        for (int j = 0; j < 4; ++j) xv[m][j] = widen_part<BF16>(c, j, SW ? 1.f : kw[0].power());
                        sx[m] = XS[xr + 16 * m];
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            xv[m][j] = *(const uint4*)(X + ((xr >> 3) + 2 * m) * 2048 + (j >> 1) * 1024 + (l16 & 7) * 128 +
                                                       16 * ((g + 4 * (j & 1)) ^ (l16 & 7)));
                    }
                }
#pragma unroll
                for (int n = 0; n < TN; ++n) {
                    between(n);
                    f32x4 p[TM] = {};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint4 w = widen_part<WIDER<XT>>(wv[n], j, XT == F16 || (XT == F8 && !SW) ? 1.f : kw[SW ? n & 1 : 0].power());
#pragma unroll
                        for (int m = 0; m < TM; ++m) p[m] = mma<WIDER<XT>>(w, xv[m][j], p[m]);
                    }
#pragma unroll
                    for (int m = 0; m < TM; ++m) {
                        const float k = XT == F16 ? sw[SW ? n & 1 : 0] : kw[SW ? n & 1 : 0].f, f = XT == F8 ? sx[m] * k : k;
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[n][m][r] = __builtin_fmaf(p[m][r], f, acc[n][m][r]);
                    }
                }
            }
        };
        if (stages == 1) end_w();
#pragma unroll
        for (int i = 0; i < G::NW; ++i) load_w(i, -1);
#pragma unroll
        for (int q = 0; q < XB - 1; ++q) {
            if (q + 1 == stages) end_x();
#pragma unroll
            for (int i = 0; i < G::NX; ++i) load_x(i, at0 + q * G::XSLOT, there(q));
        }
        int slot_x = 0;
        for (int t = 0; t < stages; ++t) {
            // the weights and x of stage t are here (the loads behind theirs are x's of stage t + 1)
            if (XB == 2 || t + 1 >= stages) wait_loads<0>();
            else wait_loads<G::NX>();
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if (t + 2 == stages) end_w();
            if (t + XB == stages) end_x();
            // the place of x of stage t - 1, read by all before the barrier
            const uint32_t to_x = at0 + (slot_x == 0 ? XB - 1 : slot_x - 1) * G::XSLOT;
            // Behind the last stage no lane loads: a branch would keep the products of one row tile from running on beside the
            // next one's (8192 tokens over 8 experts, 2816 x 2048: 123 us for 114, when one workgroup filled a CU).
            const int more_w = there(t + 1), more_x = there(t + XB - 1);
            multiply(slot_x, [&](int s) {
                constexpr int AT = SLOTS > 1 ? 1 : 0;                        // the loads follow in one to four slots
                constexpr int FOR = SLOTS - AT > 4 ? 4 : SLOTS - AT;
                if (s == AT) {                                               // every wave has read the weights
                    asm volatile("" ::: "memory");
                    __builtin_amdgcn_s_waitcnt(0xC07F);                      // lgkmcnt(0)
                    __builtin_amdgcn_s_barrier();
                    asm volatile("" ::: "memory");
                }
#pragma unroll
                for (int i = 0; i < G::NW + G::NX; ++i)
                    if (s == AT + i * FOR / (G::NW + G::NX)) {
                        if (i < G::NW) load_w(i, more_w);
                        else load_x(i - G::NW, to_x, more_x);
                    }
            });
            asm volatile("" ::: "memory");
            slot_x = slot_x + 1 == XB ? 0 : slot_x + 1;
        }
    }
    // A lane holds columns 16 n + 4 g .. + 3 of row 16 m + l16 of the wave's (SwiGLU: of gate tile 2 n and up tile 2 n + 1). PM
    // row tiles at a time cross LDS in y's type, so that whole rows of the tile go out by 16 bytes a lane (8192 tokens over 8
    // experts, 2048 x 1408: 78 us with 8 bytes a lane from each wave's own columns, 68 so; 2816 x 2048 with SwiGLU 115 and 111;
    // 2560 x 640 over 512 experts the same).
    constexpr int TO = SW ? TN / 2 : TN, OC = 16 * TO * WN, MOST = WIDE ? 4 : 2;      // (y is f32 where the codes are widened only)
    constexpr int FIT = G::LDS / (16 * (OC * MOST + 16)), PM = FIT >= TM ? TM : FIT >= 4 ? 4 : FIT >= 2 ? 2 : 1;
    static_assert(WM == 1 && FIT >= 1 && TM % PM == 0, "a pass's rows fit");
    const int size_log2 = MOST == 4 && a.y_type == EXL3C4_F32 ? 2 : 1, pitch = (OC << size_log2) + 16;
    const int per_log2 = 4 - size_log2, row_log2 = __builtin_ctz(OC) - per_log2;      // columns in 16 bytes; 16 bytes a row
    struct __attribute__((packed, aligned(2))) Part { uint32_t v[4]; };
    typedef u32x4 u32x4_at2 __attribute__((aligned(2)));
#pragma unroll
    for (int m0 = 0; m0 < TM; m0 += PM) {
        __syncthreads();                                         // the stages, or the pass before, are read
#pragma unroll
        for (int m = m0; m < m0 + PM; ++m)
#pragma unroll
            for (int n = 0; n < TO; ++n) {
                f32x4 v = SW ? acc[2 * n][m] : acc[n][m];
                if (SW) v = swiglu4(v, acc[SW ? 2 * n + 1 : n][m]);
                char* p = lds + ((m - m0) * 16 + l16) * pitch + ((wn * TO * 16 + 16 * n + 4 * g) << size_log2);
                if (size_log2 == 2) *(f32x4*)p = v;
                else *(uint2*)p = a.y_type == BF16 ? uint2{ pack2<BF16>(v[0], v[1]), pack2<BF16>(v[2], v[3]) }
                                                   : uint2{ pack2<F16>(v[0], v[1]), pack2<F16>(v[2], v[3]) };
            }
        __syncthreads();
        for (int i = threadIdx.x; i < 16 * PM << row_log2; i += 64 * WV) {
            const int q = i >> row_log2, r = 16 * m0 + q, c = (i & ((1 << row_log2) - 1)) << per_log2, col = n0 + c;
            if (r >= ch.rows || col >= a.n_out) continue;
            Part v = *(const Part*)__builtin_assume_aligned(lds + q * pitch + (c << size_log2), 16);
            if (rows_x[r] < 0) v = Part{ { 0, 0, 0, 0 } };
            char* y = a.y + (int64_t)(ch.row0 + r) * a.y_pitch + ((int64_t)col << size_log2);
            if (col + (1 << per_log2) <= a.n_out) {
                if constexpr (G::LATER) __builtin_nontemporal_store(u32x4{ v.v[0], v.v[1], v.v[2], v.v[3] }, (u32x4_at2*)y);
                else *(Part*)y = v;
            } else if (size_log2 == 2) {
#pragma unroll
                for (int u = 0; u < 3; ++u)
                    if (col + u < a.n_out) ((uint32_t*)y)[u] = v.v[u];
            } else {
#pragma unroll
                for (int u = 0; u < 7; ++u)
                    if (col + u < a.n_out) ((uint16_t*)y)[u] = (uint16_t)(v.v[u >> 1] >> (16 * (u & 1)));
            }
        }
    }
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

template <int XT, bool WIDE, bool SW, int MT_LOG2, int NT, int WM, int WN, int XB>
int launch_tile(Exl3c4DevGemm& a, hipStream_t st) {
    constexpr int cols = SW ? NT / 2 : NT;
    a.tiles = (a.n_out + cols - 1) / cols;
    const int64_t grid = (chunk_bound(a.T, a.n_expert, 1 << MT_LOG2) * a.tiles + 7) / 8 * 8;
    if (grid > THREADS / (64 * WM * WN)) return EXL3C4_E_SHAPE;
    // Weights of runs that are one chunk, which no other workgroup reads, go past the caches where those of all experts that
    // can be live are more than the one behind L2 holds (256 MiB), so that the next pass does not find them there. Through them
    // / past them, us:
    //   six sets of weights in turn    bf16 x, 32 tokens 95 / 86; F8 x, 100 158 / 138, 400 184 / 163, 613 Zipf 2560 x 640 163 /
    //                                  158, 1500 194 / 188
    //   fewer, one set again and again 8 tokens 27 / 33, 64/6 32 tokens 23 / 30: through them
    //   runs of more chunks as well    2048 Zipf 226 / 241: through them
    // The choice is a branch at each load: 3% of a batch that does not need it, hence a kernel of its own, and in tiles of 128
    // rows more than it gives (4096 tokens 218 / 226).
    const int64_t live = a.n_expert < a.T ? a.n_expert : a.T;
    const bool once = MT_LOG2 < 7 && live * a.N > ((int64_t)256 << 20) / a.K;
    const auto f = once ? k_f8_tile<XT, WIDE, SW, MT_LOG2, NT, WM, WN, XB, (MT_LOG2 < 7)>
                        : k_f8_tile<XT, WIDE, SW, MT_LOG2, NT, WM, WN, XB, false>;
    hipLaunchKernelGGL(f, dim3((unsigned)grid), dim3(64 * WM * WN), 0, st, a);
    return launched();
}

// Which kernel, and how large a tile: by the types, the sizes and the rows that an expert has at least on average, r = T /
// min(E, T) -- never by the routing, which is on the device. Larger tiles read weights and rows less often; smaller ones waste
// less of a chunk, make more workgroups and start sooner; the rows kernel splits k over its waves, so that few workgroups are
// enough. `units`: workgroups of a tile, each expert half a chunk short of whole ones. Measured on one card, us, the product
// alone (E / top-k, N x K, tokens; 512/10, 1024 x 2048 with SwiGLU where nothing else is said):
//   rows against 32        bf16 x: 1 token 8.6 / 13.3, 4 19.6 / 20.0, 8 30 / 27, 32 102 / 83; F8 x: 8 30 / 26, 16 55 / 56, 32
//                          98 / 79. 64/6, 32 tokens 30 / 23; 8/2, 200 20 / 13. One expert, bf16 x: 2048 x 2048, 77 rows 10.7 /
//                          13.2, 300 22 / 18; 8192 x 8192, 64 rows 48 / 57; 4096 x 4096, 16 rows 11.7 / 22, 300 74 / 35.
//   2 strips against 4     one row, 8192 x 8192 16.5 / 23.6; 4096 x 4096, 16 rows 11.7 / 15.5; 8192 x 8192, 64 rows 61 / 48,
//                          which read the weights once for each 16 rows, mostly from L2.
//   32 rows against 64     as codes: 400 tokens 160 / 165, 613 Zipf 2560 x 640 148 / 156, 1500 202 / 171, 8/2 800 15.9 / 21.
//                          bf16 x: 400 164 / 187, 613 Zipf 2560 x 640 156 / 172, 1500 200 / 191, 8/2 800 19 / 28. F8 x, f32 y:
//                          200 161 / 200, 1500 217 / 215.
//   64 against 128         as codes: 1500 172 / 200, 2048 Zipf 211 / 222, 4096 271 / 210, 64/6 2000 52 / 40, 8/2 8192 2816 x
//                          2048 143 / 104, 2048 x 1408, sorted rows in, 79 / 64.
// As codes a tile of 256 x 256 with a CU to itself took 131 there before the loads went among the products and 114 to 118
// since, and was slower everywhere else; 128 x 128 130 (73 for 77 at 2048 x 1408, sorted rows in); weights in two places 232 at
// 64 rows, and 2% less at 32 rows and 100 to 400 tokens. Widened: 128 x 128 in eight waves 344, 128 x 256 211 against 202 of
// 64 x 256.
// Returns a tile's rows (32, 64, 128), or for few rows an expert the strips of a workgroup (2, 4).
int choose(bool wide, bool swiglu, int64_t T, int64_t n_expert, int64_t n_out, int64_t K) {
    const int64_t live = n_expert < T ? n_expert : T;
    // workgroups of tiles of `rows` x `cols` (SwiGLU: half as many columns of y)
    auto units = [&](int rows, int cols) {
        if (swiglu) cols /= 2;
        const int64_t chunks = (T + live * rows / 2) / rows;
        return (chunks > live ? chunks : live) * ((n_out + cols - 1) / cols);
    };
    if (units(32, 128) < 64 + K / 32) return T > 16 * live && units(16, 64) >= 256 ? 4 : 2;
    if (!wide && T > 56 * live && units(128, 256) >= 256) return 128;
    if (T > 18 * live && units(64, 256) >= 256) return 64;
    return 32;
}

template <int XT, bool WIDE, bool SW>
int launch(Exl3c4DevGemm& a, hipStream_t st) {
    const int path = choose(WIDE, SW, a.T, a.n_expert, a.n_out, a.K);
    if (path == 2) return launch_rows<XT, SW, 2>(a, st);
    if (path == 4) return launch_rows<XT, SW, 4>(a, st);
    if (path == 32) return launch_tile<XT, WIDE, SW, 5, 128, 1, 4, XT == F8 ? 3 : 2>(a, st);
    if constexpr (!WIDE)
        if (path == 128) return launch_tile<XT, WIDE, SW, 7, 256, 1, 4, 2>(a, st);
    if constexpr (XT == F8 && WIDE) return launch_tile<XT, WIDE, SW, 6, 128, 1, 4, 3>(a, st);
    else return launch_tile<XT, WIDE, SW, 6, 256, 1, 4, XT == F8 ? 3 : 2>(a, st);
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
