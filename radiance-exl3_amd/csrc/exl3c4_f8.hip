// exl3c4_f8.hip -- matrices of f16, bf16 or f32 to 8-bit floats with an f32 scale for each block of 128 columns (F8: e4m3
// codes) and back, on gfx950 (include/exl3c4.h has the format). No counterpart in the reference.
//
// A block's scale is a / 448 with a = max(largest magnitude, 2^-96), its codes x (448 / a) to the nearest e4m3: both quotients
// and the product are rounded once in f32, so that another implementation of these steps gives the same codes. The largest
// magnitude is found on the bits, where infinities and NaNs are the largest. v_cvt_pk_fp8_f32 rounds to nearest even (checked
// for every tie against that rule).
//
// Blocks of one row: a lane takes 16 bytes of values, 8 columns of 16 bits or 4 of 32, so that a wave's loads and stores are
// whole lines; the 16 or 32 lanes of a block find the largest by DPP. Blocks of 128 rows: a workgroup each, 16 lanes for the
// 256 bytes or twice 256 bytes of a row and every value of the block in its registers, so that memory is read once. The same
// columns a lane on the way back.
//
// What bounds it: memory, with the VALU next to it (85% busy in rows). Each way alone, us (TB/s of both sides' bytes):
//   rows of f16       20480 x 650 10.0 (4.0), back 8.7 (4.6); 8192 x 2048 9.9 (5.1), back 8.9
//   blocks, f32       131072 x 1000 135 (4.9), back 94 (7.0, part of it into the cache behind L2); 64 x 2048 3.2, back 2.7: a
//                     launch
// What is read or written once goes past the caches (ONCE). Through them / past them, us, 131072 x 1000:
//   values back                          f32 114 / 94, f16 69 / 57
//   values in, blocks (whole lines)      f32 157 / 135, f16 105 / 91
//   codes out, blocks (a line a row)     105 / 139: through them
// Tried without a gain: a row's end shifted by selects of words in place of 64-bit shifts (20480 x 650 0.3 us less, 8192 x 2048
// 1 more: the loads' order).
#include <hip/hip_runtime.h>

#include <stdint.h>

#include "exl3c4_dev.h"

namespace {

constexpr int F32 = EXL3C4_F32, F16 = EXL3C4_F16, BF16 = EXL3C4_BF16;
constexpr int WG = 256;
constexpr int PER = 4;                                          // slots (16 bytes of values) a lane, where rows are apart
constexpr int64_t SLOTS = (int64_t)1 << 31;                     // slots a launch indexes in 32 bits
// Codes up to which rows' are stored past the caches (ONCE). Quantising alone is faster so at any size, the products that read the codes
// then are not. Codes through the caches / past them, us:
//   quantising alone    20480 x 650 f16 10.2 / 8.5, 8192 x 2048 10.0 / 7.8
//   a layer (route, quantising, products, gather)    512 experts, 2048 tokens (4 and 10 M codes) 354 / 341, 1500 334 / 326, 613 467 / 464;
//                       8 experts, 4096 tokens (8 and 11 M) 149 / 151, 8192 (16 and 22 M) 241 / 247
constexpr uint64_t ONCE_MOST = 8 << 20;
constexpr float TOP = 448.f;                                    // e4m3's largest
constexpr uint32_t LEAST = 31u << 23;                           // 2^-96, the least magnitude that sets a scale: 448 / a stays finite

typedef float float2_t __attribute__((ext_vector_type(2)));
typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_at2 __attribute__((aligned(2)));
// 16 bytes at any address their type may have
template <int DT> constexpr int COLS = DT == F32 ? 4 : 8;       // values in 16 bytes
template <int DT> constexpr int SIZE = DT == F32 ? 4 : 2;

// Columns c .. of a row at p (its column c) in 16 bytes, those from `cols` on as zeros: the row's last 16 bytes where they
// would pass its end, shifted (2-byte loads of each took 20480 x 650 f16 from 9 to 14 us).
template <int DT, bool ONCE = false> __device__ __forceinline__ void load16b(uint32_t* v, const char* p, uint32_t c, uint32_t cols) {
    constexpr uint32_t C = COLS<DT>;
    if (cols >= C) {                                             // (uniform)
        const uint32_t past = c + C > cols ? c + C - cols : 0;
        u32x4 q;
        if constexpr (ONCE) q = __builtin_nontemporal_load((const u32x4_at2*)(p - (int64_t)past * SIZE<DT>));
        else q = *(const u32x4_at2*)(p - (int64_t)past * SIZE<DT>);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = q[i];
        if (past) {
            uint64_t lo = (uint64_t)v[1] << 32 | v[0], hi = (uint64_t)v[3] << 32 | v[2];
            if (past >= C / 2) lo = hi, hi = 0;
            if (past >= C) lo = 0;
            const uint32_t bits = (past & (C / 2 - 1)) * (8 * SIZE<DT>);
            lo = lo >> bits | (hi << 1) << (63 - bits);
            hi >>= bits;
            v[0] = (uint32_t)lo, v[1] = (uint32_t)(lo >> 32), v[2] = (uint32_t)hi, v[3] = (uint32_t)(hi >> 32);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = 0;
#pragma unroll
        for (int i = 0; i < (int)C; ++i)
            if (c + i < cols) {
                if constexpr (DT == F32) v[i] = ((const uint32_t*)p)[i];
                else v[i >> 1] |= (uint32_t)((const uint16_t*)p)[i] << (16 * (i & 1));
            }
    }
}
template <int DT> __device__ __forceinline__ float value(const uint32_t* v, int i) {
    if constexpr (DT == F32) return __uint_as_float(v[i]);
    const uint32_t h = (v[i >> 1] >> (16 * (i & 1))) & 0xFFFFu;
    return DT == BF16 ? __uint_as_float(h << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}
// The largest magnitude of 16 bytes as f32 bits (of f16, an infinity or a NaN stays one).
template <int DT> __device__ __forceinline__ uint32_t magnitude(const uint32_t* v) {
    uint32_t m = 0;
    if constexpr (DT == F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) m = max(m, v[i] & 0x7FFFFFFFu);
        return m;
    } else {
        ushort2_t h = { 0, 0 };                                  // the halves apart: v_pk_max_u16
#pragma unroll
        for (int i = 0; i < 4; ++i) h = __builtin_elementwise_max(h, __builtin_bit_cast(ushort2_t, v[i] & 0x7FFF7FFFu));
        m = max((uint32_t)h[0], (uint32_t)h[1]);
        return DT == BF16 ? m << 16 : __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)m));
    }
}
// The largest of a row of 16 lanes, in each of them; and of two such rows, of lanes 0 .. 31 and of 32 .. 63.
__device__ __forceinline__ uint32_t max16(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, false));       // quad_perm: lane ^ 1
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, false));       // lane ^ 2
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, false));      // row_half_mirror: the other quad of 8
    return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xF, 0xF, false));   // row_mirror: the other 8
}
__device__ __forceinline__ uint32_t max32(uint32_t v) {
    v = max16(v);
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return max(r[0], r[1]);
}

// A block's scale a / 448 and 448 / a, each rounded once: a quotient's remainder by a multiply-add, and the quotient corrected
// by it. 448 / a is taken of a's mantissa, whose reciprocal has one step of Newton's behind the hardware's; with that one off
// by up to two steps both are right for every mantissa (all of them tried). (The compiler's division is 14 instructions for
// each, of every lane: 20480 x 650 f16 14 us with them.)
struct Scale {
    float s, inv;
    __device__ __forceinline__ explicit Scale(uint32_t top) {
        const uint32_t u = max(top, LEAST);
        const float a = __uint_as_float(u), m = __uint_as_float((u & 0x7FFFFFu) | 0x3F800000u);
        constexpr float TH = 1.f / TOP;
        const float q = a * TH;
        float y = __builtin_amdgcn_rcpf(m);
        y = __builtin_fmaf(__builtin_fmaf(-m, y, 1.f), y, y);
        const float p = TOP * y;
        s = __builtin_fmaf(__builtin_fmaf(-q, TOP, a), TH, q);
        inv = __builtin_amdgcn_ldexpf(__builtin_fmaf(__builtin_fmaf(-p, m, TOP), y, p), 127 - (int)(u >> 23));
        if (top >= 0x7F800000u) s = __uint_as_float(0x7FC00000u), inv = 0.f;
    }
};
// A value times k, rounded once: f16's by the multiply-add that widens an operand (plus -0, so that a zero keeps its sign),
// 8192 x 2048 10.4 -> 10.0 us.
template <int DT> __device__ __forceinline__ float scaled(const uint32_t* v, int i, float k) {
    if constexpr (DT == F16) {
        float r;
        if (i & 1) asm("v_fma_mix_f32 %0, %1, %2, %3 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(v[i >> 1]), "v"(k), "s"(-0.f));
        else asm("v_fma_mix_f32 %0, %1, %2, %3 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(v[i >> 1]), "v"(k), "s"(-0.f));
        return r;
    } else {
        return value<DT>(v, i) * k;
    }
}
// The codes of four values from the i-th of 16 bytes on (inv 0, of a block with an infinity or a NaN: zeros).
template <int DT> __device__ __forceinline__ uint32_t four_codes(const uint32_t* v, int i, const Scale& k) {
    int q = __builtin_amdgcn_cvt_pk_fp8_f32(scaled<DT>(v, i, k.inv), scaled<DT>(v, i + 1, k.inv), 0, false);
    q = __builtin_amdgcn_cvt_pk_fp8_f32(scaled<DT>(v, i + 2, k.inv), scaled<DT>(v, i + 3, k.inv), q, true);
    return k.inv == 0.f ? 0u : (uint32_t)q;
}
// (ONCE: past the caches)
template <int DT, bool ONCE> __device__ __forceinline__ void store_codes(uint8_t* p, const uint32_t* v, const Scale& k) {
    if constexpr (DT == F32) {
        const uint32_t q = four_codes<DT>(v, 0, k);
        if (ONCE) __builtin_nontemporal_store(q, (uint32_t*)p);
        else *(uint32_t*)p = q;
    } else {
        const uint64_t q = four_codes<DT>(v, 0, k) | (uint64_t)four_codes<DT>(v, 4, k) << 32;
        if (ONCE) __builtin_nontemporal_store(q, (uint64_t*)p);
        else *(uint64_t*)p = q;
    }
}

// Slots of a launch: lanes_row of them a row. s / lanes_row by a multiplication (s < 2^31, lanes_row at least 2; exact).
struct Slots {
    uint32_t row0, count, lanes_row, mul, shift;
    __device__ __forceinline__ uint32_t row(uint32_t s) const { return __umulhi(s, mul) >> shift; }
};
// Row r of all the matrices': matrix r / rows, its row r % rows.
struct Where { uint32_t mat, row; };
__device__ __forceinline__ Where where(const Exl3c4DevF8& a, uint32_t r) {
    if (a.n == 1) return { 0, r };
    const uint32_t m = r / a.rows;
    return { m, r - m * a.rows };
}

// Blocks of one row: whole blocks of lanes a row.
template <int DT, bool ONCE>
__global__ __launch_bounds__(WG) void k_f8_quant_rows(Exl3c4DevF8 a, Slots sl) {
    constexpr uint32_t C = COLS<DT>, BLOCK_LOG2 = DT == F32 ? 5 : 4;
    uint32_t v[PER][4], at[PER];
    const uint32_t first = blockIdx.x * (WG * PER) + threadIdx.x;
    Where w[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const uint32_t s = min(first + j * WG, sl.count - 1), row = sl.row(s);     // (a slot past the last is it again, not stored)
        at[j] = s - row * sl.lanes_row;
        w[j] = where(a, sl.row0 + row);
        load16b<DT>(v[j], a.v + w[j].mat * a.v_stride + w[j].row * a.v_pitch + (int64_t)at[j] * 16, C * at[j], a.cols);
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        // (the lanes of a block are neighbours in a wave, all inside the slots or all the last one again)
        const uint32_t m = magnitude<DT>(v[j]);
        const Scale k(DT == F32 ? max32(m) : max16(m));
        if (first + j * WG >= sl.count) continue;
        if (C * at[j] < a.code_cols)
            store_codes<DT, ONCE>(a.codes + w[j].mat * a.codes_stride + w[j].row * a.codes_pitch + C * at[j], v[j], k);
        if ((at[j] & ((1u << BLOCK_LOG2) - 1)) == 0)
            *(float*)((char*)a.scales + w[j].mat * a.scales_stride + w[j].row * a.scales_pitch + (at[j] >> BLOCK_LOG2) * 4) = k.s;
    }
}

// Blocks of 128 rows: workgroup b takes block b of the matrices' grids of down x across blocks.
template <int DT>
__global__ __launch_bounds__(WG) void k_f8_quant_blocks(Exl3c4DevF8 a, uint32_t across, uint32_t down) {
    constexpr int H = 8 / COLS<DT>;                              // 16-byte parts of 8 columns
    __shared__ uint32_t top[WG / 64];
    const uint32_t per = across * down, m = blockIdx.x / per, in = blockIdx.x - m * per, rb = in / across, cb = in - rb * across;
    const uint32_t c = 128 * cb + COLS<DT> * (threadIdx.x & 15), r0 = 128 * rb + (threadIdx.x >> 4);
    const char* p = a.v + m * a.v_stride + (int64_t)c * SIZE<DT>;
    uint32_t v[8][H][4], t = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t r = r0 + 16 * j;
#pragma unroll
        for (int h = 0; h < H; ++h) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[j][h][i] = 0;
            if (r < a.rows) load16b<DT, true>(v[j][h], p + r * a.v_pitch + 256 * h, c + 64 * h, a.cols);
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int h = 0; h < H; ++h) t = max(t, magnitude<DT>(v[j][h]));
    t = max16(t);
    t = max(max((uint32_t)__builtin_amdgcn_readlane((int)t, 0), (uint32_t)__builtin_amdgcn_readlane((int)t, 16)),
            max((uint32_t)__builtin_amdgcn_readlane((int)t, 32), (uint32_t)__builtin_amdgcn_readlane((int)t, 48)));
    if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = t;
    __syncthreads();
    const Scale k(max(max(top[0], top[1]), max(top[2], top[3])));
    uint8_t* q = a.codes + m * a.codes_stride + c;
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int h = 0; h < H; ++h)
            if (r0 + 16 * j < a.rows && c + 64 * h < a.code_cols)
                store_codes<DT, false>(q + (r0 + 16 * j) * a.codes_pitch + 64 * h, v[j][h], k);
    if (threadIdx.x == 0) *(float*)((char*)a.scales + m * a.scales_stride + rb * a.scales_pitch + cb * 4) = k.s;
}

template <int DT, bool ONCE>
__global__ __launch_bounds__(WG) void k_f8_dequant(Exl3c4DevF8 a, Slots sl) {
    constexpr uint32_t C = COLS<DT>, BLOCK_LOG2 = DT == F32 ? 5 : 4;
    uint32_t q[PER][C / 4], at[PER];
    float scale[PER];
    Where w[PER];
    const uint32_t first = blockIdx.x * (WG * PER) + threadIdx.x;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const uint32_t s = min(first + j * WG, sl.count - 1), row = sl.row(s);
        at[j] = s - row * sl.lanes_row;
        w[j] = where(a, sl.row0 + row);
        const uint32_t* p = (const uint32_t*)(a.codes + w[j].mat * a.codes_stride + w[j].row * a.codes_pitch + C * at[j]);
        if constexpr (DT == F32) q[j][0] = *p;
        else {
            const uint2 u = *(const uint2*)p;
            q[j][0] = u.x, q[j][1] = u.y;
        }
        scale[j] = *(const float*)((const char*)a.scales + w[j].mat * a.scales_stride + (w[j].row >> a.block_log2) * a.scales_pitch +
                                   (at[j] >> BLOCK_LOG2) * 4);
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        if (first + j * WG >= sl.count) continue;
        float f[C];
#pragma unroll
        for (int i = 0; i < (int)C / 4; ++i) {
            const float2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8(q[j][i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(q[j][i], true);
            f[4 * i] = lo[0] * scale[j], f[4 * i + 1] = lo[1] * scale[j], f[4 * i + 2] = hi[0] * scale[j], f[4 * i + 3] = hi[1] * scale[j];
        }
        const uint32_t c = C * at[j];
        char* p = a.v + w[j].mat * a.v_stride + w[j].row * a.v_pitch + (int64_t)at[j] * 16;
        u32x4 o;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == F32) o[i] = __float_as_uint(f[i]);
            else if constexpr (DT == F16)
                o[i] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[2 * i]) |
                       (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[2 * i + 1]) << 16;
            else
                o[i] = (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)f[2 * i]) |
                       (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)f[2 * i + 1]) << 16;
        }
        if (c + C <= a.cols) {
            if constexpr (ONCE) __builtin_nontemporal_store(o, (u32x4_at2*)p);
            else *(u32x4_at2*)p = o;
        } else {
#pragma unroll
            for (int i = 0; i < (int)C; ++i)
                if (c + i < a.cols) {
                    if constexpr (DT == F32) ((uint32_t*)p)[i] = o[i];
                    else ((uint16_t*)p)[i] = (uint16_t)(o[i >> 1] >> (16 * (i & 1)));
                }
        }
    }
}

int launched() { return hipGetLastError() == hipSuccess ? 0 : EXL3C4_E_DEVICE; }

// All the matrices' rows in launches whose slots fit 31 bits (8 G columns each: one launch in all but the largest cases).
// lanes: at least 2 a row.
template <class K>
int each_part(K kernel, const Exl3c4DevF8& a, uint32_t lanes, hipStream_t st) {
    const uint32_t all = a.n * a.rows, most = (uint32_t)((SLOTS - 1) / lanes < 1 ? 1 : (SLOTS - 1) / lanes);
    // l: ceil(log2 lanes), so that ceil(2^(31 + l) / lanes) fits 32 bits, and its product is exact below 2^31
    uint32_t l = 1;
    while (((uint32_t)1 << l) < lanes) ++l;
    const uint32_t mul = (uint32_t)((((uint64_t)1 << (31 + l)) + lanes - 1) / lanes);
    for (uint32_t r = 0; r < all;) {
        const uint32_t n = all - r < most ? all - r : most;
        const Slots sl = { r, n * lanes, lanes, mul, l - 1 };
        hipLaunchKernelGGL(kernel, dim3((sl.count + WG * PER - 1) / (WG * PER)), dim3(WG), 0, st, a, sl);
        if (const int rc = launched()) return rc;
        r += n;
    }
    return 0;
}

}  // namespace

extern "C" int exl3c4_dev_f8_quant(const Exl3c4DevF8* a, int32_t dtype, void* stream) {
    const hipStream_t st = (hipStream_t)stream;
    const uint32_t across = (a->cols + 127) / 128;
    if (a->block_log2 == 0) {
        const bool once = (uint64_t)a->n * a->rows * a->cols <= ONCE_MOST;
        const auto f = dtype == F32   ? (once ? k_f8_quant_rows<F32, true> : k_f8_quant_rows<F32, false>)
                       : dtype == F16 ? (once ? k_f8_quant_rows<F16, true> : k_f8_quant_rows<F16, false>)
                                      : (once ? k_f8_quant_rows<BF16, true> : k_f8_quant_rows<BF16, false>);
        return each_part(f, *a, (dtype == F32 ? 32 : 16) * across, st);
    }
    const uint32_t down = (a->rows + 127) / 128, blocks = a->n * across * down;
    if (blocks == 0) return 0;
    const auto f = dtype == F32 ? k_f8_quant_blocks<F32> : dtype == F16 ? k_f8_quant_blocks<F16> : k_f8_quant_blocks<BF16>;
    hipLaunchKernelGGL(f, dim3(blocks), dim3(WG), 0, st, *a, across, down);
    return launched();
}

extern "C" int exl3c4_dev_f8_dequant(const Exl3c4DevF8* a, int32_t dtype, void* stream) {
    // Past the caches what the one behind L2 (256 MiB) does not hold anyway; less may be read there by what comes next. Rows
    // that are no 16-byte units go through the caches, which join their pieces (20480 x 650 f32 14.7 us past them, 11.9 so).
    const uint64_t bytes = (uint64_t)a->n * a->rows * a->cols * (dtype == F32 ? 4 : 2);
    const bool once = bytes > 256u << 20 && (((uintptr_t)a->v | (uint64_t)a->v_pitch | (uint64_t)a->v_stride) & 15) == 0;
    const auto f = dtype == F32   ? (once ? k_f8_dequant<F32, true> : k_f8_dequant<F32, false>)
                   : dtype == F16 ? (once ? k_f8_dequant<F16, true> : k_f8_dequant<F16, false>)
                                  : (once ? k_f8_dequant<BF16, true> : k_f8_dequant<BF16, false>);
    const uint32_t per = dtype == F32 ? 4 : 8, lanes = (a->cols + per - 1) / per;
    return each_part(f, *a, lanes < 2 ? 2 : lanes, (hipStream_t)stream);      // (a second lane of a single one's row stores nothing)
}
