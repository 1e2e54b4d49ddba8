// exl3c4_f8.hip -- matrices of f16, bf16 or f32 to 8-bit floats with an f32 scale for each block of 128 columns (F8: e4m3 codes) and back, on
// gfx950 (include/exl3c4.h has the format). No counterpart in the reference.
//
// A block's scale is a / 448 with a = max(largest magnitude, 2^-96), its codes x (448 / a) to the nearest e4m3: both quotients and the product
// are rounded once in f32, so that another implementation of these steps gives the same codes. The largest magnitude is found on the bits, where
// infinities and NaNs are the largest. v_cvt_pk_fp8_f32 rounds to nearest even (checked for every tie against that rule).
//
// A lane takes 8 columns (loads of 16 or 32 bytes, stores of 8), 16 lanes a block's row. Blocks of one row: the 16 lanes find the largest by DPP.
// Blocks of 128 rows: a workgroup each, every value of the block in its registers, so that memory is read once.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include "exl3c4_dev.h"

namespace {

constexpr int F32 = EXL3C4_F32, F16 = EXL3C4_F16, BF16 = EXL3C4_BF16;
constexpr int WG = 256;
constexpr int PER = 4;                                          // slots (8 columns) a lane, where rows are apart
constexpr int64_t SLOTS = (int64_t)1 << 31;                     // slots a launch indexes in 32 bits
constexpr float TOP = 448.f;                                    // e4m3's largest
constexpr uint32_t LEAST = 31u << 23;                           // 2^-96, the least magnitude that sets a scale: 448 / a stays finite

typedef float float2_t __attribute__((ext_vector_type(2)));
// 8 elements at any address their type may have
struct __attribute__((packed, aligned(2))) Eight16 { uint32_t v[4]; };
struct __attribute__((packed, aligned(4))) Eight32 { uint32_t v[8]; };
template <int DT> constexpr int words = DT == F32 ? 8 : 4;

// Columns c .. c + 7 of a row at p (its column c), those from `cols` on as zeros.
template <int DT> __device__ __forceinline__ void load8(uint32_t* v, const char* p, uint32_t c, uint32_t cols) {
    if (c + 8 <= cols) {
        if constexpr (DT == F32) {
            const Eight32 q = *(const Eight32*)p;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = q.v[i];
        } else {
            const Eight16 q = *(const Eight16*)p;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = q.v[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < words<DT>; ++i) v[i] = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
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
// The largest magnitude of the 8 as f32 bits (of f16, an infinity or a NaN stays one).
template <int DT> __device__ __forceinline__ uint32_t magnitude(const uint32_t* v) {
    uint32_t m = 0;
    if constexpr (DT == F32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, v[i] & 0x7FFFFFFFu);
        return m;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) m = max(m, max(v[i] & 0x7FFFu, (v[i] >> 16) & 0x7FFFu));
        return DT == BF16 ? m << 16 : __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)m));
    }
}
// The largest of a row of 16 lanes, in each of them.
__device__ __forceinline__ uint32_t max16(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, false));       // quad_perm: lane ^ 1
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, false));       // lane ^ 2
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, false));      // row_half_mirror: the other quad of 8
    return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xF, 0xF, false));   // row_mirror: the other 8
}

struct Scale {
    float s, inv;
    __device__ __forceinline__ explicit Scale(uint32_t top) {
        const float a = __uint_as_float(max(top, LEAST));
        const bool bad = top >= 0x7F800000u;
        s = bad ? __uint_as_float(0x7FC00000u) : a / TOP;
        inv = bad ? 0.f : TOP / a;
    }
};
// 8 values' codes (a block with an infinity or a NaN: zeros).
template <int DT> __device__ __forceinline__ uint2 codes_of(const uint32_t* v, const Scale& k) {
    uint32_t q[2] = { 0, 0 };
    if (k.inv == 0.f) return { 0, 0 };
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        q[h] = __builtin_amdgcn_cvt_pk_fp8_f32(value<DT>(v, 4 * h) * k.inv, value<DT>(v, 4 * h + 1) * k.inv, q[h], false);
        q[h] = __builtin_amdgcn_cvt_pk_fp8_f32(value<DT>(v, 4 * h + 2) * k.inv, value<DT>(v, 4 * h + 3) * k.inv, q[h], true);
    }
    return { q[0], q[1] };
}

// Row r of all the matrices': matrix r / rows, its row r % rows.
struct Where { uint32_t mat, row; };
__device__ __forceinline__ Where where(const Exl3c4DevF8& a, uint32_t r) {
    if (a.n == 1) return { 0, r };
    const uint32_t m = r / a.rows;
    return { m, r - m * a.rows };
}

// Blocks of one row. Slots first .. slots - 1 are 8 columns each, lanes_row a row (whole blocks), from row row0 on.
template <int DT>
__global__ __launch_bounds__(WG) void k_f8_quant_rows(Exl3c4DevF8 a, uint32_t row0, uint32_t slots, uint32_t lanes_row) {
    uint32_t v[PER][words<DT>], row[PER], at[PER];
    const uint32_t first = blockIdx.x * (WG * PER) + threadIdx.x;
    Where w[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const uint32_t s = min(first + j * WG, slots - 1);       // (a slot past the last is it again, not stored)
        row[j] = s / lanes_row;
        at[j] = s - row[j] * lanes_row;
        w[j] = where(a, row0 + row[j]);
        load8<DT>(v[j], a.v + w[j].mat * a.v_stride + w[j].row * a.v_pitch + (int64_t)(8 * at[j]) * (words<DT> / 2), 8 * at[j], a.cols);
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        // (the 16 lanes of a block are in one row of lanes, all inside the slots or all the last one again)
        const Scale k(max16(magnitude<DT>(v[j])));
        if (first + j * WG >= slots) continue;
        if (8 * at[j] < a.code_cols)
            *(uint2*)(a.codes + w[j].mat * a.codes_stride + w[j].row * a.codes_pitch + 8 * at[j]) = codes_of<DT>(v[j], k);
        if ((at[j] & 15) == 0) *(float*)((char*)a.scales + w[j].mat * a.scales_stride + w[j].row * a.scales_pitch + (at[j] >> 4) * 4) = k.s;
    }
}

// Blocks of 128 rows: workgroup b takes block b of the matrices' grids of down x across blocks.
template <int DT>
__global__ __launch_bounds__(WG) void k_f8_quant_blocks(Exl3c4DevF8 a, uint32_t across, uint32_t down) {
    __shared__ uint32_t top[WG / 64];
    const uint32_t per = across * down, m = blockIdx.x / per, in = blockIdx.x - m * per, rb = in / across, cb = in - rb * across;
    const uint32_t c = 128 * cb + 8 * (threadIdx.x & 15), r0 = 128 * rb + (threadIdx.x >> 4);
    const char* p = a.v + m * a.v_stride + (int64_t)c * (words<DT> / 2);
    uint32_t v[8][words<DT>], t = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t r = r0 + 16 * j;
#pragma unroll
        for (int i = 0; i < words<DT>; ++i) v[j][i] = 0;
        if (r < a.rows) load8<DT>(v[j], p + r * a.v_pitch, c, a.cols);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) t = max(t, magnitude<DT>(v[j]));
    t = max16(t);
    t = max(max((uint32_t)__builtin_amdgcn_readlane((int)t, 0), (uint32_t)__builtin_amdgcn_readlane((int)t, 16)),
            max((uint32_t)__builtin_amdgcn_readlane((int)t, 32), (uint32_t)__builtin_amdgcn_readlane((int)t, 48)));
    if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = t;
    __syncthreads();
    const Scale k(max(max(top[0], top[1]), max(top[2], top[3])));
    uint8_t* q = a.codes + m * a.codes_stride + c;
    if (c < a.code_cols)
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (r0 + 16 * j < a.rows) *(uint2*)(q + (r0 + 16 * j) * a.codes_pitch) = codes_of<DT>(v[j], k);
    if (threadIdx.x == 0) *(float*)((char*)a.scales + m * a.scales_stride + rb * a.scales_pitch + cb * 4) = k.s;
}

template <int DT>
__global__ __launch_bounds__(WG) void k_f8_dequant(Exl3c4DevF8 a, uint32_t row0, uint32_t slots, uint32_t lanes_row) {
    uint2 q[PER];
    uint32_t at[PER];
    float scale[PER];
    Where w[PER];
    const uint32_t first = blockIdx.x * (WG * PER) + threadIdx.x;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const uint32_t s = min(first + j * WG, slots - 1), row = s / lanes_row;
        at[j] = s - row * lanes_row;
        w[j] = where(a, row0 + row);
        q[j] = *(const uint2*)(a.codes + w[j].mat * a.codes_stride + w[j].row * a.codes_pitch + 8 * at[j]);
        scale[j] = *(const float*)((const char*)a.scales + w[j].mat * a.scales_stride + (w[j].row >> a.block_log2) * a.scales_pitch + (at[j] >> 4) * 4);
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        if (first + j * WG >= slots) continue;
        float f[8];
#define CVT(i, word, hi) { const float2_t p = __builtin_amdgcn_cvt_pk_f32_fp8(word, hi); f[i] = p[0] * scale[j]; f[i + 1] = p[1] * scale[j]; }
        CVT(0, q[j].x, false) CVT(2, q[j].x, true) CVT(4, q[j].y, false) CVT(6, q[j].y, true)
#undef CVT
        const uint32_t c = 8 * at[j];
        char* p = a.v + w[j].mat * a.v_stride + w[j].row * a.v_pitch + (int64_t)c * (words<DT> / 2);
        uint32_t o[words<DT>];
#pragma unroll
        for (int i = 0; i < words<DT>; ++i) {
            if constexpr (DT == F32) o[i] = __float_as_uint(f[i]);
            else if constexpr (DT == F16)
                o[i] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[2 * i]) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[2 * i + 1]) << 16;
            else
                o[i] = (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)f[2 * i]) | (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)f[2 * i + 1]) << 16;
        }
        if (c + 8 <= a.cols) {
            if constexpr (DT == F32) {
                Eight32 e;
#pragma unroll
                for (int i = 0; i < 8; ++i) e.v[i] = o[i];
                *(Eight32*)p = e;
            } else {
                Eight16 e;
#pragma unroll
                for (int i = 0; i < 4; ++i) e.v[i] = o[i];
                *(Eight16*)p = e;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < a.cols) {
                    if constexpr (DT == F32) ((uint32_t*)p)[i] = o[i];
                    else ((uint16_t*)p)[i] = (uint16_t)(o[i >> 1] >> (16 * (i & 1)));
                }
        }
    }
}

int launched() { return hipGetLastError() == hipSuccess ? 0 : EXL3C4_E_DEVICE; }

// All the matrices' rows in launches whose slots fit 32 bits (17 G columns each: one launch in all but the largest cases).
template <class K>
int each_part(K kernel, const Exl3c4DevF8& a, uint32_t lanes, hipStream_t st) {
    const uint32_t all = a.n * a.rows, most = (uint32_t)(SLOTS / lanes < 1 ? 1 : SLOTS / lanes);
    for (uint32_t r = 0; r < all;) {
        const uint32_t n = all - r < most ? all - r : most, slots = n * lanes;
        hipLaunchKernelGGL(kernel, dim3((slots + WG * PER - 1) / (WG * PER)), dim3(WG), 0, st, a, r, slots, lanes);
        if (const int rc = launched()) return rc;
        r += n;
    }
    return 0;
}

}  // namespace

extern "C" int exl3c4_dev_f8_quant(const Exl3c4DevF8* a, int32_t dtype, void* stream) {
    const hipStream_t st = (hipStream_t)stream;
    const uint32_t across = (a->cols + 127) / 128;
    if (a->block_log2 == 0)
        return each_part(dtype == F32 ? k_f8_quant_rows<F32> : dtype == F16 ? k_f8_quant_rows<F16> : k_f8_quant_rows<BF16>, *a, 16 * across, st);
    const uint32_t down = (a->rows + 127) / 128, blocks = a->n * across * down;
    if (blocks == 0) return 0;
    const auto f = dtype == F32 ? k_f8_quant_blocks<F32> : dtype == F16 ? k_f8_quant_blocks<F16> : k_f8_quant_blocks<BF16>;
    hipLaunchKernelGGL(f, dim3(blocks), dim3(WG), 0, st, *a, across, down);
    return launched();
}

extern "C" int exl3c4_dev_f8_dequant(const Exl3c4DevF8* a, int32_t dtype, void* stream) {
    const auto f = dtype == F32 ? k_f8_dequant<F32> : dtype == F16 ? k_f8_dequant<F16> : k_f8_dequant<BF16>;
    return each_part(f, *a, (a->cols + 7) / 8, (hipStream_t)stream);
}
