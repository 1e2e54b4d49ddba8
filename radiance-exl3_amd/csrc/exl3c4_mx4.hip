// exl3c4_mx4.hip -- rows of f16, bf16 or f32 to microscaled 4-bit floats (e2m1 codes, one e8m0 scale each 32 columns)
// and back, on gfx950 (include/exl3c4.h has the format). No counterpart in the reference.
//
// A lane takes 8 columns: its loads and stores are 16 and 4 bytes (32 and 4 for f32), contiguous over the wave, and four
// lanes share a block. The scale is the exponent field of the block's largest magnitude less two (e2m1's largest
// exponent), found on the bits, where infinities and NaNs are the largest; v_cvt_scalef32_pk_fp4_* divides by it, rounds to
// nearest even and saturates (checked for every tie and every exponent against that rule), and its inverse is exact.
//
// Both are bound by memory: 131072 x 2048 f32 quantised in 261 us (1.07 GB in, 0.14 out: 4.6 TB/s) and read back in 291
// (4.2 TB/s; a large copy on this card 4.7); 20480 x 650 f16 in 9.5 and 7.4 us; 8 x 2048 in 2.5 and 1.9, a launch's least.
// Four slots a lane, 256 lanes: the loads of four are out together.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include "exl3c4_dev.h"

namespace {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf2_t __attribute__((ext_vector_type(2)));
typedef float float2_t __attribute__((ext_vector_type(2)));

constexpr int WG = 256;
constexpr int PER = 4;                                          // slots (8 columns) a lane
constexpr int64_t SLOTS = (int64_t)1 << 31;                     // slots a launch indexes in 32 bits

// 8 elements at any address their type may have
struct __attribute__((packed, aligned(2))) Eight16 { uint32_t v[4]; };
struct __attribute__((packed, aligned(4))) Eight32 { uint32_t v[8]; };

// The value of lane l ^ 1 and l ^ 2 (DPP quad_perm).
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, false));
    return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, false));
}
__device__ __forceinline__ uint32_t half_max(uint32_t a, uint32_t b) {   // of both halves
    const uint32_t lo = max(a & 0xFFFFu, b & 0xFFFFu), hi = max(a >> 16, b >> 16);
    return lo | (hi << 16);
}

// x rows [rows][cols] to codes and scales; slots = rows * lanes_row.
template <int DT>
__global__ __launch_bounds__(WG) void k_mx4_quant(const char* x, uint32_t slots, uint32_t lanes_row, uint32_t cols,
                                                  int64_t pitch, uint8_t* codes, int64_t codes_pitch, uint8_t* scales,
                                                  int64_t scales_pitch) {
    constexpr int W = DT == EXL3C4_F32 ? 8 : 4;                 // words of 8 elements
    uint32_t v[PER][W], row[PER], at[PER];
    const uint32_t first = blockIdx.x * (WG * PER) + threadIdx.x;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const uint32_t s = first + j * WG;
        row[j] = s / lanes_row;
        at[j] = s - row[j] * lanes_row;
        const uint32_t c = 8 * at[j];
        const char* p = x + (int64_t)row[j] * pitch + (int64_t)c * (W / 2);
#pragma unroll
        for (int i = 0; i < W; ++i) v[j][i] = 0;
        if (s >= slots) continue;
        if (c + 8 <= cols) {
            if constexpr (W == 4) {
                const Eight16 q = *(const Eight16*)p;
#pragma unroll
                for (int i = 0; i < 4; ++i) v[j][i] = q.v[i];
            } else {
                const Eight32 q = *(const Eight32*)p;
#pragma unroll
                for (int i = 0; i < 8; ++i) v[j][i] = q.v[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < cols) {
                    if constexpr (W == 4) v[j][i >> 1] |= (uint32_t)((const uint16_t*)p)[i] << (16 * (i & 1));
                    else v[j][i] = ((const uint32_t*)p)[i];
                }
        }
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        // the block's largest magnitude as f32 bits; past every finite value: an infinity or a NaN is in it
        uint32_t top = 0;
        bool bad;
        if constexpr (DT == EXL3C4_F32) {
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max(top, v[j][i] & 0x7FFFFFFFu);
            top = quad_max(top);
            bad = top >= 0x7F800000u;
        } else {
            uint32_t m = v[j][0] & 0x7FFF7FFFu;
#pragma unroll
            for (int i = 1; i < 4; ++i) m = half_max(m, v[j][i] & 0x7FFF7FFFu);
            m = quad_max(max(m & 0xFFFFu, m >> 16));
            bad = m >= (DT == EXL3C4_F16 ? 0x7C00u : 0x7F80u);
            top = DT == EXL3C4_F16 ? __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)m)) : m << 16;
        }
        const int e = (int)(top >> 23) - 2;                      // floor(log2) - 2, biased by 127; a subnormal's field is 0
        const uint32_t byte = bad ? 255u : (uint32_t)max(e, 0);
        const float scale = __uint_as_float(byte << 23);        // the conversion reads the exponent field alone
        uint32_t q = 0;
        if constexpr (DT == EXL3C4_F32) {
#define CVT(i) q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, __uint_as_float(v[j][2 * i]), __uint_as_float(v[j][2 * i + 1]), scale, i)
            CVT(0); CVT(1); CVT(2); CVT(3);
#undef CVT
        } else if constexpr (DT == EXL3C4_F16) {
#define CVT(i) q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, __builtin_bit_cast(half2_t, v[j][i]), scale, i)
            CVT(0); CVT(1); CVT(2); CVT(3);
#undef CVT
        } else {
#define CVT(i) q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf2_t, v[j][i]), scale, i)
            CVT(0); CVT(1); CVT(2); CVT(3);
#undef CVT
        }
        if (first + j * WG >= slots) continue;
        *(uint32_t*)(codes + (int64_t)row[j] * codes_pitch + 4 * (int64_t)at[j]) = bad ? 0u : q;
        if ((at[j] & 3) == 0) scales[(int64_t)row[j] * scales_pitch + (at[j] >> 2)] = (uint8_t)byte;
    }
}

template <int DT>
__global__ __launch_bounds__(WG) void k_mx4_dequant(const uint8_t* codes, int64_t codes_pitch, const uint8_t* scales,
                                                    int64_t scales_pitch, uint32_t slots, uint32_t lanes_row,
                                                    uint32_t cols, char* out, int64_t pitch) {
    constexpr int W = DT == EXL3C4_F32 ? 8 : 4;
    uint32_t q[PER], row[PER], at[PER];
    float scale[PER];
    const uint32_t first = blockIdx.x * (WG * PER) + threadIdx.x;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const uint32_t s = first + j * WG < slots ? first + j * WG : slots - 1;
        row[j] = s / lanes_row;
        at[j] = s - row[j] * lanes_row;
        q[j] = *(const uint32_t*)(codes + (int64_t)row[j] * codes_pitch + 4 * (int64_t)at[j]);
        scale[j] = __uint_as_float((uint32_t)scales[(int64_t)row[j] * scales_pitch + (at[j] >> 2)] << 23);
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        uint32_t v[W];
        if constexpr (DT == EXL3C4_F32) {
#define CVT(i) { const float2_t f = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[j], scale[j], i); \
                 v[2 * i] = __float_as_uint(f[0]); v[2 * i + 1] = __float_as_uint(f[1]); }
            CVT(0) CVT(1) CVT(2) CVT(3)
#undef CVT
        } else if constexpr (DT == EXL3C4_F16) {
#define CVT(i) v[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q[j], scale[j], i));
            CVT(0) CVT(1) CVT(2) CVT(3)
#undef CVT
        } else {
#define CVT(i) v[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q[j], scale[j], i));
            CVT(0) CVT(1) CVT(2) CVT(3)
#undef CVT
        }
        if (first + j * WG >= slots) continue;
        const uint32_t c = 8 * at[j];
        char* p = out + (int64_t)row[j] * pitch + (int64_t)c * (W / 2);
        if (c + 8 <= cols) {
            if constexpr (W == 4) {
                Eight16 o;
#pragma unroll
                for (int i = 0; i < 4; ++i) o.v[i] = v[i];
                *(Eight16*)p = o;
            } else {
                Eight32 o;
#pragma unroll
                for (int i = 0; i < 8; ++i) o.v[i] = v[i];
                *(Eight32*)p = o;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < cols) {
                    if constexpr (W == 4) ((uint16_t*)p)[i] = (uint16_t)(v[i >> 1] >> (16 * (i & 1)));
                    else ((uint32_t*)p)[i] = v[i];
                }
        }
    }
}

int launched() { return hipGetLastError() == hipSuccess ? 0 : EXL3C4_E_DEVICE; }

// Rows in launches whose slots fit 32 bits (17 G columns each: one launch in all but the largest cases).
template <class F>
int each_part(int64_t rows, int64_t cols, F&& f) {
    const int64_t lanes = (cols + 31) / 32 * 4;
    const int64_t most = SLOTS / lanes < 1 ? 1 : SLOTS / lanes;
    for (int64_t r = 0; r < rows; r += most) {
        const int64_t n = rows - r < most ? rows - r : most;
        const uint32_t slots = (uint32_t)(n * lanes);
        f(r, slots, (uint32_t)lanes, dim3((slots + WG * PER - 1) / (WG * PER)));
        if (const int rc = launched()) return rc;
    }
    return 0;
}

}  // namespace

extern "C" int exl3c4_dev_mx4_quant(const void* x, int32_t dtype, int64_t rows, int64_t cols, int64_t pitch,
                                    uint8_t* codes, int64_t codes_pitch, uint8_t* scales, int64_t scales_pitch,
                                    void* stream) {
    const int64_t bytes = pitch * (dtype == EXL3C4_F32 ? 4 : 2);
    const auto f = dtype == EXL3C4_F32 ? k_mx4_quant<EXL3C4_F32>
                   : dtype == EXL3C4_F16 ? k_mx4_quant<EXL3C4_F16> : k_mx4_quant<EXL3C4_BF16>;
    return each_part(rows, cols, [&](int64_t r, uint32_t slots, uint32_t lanes, dim3 grid) {
        hipLaunchKernelGGL(f, grid, dim3(WG), 0, (hipStream_t)stream, (const char*)x + r * bytes, slots, lanes,
                           (uint32_t)cols, bytes, codes + r * codes_pitch, codes_pitch, scales + r * scales_pitch,
                           scales_pitch);
    });
}

extern "C" int exl3c4_dev_mx4_dequant(const uint8_t* codes, int64_t codes_pitch, const uint8_t* scales,
                                      int64_t scales_pitch, int64_t rows, int64_t cols, void* out, int32_t dtype,
                                      int64_t out_pitch, void* stream) {
    const int64_t bytes = out_pitch * (dtype == EXL3C4_F32 ? 4 : 2);
    const auto f = dtype == EXL3C4_F32 ? k_mx4_dequant<EXL3C4_F32>
                   : dtype == EXL3C4_F16 ? k_mx4_dequant<EXL3C4_F16> : k_mx4_dequant<EXL3C4_BF16>;
    return each_part(rows, cols, [&](int64_t r, uint32_t slots, uint32_t lanes, dim3 grid) {
        hipLaunchKernelGGL(f, grid, dim3(WG), 0, (hipStream_t)stream, codes + r * codes_pitch, codes_pitch,
                           scales + r * scales_pitch, scales_pitch, slots, lanes, (uint32_t)cols,
                           (char*)out + r * bytes, bytes);
    });
}
