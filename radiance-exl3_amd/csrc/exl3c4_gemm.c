/* exl3c4_gemm.c -- the C-ABI entry points of the products of 16-bit and MX4 experts and of MX4's conversions
 * (include/exl3c4.h): the refusals, before anything is written, then the device launch (exl3c4_gemm.hip,
 * exl3c4_mx4.hip). No counterpart in the reference. */
#include <stdint.h>

#include "exl3c4.h"
#include "exl3c4_dev.h"

/* extents that the kernels hold in 32 bits, with room for a tile's rounding up */
#define MAX_EXTENT (INT32_MAX - 65536)
/* byte pitches: offsets inside an operand stay far from 64 bits, and those of a weight's 16 rows in 32 */
#define MAX_PITCH ((int64_t)1 << 40)
#define MAX_W_PITCH ((int64_t)1 << 27)

static int size_of(int32_t type) { return type == EXL3C4_F32 ? 4 : 2; }
static int is_float(int32_t type) { return type == EXL3C4_F16 || type == EXL3C4_BF16 || type == EXL3C4_F32; }

/* The MX4 planes of rows of `cols`: what both conversions refuse. */
static int mx4_check(const void* codes, int64_t codes_pitch, const void* scales, int64_t scales_pitch, const void* v,
                     int32_t dtype, int64_t rows, int64_t cols, int64_t pitch) {
    if (!is_float(dtype)) return EXL3C4_E_DTYPE;
    if (rows < 0 || cols < 1 || rows > MAX_EXTENT || cols > MAX_EXTENT) return EXL3C4_E_SHAPE;
    const int64_t blocks = (cols + 31) / 32;
    if (rows * blocks > ((int64_t)1 << 36)) return EXL3C4_E_SHAPE;      /* 2^41 columns: past any memory */
    if (rows > 0 && (!codes || !scales || !v)) return EXL3C4_E_INVAL;
    if (pitch < cols || codes_pitch < 16 * blocks || scales_pitch < blocks) return EXL3C4_E_STRIDE;
    if (pitch > MAX_PITCH || codes_pitch > MAX_PITCH || scales_pitch > MAX_PITCH) return EXL3C4_E_STRIDE;
    if ((uintptr_t)v % (uintptr_t)size_of(dtype) || (uintptr_t)codes % 16 || codes_pitch % 16 ||
        (uintptr_t)scales % 4 || scales_pitch % 4)
        return EXL3C4_E_ALIGN;
    return EXL3C4_OK;
}

int exl3c4_mx4_quant(const void* x, int32_t x_dtype, int64_t rows, int64_t cols, int64_t x_pitch, void* codes,
                     int64_t codes_pitch, void* scales, int64_t scales_pitch, void* stream) {
    const int rc = mx4_check(codes, codes_pitch, scales, scales_pitch, x, x_dtype, rows, cols, x_pitch);
    if (rc) return rc;
    return exl3c4_dev_mx4_quant(x, x_dtype, rows, cols, x_pitch, (uint8_t*)codes, codes_pitch, (uint8_t*)scales,
                                scales_pitch, stream);
}

int exl3c4_mx4_dequant(const void* codes, int64_t codes_pitch, const void* scales, int64_t scales_pitch, int64_t rows,
                       int64_t cols, void* out, int32_t out_dtype, int64_t out_pitch, void* stream) {
    const int rc = mx4_check(codes, codes_pitch, scales, scales_pitch, out, out_dtype, rows, cols, out_pitch);
    if (rc) return rc;
    return exl3c4_dev_mx4_dequant((const uint8_t*)codes, codes_pitch, (const uint8_t*)scales, scales_pitch, rows, cols,
                                  out, out_dtype, out_pitch, stream);
}

/* One operand of the product: rows of K columns, pitch as the caller gives it; *bytes: the pitch in bytes. table: p and scales are
 * device arrays of pointers. */
static int operand_check(int32_t type, const void* p, const void* scales, int table, int64_t pitch, int64_t s_pitch, int64_t K,
                         int64_t* bytes) {
    const int mx4 = type == EXL3C4_MX4;
    if (!p || (mx4 && !scales)) return EXL3C4_E_INVAL;
    if (pitch < (mx4 ? K / 2 : K) || (mx4 && s_pitch < K / 32)) return EXL3C4_E_STRIDE;      /* K in whole blocks */
    if (pitch > MAX_PITCH || s_pitch > MAX_PITCH) return EXL3C4_E_STRIDE;
    *bytes = mx4 ? pitch : 2 * pitch;
    if ((uintptr_t)p % (table ? 8 : 16) || *bytes % 16) return EXL3C4_E_ALIGN;
    if (mx4 && ((uintptr_t)scales % (table ? 8 : 4) || s_pitch % 4)) return EXL3C4_E_ALIGN;
    return EXL3C4_OK;
}

int exl3c4_moe_gemm(const Exl3c4Gemm* g, void* stream) {
    if (!g || (g->act != EXL3C4_ACT_NONE && g->act != EXL3C4_ACT_SWIGLU)) return EXL3C4_E_INVAL;
    const int wide = (g->w_type == EXL3C4_F16 || g->w_type == EXL3C4_BF16) && g->x_type == g->w_type;
    const int mx4 = g->w_type == EXL3C4_MX4 &&
                    (g->x_type == EXL3C4_F16 || g->x_type == EXL3C4_BF16 || g->x_type == EXL3C4_MX4);
    if ((!wide && !mx4) || !is_float(g->y_type)) return EXL3C4_E_DTYPE;
    const int swiglu = g->act == EXL3C4_ACT_SWIGLU;
    if (g->N < 1 || g->K < 1 || g->n_expert < 1 || g->top_k < 1 || g->T < 0 || g->x_rows < 0) return EXL3C4_E_SHAPE;
    if (g->N > MAX_EXTENT || g->K > MAX_EXTENT || g->n_expert > MAX_EXTENT || g->top_k > MAX_EXTENT ||
        g->T > MAX_EXTENT || g->x_rows > MAX_EXTENT)
        return EXL3C4_E_SHAPE;
    if (g->K % (mx4 ? 32 : 8) || (swiglu && g->N % 2)) return EXL3C4_E_SHAPE;
    const int64_t n_out = swiglu ? g->N / 2 : g->N;
    if (g->y_pitch < n_out || g->y_pitch > MAX_PITCH) return EXL3C4_E_STRIDE;
    if (!g->expert_offset) return EXL3C4_E_INVAL;
    Exl3c4DevGemm d;
    int64_t       x_bytes = 0, w_bytes = 0;
    int           rc;
    if (g->T == 0) return EXL3C4_OK;
    if (!g->y) return EXL3C4_E_INVAL;
    if (g->x_rows < (g->sorted_tok ? 1 : g->T)) return EXL3C4_E_SHAPE;
    rc = operand_check(g->x_type, g->x, g->x_scales, 0, g->x_pitch, g->xs_pitch, g->K, &x_bytes);
    if (rc) return rc;
    rc = operand_check(g->w_type, g->w, g->w_scales, g->w_stride == 0, g->w_pitch, g->ws_pitch, g->K, &w_bytes);
    if (rc) return rc;
    if (w_bytes > MAX_W_PITCH || g->ws_pitch > MAX_W_PITCH) return EXL3C4_E_STRIDE;
    /* an entry's last row ends with its last column */
    const int64_t w_row = g->w_type == EXL3C4_MX4 ? g->K / 2 : 2 * g->K;
    if (g->w_stride != 0 && g->w_stride < (g->N - 1) * w_bytes + w_row) return EXL3C4_E_STRIDE;
    if (g->w_stride % 16) return EXL3C4_E_ALIGN;
    if (g->w_type == EXL3C4_MX4) {
        if (g->ws_stride != 0 && g->ws_stride < (g->N - 1) * g->ws_pitch + (g->K / 32 + 3) / 4 * 4) return EXL3C4_E_STRIDE;
        if (g->ws_stride % 4) return EXL3C4_E_ALIGN;
        if ((g->ws_stride == 0) != (g->w_stride == 0)) return EXL3C4_E_INVAL;      /* one form for both tables */
    }
    if ((uintptr_t)g->y % (uintptr_t)size_of(g->y_type) || (uintptr_t)g->sorted_tok % 4 ||
        (uintptr_t)g->expert_offset % 4)
        return EXL3C4_E_ALIGN;
    d.x = (const char*)g->x;
    d.xs = (const uint8_t*)g->x_scales;
    d.w = (const char*)g->w;
    d.ws = (const char*)g->w_scales;
    d.sorted = g->sorted_tok;
    d.off = g->expert_offset;
    d.y = (char*)g->y;
    d.x_pitch = x_bytes;
    d.xs_pitch = g->xs_pitch;
    d.w_pitch = w_bytes;
    d.ws_pitch = g->ws_pitch;
    d.w_stride = g->w_stride;
    d.ws_stride = g->ws_stride;
    d.y_pitch = g->y_pitch * size_of(g->y_type);
    d.x_rows = (int32_t)g->x_rows;
    d.T = (int32_t)g->T;
    d.n_expert = (int32_t)g->n_expert;
    d.top_k = (int32_t)g->top_k;
    d.N = (int32_t)g->N;
    d.K = (int32_t)g->K;
    d.n_out = (int32_t)n_out;
    d.y_type = g->y_type;
    d.tiles = 0;                                              /* the launcher's */
    return exl3c4_dev_gemm(&d, g->x_type, g->w_type, g->act, stream);
}
