/* exl3c4_gemm.c -- the C-ABI entry points of the products of 16-bit, MX4 and F8 experts and of MX4's and F8's conversions
 * (include/exl3c4.h): the refusals, before anything is written, then the device launch (exl3c4_gemm.hip, exl3c4_gemm_f8.hip,
 * exl3c4_mx4.hip, exl3c4_f8.hip). No counterpart in the reference. */
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

/* Whether matrices stride apart, of rows pitch apart (at least 1) that end after `last`, overlap (pitch * rows may pass 64 bits). */
static int overlap(int64_t stride, int64_t rows, int64_t pitch, int64_t last) {
    return stride < last || (stride - last) / pitch < rows - 1;
}

/* The F8 planes of n matrices and their values: what both conversions refuse, then the launch's block. */
static int f8_check(const Exl3c4F8* q, const void* v, int32_t dtype, int64_t pitch, int64_t stride, Exl3c4DevF8* a) {
    if (!q || (q->block != 1 && q->block != 128)) return EXL3C4_E_INVAL;
    if (!is_float(dtype)) return EXL3C4_E_DTYPE;
    if (q->n < 0 || q->rows < 0 || q->cols < 1 || q->n > MAX_EXTENT || q->rows > MAX_EXTENT || q->cols > MAX_EXTENT) return EXL3C4_E_SHAPE;
    const int64_t across = (q->cols + 127) / 128, down = (q->rows + q->block - 1) / q->block, code_cols = (q->cols + 15) / 16 * 16;
    if (q->n * q->rows > MAX_EXTENT || q->n * q->rows * across > ((int64_t)1 << 34)) return EXL3C4_E_SHAPE;   /* 2^41 columns: past any memory */
    if (q->block > 1 && q->n * down * across > (1 << 23)) return EXL3C4_E_SHAPE;            /* workgroups of 256 in a launch: 2^37 columns */
    if (q->n * q->rows > 0 && (!q->codes || !q->scales || !v)) return EXL3C4_E_INVAL;
    if (pitch < q->cols || q->codes_pitch < code_cols || q->scales_pitch < across) return EXL3C4_E_STRIDE;
    if (pitch > MAX_PITCH || q->codes_pitch > MAX_PITCH || q->scales_pitch > MAX_PITCH) return EXL3C4_E_STRIDE;
    const int apart = q->n > 1 && q->rows > 0;
    if (apart) {                                              /* a matrix's last row ends with its last column */
        const int64_t most = (int64_t)1 << 60;
        if (stride > most || q->codes_stride > most || q->scales_stride > most) return EXL3C4_E_STRIDE;
        if (overlap(stride, q->rows, pitch, q->cols) || overlap(q->codes_stride, q->rows, q->codes_pitch, code_cols) ||
            overlap(q->scales_stride, down, q->scales_pitch, across))
            return EXL3C4_E_STRIDE;
    }
    if ((uintptr_t)v % (uintptr_t)size_of(dtype) || (uintptr_t)q->codes % 16 || q->codes_pitch % 16 || (apart && q->codes_stride % 16) ||
        (uintptr_t)q->scales % 4)
        return EXL3C4_E_ALIGN;
    const int64_t size = size_of(dtype);
    a->v = (char*)v;
    a->codes = q->codes;
    a->scales = q->scales;
    a->v_pitch = pitch * size;
    a->codes_pitch = q->codes_pitch;
    a->scales_pitch = q->scales_pitch * 4;
    a->v_stride = apart ? stride * size : 0;
    a->codes_stride = apart ? q->codes_stride : 0;
    a->scales_stride = apart ? q->scales_stride * 4 : 0;
    a->n = (uint32_t)q->n;
    a->rows = (uint32_t)q->rows;
    a->cols = (uint32_t)q->cols;
    a->code_cols = (uint32_t)code_cols;
    a->block_log2 = q->block == 128 ? 7 : 0;
    return EXL3C4_OK;
}

int exl3c4_f8_quant(const void* x, int32_t x_dtype, int64_t x_pitch, int64_t x_stride, const Exl3c4F8* q, void* stream) {
    Exl3c4DevF8 a;
    const int   rc = f8_check(q, x, x_dtype, x_pitch, x_stride, &a);
    return rc ? rc : exl3c4_dev_f8_quant(&a, x_dtype, stream);
}

int exl3c4_f8_dequant(const Exl3c4F8* q, void* out, int32_t out_dtype, int64_t out_pitch, int64_t out_stride, void* stream) {
    Exl3c4DevF8 a;
    const int   rc = f8_check(q, out, out_dtype, out_pitch, out_stride, &a);
    return rc ? rc : exl3c4_dev_f8_dequant(&a, out_dtype, stream);
}

/* One operand of the product: rows of K columns, pitch as the caller gives it; *bytes: the pitch in bytes. table: p and scales are
 * device arrays of pointers. */
static int operand_check(int32_t type, const void* p, const void* scales, int table, int64_t pitch, int64_t s_pitch, int64_t K,
                         int64_t* bytes) {
    const int mx4 = type == EXL3C4_MX4, f8 = type == EXL3C4_F8, scaled = mx4 || f8;
    if (!p || (scaled && !scales)) return EXL3C4_E_INVAL;
    if (pitch < (mx4 ? K / 2 : K) || (mx4 && s_pitch < K / 32)) return EXL3C4_E_STRIDE;      /* K in whole blocks */
    if (f8 && s_pitch < (K + 127) / 128 * 4) return EXL3C4_E_STRIDE;
    if (pitch > MAX_PITCH || s_pitch > MAX_PITCH) return EXL3C4_E_STRIDE;
    *bytes = scaled ? pitch : 2 * pitch;
    if ((uintptr_t)p % (table ? 8 : 16) || *bytes % 16) return EXL3C4_E_ALIGN;
    if (scaled && ((uintptr_t)scales % (table ? 8 : 4) || s_pitch % 4)) return EXL3C4_E_ALIGN;
    return EXL3C4_OK;
}

int exl3c4_moe_gemm(const Exl3c4Gemm* g, void* stream) {
    if (!g || (g->act != EXL3C4_ACT_NONE && g->act != EXL3C4_ACT_SWIGLU)) return EXL3C4_E_INVAL;
    const int wide = (g->w_type == EXL3C4_F16 || g->w_type == EXL3C4_BF16) && g->x_type == g->w_type;
    const int mx4 = g->w_type == EXL3C4_MX4 &&
                    (g->x_type == EXL3C4_F16 || g->x_type == EXL3C4_BF16 || g->x_type == EXL3C4_MX4);
    const int f8 = g->w_type == EXL3C4_F8 &&
                   (g->x_type == EXL3C4_F16 || g->x_type == EXL3C4_BF16 || g->x_type == EXL3C4_F8);
    if ((!wide && !mx4 && !f8) || !is_float(g->y_type)) return EXL3C4_E_DTYPE;
    const int swiglu = g->act == EXL3C4_ACT_SWIGLU;
    if (g->N < 1 || g->K < 1 || g->n_expert < 1 || g->top_k < 1 || g->T < 0 || g->x_rows < 0) return EXL3C4_E_SHAPE;
    if (g->N > MAX_EXTENT || g->K > MAX_EXTENT || g->n_expert > MAX_EXTENT || g->top_k > MAX_EXTENT ||
        g->T > MAX_EXTENT || g->x_rows > MAX_EXTENT)
        return EXL3C4_E_SHAPE;
    if (g->K % (mx4 ? 32 : f8 ? 16 : 8) || (swiglu && g->N % 2)) return EXL3C4_E_SHAPE;
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
    const int64_t w_row = mx4 ? g->K / 2 : f8 ? g->K : 2 * g->K;
    if (g->w_stride != 0 && g->w_stride < (g->N - 1) * w_bytes + w_row) return EXL3C4_E_STRIDE;
    if (g->w_stride % 16) return EXL3C4_E_ALIGN;
    if (mx4 || f8) {
        const int64_t rows = mx4 ? g->N : (n_out + 127) / 128 * (swiglu ? 2 : 1);             /* of scales, and bytes of one */
        const int64_t row = mx4 ? (g->K / 32 + 3) / 4 * 4 : (g->K + 127) / 128 * 4;
        if (g->ws_stride != 0 && g->ws_stride < (rows - 1) * g->ws_pitch + row) return EXL3C4_E_STRIDE;
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
    if (f8) return exl3c4_dev_gemm_f8(&d, g->x_type, g->act, stream);
    return exl3c4_dev_gemm(&d, g->x_type, g->w_type, g->act, stream);
}
