"""moe_gemm with F8 on both sides where a block's two scales multiply to numbers that f32 does not hold, or holds with fewer bits, though it holds the
sums: scales that multiply to 2^135 on the smallest codes, and to 2^-140 on the largest, zeros among them; and bf16 rows whose products with codes alone
f32 does not hold. On every kernel, against the product in 64 bits."""
import numpy as np
import pytest

import f8ref
import mx4ref
from test_gpu_moe_gemm_f8 import SIZES, TYPES, ex, path

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
PATHS = [(y, p) for y in ("f32", "bf16") for p in ((2, 4, 32, 64) if y == "f32" else (2, 4, 32, 64, 128))]
# (codes of both sides, scale of x, scale of weights): products of 2^-18 x 2^135 to 2^137, or of up to 2^17.6 x 2^-140 to 2^-138
FAR = {"above": ((0x00, 0x01, 0x80, 0x81), 2.0 ** 70, 2.0 ** 65), "weights above": ((0x00, 0x01, 0x80, 0x81), 2.0 ** 9, 2.0 ** 126),
       "below": ((0x00, 0x7E, 0x78, 0xF9, 0xFE), 2.0 ** -70, 2.0 ** -70), "x below": ((0x00, 0x7E, 0x78, 0xF9, 0xFE), 2.0 ** -104, 2.0 ** -36),
       "weights' least": ((0x00, 0x7E, 0x78, 0xF9, 0xFE), 2.0 ** 24, 2.0 ** -140), "x's least": ((0x00, 0x7E, 0x78, 0xF9, 0xFE), 2.0 ** -126, 2.0 ** 14)}


def operands(g, codes, sx, sw, T, E, N, K, swiglu, signs=False):
    """(x, its values, its peaks, w, its values, its peaks): codes drawn from `codes`, scales sx and sw times 1 to 2 (signs: of either sign), a row of x, a weight
    row and a block of weights of zeros."""
    table = torch.tensor(codes, dtype=torch.uint8)
    halves, across = (2 if swiglu else 1), (K + 127) // 128
    down = halves * ((N // halves + 127) // 128)
    cx, cw = (table[torch.randint(0, len(codes), s, generator=g)] for s in ((T, K), (E, N, K)))
    xs, ws = ((1 + torch.rand(s, generator=g, dtype=torch.float64)) * v for s, v in (((T, across), sx), ((E, down, across), sw)))
    if signs:
        xs, ws = (v * (torch.randint(0, 2, v.shape, generator=g) * 2 - 1) for v in (xs, ws))
    cx[T // 2], cw[:, N // 3], cw[0, :min(128, N // halves), :min(128, K)] = 0, 0, 0
    xs, ws = xs.float(), ws.float()
    spread = xs.double().repeat_interleave(128, 1)[:, :K]
    one = torch.full((E, N, K), 0x38, dtype=torch.uint8)
    return (cx, xs, f8ref.values(cx[None], xs[None], K, 1)[0], f8ref.peaks(cx, spread.abs()),
            cw, ws, f8ref.weights(cw, ws, halves), f8ref.peaks(cw, f8ref.weights(one, ws, halves).abs()))


def product(ex, yt, p, far, swiglu=False, signs=False):
    """(got, want, tolerance) on kernel p."""
    T, E, N, K = SIZES[p]
    assert path(ex, "f8", yt, swiglu, T, E, N // 2 if swiglu else N, K) == p
    cx, xs, xv, xp, cw, ws, wv, wp = operands(torch.Generator().manual_seed(p), *far, T, E, N, K, swiglu, signs)
    off = np.array([T * e // E for e in range(E + 1)], np.int32)
    n_out = N // 2 if swiglu else N
    y = torch.full((T, n_out), 5.0, dtype=TYPES[yt], device="cuda")
    g = ex.make_gemm(ex.F8(cx.cuda(), xs.cuda(), K, 1), ex.F8(cw.cuda(), ws.cuda(), K, 128), None, torch.from_numpy(off).cuda(), y,
                     act=ex.ACT_SWIGLU if swiglu else ex.ACT_NONE)
    assert ex.moe_gemm(g) == 0
    torch.cuda.synchronize()
    want, tol = f8ref.gemm(xv, wv, None, off, T, 1, swiglu, (xp, wp) if yt != "f32" and p >= 32 else None)
    return y.cpu(), want, tol


@pytest.mark.parametrize("yt,p", PATHS)
@pytest.mark.parametrize("far", list(FAR))
@pytest.mark.parametrize("signs", [False, True])
def test_products_of_scales_beyond_f32(ex, yt, p, far, signs):
    got, want, tol = product(ex, yt, p, FAR[far], signs=signs)
    assert (want.abs().amax() < 3e38) and (want.abs().amax() > 1e-37)
    assert mx4ref.close(got, want, tol)
    assert (got[want == 0] == 0).all()


@pytest.mark.parametrize("yt,p", PATHS)
def test_scales_of_x_below_the_normal_numbers(ex, yt, p):
    """x's scale meets a number of 1 to 2 in f32, whose step is 2^-149 there: half of that for each code times its weight."""
    T, E, N, K = SIZES[p]
    g = torch.Generator().manual_seed(p)
    cx, _, _, _, _, _, wv, _ = operands(g, FAR["below"][0], 2.0 ** -140, 2.0 ** 20, T, E, N, K, False)
    got, want, tol = product(ex, yt, p, (FAR["below"][0], 2.0 ** -140, 2.0 ** 20))
    off = [T * e // E for e in range(E + 1)]
    step, _ = f8ref.gemm(torch.from_numpy(np.abs(f8ref.decode(cx.numpy()))), wv.abs(), None, off, T, 1, False)
    assert mx4ref.close(got, want, tol + 2.0 ** -150 * step)


@pytest.mark.parametrize("yt,p", PATHS)
def test_scales_of_zero_infinity_and_nan(ex, yt, p):
    """A scale is any number: zero makes its block zeros, infinity and NaN what code times scale is (0 times infinity is NaN), in the block's own rows alone."""
    T, E, N, K = SIZES[p]
    cx, xs, xv, xp, cw, ws, wv, wp = operands(torch.Generator().manual_seed(p), (0x38, 0x3A, 0xB8), 1.0, 1.0, T, E, N, K, False)
    xs[0, 0], xs[1, 0], xs[2, 1], xs[3, :], ws[0, 1, 0] = 0.0, float("inf"), float("nan"), 0.0, 0.0
    spread = xs.double().repeat_interleave(128, 1)[:, :K]
    xv, wv = f8ref.values(cx[None], xs[None], K, 1)[0], f8ref.weights(cw, ws, 1)
    off = np.array([T * e // E for e in range(E + 1)], np.int32)
    y = torch.full((T, N), 5.0, dtype=TYPES[yt], device="cuda")
    assert ex.moe_gemm(ex.make_gemm(ex.F8(cx.cuda(), xs.cuda(), K, 1), ex.F8(cw.cuda(), ws.cuda(), K, 128), None, torch.from_numpy(off).cuda(), y)) == 0
    torch.cuda.synchronize()
    live = [r for r in range(T) if r not in (1, 2)]
    fin = xv.clone()
    fin[1:3] = 0
    want, tol = f8ref.gemm(fin, wv, None, off, T, 1, False, (f8ref.peaks(cx, spread.nan_to_num(0, 0, 0)), wp) if yt != "f32" and p >= 32 else None)
    got = y.cpu()
    assert mx4ref.close(got[live], want[live], tol[live])
    assert got[2].isnan().all() and not torch.isfinite(got[1]).any() and (got[3] == 0).all()


@pytest.mark.parametrize("yt,p", PATHS)
def test_zeros_whatever_the_scales_with_swiglu(ex, yt, p):
    got, want, _ = product(ex, yt, p, ((0x00, 0x80), 2.0 ** 70, 2.0 ** 65), swiglu=True)
    assert (want == 0).all() and (got == 0).all()


@pytest.mark.parametrize("yt,p", [(y, p) for y in ("f32", "bf16") for p in (2, 4, 32, 64)])
@pytest.mark.parametrize("swiglu", [False, True])
def test_bf16_rows_near_the_end_of_f32(ex, yt, p, swiglu):
    """x up to 3e38 against weights far below 1 by their scale, not by their codes (gate and up: 2^-130, so that their product stays in f32)."""
    T, E, N, K = SIZES[p]
    assert path(ex, "bf16", yt, swiglu, T, E, N // 2 if swiglu else N, K) == p
    g = torch.Generator().manual_seed(p)
    x = (torch.randn((T, K), generator=g).clamp(-3, 3) * 1e38).bfloat16()
    _, _, _, _, cw, ws, wv, _ = operands(g, (0x00, 0x7E, 0x78, 0xF9, 0xFE, 0x38), 1.0, 2.0 ** (-130 if swiglu else -24), T, E, N, K, swiglu)
    off = np.array([T * e // E for e in range(E + 1)], np.int32)
    n_out = N // 2 if swiglu else N
    y = torch.full((T, n_out), 5.0, dtype=TYPES[yt], device="cuda")
    gm = ex.make_gemm(x.cuda(), ex.F8(cw.cuda(), ws.cuda(), K, 128), None, torch.from_numpy(off).cuda(), y, act=ex.ACT_SWIGLU if swiglu else ex.ACT_NONE)
    assert ex.moe_gemm(gm) == 0
    torch.cuda.synchronize()
    want, tol = f8ref.gemm(x.double(), wv, None, off, T, 1, swiglu)
    assert want.abs().amax() < 3e38
    assert mx4ref.close(y.cpu(), want, tol)
