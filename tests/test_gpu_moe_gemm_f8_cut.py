"""The bound of the matrix unit's 8-bit products as include/exl3c4.h states it: of eight neighbouring columns each product may lose 2^-13 of the largest, each code's
magnitude taken as 2^-6 at least. The largest is of the products themselves, row of x by row of weights (tests/f8ref.py bounds it by the two operands' own largest)."""
import numpy as np
import pytest

import f8ref
import mx4ref
from test_gpu_moe_gemm_f8 import TYPES, ex, path

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def largest(cx, cw):
    """Sum over the eights of their largest product of magnitudes of at least 2^-6, f64 [rows of x, rows of w] of codes [.., K], by blocks of 128: [K / 128 up, .., ..]."""
    mx, mw = (torch.from_numpy(np.maximum(np.abs(f8ref.decode(c.numpy())), 2.0 ** -6)).cuda() for c in (cx, cw))
    K = cx.shape[1]
    out = torch.zeros((K + 127) // 128, len(cx), len(cw), dtype=torch.float64, device="cuda")
    for k in range(0, K, 8):
        top = mx[:, k, None] * mw[None, :, k]
        for j in range(k + 1, k + 8):
            top = torch.maximum(top, mx[:, j, None] * mw[None, :, j])
        out[k // 128] += top
    return out.cpu()


def codes(g, shape, kind):
    """wide: every code but NaN; unlike: mostly tiny ones, some of the largest, so that an operand's largest meets the other's smallest; normal: quantised values."""
    if kind == "normal":
        return f8ref.quant(torch.randn((1,) + shape, generator=g), 1)[0][0, :, :shape[1]]
    c = torch.randint(0, 254, shape, dtype=torch.uint8, generator=g)
    c = torch.where(c >= 127, c + 1, c)
    if kind == "unlike":
        tiny = torch.randint(0, 16, shape, dtype=torch.uint8, generator=g) | (c & 0x80)
        c = torch.where(torch.rand(shape, generator=g) < 0.8, tiny, c)
    return c


@pytest.mark.parametrize("yt", ["f16", "bf16"])
@pytest.mark.parametrize("p", [32, 64, 128])
@pytest.mark.parametrize("kind", ["wide", "unlike", "normal"])
def test_sums_within_the_stated_bound(ex, yt, p, kind):
    T, N, K = {32: (16, 9000, 144), 64: (300, 13330, 144), 128: (600, 13330, 272)}[p]
    assert path(ex, "f8", yt, False, T, 1, N, K) == p
    g = torch.Generator().manual_seed(p)
    cx, cw = codes(g, (T, K), kind), codes(g, (N, K), kind)
    across, down = (K + 127) // 128, (N + 127) // 128
    sx, sw = torch.rand((T, across), generator=g) * 2.0 ** -8 + 2.0 ** -9, torch.rand((1, down, across), generator=g) * 2.0 ** -4 + 2.0 ** -5
    y = torch.full((T, N), 5.0, dtype=TYPES[yt], device="cuda")
    off = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    assert ex.moe_gemm(ex.make_gemm(ex.F8(cx.cuda(), sx.cuda(), K, 1), ex.F8(cw[None].cuda(), sw.cuda(), K, 128), None, off, y)) == 0
    torch.cuda.synchronize()
    want, tol = f8ref.gemm(f8ref.values(cx[None], sx[None], K, 1)[0], f8ref.weights(cw[None], sw, 1), None, [0, T], T, 1, False)
    swn = sw[0].double().repeat_interleave(128, 0)[:N]
    for b, top in enumerate(largest(cx, cw)):
        tol += 7 * 2.0 ** -13 * top * sx[:, b, None].double() * swn[None, :, b]
    assert mx4ref.close(y.cpu(), want, tol)


def test_a_subnormal_code_counts_as_its_exponent(ex):
    """In each eight 2^-9 times 256, a product of 2^-1 of the exponents -6 and 8, beside seven of 15/8 times 3 x 2^-9, that are no multiples of 2^-11: what is lost of
    those passes 2^-13 of the eight's largest product and keeps the stated bound."""
    T, N, K = 16, 9000, 128
    assert path(ex, "f8", "f16", False, T, 1, N, K) == 32
    cx, cw = torch.full((T, K), 0x3F, dtype=torch.uint8), torch.full((1, N, K), 0x03, dtype=torch.uint8)
    cx[:, ::8], cw[..., ::8] = 0x01, 0x78
    cw[..., 8::16] = 0xF8                                            # (of either sign: the large ones cancel, and f16 holds the rest)
    cx[:, 8::16] = 0x01
    one = torch.ones
    y = torch.zeros((T, N), dtype=torch.float16, device="cuda")
    off = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    q = ex.F8(cx.cuda(), one((T, 1), device="cuda"), K, 1), ex.F8(cw.cuda(), one((1, (N + 127) // 128, 1), device="cuda"), K, 128)
    assert ex.moe_gemm(ex.make_gemm(*q, None, off, y)) == 0
    torch.cuda.synchronize()
    small = 15 / 8 * 3 * 2.0 ** -9
    want = 16 * 7 * small
    lost = (want - y.cpu().double()).abs().max().item()
    print(f"lost {lost} of {want}: {lost / (16 * 7) * 2 ** 13:.3f} of 2^-13 a small product", flush=True)
    assert lost <= 16 * 7 * 2.0 ** -13 * (2.0 ** -6 * 256) + 2.0 ** -11 * want
