"""moe_gemm over the whole range of MX4's scales, whatever x's type: the largest ones (byte 254 is 2^127, where codes 2 to 6 pass
every 16- and 32-bit float by themselves) against x so small that the sums are finite, or zero; the smallest ones beside them;
and the conversions at the same bytes."""
import pytest

import gemmpath
import mx4ref
from test_gpu_moe_gemm import ex, operand  # noqa: F401 (ex is a fixture)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

PATHS = [2, 4, 32, 64]                                                   # few rows an expert by 2 and 4 strips, tiles of 32 and 64 rows


def size_of(kind, p):
    """(T, experts, experts with weights of their own, N, K): steps of four and a rest for each wave of few rows."""
    T, E, N = gemmpath.SIZES[p]
    K = 2592 if p in (2, 4) else 416
    assert gemmpath.path((kind, "mx4"), False, T, E, N, K) == p
    return T, E, min(E, 3), N, K


def check(ex, xd, x64, wd, w64, T, E):  # noqa: F811
    N = w64.shape[1]
    w64 = gemmpath.Shared(w64, E)
    off = torch.tensor([T * e // E for e in range(E + 1)], dtype=torch.int32)
    y = torch.full((T, N), float("nan"), device="cuda")
    gm = ex.make_gemm(xd, wd, None, off.cuda(), y)
    assert ex.moe_gemm(gemmpath.share(gm, wd, E) if E > w64.w64.shape[0] else gm) == 0
    got = y.cpu()
    want, tol = mx4ref.gemm(x64, w64, None, off, T, 1, False)
    assert mx4ref.close(got, want, tol)


@pytest.mark.parametrize("kind", ["f16", "bf16", "mx4"])
@pytest.mark.parametrize("p", PATHS)
def test_the_largest_scales(ex, kind, p):  # noqa: F811
    """Scale bytes up to 254 in some rows and blocks, x about 2^-12 (sums below 2^127): finite in 64 bits and in f32."""
    T, E, n, N, K = size_of(kind, p)
    print(f"moe_gemm {kind} path {p}: scales 250 .. 254", flush=True)
    g = torch.Generator().manual_seed(1)
    s = torch.randint(250, 255, (n, N, K // 32), generator=g)
    s[:, ::3] = torch.randint(118, 123, s[:, ::3].shape, generator=g)           # rows without them
    s[:, 1::3, 1::2] = torch.randint(100, 255, s[:, 1::3, 1::2].shape, generator=g)
    wd, w64 = gemmpath.mx4_weights(g, n, N, K, s)
    xd, x64 = operand(ex, torch.randn((T, K), generator=g) * 2.0 ** -12, kind)
    check(ex, xd, x64, wd, w64, T, E)


@pytest.mark.parametrize("kind", ["f16", "bf16", "mx4"])
@pytest.mark.parametrize("p", PATHS)
def test_zeros_of_x_at_the_largest_scales(ex, kind, p):  # noqa: F811
    """Blocks of x that are zero against scales 252 .. 254: they add nothing, and the other blocks -- of ordinary scales, and of the
    smallest the format has -- make the sums."""
    T, E, n, N, K = size_of(kind, p)
    g = torch.Generator().manual_seed(2)
    x = torch.randn((T, K // 32, 32), generator=g) * 64
    x[:, ::2] = 0
    for low, high in ((110, 130), (0, 3)):
        print(f"moe_gemm {kind} path {p}: zeros, scales {low} .. {high}", flush=True)
        s = torch.randint(low, high, (n, N, K // 32), generator=g)
        s[:, :, ::2] = torch.randint(252, 255, s[:, :, ::2].shape, generator=g)
        wd, w64 = gemmpath.mx4_weights(g, n, N, K, s)
        xd, x64 = operand(ex, x.view(T, K), kind)
        check(ex, xd, x64, wd, w64, T, E)


@pytest.mark.parametrize("p", PATHS)
def test_infinities_beside_the_largest_scales(ex, p):  # noqa: F811
    """bf16 x with an infinity and a NaN, weights with a NaN block: what the definition gives, and no more."""
    T, E, n, N, K = size_of("bf16", p)
    g = torch.Generator().manual_seed(3)
    s = torch.randint(245, 255, (n, N, K // 32), generator=g)
    s[:, 5, 2] = 255
    wd, w64 = gemmpath.mx4_weights(g, n, N, K, s)
    x = torch.randn((T, K), generator=g) * 2.0 ** -14
    x[1, 7], x[2, K - 1], x[3, 40] = float("inf"), -float("inf"), float("nan")
    xd, x64 = operand(ex, x, "bf16")
    check(ex, xd, x64, wd, w64, T, E)


@pytest.mark.parametrize("out", [torch.float16, torch.bfloat16, torch.float32], ids=str)
def test_dequant_of_every_scale_and_code(ex, out):  # noqa: F811
    """All 256 scale bytes with all 16 codes: the value rounded to nearest, infinite past the type's range, NaN at 255."""
    codes = torch.tensor([2 * i % 16 | (2 * i + 1) % 16 << 4 for i in range(16)], dtype=torch.uint8).repeat(256, 1)
    s = torch.zeros(256, 4, dtype=torch.uint8)
    s[:, 0] = torch.arange(256)
    q = ex.Mx4(codes.cuda(), s.cuda(), 32)
    y = torch.zeros(256, 32, dtype=out, device="cuda")
    assert ex.mx4_dequant(q, y) == 0
    want = mx4ref.dequant(codes, s, 32).to(torch.float32).to(out)
    got = y.cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(7), want.nan_to_num(7))
