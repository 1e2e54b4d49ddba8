"""moe_gemm's SwiGLU over the whole range of its gate, sums exact by construction (x is 1 in one column, 0 in the others): silu(g) u against
64 bits where e^-g and silu itself leave f32's range, with u that brings the product back, and infinities and NaNs.

The bound, in units of 2^-24 of the value: from g = -8 up the exponent's argument is rounded once (1.22 |g| with log2 e's own rounding, at
most 9.8), exp2 and the reciprocal take 2 each, the sum and the products 1 each: 16.8. Below, the argument's rounding takes 1: 9. Then the
output's own rounding, half its least step where it is subnormal."""
import pytest

import gemmpath
import mx4ref
from test_gpu_moe_gemm import PAIRS, TYPES, ex, operand  # noqa: F401 (ex is a fixture)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
STEPS = 17 * 2.0 ** -24
INF, NAN = float("inf"), float("nan")

# (T, experts) that take each kernel with 1,000 columns of y: few rows by 2 and 4 strips, tiles of 32 to 256 rows
SIZES = {2: (6, 2), 4: (33, 33), 32: (90, 2), 64: (1100, 3), 128: (2000, 3), 256: (16000, 3)}


def takes(pair, p, n):
    """Whether p is a path of the pair (at 32 columns of k MX4 x has no tiles of 256 rows), which the size then takes."""
    if p not in gemmpath.paths(pair) or (pair[0] == "mx4" and p == 256):
        return False
    assert gemmpath.path(pair, True, *SIZES[p], n, 32) == p
    return True


def gates(pair):
    """(g, u) in f32, exact in the weights' type: MX4 has a code times a power of two, f16 no u past 2^15."""
    if pair[1] == "mx4":
        m = torch.tensor([1.0, 1.5, 2, 3])
        g = torch.cat([-m * s for s in (2.0 ** torch.arange(-3, 7)).tolist()] + [m * s for s in (0.25, 1, 4, 16, 64)])
    else:
        g = torch.cat([torch.linspace(-130, 95, 181), torch.linspace(-89.5, -86, 15), torch.tensor([-8.0, -7.96875, 0.0])])
    big = 2.0 ** 15 if pair[1] == "f16" else 2.0 ** 100
    u = torch.tensor([1.0, -1.5, big, 3 / big, 2 * big ** 0.75])
    t = TYPES.get(pair[1], torch.float32)
    g, u = g.to(t).float(), (u if pair[1] != "mx4" else torch.tensor([1.0, -1.5, 2.0 ** 100, 3 * 2.0 ** -100, 2.0 ** 76])).to(t).float()
    return g.repeat_interleave(len(u)), u.repeat(len(g))


def layer(ex, pair, T, E, g, u, yt):  # noqa: F811
    n, K = len(g), 32
    w = torch.zeros(1, 2 * n, K)
    w[0, :n, 5], w[0, n:, 5] = g, u
    x = torch.zeros(T, K)
    x[:, 5] = 1
    if pair[1] == "mx4":                                               # one expert's planes quantised, then repeated
        q, v = operand(ex, w[0], "mx4")
        assert torch.equal(v[:, 5], w[0, :, 5].double())
        wd = ex.Mx4(q.codes.repeat(E, 1, 1), q.scales.repeat(E, 1, 1), K)
    else:
        wd = w.to(TYPES[pair[1]]).repeat(E, 1, 1).cuda()
    off = torch.tensor([T * e // E for e in range(E + 1)], dtype=torch.int32).cuda()
    y = torch.full((T, n), 7.0, dtype=TYPES[yt], device="cuda")
    assert ex.moe_gemm(ex.make_gemm(operand(ex, x, pair[0])[0], wd, None, off, y, act=ex.ACT_SWIGLU)) == 0
    got = y.cpu()
    assert torch.equal(got.nan_to_num(nan=3.25), got[:1].nan_to_num(nan=3.25).expand_as(got))     # every row the same
    return got[0]


@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
@pytest.mark.parametrize("p", list(SIZES))
@pytest.mark.parametrize("yt", ["f32", "bf16"])
def test_gates_of_every_size(ex, pair, p, yt):  # noqa: F811
    g, u = gates(pair)
    assert len(g) <= 1000
    g, u = g.repeat(4)[:1000], u.repeat(4)[:1000]                      # 1,000 columns, so that the sizes take their kernels
    if not takes(pair, p, len(g)):
        return
    print(f"swiglu {pair} path {p} {yt}: {len(g)} gates", flush=True)
    got = layer(ex, pair, *SIZES[p], g, u, yt)
    want = torch.nn.functional.silu(g.double()) * u.double()
    over = want.abs() >= 2.0 ** 128
    assert torch.equal(got[over].double(), torch.sign(want[over]) * INF)
    err = ((got.double() - want).abs() - mx4ref.TINY[got.dtype])[~over] / want.abs()[~over].clamp(min=1e-300)
    print(f"worst {float(err.max()) * 2 ** 24:.1f} steps at g {float(g[~over][err.argmax()])}, u {float(u[~over][err.argmax()])}", flush=True)
    assert mx4ref.close(got[~over], want[~over], STEPS * want[~over].abs())


@pytest.mark.parametrize("pair", [p for p in PAIRS if p[1] != "mx4"], ids="-".join)
@pytest.mark.parametrize("p", list(SIZES))
def test_infinite_gates_and_what_is_beside_them(ex, pair, p):  # noqa: F811
    """g / (1 + e^-g) u of infinities and NaNs, by IEEE's rules; the columns beside them as always."""
    g = torch.tensor([INF, INF, -INF, NAN, 2.0, -3.0, -120.0, 1.0, -65504.0, 60000.0]).repeat(100)
    u = torch.tensor([2.0, -3.0, 1.0, 1.0, INF, NAN, -INF, 0.5, 1024.0, 2.0]).repeat(100)
    assert takes(pair, p, len(g))
    t = TYPES[pair[1]]
    g, u = g.to(t).float(), u.to(t).float()
    # a zero of x times an infinity is a NaN, so x has one column only that is not a weight's zero: K = 32, the others 0 x 0
    got = layer(ex, pair, *SIZES[p], g, u, "f32")
    want = g.double() / (1 + torch.exp(-g.double())) * u.double()
    assert mx4ref.close(got, want, STEPS * want.abs().nan_to_num(0, 0, 0))


def test_a_row_goes_by_itself(ex):  # noqa: F811
    """A row's bits do not change with the gates of the rows and columns beside it."""
    rng = torch.Generator().manual_seed(1)
    for p, (T, E) in SIZES.items():
        n, K = 1000, 32
        w = (torch.randn(1, 2 * n, K, generator=rng) / 4).bfloat16().repeat(E, 1, 1).cuda()
        x = torch.randn(T, K, generator=rng).bfloat16()
        off = torch.tensor([T * e // E for e in range(E + 1)], dtype=torch.int32).cuda()
        got = []
        for scale in (1, 64):
            v = x.clone()
            v[1::2] *= scale
            y = torch.zeros(T, n, device="cuda")
            assert ex.moe_gemm(ex.make_gemm(v.cuda(), w, None, off, y, act=ex.ACT_SWIGLU)) == 0
            got.append(y.cpu())
        assert torch.equal(got[0][::2], got[1][::2]) and not torch.equal(got[0][1::2], got[1][1::2]), p
