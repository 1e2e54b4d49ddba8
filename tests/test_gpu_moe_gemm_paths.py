"""moe_gemm on the device, every kernel on purpose (tests/gemmpath.py: the library's own rule says that a size takes it): edges in rows, columns
and k, dropped rows, infinities and NaNs, scales far apart, offsets past 32 bits, graphs and streams; against the product in 64 bits."""
import pytest

import gemmpath
import mx4ref
from test_gpu_moe_gemm import PAIRS, ex, operand  # noqa: F401 (ex is a fixture)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
PATHS = [pytest.param(pair, p, id=f"{'-'.join(pair)}-{p}") for pair in PAIRS for p in gemmpath.paths(pair)]
NAN, INF = float("nan"), float("inf")


def k_of(pair, p):
    """Columns that end inside a step and a stage: each of the four waves of few rows has four steps and more."""
    if p == 256 and pair[0] == "mx4":
        return 2080
    return (2592 if p in (2, 4) else 416) if pair[1] == "mx4" else 616 if p in (2, 4) else 136


class Layer:
    """T sorted rows of `tokens` x 2 over E experts (the first rows and the last in no run, expert 1 empty), at a size that takes path p.
    E experts share three experts' weights."""
    def __init__(self, ex, pair, p, swiglu, x=None, w=None, seed=0, extra=3):  # noqa: F811
        T, E, n = gemmpath.SIZES[p]
        K = k_of(pair, p)
        self.ex, self.T, self.E, self.n, self.K, self.swiglu, self.tokens = ex, T, E, n, K, swiglu, T // 2 + 1
        assert gemmpath.path(pair, swiglu, T, E, n, K) == p
        g = torch.Generator().manual_seed(seed + p)
        N, n_w = (2 * n if swiglu else n), min(E, 3)
        if w is not None:
            self.wd, self.w64 = w(g, n_w, N, K)
        elif pair[1] == "mx4":
            self.wd, self.w64 = gemmpath.mx4_weights(g, n_w, N, K, torch.randint(117, 122, (n_w, N, K // 32), generator=g))
        else:
            self.wd, self.w64 = operand(ex, torch.randn((n_w, N, K), generator=g) / K ** 0.5, pair[1])
        x = torch.randn((self.tokens, K), generator=g) if x is None else x(g, self.tokens, K)
        self.xd, self.x64 = operand(ex, x, pair[0])
        cut = torch.sort(torch.randint(3, T - 2, (E + 1,), generator=g)).values.to(torch.int32)
        cut[0], cut[1], cut[2], cut[-1] = 3, max(3, int(cut[1])), max(3, int(cut[1])), T - 2
        self.off = torch.cummax(cut, 0).values.to(torch.int32)
        self.st = torch.randperm(T, generator=g).to(torch.int32)
        self.st[T // 2], self.st[T // 3] = -7, 2 * self.tokens + 11               # a dropped slot, and a token that x does not have
        self.y = torch.full((T + 1, n + extra), NAN, device="cuda")
        self.gm = self.descriptor(self.y)

    def descriptor(self, y):
        ex = self.ex  # noqa: F811
        gm = ex.make_gemm(self.xd, self.wd, self.st.cuda(), self.off.cuda(), y[:self.T, :self.n], top_k=2,
                          act=ex.ACT_SWIGLU if self.swiglu else ex.ACT_NONE)
        return gemmpath.share(gm, self.wd, self.E) if self.E > self.w64.shape[0] else gm

    def run(self):
        self.y.fill_(NAN)
        assert self.ex.moe_gemm(self.gm) == 0
        got = self.y.cpu()
        assert torch.isnan(got[self.T:]).all() and torch.isnan(got[:, self.n:]).all()
        return got[:self.T, :self.n]

    def want(self):
        return mx4ref.gemm(self.x64, gemmpath.Shared(self.w64, self.E), self.st, self.off, self.T, 2, self.swiglu)

    def dead(self):
        """Rows that are zeros whatever x and the weights hold."""
        i = torch.arange(self.T)
        return (i < 3) | (i >= self.T - 2) | (i == self.T // 2) | (i == self.T // 3)


@pytest.mark.parametrize("pair,p", PATHS)
@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("extra", [3, 8])
def test_products(ex, pair, p, swiglu, extra):  # noqa: F811
    """Rows of y off every alignment, and on one (n + extra in multiples of 2 only where n is)."""
    print(f"moe_gemm {pair} path {p} swiglu {swiglu}", flush=True)
    lay = Layer(ex, pair, p, swiglu, extra=extra)
    got = lay.run()
    assert mx4ref.close(got, *lay.want())
    assert (got[lay.dead()] == 0).all()


@pytest.mark.parametrize("pair,p", [c for c in PATHS if c.values[0][1] == "mx4"])
def test_scales_far_apart(ex, pair, p):  # noqa: F811
    """Scales 2^-60 to 2^60 apart inside one word of four and from step to step, x zero under the large ones in half the rows, so that the
    small ones make those rows' sums; rows of blocks of zero codes; a NaN block, which makes its own row's outputs NaN."""
    def w(g, n, N, K):
        s = torch.randint(60, 180, (n, N, K // 32), generator=g)
        s[:, ::4] = torch.randint(110, 116, s[:, ::4].shape, generator=g) + 14 * torch.randint(0, 3, s[:, ::4].shape, generator=g)
        s[:, 1::4, ::2] = 200
        wd, v = gemmpath.mx4_weights(g, n, N, K, s)
        wd.codes[:, 2::8] = 0
        wd.scales[1, 9, 3] = 255
        v[:, 2::8] = 0
        v[1, 9, 96:128] = NAN
        return wd, v

    def x(g, tokens, K):
        v = torch.randn((tokens, K // 32, 32), generator=g)
        v[::2, ::2] = 0
        return v.view(tokens, K)
    print(f"moe_gemm {pair} path {p}: scales far apart", flush=True)
    lay = Layer(ex, pair, p, False, x=x, w=w)
    assert mx4ref.close(lay.run(), *lay.want())


@pytest.mark.parametrize("pair,p", PATHS)
@pytest.mark.parametrize("swiglu", [False, True])
def test_infinities_and_nans_stay_in_their_rows(ex, pair, p, swiglu):  # noqa: F811
    """Tokens with an infinity and with a NaN: every output of their rows is no number or infinite, every other row keeps its bits."""
    lay = Layer(ex, pair, p, swiglu)
    base = lay.run()

    def x(g, tokens, K):
        v = torch.randn((tokens, K), generator=g)
        v[5, K - 3], v[6, 1] = INF, NAN
        return v
    bad = Layer(ex, pair, p, swiglu, x=x)
    assert torch.equal(lay.st, bad.st)
    got = bad.run()
    hit = (torch.div(bad.st, 2, rounding_mode="floor") == 5) | (torch.div(bad.st, 2, rounding_mode="floor") == 6)
    hit &= ~bad.dead()
    assert hit.any() and not torch.isfinite(got[hit]).any()
    assert torch.equal(got[~hit], base[~hit])


@pytest.mark.parametrize("pair", [p for p in PAIRS if p[1] != "mx4"], ids="-".join)
@pytest.mark.parametrize("K", [8, 24, 40, 72, 1000, 1544])
@pytest.mark.parametrize("p", [4, 32, 64])
def test_columns_that_end_inside_a_step(ex, pair, K, p, monkeypatch):  # noqa: F811
    monkeypatch.setattr("test_gpu_moe_gemm_paths.k_of", lambda *_: K)
    lay = Layer(ex, pair, p, p == 32)
    assert mx4ref.close(lay.run(), *lay.want())


@pytest.mark.parametrize("pair,p", PATHS)
def test_graphs_and_streams(ex, pair, p):  # noqa: F811
    """The same bits eagerly, from two captured graphs replayed between eager launches, and from two streams at once."""
    lay = Layer(ex, pair, p, True)
    base = lay.run()
    y2 = torch.zeros_like(lay.y)
    other = lay.descriptor(y2)
    graphs = []
    for gm in (lay.gm, other):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            assert ex.moe_gemm(gm) == 0
    for _ in range(3):
        lay.y.fill_(3)
        y2.fill_(4)
        for graph in graphs:
            graph.replay()
        assert torch.equal(lay.y[:lay.T, :lay.n].cpu(), base) and torch.equal(y2[:lay.T, :lay.n].cpu(), base)
        assert torch.equal(lay.run(), base)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    lay.y.fill_(1)
    y2.fill_(1)
    torch.cuda.synchronize()
    for _ in range(4):
        assert ex.moe_gemm(lay.gm, s1) == 0 and ex.moe_gemm(other, s2) == 0
    torch.cuda.synchronize()
    assert torch.equal(lay.y[:lay.T, :lay.n].cpu(), base) and torch.equal(y2[:lay.T, :lay.n].cpu(), base)


def spread(t, pitch):
    """t's rows (its last but one dimension, all before it as one) `pitch` elements apart, in memory of their own."""
    rows = t.shape[:-1].numel()
    big = torch.zeros(rows * pitch, dtype=t.dtype, device=t.device).as_strided((rows, t.shape[-1]), (pitch, 1))
    big.copy_(t.reshape(rows, -1))
    return big if t.dim() == 2 else big.as_strided(t.shape, (t.shape[1] * pitch, pitch, 1))


@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
@pytest.mark.parametrize("p", [2, 4, 32])
def test_operands_past_32_bits_of_offset(ex, pair, p):  # noqa: F811
    """x, weights and y each over more than 4 GiB by their pitches (weights of one expert too), in a tile and in few rows."""
    T, E, n = gemmpath.SIZES[p]
    K, n_w = 160, min(E, 3)
    assert gemmpath.path(pair, False, T, E, n, K) == p
    g = torch.Generator().manual_seed(p)
    xd, x64 = operand(ex, torch.randn((T, K), generator=g), pair[0])
    wd, w64 = operand(ex, torch.randn((n_w, n, K), generator=g) / K ** 0.5, pair[1])
    far_x, far_w = -(-(9 << 29) // T) // 32 * 32, min(-(-(9 << 29) // n) // 32 * 32, 1 << 26)       # bytes
    if pair[0] == "mx4":
        xd = ex.Mx4(spread(xd.codes, far_x), spread(xd.scales, far_x), K)
    else:
        xd = spread(xd, far_x // 2)
    if pair[1] == "mx4":
        wd = ex.Mx4(spread(wd.codes, far_w), spread(wd.scales, 4096), K)
    else:
        wd = spread(wd, far_w // 2)
    off = torch.tensor([T * e // E for e in range(E + 1)], dtype=torch.int32)
    y = torch.zeros(T * (far_x // 4) + n, device="cuda").as_strided((T, n), (far_x // 4, 1))
    gm = ex.make_gemm(xd, wd, None, off.cuda(), y)
    if E > n_w:
        gemmpath.share(gm, wd, E)
    assert ex.moe_gemm(gm) == 0
    got = y.cpu()
    assert mx4ref.close(got, *mx4ref.gemm(x64, gemmpath.Shared(w64, E), None, off, T, 1, False))
