"""A routed layer as a user runs it: the router's logits (a 16-bit linear layer), moe_route, f8_quant, gate and up with SwiGLU, f8_quant, down and the
gather; each step against its definition in 64 bits on what the step before left, the weights quantised on the device as a loader does, and the whole
captured into a graph that is replayed on other tokens."""
import numpy as np
import pytest

import f8ref
import mx4ref
import routeref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
H, W, E, TOP_K, GROUPS, TOP_GROUP = 384, 208, 40, 6, 5, 3


@pytest.fixture(scope="module")
def ex():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import exl3c4
    exl3c4.lib()
    return exl3c4


class Layer:
    def __init__(self, ex, n_tok, f8_x):
        g = torch.Generator().manual_seed(1)
        rand = lambda *s: torch.randn(s, generator=g).cuda()
        self.ex, self.n_tok, self.f8_x = ex, n_tok, f8_x
        T = n_tok * TOP_K
        i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
        self.router = (rand(1, E, H) / H ** 0.5).bfloat16()
        self.bias = rand(E) * 0.1
        # a loader: gate and up as the two matrices that they are, one behind the other in an expert's rows
        gu, dn = ex.f8_empty((E, 2, W, H), 128), ex.f8_empty((E, H, W), 128)
        assert ex.f8_quant((rand(E, 2, W, H) / H ** 0.5).bfloat16(), gu) == 0 and ex.f8_quant((rand(E, H, W) / W ** 0.5).bfloat16(), dn) == 0
        self.gu = ex.F8(gu.codes.view(E, 2 * W, H), gu.scales.view(E, -1, gu.scales.shape[-1]), H, 128)
        self.dn = dn
        self.x = torch.zeros(n_tok, H, dtype=torch.bfloat16, device="cuda")
        self.logits = torch.zeros(n_tok, E, device="cuda")
        self.ids, self.w, self.st, self.off, self.row = i32(n_tok, TOP_K), torch.zeros(n_tok, TOP_K, device="cuda"), i32(T), i32(E + 1), i32(T)
        self.h, self.y = torch.zeros(T, W, dtype=torch.bfloat16, device="cuda"), torch.zeros(T, H, dtype=torch.bfloat16, device="cuda")
        self.out = torch.zeros(n_tok, H, dtype=torch.float16, device="cuda")
        self.xq, self.hq = ex.f8_empty((n_tok, H), 1), ex.f8_empty((T, W), 1)
        one = torch.tensor([0, n_tok], dtype=torch.int32, device="cuda")
        self.g_router = ex.make_gemm(self.x, self.router, None, one, self.logits)
        self.route = ex.make_route(self.logits, TOP_K, self.ids, self.w, score=ex.SCORE_SIGMOID, bias=self.bias, n_group=GROUPS, top_group=TOP_GROUP,
                                   group_score=ex.GROUP_TOP2, scale=2.5, sorted_tok=self.st, expert_offset=self.off, row_of=self.row)
        self.g_gu = ex.make_gemm(self.xq if f8_x else self.x, self.gu, self.st, self.off, self.h, top_k=TOP_K, act=ex.ACT_SWIGLU)
        self.g_dn = ex.make_gemm(self.hq if f8_x else self.h, self.dn, None, self.off, self.y)

    def run(self):
        ex = self.ex
        rc = [ex.moe_gemm(self.g_router), ex.moe_route(self.route)]
        if self.f8_x:
            rc.append(ex.f8_quant(self.x, self.xq))
        rc.append(ex.moe_gemm(self.g_gu))
        if self.f8_x:
            rc.append(ex.f8_quant(self.h, self.hq))
        rc.append(ex.moe_gemm(self.g_dn))
        rc.append(ex.moe_gather(self.y.view(torch.int16), True, self.w, self.row, self.out.view(torch.int16)))
        assert rc == [0] * len(rc)

    def check(self):
        T = self.n_tok * TOP_K
        x = self.x.cpu()
        want, tol = mx4ref.gemm(x.double(), self.router.cpu().double(), None, [0, self.n_tok], self.n_tok, 1, False)
        assert mx4ref.close(self.logits.cpu(), want, tol)
        ids, w = routeref.route(self.logits.cpu().numpy(), TOP_K, "sigmoid", self.bias.cpu().numpy(), GROUPS, TOP_GROUP, "top2", True, 2.5)
        st, off, _, row = routeref.scatter(ids, E)
        assert np.array_equal(self.ids.cpu().numpy(), ids) and np.array_equal(self.st.cpu().numpy(), st)
        assert np.array_equal(self.off.cpu().numpy(), off) and np.array_equal(self.row.cpu().numpy(), row)
        assert (np.abs(self.w.cpu().numpy() - w) <= 2.0 ** -23 * np.abs(w)).all()

        def operand(v, q):
            """(values, peaks) of x as the product has them."""
            if not self.f8_x:
                return v.double(), None
            c, s = f8ref.quant(v[None], 1)
            assert torch.equal(q.codes.cpu() & 127, c[0] & 127) and torch.equal(q.scales.cpu(), s[0])
            return f8ref.values(c, s, v.shape[1], 1)[0], f8ref.peaks(c[0], s[0].double().repeat_interleave(128, 1)[:, :v.shape[1]])

        def weights(q, halves):
            c, s = q.codes.cpu(), q.scales.cpu()
            return f8ref.weights(c, s, halves), f8ref.peaks(c, f8ref.weights(torch.full_like(c, 0x38), s, halves))
        for v, q, wq, halves, got, gather in ((x, self.xq, self.gu, 2, self.h, True), (self.h.cpu(), self.hq, self.dn, 1, self.y, False)):
            (xv, xp), (wv, wp) = operand(v, q), weights(wq, halves)
            want, tol = f8ref.gemm(xv, wv, st if gather else None, off, T, TOP_K if gather else 1, halves == 2, (xp, wp) if self.f8_x else None)
            assert mx4ref.close(got.cpu(), want, tol)
        y, wt = self.y.cpu().double(), self.w.cpu().double()
        want = torch.zeros(self.n_tok, H, dtype=torch.float64)
        mag = torch.zeros_like(want)
        for s in range(TOP_K):                                   # a product and an addition in f32 a slot, then f16
            p = wt[:, s:s + 1] * y[torch.from_numpy(row).view(self.n_tok, TOP_K)[:, s].long()]
            want, mag = want + p, mag + p.abs()
        assert ((self.out.cpu().double() - want).abs() <= 2.0 ** -11 * want.abs() + (TOP_K + 1) * 2.0 ** -24 * mag * 1.01 + 2.0 ** -25).all()


@pytest.mark.parametrize("n_tok", [1, 16, 37, 400])
@pytest.mark.parametrize("f8_x", [False, True])
def test_a_layer(ex, n_tok, f8_x):
    layer = Layer(ex, n_tok, f8_x)
    layer.x.copy_(torch.randn(n_tok, H, generator=torch.Generator().manual_seed(n_tok)))
    layer.run()
    torch.cuda.synchronize()
    layer.check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.run()
    for seed in (5, 6):
        layer.x.copy_(torch.randn(n_tok, H, generator=torch.Generator().manual_seed(seed)))
        layer.out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        layer.check()


@pytest.mark.parametrize("n_tok", [9, 37, 400])
@pytest.mark.parametrize("f8_x", [False, True])
def test_a_padded_batch(ex, n_tok, f8_x):
    """Tokens of NaN (the first, some in between, the last) have no expert and come out as zeros; the others' bits are those of a batch without such tokens."""
    layer = Layer(ex, n_tok, f8_x)
    x = torch.randn(n_tok, H, generator=torch.Generator().manual_seed(n_tok))
    layer.x.copy_(x)
    layer.run()
    torch.cuda.synchronize()
    whole = layer.out.clone()
    bad = torch.zeros(n_tok, dtype=torch.bool)
    bad[0] = bad[n_tok // 2] = bad[-3:] = True
    x[bad] = float("nan")
    layer.x.copy_(x)
    for t in (layer.h, layer.y, layer.out):
        t.fill_(float("nan"))
    layer.run()
    torch.cuda.synchronize()
    live = TOP_K * int((~bad).sum())
    assert (layer.ids.cpu()[bad] == -1).all() and (layer.w.cpu()[bad] == 0).all() and int(layer.off[-1]) == live
    assert (layer.st[live:] == -1).all() and not layer.h[live:].any() and not layer.y[live:].any()
    assert not layer.out[bad.cuda()].any() and torch.equal(layer.out[~bad.cuda()], whole[~bad.cuda()])
