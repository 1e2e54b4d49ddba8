"""moe_gemm on the device against the product in 64 bits (tests/mx4ref.py), through the binding: every pair of types, with
and without SwiGLU, x by token or by sorted row; within the bound that f32 sums and one rounding leave."""
import ctypes as C

import numpy as np
import pytest

import mx4ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
PAIRS = [("f16", "f16"), ("bf16", "bf16"), ("f16", "mx4"), ("bf16", "mx4"), ("mx4", "mx4")]


@pytest.fixture(scope="module")
def ex():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import exl3c4
    exl3c4.lib()
    return exl3c4


def operand(ex, v, kind):
    """(the operand on the device, its values in f64): v [..., K] f32 on the CPU; MX4 with rows wider than K's blocks,
    what lies behind them poisoned (codes 6, scales NaN)."""
    if kind != "mx4":
        t = v.to(TYPES[kind])
        return t.cuda(), t.double()
    K = v.shape[-1]
    c, s = mx4ref.quant(v.reshape(-1, K))
    codes = torch.full((c.shape[0], c.shape[1] + 16), 0x77, dtype=torch.uint8)
    scales = torch.full((s.shape[0], (s.shape[1] + 3) // 4 * 4 + 4), 255, dtype=torch.uint8)
    codes[:, :c.shape[1]], scales[:, :s.shape[1]] = c, s
    shape = v.shape[:-1]
    return (ex.Mx4(codes.view(*shape, -1).cuda(), scales.view(*shape, -1).cuda(), K),
            mx4ref.dequant(c, s, K).view(*shape, K))


def routing(rng, tokens, top_k, n_expert, lo=0, hi=None):
    """sorted_tok and expert_offset of `tokens` x `top_k` random pairs over experts lo .. hi - 1 (the others are empty)."""
    ids = rng.integers(lo, hi or n_expert, tokens * top_k)
    order = np.argsort(ids, kind="stable").astype(np.int32)
    off = np.zeros(n_expert + 1, np.int32)
    off[1:] = np.cumsum(np.bincount(ids, minlength=n_expert))
    return order, off


def run(ex, pair, yt, swiglu, tokens, top_k, E, N, K, gather=True, seed=0, route=None, scale=None, x=None, w=None, T=None):
    rng = np.random.default_rng(seed)
    g = torch.Generator().manual_seed(seed)
    order, off = route if route is not None else routing(rng, tokens, top_k, E)
    T = len(order) if T is None else T
    x = torch.randn((tokens if gather else T, K), generator=g) if x is None else x
    w = torch.randn((E, N, K), generator=g) / K ** 0.5 if w is None else w
    xd, xv = operand(ex, x, pair[0])
    wd, wv = operand(ex, w, pair[1])
    n_out = N // 2 if swiglu else N
    yd = torch.full((T + 4, n_out + 5), float("nan"), dtype=TYPES[yt], device="cuda")
    st = torch.from_numpy(order).cuda() if gather else None
    gm = ex.make_gemm(xd, wd, st, torch.from_numpy(off).cuda(), yd[:T, :n_out], top_k=top_k,
                      act=ex.ACT_SWIGLU if swiglu else ex.ACT_NONE)
    gm.keep = (xd, wd, st, yd)
    assert ex.moe_gemm(gm) == 0
    torch.cuda.synchronize()
    y, tol = mx4ref.gemm(xv, wv, order if gather else None, off, T, top_k, swiglu)
    got = yd[:T, :n_out].cpu()
    assert torch.isnan(yd[T:]).all() and torch.isnan(yd[:, n_out:]).all()       # nothing past the rows and columns
    return got, y, tol, gm


def check(ex, *a, **kw):
    got, y, tol, _ = run(ex, *a, **kw)
    worst = ((got.double() - y).abs() / (tol + mx4ref.EPS[got.dtype] * y.abs() + 1e-300)).max() if y.numel() else 0
    print(f"moe_gemm {a} {kw.get('gather', True)}: {float(worst):.3f} of the bound", flush=True)
    assert mx4ref.close(got, y, tol)


@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
@pytest.mark.parametrize("tokens,top_k,E,N,K", [
    (1, 1, 1, 32, 64), (1, 2, 3, 34, 128), (3, 2, 5, 62, 160), (9, 4, 8, 130, 32), (40, 2, 3, 96, 416), (2, 3, 40, 64, 2048),
    (150, 2, 4, 72, 96), (300, 1, 1, 258, 352), (700, 2, 3, 320, 288)])
def test_products(ex, pair, tokens, top_k, E, N, K):
    yt = {"mx4": "f32", "f16": "f16", "bf16": "bf16"}[pair[0]]
    check(ex, pair, yt, False, tokens, top_k, E, N, K)
    check(ex, pair, yt, True, tokens, top_k, E, N, K, gather=tokens % 2 == 0)
    check(ex, pair, "f32", False, tokens, top_k, E, N - 1, K, gather=False, seed=1)


# (T, E, N) that take each kernel and tile: few rows an expert in narrow and wide workgroups, 32, 64, 128 and 256 rows a tile
PATHS = {"rows": (40, 3, 200), "rows wide": (60, 4, 11000), "32": (150, 2, 1450), "64": (250, 4, 3700), "128": (260, 2, 5510), "256": (700, 2, 13320)}


@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
@pytest.mark.parametrize("path", list(PATHS))
@pytest.mark.parametrize("swiglu", [False, True])
def test_each_tile(ex, pair, path, swiglu):
    """Sizes that take each kernel and tile, their last tiles partly past the rows and columns, k ending inside a stage (MX4's
    largest tile is taken from K = 2048 on)."""
    T, E, N = PATHS[path]
    K = 2080 if path == "256" and pair[0] == "mx4" else 160 if pair[1] == "mx4" else 136
    N *= 2 if swiglu else 1
    g = torch.Generator().manual_seed(T)
    x = torch.randn((T, K), generator=g)
    if pair[1] == "mx4":                                            # random codes at once: rounding so many is slow here
        codes = torch.randint(0, 256, (E, N, K // 2), dtype=torch.uint8, generator=g)
        scales = torch.randint(118, 122, (E, N, (K // 32 + 3) // 4 * 4), dtype=torch.uint8, generator=g)
        scales[..., K // 32:] = 255
        w = ex.Mx4(codes.cuda(), scales.cuda(), K), mx4ref.dequant(codes, scales, K)
    else:
        w = operand(ex, torch.randn((E, N, K), generator=g) / K ** 0.5, pair[1])
    xd, xv = operand(ex, x, pair[0])
    off = torch.tensor([0] + [T * (e + 1) // E - (e == 0) for e in range(E)], dtype=torch.int32)
    off[-1] = T - 2
    st = torch.randperm(T, generator=g).to(torch.int32)
    n_out = N // 2 if swiglu else N
    y = torch.full((T + 1, n_out + 3), float("nan"), dtype=torch.float32, device="cuda")
    assert ex.moe_gemm(ex.make_gemm(xd, w[0], st.cuda(), off.cuda(), y[:T, :n_out], act=ex.ACT_SWIGLU if swiglu else ex.ACT_NONE)) == 0
    torch.cuda.synchronize()
    want, tol = mx4ref.gemm(xv, w[1], st, off, T, 1, swiglu)
    assert mx4ref.close(y[:T, :n_out].cpu(), want, tol)
    assert torch.isnan(y[T]).all() and torch.isnan(y[:, n_out:]).all()


@pytest.mark.parametrize("pair", [("f16", "f16"), ("bf16", "bf16")], ids="-".join)
@pytest.mark.parametrize("K", [8, 24, 40, 72, 1000, 1544])
def test_columns_that_end_inside_a_step(ex, pair, K):
    check(ex, pair, "f32", False, 5, 3, 4, 33, K)
    check(ex, pair, "f32", True, 130, 1, 2, 66, K)


@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
@pytest.mark.parametrize("yt", list(TYPES))
def test_output_types(ex, pair, yt):
    check(ex, pair, yt, True, 20, 2, 6, 96, 256)
    check(ex, pair, yt, False, 200, 2, 2, 150, 256)


@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
@pytest.mark.parametrize("n", [3, 200])
def test_rows_outside_the_runs_and_dropped_rows_are_zeros(ex, pair, n):
    """Runs that start behind row 0 and end before T, empty experts, dropped slots, tokens that x does not have; and rows
    with infinities and NaNs beside others, which stay alone."""
    rng = np.random.default_rng(5)
    E, T, tokens, K, N = 4, n + 20, 30, 96, 48
    off = np.array([7, 7, 7 + n // 3, 7 + n, 7 + n], np.int32)
    order = rng.integers(0, tokens * 2, T).astype(np.int32)
    order[8] = -1
    order[7 + n // 2] = tokens * 2 + 5
    x = torch.randn((tokens, K), generator=torch.Generator().manual_seed(1))
    got, y, tol, _ = run(ex, pair, "f32", False, tokens, 2, E, N, K, route=(order, off), x=x)
    assert mx4ref.close(got, y, tol)
    dead = [i for i in range(T) if i < 7 or i >= 7 + n or i == 8 or i == 7 + n // 2]
    assert (got[dead] == 0).all()
    bad = x.clone()
    bad[3, 5], bad[4, 9] = float("nan"), float("inf")
    got2, _, _, _ = run(ex, pair, "f32", False, tokens, 2, E, N, K, route=(order, off), x=bad)
    hit = torch.tensor([order[i] // 2 in (3, 4) and i not in dead for i in range(T)])
    assert torch.equal(got2[~hit], got[~hit])
    assert not torch.isfinite(got2[hit]).all() if hit.any() else True
    assert (got2[dead] == 0).all()


@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
def test_offsets_that_are_no_routing_write_only_their_rows(ex, pair):
    """Descending, negative and too large offsets: wrong rows, but none outside y (its guard rows stay), and every launch
    of the same table writes rows that the definition gives for some run, or zeros."""
    E, T, K, N = 6, 64, 64, 40
    order = np.arange(T, dtype=np.int32)
    for off in ([0, 10, 5, 64, 64, 64, 64], [-5, 3, 900, 20, 64, 70, 80], [70, 70, 70, 70, 70, 70, 70], [0] * 7):
        run(ex, pair, "f32", False, T, 1, E, N, K, route=(order, np.array(off, np.int32)))


def test_no_rows_and_no_live_rows(ex):
    x, w = torch.zeros(4, 64, device="cuda").half(), torch.zeros(2, 8, 64, device="cuda").half()
    off = torch.zeros(3, dtype=torch.int32, device="cuda")
    y = torch.full((0, 8), 1.0, device="cuda")
    assert ex.moe_gemm(ex.make_gemm(x, w, None, off, y)) == 0
    y = torch.full((4, 8), 1.0, device="cuda")
    assert ex.moe_gemm(ex.make_gemm(x, w, None, off, y)) == 0
    assert (y == 0).all()


@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
def test_more_experts_than_one_scan_holds(ex, pair):
    """1,500 experts (the search takes 512 segments at a time), rows in a few of them far apart."""
    E, T = 1500, 90
    ids = np.sort(np.random.default_rng(2).choice([0, 5, 509, 510, 511, 512, 1021, 1022, 1023, 1400, 1499], T))
    off = np.zeros(E + 1, np.int32)
    off[1:] = np.cumsum(np.bincount(ids, minlength=E))
    check(ex, pair, "f32", False, T, 1, E, 36, 32, route=(np.arange(T, dtype=np.int32), off))


@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
def test_pointer_tables_give_the_stacked_buffers_bits(ex, pair):
    got, y, tol, gm = run(ex, pair, "f32", True, 20, 2, 5, 64, 128)
    _, wd, _, yd = gm.keep
    table = lambda t: torch.tensor([t[e].data_ptr() for e in range(t.shape[0])], dtype=torch.int64, device="cuda")
    v = wd.codes if pair[1] == "mx4" else wd
    tw = table(v)
    gm.w, gm.w_stride = tw.data_ptr(), 0
    if pair[1] == "mx4":
        ts = table(wd.scales)
        gm.w_scales, gm.ws_stride = ts.data_ptr(), 0
    yd.fill_(7)
    assert ex.moe_gemm(gm) == 0
    torch.cuda.synchronize()
    assert torch.equal(yd[:40, :32].cpu(), got)


@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
@pytest.mark.parametrize("tokens", [20, 600])
def test_a_pointer_table_that_starts_between_16_bytes(ex, pair, tokens):
    got, y, tol, gm = run(ex, pair, "f32", False, tokens, 2, 5, 640, 128)
    _, wd, _, yd = gm.keep
    table = lambda t: torch.tensor([0] + [t[e].data_ptr() for e in range(t.shape[0])], dtype=torch.int64, device="cuda")
    tw = table(wd.codes if pair[1] == "mx4" else wd)
    gm.w, gm.w_stride = tw.data_ptr() + 8, 0
    if pair[1] == "mx4":
        ts = table(wd.scales)
        gm.w_scales, gm.ws_stride = ts.data_ptr() + 8, 0
    yd.fill_(7)
    assert ex.moe_gemm(gm) == 0
    torch.cuda.synchronize()
    assert torch.equal(yd[:2 * tokens, :640].cpu(), got)


@pytest.mark.parametrize("pair", [p for p in PAIRS if p[1] == "mx4"], ids="-".join)
@pytest.mark.parametrize("tokens", [3, 150])
@pytest.mark.parametrize("K", [256, 2304])
def test_extreme_scales(ex, pair, tokens, K):
    """Scales over the format's whole range: a row's blocks from 2^-120 to 2^20, where f16 could not hold the weights; x zero
    where the largest are, so that the small ones make the sums; and a NaN block, which makes its own rows' outputs
    NaN and no others."""
    g = torch.Generator().manual_seed(3)
    N, E = 40, 2
    e = torch.randint(-118, 18, (E, N, K // 32, 1), generator=g)
    e[:, :, 1::2] = torch.randint(-118, -30, (E, N, K // 32, 1), generator=g)[:, :, 1::2]
    e[:, ::3] = torch.randint(-3, 4, (E, N, K // 32, 1), generator=g)[:, ::3]
    w = (torch.randn((E, N, K // 32, 32), generator=g) * torch.exp2(e.float())).reshape(E, N, K)
    check(ex, pair, "f32", False, tokens, 1, E, N, K, w=w)
    x = torch.randn((tokens, K // 64, 2, 32), generator=g)
    x[:, :, 0] = 0
    check(ex, pair, "f32", False, tokens, 1, E, N, K, w=w, x=x.reshape(tokens, K))
    w[1, 7, 40] = float("nan")
    check(ex, pair, "f32", False, tokens, 1, E, N, K, w=w, seed=4)


@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
def test_rows_far_apart(ex, pair):
    """Pitches that take x, w and y past 32 bits of byte offset."""
    K, N, T = 64, 20, 3
    far = 1 << 30                                                   # elements between rows
    xv = torch.randn(T, K)
    wv = torch.randn(2, N, K) / 8
    xd, x64 = operand(ex, xv, pair[0])
    wd, w64 = operand(ex, wv, pair[1])
    buf = torch.zeros(2 * far + 4096, dtype=torch.float16, device="cuda")
    y = buf.as_strided((T, N), (far, 1))
    if pair[0] != "mx4":
        big = torch.zeros(2 * far + 4096, dtype=xd.dtype, device="cuda").as_strided((T, K), (far, 1))
        big.copy_(xd)
        xd = big
    if pair[1] != "mx4":
        big = torch.zeros((2 * far + 4096), dtype=wd.dtype, device="cuda").as_strided((2, N, K), (far, 128, 1))
        big.copy_(wd)
        wd = big
    off = torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda")
    assert ex.moe_gemm(ex.make_gemm(xd, wd, None, off, y)) == 0
    want, tol = mx4ref.gemm(x64, w64, None, [0, 1, 3], T, 1, False)
    assert mx4ref.close(y.cpu(), want, tol)


@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
@pytest.mark.parametrize("tokens", [4, 300])
def test_captured_replayed_and_on_two_streams(ex, pair, tokens):
    """The same bits eagerly, from a graph replayed between eager launches, and from two streams at once."""
    got, y, tol, gm = run(ex, pair, "bf16", True, tokens, 2, 7, 64, 288)
    yd = gm.keep[3]
    n = tokens * 2
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert ex.moe_gemm(gm) == 0
    for _ in range(3):
        yd.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(yd[:n, :32].cpu(), got)
        yd.fill_(5)
        assert ex.moe_gemm(gm) == 0
        torch.cuda.synchronize()
        assert torch.equal(yd[:n, :32].cpu(), got)
    other = ex.Gemm.from_buffer_copy(gm)
    y2 = torch.zeros_like(yd)
    other.y, other.device = y2.data_ptr(), yd.device
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    yd.fill_(1)
    torch.cuda.synchronize()
    for _ in range(5):
        assert ex.moe_gemm(gm, s1) == 0 and ex.moe_gemm(other, s2) == 0
    torch.cuda.synchronize()
    assert torch.equal(yd[:n, :32].cpu(), got) and torch.equal(y2[:n, :32].cpu(), got)


@pytest.mark.parametrize("tokens", [1, 9, 130])
@pytest.mark.parametrize("kind", ["mx4w", "mx4", "16"])
def test_a_layer_of_them(ex, tokens, kind):
    """Router, scatter, gate and up with SwiGLU, down, gather, as a layer runs them: against 64 bits of the device's own
    routing. MX4 x rounds its rows (and h its own) to 4 bits by the same rule on both sides; where h's 16-bit value and the
    64-bit one fall on two sides of a tie, one step of the code apart, so the layer is compared as a whole: each of h's
    roundings to bf16 is 2^-8 at most, a step of a code at most half its value, met by the share 2^-8 of values that near a tie."""
    E, H, W, k = 16, 160, 96, 4
    g = torch.Generator().manual_seed(tokens)
    x = torch.randn((tokens, H), generator=g).bfloat16().cuda()
    logits = torch.randn((tokens, E), generator=g).cuda()
    T = tokens * k
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
    ids, w, st, off, row_of = i32(tokens, k), torch.zeros(tokens, k, device="cuda"), i32(T), i32(E + 1), i32(T)
    assert ex.router_topk_scatter(logits, k, True, ids, w, st, off, None, row_of) == 0
    wk = "bf16" if kind == "16" else "mx4"
    gu, gu64 = operand(ex, torch.randn((E, 2 * W, H), generator=g) / H ** 0.5, wk)
    dn, dn64 = operand(ex, torch.randn((E, H, W), generator=g) / W ** 0.5, wk)
    h = torch.zeros((T, W), dtype=torch.bfloat16, device="cuda")
    y = torch.zeros((T, H), dtype=torch.bfloat16, device="cuda")
    out = torch.zeros((tokens, H), dtype=torch.int16, device="cuda")
    x_in, h_in = x, h
    if kind == "mx4":
        x_in, h_in = ex.mx4_empty(x.shape), ex.mx4_empty(h.shape)
        assert ex.mx4_quant(x, x_in) == 0
    assert ex.moe_gemm(ex.make_gemm(x_in, gu, st, off, h, top_k=k, act=ex.ACT_SWIGLU)) == 0
    if kind == "mx4":
        assert ex.mx4_quant(h, h_in) == 0
    assert ex.moe_gemm(ex.make_gemm(h_in, dn, None, off, y, top_k=k)) == 0
    assert ex.moe_gather(y.view(torch.int16), True, w, row_of, out) == 0
    torch.cuda.synchronize()
    x64 = x.double().cpu()
    if kind == "mx4":
        x64 = mx4ref.dequant(*mx4ref.quant(x.cpu()), H)
    h64, _ = mx4ref.gemm(x64, gu64, st.tolist(), off.tolist(), T, k, True)
    if kind == "mx4":
        h64 = mx4ref.dequant(*mx4ref.quant(h64), W)
    y64, _ = mx4ref.gemm(h64, dn64, None, off.tolist(), T, k, False)
    r, wt = row_of.cpu().view(tokens, k).long(), w.double().cpu()
    want = (wt[..., None] * y64[r]).sum(1)
    got = out.view(torch.float16).double().cpu()
    rel = float((got - want).norm() / want.norm())
    print(f"layer {kind} {tokens}: relative L2 {rel:.2e}", flush=True)
    # h and y rounded to bf16, out to f16 (2^-8, 2^-8, 2^-11 at most); MX4: of h's values the share 2^-8 / 2^-3 that lie within
    # their bf16 rounding of a tie, by a step of up to 1/2 of the value: sqrt(2^-5) / 2 of the norm at the very most
    assert rel <= 2 * 2.0 ** -8 + 2.0 ** -11 + (2.0 ** -2.5 / 2 if kind == "mx4" else 0)
