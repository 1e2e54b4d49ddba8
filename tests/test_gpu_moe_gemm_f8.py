"""moe_gemm with F8 weights on the device against the product in 64 bits (tests/f8ref.py), through the binding: x in F8, f16 and bf16, with and
without SwiGLU, by token or by sorted row, on every kernel; within the bound that f32 sums (F8 x, many rows and y in 16 bits: the matrix unit's
8-bit products) and one rounding leave."""
import ctypes as C

import numpy as np
import pytest

import f8ref
import mx4ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
XS = ["f16", "bf16", "f8"]


@pytest.fixture(scope="module")
def ex():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import exl3c4
    exl3c4.lib()
    return exl3c4


def path(ex, xt, yt, swiglu, T, E, n_out, K):
    f = ex.lib().exl3c4_dev_gemm_f8_path
    f.restype, f.argtypes = C.c_int, [C.c_int32] * 3 + [C.c_int64] * 4
    code = {"f16": ex.F16, "bf16": ex.BF16, "f32": ex.F32, "f8": ex.TYPE_F8}
    return f(code[xt], code[yt], ex.ACT_SWIGLU if swiglu else ex.ACT_NONE, T, E, 2 * n_out if swiglu else n_out, K)


def x_operand(ex, v, kind):
    """(x on the device, its values in f64, its eights' peaks or None); F8 with rows wider than its columns, what lies behind them poisoned (NaN codes and scales)."""
    if kind != "f8":
        t = v.to(TYPES[kind])
        return t.cuda(), t.double(), None
    c, s = f8ref.quant(v[None], 1)
    codes = torch.full((c.shape[1], c.shape[2] + 16), 0x7F, dtype=torch.uint8)
    scales = torch.full((s.shape[1], s.shape[2] + 2), float("nan"))
    codes[:, :c.shape[2]], scales[:, :s.shape[2]] = c[0], s[0]
    spread = s[0].double().repeat_interleave(128, 1)[:, :v.shape[1]].nan_to_num(0)
    return ex.F8(codes.cuda(), scales.cuda(), v.shape[1], 1), f8ref.values(c, s, v.shape[1], 1)[0], f8ref.peaks(c[0], spread)


def w_operand(ex, g, E, N, K, swiglu, scale=None):
    """(w on the device, its values in f64, its eights' peaks): random codes of every kind but NaN, each block's scale at random (or `scale`); planes wider than they
    need be, poisoned behind."""
    halves = 2 if swiglu else 1
    rows = N // halves
    c = torch.randint(0, 254, (E, N, K), dtype=torch.uint8, generator=g)
    c = torch.where(c >= 127, c + 1, c)                             # 127 and 255 are NaN
    down, across = halves * ((rows + 127) // 128), (K + 127) // 128
    s = torch.rand((E, down, across), generator=g) * 0.01 + 0.0005 if scale is None else scale
    codes = torch.full((E, N + 1, K + 16), 0x7F, dtype=torch.uint8)
    scales = torch.full((E, down, across + 1), float("nan"))
    codes[:, :N, :K], scales[..., :across] = c, s
    one = torch.full((E, N, K), 0x38, dtype=torch.uint8)                # 1 everywhere: each code's scale
    return ex.F8(codes.cuda()[:, :N], scales.cuda(), K, 128), f8ref.weights(c, s, halves), f8ref.peaks(c, f8ref.weights(one, s, halves))


def routing(rng, tokens, top_k, n_expert):
    ids = rng.integers(0, n_expert, tokens * top_k)
    order = np.argsort(ids, kind="stable").astype(np.int32)
    off = np.zeros(n_expert + 1, np.int32)
    off[1:] = np.cumsum(np.bincount(ids, minlength=n_expert))
    return order, off


def run(ex, xt, yt, swiglu, tokens, top_k, E, N, K, gather=True, seed=0, route=None, x=None, T=None, w=None):
    rng = np.random.default_rng(seed)
    g = torch.Generator().manual_seed(seed)
    order, off = route if route is not None else routing(rng, tokens, top_k, E)
    T = len(order) if T is None else T
    x = torch.randn((tokens if gather else T, K), generator=g) if x is None else x
    xd, xv, xp = x_operand(ex, x, xt)
    wd, wv, wp = w if w is not None else w_operand(ex, g, E, N, K, swiglu)
    n_out = N // 2 if swiglu else N
    yd = torch.full((T + 4, n_out + 5), float("nan"), dtype=TYPES[yt], device="cuda")
    st = torch.from_numpy(order).cuda() if gather else None
    gm = ex.make_gemm(xd, wd, st, torch.from_numpy(off).cuda(), yd[:T, :n_out], top_k=top_k, act=ex.ACT_SWIGLU if swiglu else ex.ACT_NONE)
    assert ex.moe_gemm(gm) == 0
    torch.cuda.synchronize()
    # the rows kernels widen, and so do tiles where y is f32
    cut = (xp, wp) if xt == "f8" and yt != "f32" and path(ex, xt, yt, swiglu, T, E, n_out, K) >= 32 else None
    y, tol = f8ref.gemm(xv, wv, order if gather else None, off, T, top_k, swiglu, cut)
    got = yd[:T, :n_out].cpu()
    assert torch.isnan(yd[T:]).all() and torch.isnan(yd[:, n_out:]).all()       # nothing past the rows and columns
    return got, y, tol, gm


def check(ex, *a, **kw):
    got, y, tol, _ = run(ex, *a, **kw)
    worst = ((got.double() - y).abs() / (tol + mx4ref.EPS[got.dtype] * y.abs() + 1e-300)).max() if y.numel() else 0
    print(f"moe_gemm f8 {a} {kw.get('gather', True)}: {float(worst):.3f} of the bound", flush=True)
    assert mx4ref.close(got, y, tol)


@pytest.mark.parametrize("xt", XS)
@pytest.mark.parametrize("tokens,top_k,E,N,K", [
    (1, 1, 1, 32, 16), (1, 2, 3, 34, 128), (3, 2, 5, 62, 160), (9, 4, 8, 130, 32), (40, 2, 3, 300, 416), (2, 3, 40, 64, 2048),
    (150, 2, 4, 72, 96), (300, 1, 1, 258, 352), (700, 2, 3, 320, 272)])
def test_products(ex, xt, tokens, top_k, E, N, K):
    yt = {"f8": "bf16", "f16": "f16", "bf16": "bf16"}[xt]
    check(ex, xt, yt, False, tokens, top_k, E, N, K)
    check(ex, xt, yt, True, tokens, top_k, E, N, K, gather=tokens % 2 == 0)
    check(ex, xt, "f32", False, tokens, top_k, E, N - 1, K, gather=False, seed=1)


# (T, experts, weight rows, K) that take each kernel and tile; the last column tile is not whole, and k ends inside a block
SIZES = {2: (40, 3, 200, 144), 4: (200, 3, 1650, 2064), 32: (150, 2, 1810, 144), 64: (250, 4, 13330, 144), 128: (700, 4, 9500, 272)}


@pytest.mark.parametrize("xt,yt,p", [(x, y, p) for x, y in (("f16", "f32"), ("bf16", "f32"), ("f8", "f32"), ("f8", "f16"))
                                     for p in ((2, 4, 32, 64) if y == "f32" else (2, 4, 32, 64, 128))])
@pytest.mark.parametrize("swiglu", [False, True])
def test_each_kernel(ex, xt, yt, p, swiglu):
    """Sizes that take each kernel, their last tiles partly past the rows and columns, runs that leave rows out."""
    T, E, N, K = SIZES[p]
    assert path(ex, xt, yt, swiglu, T, E, N // 2 if swiglu else N, K) == p
    off = np.array([0] + [T * (e + 1) // E - (e == 0) for e in range(E)], np.int32)
    off[-1] = T - 2
    order = np.random.default_rng(T).permutation(T).astype(np.int32)
    check(ex, xt, yt, swiglu, T, 1, E, N, K, route=(order, off))


@pytest.mark.parametrize("xt,yt,p", [("bf16", "f32", 32), ("bf16", "f32", 64), ("f8", "f32", 32), ("f8", "f32", 64), ("f8", "bf16", 32),
                                     ("f8", "bf16", 64), ("f8", "bf16", 128)])
@pytest.mark.parametrize("K", [16, 128, 240, 256, 384, 400, 512, 1040])
def test_each_tile_by_stages(ex, xt, yt, p, K):
    """One stage, two, three and more, whole and partly past K: the loads' places in turn, and none behind the last."""
    T, E, N, _ = SIZES[p]
    N += 800 if K >= 384 and p == 32 else 0                         # a longer k asks for more workgroups
    assert path(ex, xt, yt, False, T, E, N, K) == p
    g = torch.Generator().manual_seed(K)
    w = w_operand(ex, g, 1, N, K, False)
    x = torch.randn((T, K), generator=g)
    off = np.array([T * e // E for e in range(E + 1)], np.int32)
    # experts that share one matrix, by a table of pointers
    xd, xv, xp = x_operand(ex, x, xt)
    y = torch.full((T + 1, N + 3), float("nan"), dtype=TYPES[yt], device="cuda")
    gm = ex.make_gemm(xd, w[0], None, torch.from_numpy(off).cuda(), y[:T, :N])
    tw = torch.full((E,), w[0].codes.data_ptr(), dtype=torch.int64, device="cuda")
    ts = torch.full((E,), w[0].scales.data_ptr(), dtype=torch.int64, device="cuda")
    gm.n_expert, gm.w, gm.w_scales, gm.w_stride, gm.ws_stride = E, tw.data_ptr(), ts.data_ptr(), 0, 0
    assert ex.moe_gemm(gm) == 0
    torch.cuda.synchronize()
    want, tol = f8ref.gemm(xv, w[1], None, [0, T], T, 1, False, (xp, w[2]) if xt == "f8" and yt != "f32" else None)
    assert mx4ref.close(y[:T, :N].cpu(), want, tol)
    assert torch.isnan(y[T]).all() and torch.isnan(y[:, N:]).all()


@pytest.mark.parametrize("xt", XS)
@pytest.mark.parametrize("K", [16, 48, 112, 144, 640, 1040, 1552])
def test_columns_that_end_inside_a_block(ex, xt, K):
    check(ex, xt, "f32", False, 5, 3, 4, 33, K)
    check(ex, xt, "f32", True, 130, 1, 2, 66, K)


@pytest.mark.parametrize("xt", XS)
@pytest.mark.parametrize("yt", list(TYPES))
def test_output_types(ex, xt, yt):
    check(ex, xt, yt, True, 20, 2, 6, 96, 256)
    check(ex, xt, yt, False, 200, 2, 2, 150, 256)


@pytest.mark.parametrize("xt", XS)
@pytest.mark.parametrize("half", [1, 15, 100, 129, 135, 200, 257])
def test_gate_and_up_have_blocks_of_their_own(ex, xt, half):
    """Halves that are no whole blocks, scales a thousandfold apart from block to block; few rows and many."""
    g = torch.Generator().manual_seed(half)
    down = 2 * ((half + 127) // 128)
    scale = torch.pow(10.0, torch.randint(-4, 0, (2, down, 3), generator=g).float())
    for tokens in (3, 150):
        check(ex, xt, "f32", True, tokens, 2, 2, 2 * half, 272, w=w_operand(ex, g, 2, 2 * half, 272, True, scale))


@pytest.mark.parametrize("xt", XS)
@pytest.mark.parametrize("n", [3, 200])
def test_rows_outside_the_runs_and_dropped_rows_are_zeros(ex, xt, n):
    """Runs that start behind row 0 and end before T, empty experts, dropped slots, tokens that x does not have; and rows with infinities and NaNs
    beside others, which stay alone."""
    rng = np.random.default_rng(5)
    E, T, tokens, K, N = 4, n + 20, 30, 96, 48
    off = np.array([7, 7, 7 + n // 3, 7 + n, 7 + n], np.int32)
    order = rng.integers(0, tokens * 2, T).astype(np.int32)
    order[8] = -1
    order[7 + n // 2] = tokens * 2 + 5
    x = torch.randn((tokens, K), generator=torch.Generator().manual_seed(1))
    got, y, tol, _ = run(ex, xt, "f32", False, tokens, 2, E, N, K, route=(order, off), x=x)
    assert mx4ref.close(got, y, tol)
    dead = [i for i in range(T) if i < 7 or i >= 7 + n or i == 8 or i == 7 + n // 2]
    assert (got[dead] == 0).all()
    bad = x.clone()
    bad[3, 5], bad[4, 9] = float("nan"), float("inf")
    got2, _, _, _ = run(ex, xt, "f32", False, tokens, 2, E, N, K, route=(order, off), x=bad)
    hit = torch.tensor([order[i] // 2 in (3, 4) and i not in dead for i in range(T)])
    assert torch.equal(got2[~hit], got[~hit])
    assert not torch.isfinite(got2[hit]).all() if hit.any() else True
    assert (got2[dead] == 0).all()


@pytest.mark.parametrize("xt", XS)
@pytest.mark.parametrize("T", [5, 300])
def test_a_weights_infinite_block_stays_alone(ex, xt, T):
    """A block of weights with the scale NaN: its 128 columns of y are NaN, the others are what they were."""
    g = torch.Generator().manual_seed(2)
    wd, wv, wp = w_operand(ex, g, 1, 400, 272, False)
    wd.scales[0, 1, 1] = float("nan")
    wv[0, 128:256, 128:256] = float("nan")
    check(ex, xt, "f32", False, T, 1, 1, 400, 272, w=(wd, wv, wp))


@pytest.mark.parametrize("xt", XS)
def test_offsets_that_are_no_routing_write_only_their_rows(ex, xt):
    E, T, K, N = 6, 64, 64, 40
    order = np.arange(T, dtype=np.int32)
    for off in ([0, 10, 5, 64, 64, 64, 64], [-5, 3, 900, 20, 64, 70, 80], [70, 70, 70, 70, 70, 70, 70], [0] * 7):
        run(ex, xt, "f32", False, T, 1, E, N, K, route=(order, np.array(off, np.int32)))


@pytest.mark.parametrize("xt", XS)
def test_more_experts_than_one_scan_holds(ex, xt):
    E, T = 1500, 90
    ids = np.sort(np.random.default_rng(2).choice([0, 5, 509, 510, 511, 512, 1021, 1022, 1023, 1400, 1499], T))
    off = np.zeros(E + 1, np.int32)
    off[1:] = np.cumsum(np.bincount(ids, minlength=E))
    check(ex, xt, "f32", False, T, 1, E, 36, 32, route=(np.arange(T, dtype=np.int32), off))


@pytest.mark.parametrize("xt", XS)
@pytest.mark.parametrize("tokens", [20, 400])
def test_pointer_tables_give_the_stacked_buffers_bits(ex, xt, tokens):
    g = torch.Generator().manual_seed(1)
    w = w_operand(ex, g, 5, 300, 272, True)
    got, y, tol, gm = run(ex, xt, "f32", True, tokens, 2, 5, 300, 272, w=w)
    table = lambda t: torch.tensor([t[e].data_ptr() for e in range(t.shape[0])], dtype=torch.int64, device="cuda")
    tw, ts = table(w[0].codes), table(w[0].scales)
    yd = gm.tensors[-1]
    yd.fill_(0)
    gm.w, gm.w_scales, gm.w_stride, gm.ws_stride = tw.data_ptr(), ts.data_ptr(), 0, 0
    assert ex.moe_gemm(gm) == 0
    torch.cuda.synchronize()
    assert torch.equal(yd.cpu(), got)


@pytest.mark.parametrize("xt", XS)
def test_large_numbers_in_16_bit_rows(ex, xt):
    """The largest codes against x near its type's end (F8: a scale near f32's): products and sums that 16 bits would not hold."""
    g = torch.Generator().manual_seed(4)
    w = w_operand(ex, g, 1, 64, 256, False, torch.full((1, 1, 2), 2.0 ** -20))
    x = torch.randn((40, 256), generator=g).clamp(-3, 3) * {"f16": 2e4, "bf16": 1e33, "f8": 1e33}[xt]
    check(ex, xt, "f32", False, 40, 1, 1, 64, 256, x=x, w=w)


def test_same_bits_on_two_streams_and_in_a_replayed_graph(ex):
    """One descriptor's operands, two outputs: launches on two streams at once, and a captured chain (quantise, product) replayed on new rows."""
    g = torch.Generator().manual_seed(7)
    wd, wv, _ = w_operand(ex, g, 3, 256, 272, True)
    x = torch.randn((200, 272), generator=g).bfloat16().cuda()
    q = ex.f8_empty((200, 272), 1)
    order, off = routing(np.random.default_rng(0), 200, 2, 3)
    st, of = torch.from_numpy(order).cuda(), torch.from_numpy(off).cuda()
    ys = [torch.zeros(400, 128, device="cuda") for _ in range(3)]
    gs = [ex.make_gemm(q, wd, st, of, y, top_k=2, act=ex.ACT_SWIGLU) for y in ys]
    assert ex.f8_quant(x, q) == 0
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for i, s in enumerate(streams):
            assert ex.moe_gemm(gs[i], s) == 0
    torch.cuda.synchronize()
    assert torch.equal(ys[0], ys[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert ex.f8_quant(x, q) == 0 and ex.moe_gemm(gs[2]) == 0
    for seed in range(3):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(seed)))
        ys[2].fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert ex.f8_quant(x, q) == 0 and ex.moe_gemm(gs[0]) == 0
        torch.cuda.synchronize()
        assert torch.equal(ys[2], ys[0])
        c, s = f8ref.quant(x.cpu()[None], 1)
        y, tol = f8ref.gemm(f8ref.values(c, s, 272, 1)[0], wv, order, off, 400, 2, True)
        assert mx4ref.close(ys[2].cpu(), y, tol)


def far(t, pitch):
    """t with its rows `pitch` bytes apart."""
    n, size = t.shape[:-1].numel(), t.element_size()
    strides = [pitch // size, 1]
    for d in t.shape[1:-1][::-1]:
        strides.insert(0, strides[0] * d)
    v = torch.empty(n * pitch // size, dtype=t.dtype, device="cuda").as_strided(t.shape, strides)
    return v.copy_(t)


@pytest.mark.parametrize("xt,yt", [("f16", "f16"), ("bf16", "f32"), ("f8", "f32"), ("f8", "bf16")])
@pytest.mark.parametrize("T,pitch", [(6, 1 << 30), (2600, 1 << 22)])
def test_offsets_past_32_bits(ex, xt, yt, T, pitch):
    """Rows of x, of y and of weights, scales and experts that lie more than 4 GiB apart: the bits of the same operands without gaps."""
    E, N, K = 2, 40, 256
    assert path(ex, xt, yt, False, T, E, N, K) == (2 if T == 6 else 32)
    g = torch.Generator().manual_seed(7)
    off = torch.tensor([0, T // 3, T], dtype=torch.int32, device="cuda")
    x = torch.randn((T, K), generator=g).cuda()
    if xt == "f8":
        q = ex.f8_empty((T, K), 1)
        assert ex.f8_quant(x, q) == 0
        xs = q, ex.F8(far(q.codes, pitch), far(q.scales, pitch), K, 1)
    else:
        x = x.to(TYPES[xt])
        xs = x, far(x, pitch)
    w = w_operand(ex, g, E, N, K, False)[0]
    wf = ex.F8(far(w.codes, 1 << 27), far(w.scales, 1 << 27), K, 128)
    outs = []
    for xq, wq, y in ((xs[0], w, torch.empty((T, N), dtype=TYPES[yt], device="cuda")), (xs[1], wf, far(torch.zeros((T, N), dtype=TYPES[yt], device="cuda"), pitch))):
        assert ex.moe_gemm(ex.make_gemm(xq, wq, None, off, y)) == 0
        torch.cuda.synchronize()
        outs.append(y.cpu())
    assert not outs[0].isnan().any() and torch.equal(*outs)
    del xs, w, wf, x, xq, wq, y
    torch.cuda.empty_cache()


@pytest.mark.parametrize("xt,yt", [("bf16", "bf16"), ("f16", "f32"), ("f8", "bf16"), ("f8", "f32")])
@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("others,p", [(2, 32), (20, 64)])
def test_weights_that_go_past_the_caches(ex, xt, yt, swiglu, others, p):
    """More weights than the cache behind L2 holds (287 MB): runs of one chunk, of no row, of a chunk and a row, of whole chunks and of several, against the product
    of their experts in 64 bits; the other experts' rows are written."""
    E, N, K = 80, 3500, 1024
    lens = [others] * E
    some = {0: 1, 3: 0, 4: 33, 5: 64, 6: 65, 40: 32, 79: 130}
    for e, n in some.items():
        lens[e] = n
    off = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    T, n_out = int(off[-1]), N // 2 if swiglu else N
    assert path(ex, xt, yt, swiglu, T, E, n_out, K) == p
    g = torch.Generator().manual_seed(p)
    dg = torch.Generator(device="cuda").manual_seed(p)
    codes = torch.randint(0, 254, (E, N, K), dtype=torch.uint8, device="cuda", generator=dg)
    codes += (codes >= 127).to(torch.uint8)                       # 127 and 255 are NaN
    halves = 2 if swiglu else 1
    scales = torch.rand((E, halves * ((N // halves + 127) // 128), K // 128), generator=g) * 0.01 + 0.0005
    x = torch.randn((T, K), generator=g)
    xd, xv, xp = x_operand(ex, x, xt)
    y = torch.full((T, n_out), float("nan"), dtype=TYPES[yt], device="cuda")
    gm = ex.make_gemm(xd, ex.F8(codes, scales.cuda(), K, 128), None, torch.from_numpy(off).cuda(), y, act=ex.ACT_SWIGLU if swiglu else ex.ACT_NONE)
    for _ in range(2):
        assert ex.moe_gemm(gm) == 0
        torch.cuda.synchronize()
        got = y.cpu()
        assert not got.isnan().any()
        for e in some:
            rows = slice(off[e], off[e + 1])
            c, s = codes[e:e + 1].cpu(), scales[e:e + 1]
            cut = (xp[rows], f8ref.peaks(c, f8ref.weights(torch.full_like(c, 0x38), s, halves))) if xt == "f8" and yt != "f32" else None
            want, tol = f8ref.gemm(xv[rows], f8ref.weights(c, s, halves), None, [0, lens[e]], lens[e], 1, swiglu, cut)
            assert mx4ref.close(got[rows], want, tol), e
        y.fill_(float("nan"))
