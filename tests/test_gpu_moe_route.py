"""moe_route on the device against its definition in 64 bits (tests/routeref.py): experts equal, in order and with ties, the scatter equal, weights
within their one rounding to f32 (what is behind it is in f64, some 2^-45 off at most)."""
import numpy as np
import pytest

import routeref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


@pytest.fixture(scope="module")
def ex():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import exl3c4
    exl3c4.lib()
    return exl3c4


def outputs(n_tok, E, top_k, spare=3):
    """(ids, w, sorted_tok, offset, count, row_of) as the routing writes them, each with guards behind."""
    i32 = lambda n: torch.full((n + spare,), -77, dtype=torch.int32, device="cuda")
    return (i32(n_tok * top_k), torch.full((n_tok * top_k + spare,), -77.0, device="cuda"), i32(n_tok * top_k), i32(E + 1), i32(E), i32(n_tok * top_k))


def check(ex, l, top_k, score="sigmoid", bias=None, n_group=1, top_group=1, group="max", renorm=True, scale=1.0, scatter=True, stream=None):
    """l [n_tok, n_expert] on the device, of any pitch."""
    n_tok, E = l.shape
    ids, w, st, off, cnt, row = outputs(n_tok, E, top_k)
    more = dict(sorted_tok=st, expert_offset=off, expert_count=cnt, row_of=row) if scatter else {}
    n = n_tok * top_k
    r = ex.make_route(l, top_k, ids[:n].view(n_tok, top_k), w[:n].view(n_tok, top_k), score=ex.SCORE_SIGMOID if score == "sigmoid" else ex.SCORE_SOFTMAX,
                      bias=bias, n_group=n_group, top_group=top_group, group_score=ex.GROUP_TOP2 if group == "top2" else ex.GROUP_MAX, renorm=renorm,
                      scale=scale, **more)
    assert ex.moe_route(r, stream) == 0
    torch.cuda.synchronize()
    wi, ww = routeref.route(l.float().cpu().numpy(), top_k, score, None if bias is None else bias.cpu().numpy(), n_group, top_group, group, renorm, scale)
    gi, gw = ids[:n].view(n_tok, top_k).cpu().numpy(), w[:n].view(n_tok, top_k).cpu().numpy().astype(np.float64)
    assert np.array_equal(gi, wi), (np.argwhere(gi != wi)[:5], gi[(gi != wi).any(1)][:2], wi[(gi != wi).any(1)][:2])
    assert (np.abs(gw - ww) <= 2.0 ** -24 * (1 + 2.0 ** -18) * np.abs(ww) + 2.0 ** -150).all()
    assert (ids[n:] == -77).all() and (w[n:] == -77).all()
    if scatter:
        for got, want in zip((st, off, cnt, row), routeref.scatter(wi, E)):
            assert np.array_equal(got[:len(want)].cpu().numpy(), want) and (got[len(want):] == -77).all()
    return gi, gw


CASES = [  # n_tok, n_expert, top_k, n_group, top_group
    (1, 1, 1, 1, 1), (1, 256, 8, 8, 4), (3, 8, 2, 1, 1), (16, 20, 5, 5, 2), (17, 20, 20, 5, 5), (5, 64, 6, 64, 8), (16, 64, 1, 2, 1), (33, 160, 6, 8, 3),
    (300, 256, 8, 8, 4), (20, 384, 64, 16, 8), (64, 512, 10, 1, 1), (9, 512, 10, 4, 2), (40, 1000, 7, 10, 3), (16, 1024, 64, 2, 1), (70, 1024, 33, 64, 40),
    (4, 66, 3, 33, 2)]


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_sizes(ex, case, score):
    n_tok, E, top_k, n_group, top_group = case
    print(f"route {case} {score}", flush=True)
    g = torch.Generator().manual_seed(E + n_tok)
    l = torch.randn((n_tok, E), generator=g) * 2
    bias = (torch.randn(E, generator=g) * (0.2 if score == "sigmoid" else 1 / E)).cuda()
    for b in (None, bias):
        for group in (("max", "top2") if n_group > 1 else ("max",)):
            check(ex, l.cuda(), top_k, score, b, n_group, top_group, group, renorm=b is None, scale=2.5, scatter=group == "max")


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("n_tok", [1, 16, 50])
def test_types_pitches_and_alignment(ex, t, n_tok):
    """Logits of each type from an odd element on, rows apart by an odd pitch; in 16 bits equal ones are common."""
    buf = (torch.randn(40000, generator=torch.Generator().manual_seed(n_tok)) * 1.5).to(TYPES[t]).cuda()
    l = buf[1:].as_strided((n_tok, 192), (301, 1))
    bias = torch.round(torch.randn(192, generator=torch.Generator().manual_seed(2)) * 4).cuda() / 4
    for score in ("sigmoid", "softmax"):
        check(ex, l, 8, score)
        check(ex, l, 8, score, n_group=6, top_group=2, group="top2")
        check(ex, l, 8, score, bias, 6, 2, "top2")


def test_ties_go_to_the_lower_id(ex):
    """Equal logits (all of them: more candidates than a wave holds), equal biases, equal groups, zeros of both signs."""
    for n_tok in (2, 30):
        l = torch.zeros(n_tok, 300, device="cuda")
        gi, gw = check(ex, l, 40)
        assert (gi == np.arange(40)).all()
        check(ex, l, 40, bias=torch.full((300,), 0.3, device="cuda"))
        check(ex, l, 12, n_group=30, top_group=2, group="top2")
        l[:, ::2] = -0.0
        check(ex, l, 64, "softmax")
        l = torch.randint(-2, 3, (n_tok, 300), generator=torch.Generator().manual_seed(1)).float().cuda()
        check(ex, l, 64)
        check(ex, l, 20, bias=(torch.arange(300) % 3).float().cuda() / 8)
        check(ex, l, 9, "softmax", n_group=20, top_group=3, group="top2")


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_values_that_32_bits_do_not_tell_apart(ex, score):
    """Biases that bring the choices of all experts within some 2^-28 of each other, and groups' sums too."""
    g = torch.Generator().manual_seed(5)
    l = torch.randn((40, 256), generator=g)
    s = torch.sigmoid(l.double()) if score == "sigmoid" else torch.softmax(l.double(), 1)
    for n_group, group in ((1, "max"), (8, "max"), (8, "top2")):
        for t in range(0, 40, 8):
            check(ex, l[t:t + 1].cuda(), 8, score, (0.75 - s[t]).float().cuda(), n_group, max(1, n_group // 2), group)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("n_tok", [7, 40])
def test_experts_that_are_out(ex, score, n_tok):
    """-infinity and NaN in logits and biases: rows without an expert, groups without one, fewer experts than slots, one expert in a group."""
    g = torch.Generator().manual_seed(n_tok)
    l = torch.randn((n_tok, 96), generator=g)
    l[0] = -float("inf")
    l[1] = float("nan")
    l[2, 3:] = -float("inf")
    l[3, :90] = float("nan")
    l[4][torch.rand(96, generator=g) < 0.9] = -float("inf")
    l[5, 12:24] = -float("inf")
    l[6, 0:11] = float("nan")
    bias = torch.randn(96, generator=g) * 0.1
    bias[7], bias[8], bias[24:36] = -float("inf"), float("nan"), -float("inf")
    for b in (None, bias.cuda()):
        for n_group, top_group, group in ((1, 1, "max"), (8, 3, "max"), (8, 3, "top2"), (8, 8, "top2")):
            for renorm in (False, True):
                gi, gw = check(ex, l.cuda(), 6, score, b, n_group, top_group, group, renorm, 1.5)
                assert (gi[:2] == -1).all() and (gw[gi < 0] == 0).all()
    check(ex, torch.full((n_tok, 96), -float("inf"), device="cuda"), 6, score)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_infinities_and_far_logits(ex, score):
    """+infinity (once, several times), logits far beyond where a score leaves f32 and f64, a bias of +infinity."""
    l = torch.randn((20, 64), generator=torch.Generator().manual_seed(3))
    l[0, 9] = float("inf")
    l[1, 5:8] = float("inf")
    l[2] *= 1e30
    l[3] -= 200.0
    l[4] -= 2000.0
    l[5] += 3e38
    l[6] *= 30
    for renorm in (False, True):
        check(ex, l.cuda(), 5, score, renorm=renorm)
    b = torch.zeros(64)
    b[40] = float("inf")
    check(ex, l[6:].cuda(), 5, score, b.cuda(), 4, 2, "max")


def test_no_tokens_and_one_expert(ex):
    for top in (1, 3):
        l = torch.zeros(0, 64, device="cuda")
        off = torch.full((65,), 9, dtype=torch.int32, device="cuda")
        ids, w = torch.zeros(0, top, dtype=torch.int32, device="cuda"), torch.zeros(0, top, device="cuda")
        assert ex.moe_route(ex.make_route(l, top, ids, w, expert_offset=off, sorted_tok=ids.view(-1))) == 0
        assert (off == 0).all()
    check(ex, torch.tensor([[-3.0]]).cuda(), 1, "softmax")


def test_streams_and_a_replayed_graph(ex):
    """On a stream of the caller's, two routings at once, and captured (16 tokens: one launch, 40: two), replayed on new logits."""
    st = torch.cuda.Stream()
    l = torch.randn(40, 256, device="cuda")
    st.wait_stream(torch.cuda.current_stream())
    check(ex, l, 8, n_group=8, top_group=4, group="top2", stream=st)
    for n_tok in (16, 40):
        ids, w, so, off, cnt, row = outputs(n_tok, 256, 8, 0)
        r = ex.make_route(l[:n_tok], 8, ids.view(n_tok, 8), w.view(n_tok, 8), score=ex.SCORE_SIGMOID, n_group=8, top_group=4, group_score=ex.GROUP_TOP2,
                          sorted_tok=so, expert_offset=off, row_of=row)
        assert ex.moe_route(r) == 0
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            assert ex.moe_route(r) == 0
        for seed in range(3):
            l.copy_(torch.randn(l.shape, generator=torch.Generator().manual_seed(seed)))
            for o in (ids, so, off, row):
                o.fill_(-5)
            graph.replay()
            torch.cuda.synchronize()
            wi, _ = routeref.route(l[:n_tok].cpu().numpy(), 8, "sigmoid", None, 8, 4, "top2")
            want = routeref.scatter(wi, 256)
            assert np.array_equal(ids.view(n_tok, 8).cpu().numpy(), wi)
            assert np.array_equal(so.cpu().numpy(), want[0]) and np.array_equal(off.cpu().numpy(), want[1]) and np.array_equal(row.cpu().numpy(), want[3])


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_groups_whose_sums_32_bits_do_not_tell_apart(ex, score):
    """Biases of unlike sign and size whose pairs bring each group's sum to within some 2^-28 of the others', among them exactly equal ones."""
    g = torch.Generator().manual_seed(8)
    l = torch.randn((12, 64), generator=g)
    s = torch.sigmoid(l.double()) if score == "sigmoid" else torch.softmax(l.double(), 1)
    for t in range(12):
        for big in (0.0, 3.0, 40.0):
            b = torch.full((64,), -100.0, dtype=torch.float64)
            for grp in range(16):                                # two experts a group that count: one up, one down
                b[4 * grp] = big + 0.5 - s[t, 4 * grp]
                b[4 * grp + 1] = -big + 0.25 - s[t, 4 * grp + 1]
            check(ex, l[t:t + 1].cuda(), 6, score, b.float().cuda(), 16, 5, "top2")
            check(ex, l[t:t + 1].cuda(), 6, score, b.float().cuda(), 16, 5, "max")
    same = torch.randn((1, 4), generator=g).repeat(3, 16)            # every group the same
    check(ex, same.cuda(), 9, score, None, 16, 3, "top2")
    check(ex, same.cuda(), 9, score, torch.randn(4, generator=g).repeat(16).cuda(), 16, 3, "top2")


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("n_tok", [16, 4000])
def test_groups_of_which_one_is_less_certain_in_32_bits(ex, score, n_tok):
    """The sums of two groups differ by less than 2^-14, where the second's is one of 1000 and -1000: far less certain than the first's."""
    g = torch.Generator().manual_seed(n_tok)
    l = torch.randn((n_tok, 12), generator=g)
    l[:, 4:6] = l[:, 0:2] + (torch.rand((n_tok, 2), generator=g) - 0.5) * 2.0 ** -12
    out = -float("inf")
    bias = torch.tensor([0.0, 0.0, out, out, 1000.0, -1000.0, out, out, -3.0, -3.0, out, out]).cuda()
    check(ex, l.cuda(), 2, score, bias, 3, 1, "top2", scatter=n_tok == 16)
    check(ex, l.cuda(), 3, score, bias, 3, 2, "top2", scatter=False)


@pytest.mark.parametrize("n_tok", [3, 40])
@pytest.mark.parametrize("E", [65, 100, 129, 192, 193, 257, 320, 511, 513, 700, 961])
def test_experts_that_do_not_fill_the_registers(ex, n_tok, E):
    g = torch.Generator().manual_seed(E)
    l = torch.randn((n_tok, E), generator=g)
    l[:, -1] += 3                                                   # the last one is often chosen
    b = (torch.randn(E, generator=g) * 0.1).cuda()
    check(ex, l.cuda(), min(8, E), "sigmoid", b)
    check(ex, l.bfloat16().cuda(), min(8, E), "softmax", b)
    check(ex, l.half().cuda(), min(8, E), "softmax")


@pytest.mark.parametrize("base", [-2 ** 31 - 2, -2 ** 31, -5, 2 ** 31 - 40, 2 ** 31 - 1, 2 ** 31, 2 ** 40, -2 ** 40])
def test_the_scatters_base_over_its_range(ex, base):
    """Ids over the whole of 32 bits against bases at its ends and beyond."""
    rng = np.random.default_rng(1)
    ids = rng.integers(-2 ** 31, 2 ** 31, (300, 6)).astype(np.int32)
    near = np.clip(base + rng.integers(-3, 60, ids.shape), -2 ** 31, 2 ** 31 - 1).astype(np.int32)
    ids = np.where(rng.random(ids.shape) < 0.7, near, ids)
    E, T = 50, ids.size
    g = ids.reshape(-1).astype(np.int64) - base
    want = routeref.scatter(np.where((g >= 0) & (g < E), g, -1).reshape(ids.shape), E)
    i = torch.from_numpy(ids).cuda()
    st, off, cnt, row = (torch.full((n,), -9, dtype=torch.int32, device="cuda") for n in (T, E + 1, E, T))
    assert ex.moe_scatter(i, E, st, off, cnt, row, base) == 0
    torch.cuda.synchronize()
    for got, w in zip((st, off, cnt, row), want):
        assert np.array_equal(got.cpu().numpy(), w)


@pytest.mark.parametrize("n_tok", [16, 20])
@pytest.mark.parametrize("t", list(TYPES))
def test_rows_past_32_bits(ex, t, n_tok):
    """Rows of logits 512 MiB apart."""
    pitch = (1 << 29) // torch.empty((), dtype=TYPES[t]).element_size()
    l = torch.empty(n_tok * pitch, dtype=TYPES[t], device="cuda").as_strided((n_tok, 96), (pitch, 1))
    l.copy_(torch.randn((n_tok, 96), generator=torch.Generator().manual_seed(3)) * 2)
    check(ex, l, 6, "sigmoid", (torch.arange(96) % 7).float().cuda() * 0.01, 8, 3, "top2")
    del l
    torch.cuda.empty_cache()


def scatter_check(ex, ids, E, base=0, count=True, rows=True):
    """moe_scatter of ids i32 [n_tok, top_k] on the device (of any 4-byte alignment) against the stable sort."""
    n_tok, top_k = ids.shape
    _, _, st, off, cnt, row = outputs(n_tok, E, top_k)
    assert ex.moe_scatter(ids, E, st[:-3], off[:-3], cnt[:-3] if count else None, row[:-3] if rows else None, base) == 0
    torch.cuda.synchronize()
    e = ids.cpu().numpy().astype(np.int64).reshape(-1) - base
    e = np.where((e >= 0) & (e < E), e, E)
    order = np.argsort(e, kind="stable")
    counts = np.bincount(e, minlength=E + 1)[:E]
    live = int(counts.sum())
    want = np.full(e.size, -1), np.concatenate(([0], np.cumsum(counts))), counts, np.full(e.size, -1)
    want[0][:live] = order[:live]
    want[3][order[:live]] = np.arange(live)
    for got, w, there in zip((st, off, cnt, row), want, (True, True, count, rows)):
        got = got.cpu().numpy()
        assert (got[len(w):] == -77).all()
        assert np.array_equal(got[:len(w)], w) if there else (got == -77).all()


@pytest.mark.parametrize("E", [1, 3, 8, 64, 255, 256, 257, 512, 513, 768, 769, 1000, 1024])
@pytest.mark.parametrize("n_tok,top_k", [(32, 1), (33, 1), (51, 5), (1024, 4), (4097, 1), (409, 10), (410, 10), (1640, 10), (8192, 9)])
def test_the_scatter_by_experts(ex, E, n_tok, top_k):
    """Numbers of experts around those that one, two, three and four a workgroup take, pairs around those of a wave's load and of its four loads together;
    ids at an odd word, some of them no expert's."""
    rng = np.random.default_rng(E * 7 + n_tok)
    store = torch.zeros(n_tok * top_k + 1, dtype=torch.int32, device="cuda")
    ids = store[1:].view(n_tok, top_k)
    ids.copy_(torch.from_numpy(rng.integers(-2, E + 3, (n_tok, top_k)).astype(np.int32)))
    scatter_check(ex, ids, E)
    scatter_check(ex, ids, E, count=False, rows=False)
    scatter_check(ex, ids, max(E // 4, 1), base=E // 3)
    ids += 1 << 29
    scatter_check(ex, ids, E, base=1 << 29)


@pytest.mark.parametrize("n_tok,top_k,E", [(4096, 2, 8), (20000, 4, 20), (20000, 4, 100), (13107, 10, 512), (65536, 8, 512), (65536, 2, 8)])
def test_scatters_of_one_expert_and_of_none(ex, n_tok, top_k, E):
    """More pairs of an expert than a wave's list holds (2,048 of the 16th of the pairs): all of them, three quarters, nearly all; and no expert's at all."""
    ids = torch.full((n_tok, top_k), E - 1, dtype=torch.int32, device="cuda")
    scatter_check(ex, ids, E)
    ids[:, 0] = torch.arange(n_tok, device="cuda") % E
    scatter_check(ex, ids, E)
    ids.fill_(0)
    ids[n_tok // 2:, 1] = E // 2
    scatter_check(ex, ids, E)
    ids.fill_(-1)
    scatter_check(ex, ids, E)
    ids.fill_(-2 ** 31)
    ids[5] = 2 ** 31 - 1
    scatter_check(ex, ids, E, base=1 << 30)
    scatter_check(ex, ids, E, base=-(1 << 30))
