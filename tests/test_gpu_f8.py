"""f8_quant and f8_dequant on the device against the format's rule (tests/f8ref.py): codes and scales equal to the bit, values to a rounding,
whatever the type, the columns, the block, the pitches and the alignment."""
import pytest

import f8ref

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


def special(dt):
    """Rows of two blocks of what a conversion can get wrong: every code's value and every tie between codes at several scales, zeros of both
    signs, subnormals, the largest and smallest numbers, a lone value among zeros, infinities and NaNs."""
    grid = torch.from_numpy(f8ref.GRID)
    ties = (grid[1:] + grid[:-1]) / 2
    base = torch.cat([grid, -grid[:1], grid[126:], -ties, ties[-2:]])[:256]                      # 448 among them in both blocks
    base[0] = 448.0
    rows = [torch.ldexp(base, torch.tensor(e)) for e in (0, -9, 6, -30, -100, -140, 80, 117)]
    rows += [torch.zeros(256), -torch.zeros(256), torch.full((256,), 1e-45), torch.full((256,), 3.4e38), torch.full((256,), 65504.0)]
    lone = torch.zeros(256)
    lone[77], lone[200] = 1e-3, -2.0 ** -97
    rows.append(lone)
    for bad in (float("inf"), -float("inf"), float("nan")):
        r = torch.arange(256).double()
        r[130] = bad
        rows.append(r)
    x = torch.stack([r.double() for r in rows])
    return x.to(dt) if dt != torch.float16 else x.clamp(-7e4, 7e4).to(dt)                      # past f16's range: infinities again


def check(ex, x, block, extra=(0, 0, 0)):
    """x [mats, rows, cols] on the device; planes `extra` columns of codes (in 16s), of scales and rows of codes larger than they need be."""
    m, R, C = x.shape
    c, s = f8ref.quant(x.cpu(), block)
    codes = torch.full((m, R + extra[2], c.shape[2] + extra[0]), 0xA5, dtype=torch.uint8, device="cuda")
    scales = torch.full((m, s.shape[1], s.shape[2] + extra[1]), -7.0, device="cuda")
    q = ex.F8(codes[:, :R], scales, C, block)
    assert ex.f8_quant(x, q) == 0
    torch.cuda.synchronize()
    got = codes[:, :R, :c.shape[2]].cpu()
    same = (got == c) | ((got & 127 == 0) & (c & 127 == 0))                                  # a zero's sign is open
    assert same.all(), (got != c).nonzero()[:5]
    gs = scales[..., :s.shape[2]].cpu()
    assert torch.equal(gs.isnan(), s.isnan()) and torch.equal(gs.nan_to_num(1.5), s.nan_to_num(1.5))
    assert (codes[:, :R, c.shape[2]:] == 0xA5).all() and (codes[:, R:] == 0xA5).all() and (scales[..., s.shape[2]:] == -7).all()
    v = f8ref.values(c, s, C, block)
    for t in TYPES.values():
        out = torch.full((m, R + 1, C + 3), -7.0, dtype=t, device="cuda")
        assert ex.f8_dequant(q, out[:, :R, :C]) == 0
        torch.cuda.synchronize()
        o = out[:, :R, :C].cpu()
        # the product in f32, then its rounding to t: two halves of a step, and of the smallest step below the normal numbers
        step = torch.finfo(t).eps / 2 + 2.0 ** -24
        tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[t] * (1 + 2.0 ** -10)
        top = torch.finfo(t).max * (1 + torch.finfo(t).eps / 4)
        fits = v.abs() <= top
        assert torch.equal(o.isnan(), v.isnan())
        assert ((o.double() - v).abs() <= step * v.abs() + tiny)[fits].all()
        assert (o.isinf() | v.isnan() | fits).all()
        assert (out[:, :R, C:] == -7).all() and (out[:, R:] == -7).all()


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("block", [1, 128])
def test_special_values(ex, t, block):
    x = special(TYPES[t])
    if block == 1:
        check(ex, x[None].cuda(), 1)
    else:                                                          # a matrix each: its first row the values, the others a 300th of them
        y = torch.cat([x[:, None], (x[:, None].float() / 300).to(x.dtype).expand(-1, 130, -1)], 1)
        check(ex, y.cuda(), 128)


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("mats,rows,cols,block", [
    (1, 1, 1, 1), (1, 1, 1, 128), (1, 3, 7, 1), (1, 5, 128, 1), (2, 9, 129, 1), (1, 4, 650, 1), (3, 127, 127, 128), (2, 128, 128, 128),
    (2, 129, 257, 128), (1, 300, 16, 128), (5, 1, 640, 128), (1, 700, 2048, 1), (2, 333, 1000, 128)])
def test_sizes(ex, t, mats, rows, cols, block):
    print(f"f8 {mats} x {rows} x {cols} block {block} {t}", flush=True)
    g = torch.Generator().manual_seed(rows * cols)
    x = torch.randn((mats, rows, cols), generator=g) * (torch.rand((mats, rows, 1), generator=g) * 3 + 0.01)
    check(ex, x.to(TYPES[t]).cuda(), block, extra=(16, 1, 2))


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("block", [1, 128])
def test_any_alignment_and_pitch(ex, t, block):
    """Values from an odd element on, rows of an odd pitch, matrices an odd stride apart."""
    buf = torch.randn(40000, generator=torch.Generator().manual_seed(3)).to(TYPES[t]).cuda()
    x = buf[1:].as_strided((3, 30, 277), (9001, 293, 1))
    check(ex, x, block)


def test_the_whole_range_of_16_bit_inputs(ex):
    """Every finite bf16 and f16 number, each block a stretch of the numbers in order (blocks of one row and of 128 rows)."""
    for dt, n in ((torch.bfloat16, 0x7F80), (torch.float16, 0x7C00)):
        b = torch.arange(n, dtype=torch.int32).to(torch.int16).view(dt)
        x = torch.cat([b, -b]).view(1, -1, 256)
        for block in (1, 128):
            check(ex, x.cuda(), block)


def test_nothing_to_convert(ex):
    for shape in ((0, 4, 128), (2, 0, 128)):
        q = ex.f8_empty(shape, 128)
        x = torch.zeros(shape, device="cuda")
        assert ex.f8_quant(x, q) == 0 and ex.f8_dequant(q, x) == 0


def test_planes_of_e4m3_tensors_and_another_stream(ex):
    """Codes that torch holds as float8_e4m3fn, on a stream of the caller's, and in a graph that is replayed on new values."""
    x = torch.randn(1, 40, 256, device="cuda")
    q = ex.F8(torch.zeros(1, 40, 256, dtype=torch.float8_e4m3fn, device="cuda"), torch.zeros(1, 40, 2, device="cuda"), 256, 1)
    out = torch.zeros_like(x)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    assert ex.f8_quant(x, q, st) == 0 and ex.f8_dequant(q, out, st) == 0
    st.synchronize()
    assert torch.equal(out, q.codes.float() * q.scales.repeat_interleave(128, 2))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        assert ex.f8_quant(x, q) == 0 and ex.f8_dequant(q, out) == 0
    for seed in range(3):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(seed)))
        g.replay()
        torch.cuda.synchronize()
        c, s = f8ref.quant(x.cpu(), 1)
        v = f8ref.values(c, s, 256, 1)
        assert ((out.cpu().double() - v).abs() <= 2.0 ** -24 * v.abs()).all()


def far(t, pitch, stride):
    """t [mats, rows, cols] with its rows `pitch` and its matrices `stride` bytes apart."""
    size = t.element_size()
    v = torch.empty(t.shape[0] * stride // size, dtype=t.dtype, device="cuda").as_strided(t.shape, (stride // size, pitch // size, 1))
    return v.copy_(t)


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("block,rows,pitch,stride", [(1, 3, 1 << 31, 3 << 31), (128, 130, 1 << 25, 130 << 25), (1, 5, 1 << 12, 5 << 30), (128, 5, 1 << 12, 5 << 30)])
def test_offsets_past_32_bits(ex, t, block, rows, pitch, stride):
    """Rows and matrices more than 4 GiB apart: the codes, scales and values of the same without gaps."""
    x = torch.randn((2, rows, 300), generator=torch.Generator().manual_seed(1)).to(TYPES[t]).cuda()
    q = ex.f8_empty(x.shape, block)
    assert ex.f8_quant(x, q) == 0
    fq = ex.F8(far(torch.zeros_like(q.codes), pitch, stride), far(torch.zeros_like(q.scales), pitch, stride), 300, block)
    assert ex.f8_quant(far(x, pitch, stride), fq) == 0
    out, fout = torch.empty_like(x), far(torch.zeros_like(x), pitch, stride)
    assert ex.f8_dequant(q, out) == 0 and ex.f8_dequant(fq, fout) == 0
    torch.cuda.synchronize()
    assert torch.equal(q.codes, fq.codes) and torch.equal(q.scales, fq.scales) and torch.equal(out, fout)
    del fq, fout
    torch.cuda.empty_cache()


def test_more_values_than_one_launch_indexes(ex):
    """2^17 slots of 16 bytes a row and 16,400 rows: a second launch from row 16,383 on."""
    rows, cols, some = 16400, 1 << 20, [0, 5, 16382, 16383, 16384, 16399]
    x = torch.empty((rows, cols), dtype=torch.float16, device="cuda").zero_()
    part = torch.randn((len(some), cols), device="cuda").half()
    for i, r in enumerate(some):
        x[r] = part[i]
    few, q = ex.f8_empty((len(some), cols), 1), ex.f8_empty((rows, cols), 1)
    q.codes.fill_(0xA5)
    assert ex.f8_quant(part, few) == 0 and ex.f8_quant(x, q) == 0
    out = x.view(torch.bfloat16)
    out.fill_(-7.0)
    want = torch.empty((len(some), cols), dtype=torch.bfloat16, device="cuda")
    assert ex.f8_dequant(few, want) == 0 and ex.f8_dequant(q, out) == 0
    torch.cuda.synchronize()
    for i, r in enumerate(some):
        assert torch.equal(q.codes[r], few.codes[i]) and torch.equal(q.scales[r], few.scales[i]) and torch.equal(out[r], want[i])
    for a, b in zip([-1] + some, some + [rows]):
        for r in range(a + 1, b, 2048):
            assert not q.codes[r:min(r + 2048, b)].any() and not out[r:min(r + 2048, b)].any()
    del x, out, q
    torch.cuda.empty_cache()


@pytest.mark.parametrize("block", [1, 128])
def test_replayed_graphs_beside_each_other(ex, block):
    """Two captured graphs of both conversions, replayed on two streams at once several times, with new values in between."""
    sets = []
    for i in range(2):
        x = torch.empty((2, 200 + i, 650), dtype=torch.bfloat16, device="cuda")
        q, out, st, graph = ex.f8_empty(x.shape, block), torch.empty_like(x, dtype=torch.float32), torch.cuda.Stream(), torch.cuda.CUDAGraph()
        x.zero_()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=st):
            assert ex.f8_quant(x, q, st) == 0 and ex.f8_dequant(q, out, st) == 0
        sets.append((x, q, out, st, graph))
    for k in range(4):
        for i, (x, q, out, st, graph) in enumerate(sets):
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(10 * k + i)) * 2.0 ** (k - 2))
        torch.cuda.synchronize()
        for _, _, _, st, graph in sets:
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for x, q, out, _, _ in sets:
            own, values = ex.f8_empty(x.shape, block), torch.empty_like(out)
            assert ex.f8_quant(x, own) == 0 and ex.f8_dequant(own, values) == 0
            torch.cuda.synchronize()
            assert torch.equal(q.codes, own.codes) and torch.equal(q.scales, own.scales) and torch.equal(out, values)


@pytest.mark.parametrize("t", list(TYPES))
def test_zeros_keep_their_sign(ex, t):
    x = torch.zeros((2, 256), dtype=TYPES[t], device="cuda")
    x[0, 1::2] = -0.0
    x[1, ::3] = -0.0
    x[1, 5] = -2.0
    q = ex.f8_empty(x.shape, 1)
    assert ex.f8_quant(x, q) == 0
    torch.cuda.synchronize()
    assert torch.equal(q.codes.cpu() >> 7, torch.signbit(x.cpu()).byte())


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("cols", [1024, 1022])
def test_large_matrices_are_what_their_parts_are(ex, t, block, cols):
    """More codes and values than the caches are meant to keep, which are stored past them: the same as of 1,280 rows at a time."""
    rows = 1280 * 110
    x = torch.randn((rows, cols), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(TYPES[t])
    q, out = ex.f8_empty(x.shape, block), torch.empty_like(x)
    assert ex.f8_quant(x, q) == 0 and ex.f8_dequant(q, out) == 0
    part, values = ex.f8_empty((1280, cols), block), torch.empty((1280, cols), dtype=TYPES[t], device="cuda")
    for r in range(0, rows, 1280 * 7):
        assert ex.f8_quant(x[r:r + 1280], part) == 0 and ex.f8_dequant(part, values) == 0
        torch.cuda.synchronize()
        assert torch.equal(q.codes[r:r + 1280], part.codes) and torch.equal(out[r:r + 1280], values)
        assert torch.equal(q.scales[r // block:(r + 1280) // block], part.scales)
