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
