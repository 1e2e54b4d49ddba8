"""mx4_quant and mx4_dequant on the device against the format's rule in 64 bits (tests/mx4ref.py): codes, scale bytes and
values equal to the bit, whatever the type, the columns, the pitches and the alignment."""
import numpy as np
import pytest

import mx4ref

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


def bits(t):
    return t.view({2: torch.int16, 4: torch.int32}[t.element_size()])


def special(dt):
    """Blocks of what a conversion can get wrong: every tie of every code at several scales, subnormals, the largest and
    smallest numbers, zeros of both signs, infinities and NaNs."""
    ties = [0, 0.25, 0.5, 0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7, 7.9]
    rows = []
    for e in (-24, -14, -3, 0, 9, -126, -133, -149, 100, 125):
        v = torch.tensor([t * 2.0 ** e for t in ties[:16]], dtype=torch.float64)
        rows.append(torch.cat([v, -v]))
    rows += [torch.zeros(32), -torch.zeros(32), torch.full((32,), 1e-45), torch.full((32,), 3.4e38), torch.full((32,), 65504.0)]
    for bad in (float("inf"), -float("inf"), float("nan")):
        r = torch.arange(32).double()
        r[17] = bad
        rows.append(r)
    x = torch.stack([r.double() for r in rows])
    return x.to(dt) if dt != torch.float16 else x.clamp(-7e4, 7e4).to(dt)      # past f16's range: infinities again


def check(ex, x, cols, pitch_c, pitch_s):
    rows = x.shape[0]
    codes = torch.full((rows, pitch_c), 0xA5, dtype=torch.uint8, device="cuda")
    scales = torch.full((rows, pitch_s), 0xA5, dtype=torch.uint8, device="cuda")
    q = ex.Mx4(codes, scales, cols)
    assert ex.mx4_quant(x, q) == 0
    torch.cuda.synchronize()
    c, s = mx4ref.quant(x.cpu())
    nb = s.shape[1]
    assert torch.equal(scales[:, :nb].cpu(), s)
    got = codes[:, :16 * nb].cpu()
    # a code of a zero may carry either sign's bit: the values are what the format says
    v, w = mx4ref.dequant(got, s, 32 * nb), mx4ref.dequant(c, s, 32 * nb)
    assert torch.equal(torch.isnan(v), torch.isnan(w)) and torch.equal(v.nan_to_num(7), w.nan_to_num(7))
    assert (got[s.repeat_interleave(16, 1) == 255] == 0).all()
    assert (codes[:, 16 * nb:] == 0xA5).all() and (scales[:, nb:] == 0xA5).all()
    for t in (torch.float32, torch.bfloat16, torch.float16):
        out = torch.full((rows, cols + 3), -7.0, dtype=t, device="cuda")
        assert ex.mx4_dequant(q, out[:, :cols]) == 0
        want = w[:, :cols].to(torch.float32).to(t)
        o = out[:, :cols].cpu()
        assert torch.equal(torch.isnan(o), torch.isnan(want)) and torch.equal(o.nan_to_num(7), want.nan_to_num(7)), t
        assert (out[:, cols:] == -7).all()


@pytest.mark.parametrize("dt", list(TYPES))
def test_special_blocks(ex, dt):
    x = special(TYPES[dt]).cuda()
    check(ex, x, 32, 32, 8)


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 31), (1, 32), (7, 33), (64, 64), (33, 650), (8, 2048), (2, 5003)])
def test_rows(ex, dt, rows, cols):
    print(f"mx4 {dt} {rows} x {cols}", flush=True)
    g = torch.Generator().manual_seed(rows * 1000 + cols)
    x = (torch.randn((rows, cols), generator=g) * torch.exp(2 * torch.randn((rows, 1), generator=g))).to(TYPES[dt])
    nb = (cols + 31) // 32
    check(ex, x.cuda(), cols, 16 * nb, (nb + 3) // 4 * 4)
    wide = torch.zeros((rows, cols + 5), dtype=x.dtype, device="cuda")          # a pitch and a start off every alignment
    wide[:, 3:3 + cols] = x.cuda()
    check(ex, wide[:, 3:3 + cols], cols, 16 * nb + 32, (nb + 3) // 4 * 4 + 4)


def test_stacked_weights_and_empty(ex):
    x = torch.randn(3, 5, 96, device="cuda")
    q = ex.mx4_empty(x.shape)
    assert ex.mx4_quant(x, q) == 0
    c, s = mx4ref.quant(x.reshape(15, 96).cpu())
    assert torch.equal(q.codes.reshape(15, -1).cpu(), c) and torch.equal(q.scales.reshape(15, -1)[:, :3].cpu(), s)
    assert ex.mx4_quant(torch.zeros(0, 96, device="cuda"), ex.mx4_empty((0, 96))) == 0


def test_rounded_values_round_to_themselves(ex):
    x = torch.randn(64, 512, device="cuda").half()
    q, out = ex.mx4_empty(x.shape), torch.empty_like(x)
    q2, out2 = ex.mx4_empty(x.shape), torch.empty_like(x)
    assert ex.mx4_quant(x, q) == 0 and ex.mx4_dequant(q, out) == 0
    assert ex.mx4_quant(out, q2) == 0 and ex.mx4_dequant(q2, out2) == 0
    assert torch.equal(out, out2)


def test_rows_past_32_bits_of_slots_and_bytes(ex):
    """17.3 G columns: more than one launch indexes in 32 bits, and offsets past 2^34 bytes. The last rows and the rows
    around the launches' seam, against the rule."""
    cols, rows = 4096, (1 << 31) // 512 + 1000
    x = torch.zeros((rows, cols), dtype=torch.float16, device="cuda")
    seam = (1 << 31) // 512
    at = [0, 1, seam - 2, seam - 1, seam, seam + 1, rows - 2, rows - 1]
    x[at] = torch.randn(len(at), cols, device="cuda").half()
    q = ex.mx4_empty(x.shape)
    assert ex.mx4_quant(x, q) == 0
    c, s = mx4ref.quant(x[at].cpu())
    assert torch.equal(q.codes[at].cpu(), c) and torch.equal(q.scales[at].cpu(), s)
    x.fill_(1)
    assert ex.mx4_dequant(q, x) == 0
    assert torch.equal(x[at].double().cpu(), mx4ref.dequant(c, s, cols))
    assert int(torch.count_nonzero(x[1000:2000])) == 0


def test_captured_and_on_another_stream(ex):
    x = torch.randn(40, 200, device="cuda").bfloat16()
    q, out = ex.mx4_empty(x.shape), torch.empty_like(x)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert ex.mx4_quant(x, q) == 0                             # by default on the current stream
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        assert ex.mx4_quant(x, q) == 0 and ex.mx4_dequant(q, out) == 0
    for seed in range(4):
        x.copy_(torch.randn(40, 200, generator=torch.Generator().manual_seed(seed)).bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        c, s = mx4ref.quant(x.cpu())
        assert torch.equal(out.double().cpu(), mx4ref.dequant(c, s, 200))
