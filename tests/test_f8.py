"""F8 (8-bit floats in blocks of 128) on the CPU: the refusals of f8_quant, f8_dequant and of moe_gemm with F8 operands, the binding, and the
reference that the device tests use (nothing is launched, every refusal is decided on the host)."""
import copy
import ctypes as C

import numpy as np
import pytest
import torch

import exl3c4
import f8ref

P = 0x100000                                                       # an address nothing reads
SHAPE, DTYPE, ALIGN, STRIDE, INVAL = -1, -2, -3, -4, -12


# ------------------------------------------------------------------------------------------ the conversions
def conv(dt=0, x=P, pitch=300, xs=300 * 200, **kw):
    """Both conversions of 3 matrices of 200 x 300 in blocks of 128; they refuse the same."""
    d = dict(n=3, rows=200, cols=300, block=128, codes=P, codes_pitch=304, codes_stride=304 * 200, scales=P, scales_pitch=3, scales_stride=6)
    d.update(kw)
    q = exl3c4.F8Planes(**d)
    L = exl3c4.lib()
    a = L.exl3c4_f8_quant(x, dt, pitch, xs, C.byref(q), None)
    assert a == L.exl3c4_f8_dequant(C.byref(q), x, dt, pitch, xs, None)
    return a


@pytest.mark.parametrize("change,want", [
    ({"dt": 3}, DTYPE), ({"dt": -1}, DTYPE), ({"dt": 4}, DTYPE), ({"block": 0}, INVAL), ({"block": 64}, INVAL),
    ({"n": -1}, SHAPE), ({"rows": -1}, SHAPE), ({"cols": 0}, SHAPE), ({"rows": 1 << 40}, SHAPE), ({"n": 1 << 24, "rows": 1 << 24}, SHAPE),
    ({"n": 1 << 20, "rows": 1 << 10, "cols": 1 << 14, "pitch": 1 << 14, "xs": 1 << 40}, SHAPE),
    ({"x": None}, INVAL), ({"codes": None}, INVAL), ({"scales": None}, INVAL),
    ({"pitch": 299}, STRIDE), ({"codes_pitch": 288}, STRIDE), ({"scales_pitch": 2}, STRIDE), ({"pitch": -300}, STRIDE), ({"pitch": 1 << 50}, STRIDE),
    ({"xs": 300 * 200 - 1}, STRIDE), ({"codes_stride": 304 * 199}, STRIDE), ({"scales_stride": 5}, STRIDE), ({"xs": 0}, STRIDE), ({"xs": 1 << 62}, STRIDE),
    ({"x": P + 1}, ALIGN), ({"dt": 2, "x": P + 2}, ALIGN), ({"codes": P + 8}, ALIGN), ({"codes_pitch": 312, "codes_stride": 1 << 20}, ALIGN),
    ({"codes_stride": (1 << 20) + 8}, ALIGN), ({"scales": P + 2}, ALIGN),
    ({"rows": 0, "x": None, "codes": None, "scales": None}, 0), ({"n": 0, "x": None, "codes": None, "scales": None}, 0),
], ids=str)
def test_conversions_refuse(change, want):
    assert conv(**change) == want


@pytest.mark.parametrize("change", [{"pitch": 1 << 35, "xs": 1 << 40}, {"codes_pitch": 1 << 35, "codes_stride": 1 << 40},
                                    {"scales_pitch": 1 << 40, "scales_stride": 1 << 41}, {"xs": -1}, {"codes_stride": -(1 << 62)}], ids=str)
def test_matrices_that_overlap_are_refused_whatever_64_bits_hold(change):
    """2^29 rows, 2^22 rows of blocks: (rows - 1) * pitch is 2^64 less the pitch (2^62 less it for the scales)."""
    d = dict(n=2, rows=1 << 29, cols=100, pitch=100, xs=1 << 60, codes_pitch=112, codes_stride=1 << 60, scales_pitch=1, scales_stride=1 << 60)
    assert conv(**d | change) == STRIDE


def test_a_conversion_without_planes_is_refused():
    L = exl3c4.lib()
    assert L.exl3c4_f8_quant(P, 0, 300, 0, None, None) == INVAL and L.exl3c4_f8_dequant(None, P, 0, 300, 0, None) == INVAL


# ------------------------------------------------------------------------------------------ the product
def gemm(**kw):
    """A well-formed product of 4 experts: F8 x [8, 272], w [4, 300, 272] (3 x 3 blocks an expert), 16 sorted rows."""
    g = exl3c4.Gemm()
    d = dict(x_type=4, w_type=4, y_type=1, act=0, N=300, K=272, n_expert=4, top_k=2, T=16, x=P, x_rows=8, x_pitch=272, x_scales=P, xs_pitch=12,
             w=P, w_pitch=272, w_stride=300 * 272, w_scales=P, ws_pitch=12, ws_stride=36, sorted_tok=P, expert_offset=P, y=P, y_pitch=300)
    d.update(kw)
    for k, v in d.items():
        setattr(g, k, v)
    return g


def rc(g):
    return exl3c4.lib().exl3c4_moe_gemm(C.byref(g), None)


@pytest.mark.parametrize("change,want", [
    ({"x_scales": None}, INVAL), ({"w_scales": None}, INVAL), ({"w_stride": 0}, INVAL), ({"ws_stride": 0}, INVAL),
    ({"x_type": 2}, DTYPE), ({"x_type": 3}, DTYPE), ({"w_type": 1}, DTYPE), ({"y_type": 4}, DTYPE), ({"w_type": 3}, DTYPE),
    ({"K": 264, "x_pitch": 288}, SHAPE), ({"act": 1, "N": 301}, SHAPE), ({"x_rows": 0}, SHAPE),
    ({"x_pitch": 256}, STRIDE), ({"xs_pitch": 8}, STRIDE), ({"ws_pitch": 8}, STRIDE), ({"w_pitch": 256}, STRIDE), ({"ws_stride": 32}, STRIDE),
    ({"w_stride": 300 * 272 - 16}, STRIDE), ({"x_type": 0, "x_pitch": 264}, STRIDE), ({"w_pitch": (1 << 27) + 16, "w_stride": 1 << 40}, STRIDE),
    # with SwiGLU gate and up have two rows of blocks each
    ({"act": 1, "y_pitch": 150, "ws_stride": 44}, STRIDE), ({"act": 1, "y_pitch": 149}, STRIDE),
    ({"x_pitch": 280}, ALIGN), ({"x": P + 8}, ALIGN), ({"w": P + 8}, ALIGN), ({"x_scales": P + 2}, ALIGN), ({"w_scales": P + 1}, ALIGN),
    ({"xs_pitch": 14}, ALIGN), ({"ws_pitch": 14, "ws_stride": 48}, ALIGN), ({"ws_stride": 38}, ALIGN),
    ({"w_stride": 0, "ws_stride": 0, "w_scales": P + 4}, ALIGN),
], ids=str)
def test_moe_gemm_refuses(change, want):
    assert rc(gemm(**change)) == want


def test_no_rows_launch_nothing():
    assert rc(gemm(T=0, x=None, w=None, y=None)) == 0


@pytest.mark.parametrize("change", [{"T": 1 << 20, "x_rows": 1 << 20, "n_expert": 1 << 20}, {"T": 1 << 30, "x_rows": 1 << 30, "n_expert": 1}],
                         ids=["rows", "tiles"])
def test_more_threads_than_a_launch_holds_are_refused(change):
    n = 1 << 14 if change["n_expert"] > 1 else 1 << 16
    assert rc(gemm(N=n, y_pitch=n, w_stride=n * 272, ws_stride=n // 128 * 12, **change)) == SHAPE


# ------------------------------------------------------------------------------------------ the binding
@pytest.fixture
def calls(monkeypatch):
    got = []

    def record(device, stream, fn, *args):
        got.append([a._obj if hasattr(a, "_obj") else a for a in args])
        return 0
    monkeypatch.setattr(exl3c4, "_launch_on", record)
    return got


@pytest.mark.parametrize("name", ["codes", "scales", "cols", "block", "shape", "rows", "mats", "device"])
def test_the_parts_of_an_f8_cannot_be_replaced(name):
    q = exl3c4.f8_empty((2, 100, 300), 128, device="cpu")
    was = getattr(q, name)
    with pytest.raises(AttributeError):
        setattr(q, name, 1)
    with pytest.raises(AttributeError):
        delattr(q, name)
    assert getattr(q, name) is was


def test_a_conversion_takes_the_planes_as_they_are_at_the_call(calls):
    q = exl3c4.f8_empty((2, 100, 300), 128, device="cpu")
    x = torch.zeros(2, 100, 300)
    assert exl3c4.f8_quant(x, q) == 0
    assert calls[0][:4] == [x.data_ptr(), exl3c4.F32, 300, 30000] and calls[0][4].codes == q.codes.data_ptr()
    other = torch.zeros(2, 100, 304, dtype=torch.uint8)
    q.codes.set_(other.untyped_storage(), 0, (2, 100, 304), (30400, 304, 1))
    assert exl3c4.f8_dequant(q, x.half()) == 0
    p = calls[1][0]
    assert (p.codes, p.codes_pitch, p.codes_stride, p.scales, p.scales_pitch, p.scales_stride) == (
        other.data_ptr(), 304, 30400, q.scales.data_ptr(), 3, 3)
    c = copy.deepcopy(q)
    assert c.codes.data_ptr() != q.codes.data_ptr() and c.block == 128 and copy.copy(q).codes is q.codes


def test_pitches_and_strides_of_views(calls):
    """Rows of a wider buffer, matrices of a larger one, two leading dimensions that step as one."""
    big = torch.zeros(2, 3, 128, 512)
    q = exl3c4.F8(torch.zeros(2, 3, 130, 320, dtype=torch.uint8)[:, :, :128], torch.zeros(2, 3, 2, 3)[:, :, :1], 300, 128)
    assert exl3c4.f8_quant(big[..., :300], q) == 0
    p = calls[0][4]
    assert calls[0][2:4] == [512, 128 * 512] and (p.n, p.rows, p.codes_pitch, p.codes_stride, p.scales_pitch, p.scales_stride) == (6, 128, 320, 130 * 320, 3, 6)
    with pytest.raises(ValueError):
        exl3c4.f8_quant(big[:, :2, :, :300], exl3c4.f8_empty((2, 2, 128, 300), 128, device="cpu"))
    with pytest.raises(ValueError):
        exl3c4.f8_quant(big.transpose(2, 3), exl3c4.f8_empty((2, 3, 512, 128), 128, device="cpu"))


def test_the_binding_refuses_what_does_not_fit():
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)
    for bad in (lambda: exl3c4.F8(u8(4, 304), torch.zeros(4, 3), 300, 2),
                lambda: exl3c4.F8(u8(4, 300), torch.zeros(4, 3), 300, 1),
                lambda: exl3c4.F8(u8(4, 304), torch.zeros(3, 3), 300, 1),
                lambda: exl3c4.F8(u8(4, 304), torch.zeros(4, 2), 300, 1),
                lambda: exl3c4.F8(u8(4, 304), torch.zeros(4, 3).half(), 300, 1),
                lambda: exl3c4.F8(u8(4, 304), torch.zeros(4, 3, dtype=torch.int32), 300, 1),
                lambda: exl3c4.F8(u8(2, 4, 304), torch.zeros(4, 3), 300, 1),
                lambda: exl3c4.F8(u8(304), torch.zeros(3), 300, 1),
                lambda: exl3c4.F8(torch.zeros(4, 304), torch.zeros(4, 3), 300, 1),
                lambda: exl3c4.f8_quant(torch.zeros(4, 299), exl3c4.f8_empty((4, 300), 1, device="cpu")),
                # gate and up quantised as one matrix, or read back as one
                lambda: exl3c4.f8_quant(torch.zeros(1, 384, 128), exl3c4.F8(u8(1, 384, 128), torch.zeros(1, 4, 1), 128, 128))):
        with pytest.raises(ValueError):
            bad()
    i, y = torch.zeros(4, dtype=torch.int32), torch.zeros(4, 384)
    x, w = exl3c4.f8_empty((4, 256), 1, device="cpu"), exl3c4.f8_empty((3, 384, 256), 128, device="cpu")
    h = exl3c4.F8(w.codes, torch.zeros(3, 4, 2), 256, 128)
    g = exl3c4.make_gemm(x, w, i, i, y)
    assert (g.xs_pitch, g.ws_pitch, g.ws_stride, g.w_stride) == (8, 8, 24, 384 * 256)
    assert exl3c4.make_gemm(x, h, i, i, y[:, :192], act=exl3c4.ACT_SWIGLU).ws_stride == 32
    one = exl3c4.make_gemm(x, exl3c4.f8_empty((1, 384, 256), 128, device="cpu"), None, i, y)
    assert one.ws_stride == 24 and one.w_stride == 384 * 256
    for bad in (lambda: exl3c4.make_gemm(exl3c4.f8_empty((4, 256), 128, device="cpu"), w, i, i, y),
                lambda: exl3c4.make_gemm(x, exl3c4.f8_empty((3, 384, 256), 1, device="cpu"), i, i, y),
                lambda: exl3c4.make_gemm(x, h, i, i, y),
                lambda: exl3c4.make_gemm(x, w, i, i, y[:, :192], act=exl3c4.ACT_SWIGLU)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("t", [torch.int8, torch.float8_e5m2, torch.float8_e4m3fnuz, torch.bool])
def test_codes_of_another_type_are_refused(t):
    with pytest.raises(ValueError):
        exl3c4.F8(torch.zeros(4, 304, dtype=torch.uint8).view(t), torch.zeros(4, 3), 300, 1)
    exl3c4.F8(torch.zeros(4, 304, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros(4, 3), 300, 1)


# ------------------------------------------------------------------------------------------ the reference
def test_the_reference_rounds_to_the_nearest_code():
    """Every code's value comes back as itself, and every tie between neighbours goes to the even code; torch's own e4m3 agrees."""
    v = f8ref.GRID.astype(np.float32)
    assert (f8ref.encode(v) == np.arange(127)).all() and (f8ref.encode(-v)[1:] == np.arange(129, 255)).all()
    ties = ((f8ref.GRID[1:] + f8ref.GRID[:-1]) / 2).astype(np.float32)
    lo = np.arange(126)
    assert (f8ref.encode(ties) == np.where(lo % 2 == 0, lo, lo + 1)).all()
    x = torch.randn(100000, generator=torch.Generator().manual_seed(1)) * 30
    assert (f8ref.encode(x.numpy()) == x.to(torch.float8_e4m3fn).view(torch.uint8).numpy()).all()
    assert (f8ref.decode(np.arange(127, dtype=np.uint8)) == torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()).all()


def test_the_reference_by_blocks():
    x = torch.zeros(1, 130, 130)
    x[0, 0, 0], x[0, 129, 0], x[0, 5, 129], x[0, 128, 129] = 896.0, 3.0, float("inf"), 1e-36
    c, s = f8ref.quant(x, 128)
    assert c.shape == (1, 130, 144) and s.shape == (1, 2, 2) and s[0, 0, 0] == 2 and torch.isnan(s[0, 0, 1])
    assert c[0, 0, 0] == 126 and c[0, 129, 0] == 126 and (c[0, :, 128:] == 0).sum() == 130 * 16
    assert f8ref.values(c, s, 130, 128)[0, 0, 0] == 896
    c, s = f8ref.quant(x, 1)
    assert s.shape == (1, 130, 2) and s[0, 1, 0] == np.float32(2.0 ** -96) / np.float32(448) and torch.isnan(s[0, 5, 1])
