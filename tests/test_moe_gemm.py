"""The refusals of mx4_quant, mx4_dequant and moe_gemm, and the 64-bit reference that the device tests use (CPU: nothing is
launched, every refusal is decided on the host)."""
import ctypes as C

import pytest
import torch

import exl3c4
import mx4ref

P = 0x100000                                                       # an address nothing reads
SHAPE, DTYPE, ALIGN, STRIDE, INVAL = -1, -2, -3, -4, -12


def gemm(**kw):
    """A well-formed product of 4 experts: bf16 x [8, 64], w [4, 48, 64], 16 sorted rows."""
    g = exl3c4.Gemm()
    d = dict(x_type=1, w_type=1, y_type=1, act=0, N=48, K=64, n_expert=4, top_k=2, T=16, x=P, x_rows=8, x_pitch=64, w=P,
             w_pitch=64, w_stride=48 * 64 * 2, sorted_tok=P, expert_offset=P, y=P, y_pitch=48)
    d.update(kw)
    for k, v in d.items():
        setattr(g, k, v)
    return g


def mx4(**kw):
    d = dict(x_type=3, w_type=3, x_scales=P, xs_pitch=4, x_pitch=32, w_scales=P, ws_pitch=4, w_pitch=32, w_stride=48 * 32,
             ws_stride=48 * 4)
    d.update(kw)
    return gemm(**d)


def rc(g):
    return exl3c4.lib().exl3c4_moe_gemm(C.byref(g), None)


@pytest.mark.parametrize("change,want", [
    ({"act": 2}, INVAL), ({"act": -1}, INVAL), ({"x": None}, INVAL), ({"w": None}, INVAL), ({"y": None}, INVAL),
    ({"expert_offset": None}, INVAL),
    ({"x_type": 0}, DTYPE), ({"x_type": 2, "w_type": 2}, DTYPE), ({"x_type": 3}, DTYPE), ({"y_type": 3}, DTYPE), ({"y_type": 7}, DTYPE),
    ({"w_type": 9}, DTYPE),
    ({"N": 0}, SHAPE), ({"K": 0}, SHAPE), ({"K": 60}, SHAPE), ({"T": -1}, SHAPE), ({"n_expert": 0}, SHAPE), ({"top_k": 0}, SHAPE),
    ({"x_rows": 0}, SHAPE), ({"x_rows": 15, "sorted_tok": None}, SHAPE), ({"T": 1 << 31}, SHAPE), ({"K": 1 << 32}, SHAPE),
    ({"act": 1, "N": 47, "w_stride": 1 << 20}, SHAPE),
    ({"x_pitch": 56}, STRIDE), ({"w_pitch": 56}, STRIDE), ({"w_stride": 47 * 128}, STRIDE), ({"w_stride": -16}, STRIDE), ({"y_pitch": 47}, STRIDE),
    ({"w_pitch": (1 << 26) + 8, "w_stride": 1 << 34}, STRIDE), ({"x_pitch": -64}, STRIDE), ({"x_pitch": 1 << 62}, STRIDE),
    ({"x": P + 8}, ALIGN), ({"w": P + 2}, ALIGN), ({"x_pitch": 68}, ALIGN), ({"w_pitch": 68, "w_stride": 1 << 20}, ALIGN),
    ({"w_stride": 48 * 128 + 8}, ALIGN), ({"y": P + 1}, ALIGN), ({"y_type": 2, "y": P + 2}, ALIGN), ({"sorted_tok": P + 2}, ALIGN),
    ({"expert_offset": P + 1}, ALIGN),
], ids=str)
def test_moe_gemm_refuses(change, want):
    assert rc(gemm(**change)) == want


@pytest.mark.parametrize("change,want", [
    ({"x_scales": None}, INVAL), ({"w_scales": None}, INVAL), ({"w_stride": 0}, INVAL), ({"ws_stride": 0}, INVAL),
    ({"K": 48}, SHAPE), ({"x_type": 2}, DTYPE), ({"x_type": 1, "x_pitch": 48}, STRIDE),
    ({"x_pitch": 16}, STRIDE), ({"K": 160, "x_pitch": 80, "w_pitch": 80, "w_stride": 1 << 20, "ws_stride": 1 << 10}, STRIDE),
    ({"ws_stride": 47 * 4}, STRIDE), ({"xs_pitch": 6}, ALIGN), ({"ws_pitch": 6, "ws_stride": 1 << 10}, ALIGN),
    ({"x_scales": P + 2}, ALIGN), ({"w_scales": P + 1}, ALIGN), ({"x_pitch": 40}, ALIGN), ({"ws_stride": 48 * 4 + 2}, ALIGN),
    ({"w_stride": 0, "ws_stride": 0, "w_scales": P + 4}, ALIGN),
], ids=str)
def test_moe_gemm_refuses_mx4(change, want):
    assert rc(mx4(**change)) == want


def test_a_pointer_table_needs_a_pointers_alignment():
    """A row of a layers x experts table may start at any pointer: what is refused is what comes behind (here the pitch), not it."""
    far = {"w_stride": 0, "w": P + 8, "w_pitch": (1 << 26) + 8}
    assert rc(gemm(**far)) == STRIDE and rc(gemm(**dict(far, w=P + 4))) == ALIGN
    far = {"w_stride": 0, "ws_stride": 0, "w": P + 8, "w_scales": P + 8, "w_pitch": (1 << 27) + 16}
    assert rc(mx4(**far)) == STRIDE and rc(mx4(**dict(far, w=P + 4))) == ALIGN


@pytest.mark.parametrize("change", [{"T": 1 << 20, "x_rows": 1 << 20, "n_expert": 1 << 20}, {"T": 1 << 30, "x_rows": 1 << 30, "n_expert": 1}],
                         ids=["rows", "tiles"])
def test_more_threads_than_a_launch_holds_are_refused(change):
    """17.8 M workgroups of 256 threads and 2^29 of 512: past 2^32 threads, before anything is launched."""
    n = 1024 if change["n_expert"] > 1 else 1 << 15
    assert rc(gemm(N=n, y_pitch=n, w_stride=n * 128, **change)) == SHAPE


def test_no_rows_launch_nothing():
    assert rc(gemm(T=0, x=None, w=None, y=None)) == 0
    assert rc(mx4(T=0, x=None, w=None, y=None)) == 0
    assert exl3c4.lib().exl3c4_moe_gemm(None, None) == INVAL


def conv(rows=4, cols=100, pitch=100, dt=0, x=P, codes=P, cp=64, scales=P, sp=4):
    L = exl3c4.lib()
    a = L.exl3c4_mx4_quant(x, dt, rows, cols, pitch, codes, cp, scales, sp, None)
    b = L.exl3c4_mx4_dequant(codes, cp, scales, sp, rows, cols, x, dt, pitch, None)
    assert a == b
    return a


@pytest.mark.parametrize("change,want", [
    ({"dt": 3}, DTYPE), ({"dt": -1}, DTYPE), ({"rows": -1}, SHAPE), ({"cols": 0}, SHAPE), ({"rows": 1 << 40}, SHAPE),
    ({"rows": (1 << 31) - (1 << 17), "cols": 4096, "pitch": 4096, "cp": 2048, "sp": 128}, SHAPE),
    ({"x": None}, INVAL), ({"codes": None}, INVAL), ({"scales": None}, INVAL),
    ({"pitch": 99}, STRIDE), ({"cp": 48}, STRIDE), ({"cols": 129, "pitch": 129, "cp": 80, "sp": 4}, STRIDE), ({"pitch": -100}, STRIDE),
    ({"x": P + 1}, ALIGN), ({"dt": 2, "x": P + 2}, ALIGN), ({"codes": P + 8}, ALIGN), ({"cp": 72}, ALIGN), ({"scales": P + 2}, ALIGN),
    ({"sp": 6}, ALIGN), ({"rows": 0, "x": None, "codes": None, "scales": None}, 0),
], ids=str)
def test_conversions_refuse(change, want):
    assert conv(**change) == want


def test_the_binding_refuses_what_does_not_fit():
    q = exl3c4.mx4_empty((4, 100), device="cpu")
    assert q.codes.shape == (4, 64) and q.scales.shape == (4, 4)
    with pytest.raises(ValueError):
        exl3c4.mx4_quant(torch.zeros(4, 96), q)
    with pytest.raises(ValueError):
        exl3c4.mx4_quant(torch.zeros(5, 100), q)
    with pytest.raises(ValueError):
        exl3c4.mx4_quant(torch.zeros(100, 4).T, q)
    i = torch.zeros(4, dtype=torch.int32)
    x, w, y = torch.zeros(4, 64).half(), torch.zeros(3, 8, 64).half(), torch.zeros(4, 8)
    exl3c4.make_gemm(x, w, i, i, y)
    for bad in (lambda: exl3c4.make_gemm(x, w, i, i, torch.zeros(4, 9)),
                lambda: exl3c4.make_gemm(x[:, :32], w, i, i, y),
                lambda: exl3c4.make_gemm(x, w, i[:3], i, y),
                lambda: exl3c4.make_gemm(x, w, i, i[:3], y),
                lambda: exl3c4.make_gemm(x, w, i.long(), i, y),
                lambda: exl3c4.make_gemm(x, w, i.float(), i, y),
                lambda: exl3c4.make_gemm(x, w[:1].expand(3, 8, 64), i, i, y),          # a stride of 0 is a pointer array
                lambda: exl3c4.make_gemm(x, w, i, i, torch.zeros(8, 4).T)):
        with pytest.raises(ValueError):
            bad()


def test_the_binding_refuses_operands_of_another_rank():
    """x of a batch and a sequence, weights of one expert as they are, y by head: their strides are not a row's, and the call would
    have read every other sequence's first token."""
    i = torch.zeros(4, dtype=torch.int32)
    x, w, y = torch.zeros(4, 64).half(), torch.zeros(3, 8, 64).half(), torch.zeros(4, 8)
    m = exl3c4.mx4_empty((2, 2, 64), device="cpu")
    for bad in (lambda: exl3c4.make_gemm(x.reshape(2, 2, 64), w, i, i, y),
                lambda: exl3c4.make_gemm(x, w[0], i, i, torch.zeros(4, 64)),
                lambda: exl3c4.make_gemm(x, w, i, i, torch.zeros(4, 8, 2)),
                lambda: exl3c4.make_gemm(m, exl3c4.mx4_empty((3, 8, 64), device="cpu"), i, i, y)):
        with pytest.raises(ValueError):
            bad()


def test_the_reference_rounds_to_the_nearest_code():
    """mx4ref.quant on every tie and neighbour of a tie, against the format's list."""
    x = torch.zeros(1, 32)
    vals = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.9, 0.2500001, 0.7499999, -0.25, -0.75]
    x[0, :len(vals)] = torch.tensor(vals)
    codes, scales = mx4ref.quant(x)
    assert scales[0, 0] == 127
    v = mx4ref.dequant(codes, scales, 32)[0, :len(vals)].tolist()
    assert v == [0, 1, 1, 2, 2, 4, 4, 6, 6, 0.5, 0.5, 0, -1]
    big = torch.full((1, 32), 2.0 ** 100)
    assert mx4ref.quant(big)[1][0, 0] == 225 and mx4ref.dequant(*mx4ref.quant(big), 32).eq(2.0 ** 100).all()
    assert mx4ref.quant(torch.zeros(1, 5))[1][0, 0] == 0
    assert mx4ref.quant(torch.tensor([[float("inf"), 1.0]]))[1][0, 0] == 255
