"""moe_route on the CPU: its refusals and its binding (nothing is launched), and the reference that the device tests use."""
import ctypes as C

import numpy as np
import pytest
import torch

import exl3c4
import routeref

P = 0x100000                                                       # an address nothing reads
SHAPE, DTYPE, ALIGN, STRIDE, INVAL, UNSUPPORTED = -1, -2, -3, -4, -12, -18


def route(**kw):
    """A well-formed routing of 20 tokens to 6 of 96 experts in 8 groups, with its scatter."""
    r = exl3c4.Route()
    d = dict(logits_type=2, score=1, group_score=1, renorm=1, top_k=6, n_group=8, top_group=3, scale=2.5, n_tok=20, n_expert=96, pitch=96, logits=P,
             bias=P, expert_ids=P, expert_w=P, sorted_tok=P, expert_offset=P, expert_count=P, row_of=P + 4096)
    d.update(kw)
    for k, v in d.items():
        setattr(r, k, v)
    return exl3c4.lib().exl3c4_moe_route(C.byref(r), None)


@pytest.mark.parametrize("change,want", [
    ({"logits_type": 3}, DTYPE), ({"logits_type": -1}, DTYPE), ({"score": 2}, INVAL), ({"score": -1}, INVAL), ({"group_score": 2}, INVAL),
    ({"renorm": 2}, INVAL), ({"scale": float("nan")}, INVAL), ({"scale": float("inf")}, INVAL),
    ({"n_tok": -1}, SHAPE), ({"n_tok": 1 << 30}, SHAPE), ({"n_expert": 0}, SHAPE), ({"n_expert": 2048, "pitch": 2048}, UNSUPPORTED),
    ({"top_k": 0}, SHAPE), ({"top_k": 65}, SHAPE), ({"top_k": 37}, SHAPE), ({"n_group": 0}, SHAPE), ({"n_group": 7}, SHAPE), ({"n_group": 96}, SHAPE),
    ({"top_group": 0}, SHAPE), ({"top_group": 9}, SHAPE),
    ({"logits": None}, INVAL), ({"expert_ids": None}, INVAL), ({"expert_w": None}, INVAL), ({"sorted_tok": None}, INVAL),
    ({"expert_offset": None}, INVAL), ({"row_of": P}, INVAL), ({"pitch": 95}, STRIDE), ({"pitch": -96}, STRIDE),
    ({"logits": P + 2}, ALIGN), ({"logits_type": 0, "logits": P + 1}, ALIGN), ({"bias": P + 2}, ALIGN), ({"expert_ids": P + 1}, ALIGN),
    ({"expert_w": P + 2}, ALIGN), ({"sorted_tok": P + 2}, ALIGN), ({"expert_offset": P + 2}, ALIGN), ({"expert_count": P + 2}, ALIGN),
    ({"row_of": P + 2}, ALIGN),
], ids=str)
def test_moe_route_refuses(change, want):
    assert route(**change) == want


def test_a_pitch_past_any_memory_is_refused():
    assert route(pitch=(1 << 36) + 1) == STRIDE and route(pitch=1 << 62) == STRIDE


def test_no_tokens_without_a_scatter_launch_nothing():
    none = dict(sorted_tok=None, expert_offset=None, expert_count=None, row_of=None)
    assert route(n_tok=0, logits=None, expert_ids=None, expert_w=None, **none) == 0
    assert exl3c4.lib().exl3c4_moe_route(None, None) == INVAL


def test_the_binding_refuses_what_does_not_fit():
    l, ids, w = torch.zeros(5, 32), torch.zeros(5, 4, dtype=torch.int32), torch.zeros(5, 4)
    r = exl3c4.make_route(l, 4, ids, w, bias=torch.zeros(32), expert_offset=torch.zeros(33, dtype=torch.int32), sorted_tok=ids.view(-1))
    assert (r.n_tok, r.n_expert, r.pitch, r.logits, r.expert_w, r.top_k) == (5, 32, 32, l.data_ptr(), w.data_ptr(), 4)
    assert exl3c4.make_route(torch.zeros(5, 40)[:, :32], 4, ids, w).pitch == 40
    for bad in (lambda: exl3c4.make_route(l[0], 4, ids, w), lambda: exl3c4.make_route(l.T, 4, ids, w),
                lambda: exl3c4.make_route(l, 4, ids.long(), w), lambda: exl3c4.make_route(l, 4, ids, w.double()),
                lambda: exl3c4.make_route(l, 4, ids[:, :3], w), lambda: exl3c4.make_route(l, 4, ids, w[:4]),
                lambda: exl3c4.make_route(l, 4, ids.T.contiguous(), w),
                lambda: exl3c4.make_route(l, 4, ids, w, bias=torch.zeros(31)), lambda: exl3c4.make_route(l, 4, ids, w, bias=torch.zeros(32).half()),
                lambda: exl3c4.make_route(l, 4, ids, w, bias=torch.zeros(64)[::2]),
                lambda: exl3c4.make_route(l, 4, ids, w, expert_offset=torch.zeros(32, dtype=torch.int32)),
                lambda: exl3c4.make_route(l, 4, ids, w, row_of=torch.zeros(19, dtype=torch.int32)),
                lambda: exl3c4.make_route(l, 4, ids, torch.zeros(5, 4, device="meta"))):
        with pytest.raises(ValueError):
            bad()


# ------------------------------------------------------------------------------------------ the reference
def test_the_reference_on_a_hand_made_row():
    l = np.array([[0.0, 2.0, 1.0, -np.inf, 3.0, np.nan, 1.0, 1.0]])
    sig = lambda v: 1 / (1 + np.exp(-v))
    ids, w = routeref.route(l, 3, "sigmoid", renorm=False, scale=2.0)
    assert ids.tolist() == [[4, 1, 2]] and np.allclose(w, 2 * sig(np.array([[3.0, 2.0, 1.0]])), rtol=1e-15)
    # groups of two: 0+2, 1, 3, 1+1 in logits; by the two best scores (1, 1) is first, then (0, 2)
    ids, _ = routeref.route(l, 2, "sigmoid", n_group=4, top_group=1, group="top2")
    assert ids.tolist() == [[6, 7]]
    ids, _ = routeref.route(l, 2, "sigmoid", n_group=4, top_group=1, group="max")
    assert ids.tolist() == [[4, -1]]
    bias = np.array([10.0, -np.inf, 0, 50, 0, 50, 0, 0.001])
    ids, w = routeref.route(l, 4, "softmax", bias=bias)
    p = np.exp([0.0, 2.0, 1.0, 3.0, 1.0, 1.0]) / np.exp([0.0, 2.0, 1.0, 3.0, 1.0, 1.0]).sum()
    assert ids.tolist() == [[0, 4, 7, 2]] and np.allclose(w, p[[0, 3, 5, 2]] / p[[0, 3, 5, 2]].sum(), rtol=1e-15)
    ids, w = routeref.route(np.full((1, 4), -np.inf), 2, "softmax")
    assert ids.tolist() == [[-1, -1]] and w.tolist() == [[0, 0]]
    st, off, cnt, row = routeref.scatter(np.array([[2, -1], [0, 2]], np.int32), 3)
    assert st.tolist() == [2, 0, 3, -1] and off.tolist() == [0, 1, 1, 3] and cnt.tolist() == [1, 0, 2] and row.tolist() == [1, -1, 0, 2]
