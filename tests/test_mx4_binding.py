"""Mx4, the binding's pair of planes: what a conversion is given is what the object's planes are at the call (CPU: the launch is
replaced by a record of its arguments)."""
import copy

import pytest
import torch

import exl3c4


@pytest.fixture
def calls(monkeypatch):
    got = []

    def record(device, stream, fn, *args):
        got.append(args)
        return 0
    monkeypatch.setattr(exl3c4, "_launch_on", record)
    return got


def conversions(q, calls):
    """The (codes, codes pitch, scales, scales pitch) that each conversion of q passes on."""
    v = torch.zeros(q.shape)
    del calls[:]
    assert exl3c4.mx4_quant(v, q) == 0 and exl3c4.mx4_dequant(q, v) == 0
    return [calls[0][5:9], calls[1][0:4]]


@pytest.mark.parametrize("name", ["codes", "scales", "cols", "shape", "rows", "device"])
def test_the_parts_of_an_mx4_cannot_be_replaced(name):
    """Another plane under the same object would leave its sizes, pitches and device those of the old one."""
    q = exl3c4.mx4_empty((4, 100), device="cpu")
    was = getattr(q, name)
    with pytest.raises(AttributeError):
        setattr(q, name, exl3c4.mx4_empty((4, 100), device="cpu").codes)
    with pytest.raises(AttributeError):
        delattr(q, name)
    assert getattr(q, name) is was


@pytest.mark.parametrize("wide", [0, 32])
def test_a_conversion_takes_the_planes_as_they_are_at_the_call(calls, wide):
    """Planes given other memory in place (set_, or .data): the next call writes there, not to what they had before."""
    c, s = torch.zeros(4, 64 + wide, dtype=torch.uint8)[:, :64], torch.zeros(4, 4 + wide, dtype=torch.uint8)[:, :4]
    q = exl3c4.Mx4(c, s, 100)
    old = (c.data_ptr(), 64 + wide, s.data_ptr(), 4 + wide)
    assert conversions(q, calls) == [old, old]
    other = torch.zeros(4, 64 + wide, dtype=torch.uint8), torch.zeros(4, 4 + wide, dtype=torch.uint8)
    q.codes.set_(other[0].untyped_storage(), 0, (4, 64), (64 + wide, 1))
    q.scales.data = other[1][:, :4]
    new = (other[0].data_ptr(), 64 + wide, other[1].data_ptr(), 4 + wide)
    assert new[0] != old[0] and new[2] != old[2]
    assert conversions(q, calls) == [new, new]


def test_a_deep_copy_is_of_its_own_planes(calls):
    q = exl3c4.mx4_empty((4, 100), device="cpu")
    p, shared = copy.deepcopy(q), copy.copy(q)
    assert p.shape == q.shape and p.codes.data_ptr() != q.codes.data_ptr() and shared.codes is q.codes
    assert conversions(p, calls) == [(p.codes.data_ptr(), 64, p.scales.data_ptr(), 4)] * 2
