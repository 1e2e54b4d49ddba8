"""moe_route with biases at the ends of f32, as masks are made (torch.finfo(float32).min): the sum of a group's two best leaves f32 where 64 bits hold
it, and a group of masked experts is still one that has experts. Against the definition in 64 bits, as tests/test_gpu_moe_route.py."""
import numpy as np
import pytest

from test_gpu_moe_route import check, ex

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
LOW, TOP, OUT = torch.finfo(torch.float32).min, torch.finfo(torch.float32).max, -float("inf")


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("n_tok", [5, 40])
def test_sums_below_f32(ex, score, n_tok):
    """Groups by four whose two best sum to -6.8e38, -6.6e38, -4e38 and about 1: the last two stay, in that order."""
    l = torch.randn((n_tok, 16), generator=torch.Generator().manual_seed(n_tok)).cuda()
    bias = torch.tensor([-3.4e38, -3.3e38, -2e38, 0.0]).repeat_interleave(4).cuda()
    gi, _ = check(ex, l, 8, score, bias, 4, 2, "top2")
    assert (gi[:, :4] >= 12).all() and ((gi[:, 4:] >= 8) & (gi[:, 4:] < 12)).all()
    check(ex, l, 8, score, bias, 4, 3, "top2")
    check(ex, l, 4, score, bias.flip(0), 4, 1, "top2")
    check(ex, l, 12, score, -bias, 4, 3, "top2")                     # and above it


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("n_tok", [5, 40])
def test_masked_groups_come_before_empty_ones(ex, score, n_tok):
    """Group 0 has no expert that can be chosen, groups 1 and 2 are masked by the type's lowest value."""
    l = torch.randn((n_tok, 16), generator=torch.Generator().manual_seed(n_tok))
    l[:, :4] = OUT
    bias = torch.tensor([0.0, LOW, LOW, 0.0]).repeat_interleave(4).cuda()
    gi, _ = check(ex, l.cuda(), 8, score, bias, 4, 2, "top2")
    assert (gi[:, 4:] >= 4).all() and (gi[:, 4:] < 8).all()
    check(ex, l.cuda(), 8, score, bias, 4, 3, "top2")
    check(ex, l.cuda(), 8, score, bias, 4, 2, "max")
    l[:, 12:] = OUT                                                  # nothing but masked experts
    check(ex, l.cuda(), 8, score, bias, 4, 2, "top2")


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("E,n_group", [(12, 6), (64, 64), (96, 8), (256, 32), (1024, 4)])
def test_masks_of_every_kind(ex, score, E, n_group):
    """Biases drawn from the type's ends, their halves and neighbours, infinities, NaN and ordinary ones, by expert and by whole groups."""
    g = torch.Generator().manual_seed(E)
    kinds = torch.tensor([0.0, 0.1, -0.1, LOW, LOW / 2, LOW * (1 - 2.0 ** -24), -2e38, 1e30, -1e30, OUT, float("nan"), TOP, TOP / 2, -float(OUT)])
    size = E // n_group
    for seed in range(12):
        few = kinds[torch.randperm(len(kinds), generator=g)[:2 + seed % 4]]
        b = few[torch.randint(0, len(few), (E,), generator=g)] if seed % 2 else few[torch.randint(0, len(few), (n_group,), generator=g)].repeat_interleave(size)
        b = torch.where(torch.rand(E, generator=g) < 0.2, torch.randn(E, generator=g) * 0.1, b)
        l = torch.randn((7 if seed % 3 else 30, E), generator=g)
        l[torch.rand(l.shape, generator=g) < 0.1] = OUT
        top_group = 1 + seed % (n_group - 1)
        for group in ("top2", "max"):
            check(ex, l.cuda(), min(6, top_group * size), score, b.cuda(), n_group, top_group, group, renorm=seed % 2 == 0)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_one_group_far_from_the_others(ex, score):
    """A group of one ordinary expert and masked ones (a sum of -3.4e38) beside ordinary groups, some within 2^-28 of each other: f32 tells it from them and
    leaves only those open."""
    g = torch.Generator().manual_seed(8)
    l = torch.randn((12, 64), generator=g)
    s = torch.sigmoid(l.double()) if score == "sigmoid" else torch.softmax(l.double(), 1)
    for t in range(12):
        b = 0.5 - s[t]
        b[0:3], b[20:23] = LOW, LOW
        check(ex, l[t:t + 1].cuda(), 6, score, b.float().cuda(), 16, 5, "top2")
        check(ex, l[t:t + 1].cuda(), 6, score, b.float().cuda(), 16, 5, "max")
