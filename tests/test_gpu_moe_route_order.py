"""How close choices may come before moe_route's order is open (include/exl3c4.h: scores are within 2^-51 of their values by sigmoid, 2^-48 by softmax): choices that
differ by eight times that or so are in order, in one launch with the scatter and in two, with and without groups."""
import pytest

from test_gpu_moe_route import check, ex

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("score,step", [("sigmoid", 2.0 ** -46), ("softmax", 2.0 ** -38)])
@pytest.mark.parametrize("n_tok", [4, 40])
@pytest.mark.parametrize("bias", [0.0, 0.3, -0.7])
def test_choices_next_to_each_other(ex, score, step, n_tok, bias):
    """Logits of k step, k = 0 .. 255 in any order: sigmoid's scores are 1/2 + k 2^-48, softmax's about 1/256 and 2^-46 apart, all with one bias."""
    g = torch.Generator().manual_seed(n_tok)
    l = torch.stack([torch.randperm(256, generator=g) for _ in range(n_tok)]).double().mul(step).float().cuda()
    b = torch.full((256,), bias).cuda()
    gi, _ = check(ex, l, 16, score, b)
    assert (l.cpu().gather(1, torch.from_numpy(gi).long()).diff(dim=1) < 0).all()
    check(ex, l, 16, score, b, 8, 3, "top2")
    check(ex, l, 16, score, b, 8, 3, "max")
    check(ex, l, 16, score, None, 32, 5, "top2")
