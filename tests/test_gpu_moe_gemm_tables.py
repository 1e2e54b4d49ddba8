"""moe_gemm under offset tables that are no routing: an offset below an earlier one counts as that one, so the runs are disjoint,
every row of y is written once -- by its run's expert, or as zeros -- and every launch gives the same bits."""
import numpy as np
import pytest

import gemmpath
import mx4ref
from test_gpu_moe_gemm import PAIRS, ex, operand  # noqa: F401 (ex is a fixture)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def tables(E, T, rng):
    """Offset tables of E experts: overlapping, descending, repeated, negative and too large, and wholly random ones."""
    up = np.sort(rng.integers(0, T + 1, E + 1))
    whole = np.where(np.arange(E + 1) % 2 == 0, 0, T)               # every other run all of the rows
    late = up.copy()
    late[E // 2:] = up[E // 2:] // 3
    yield from (up[::-1], whole, late, rng.integers(-T, 2 * T, E + 1), np.full(E + 1, T + 9), np.zeros(E + 1),
                rng.integers(-2 ** 31, 2 ** 31 - 1, E + 1))
    yield np.where(rng.random(E + 1) < 0.05, rng.integers(-5, T + 5, E + 1), up)


def disjoint(off, T):
    return np.maximum.accumulate(np.clip(np.asarray(off, np.int64), 0, T))


@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
@pytest.mark.parametrize("E,T,N,tile", [(6, 64, 40, False), (6, 400, 1450, True), (1500, 90, 36, False), (520, 4200, 160, True)], ids=str)
def test_every_row_is_written_once(ex, pair, E, T, N, tile):  # noqa: F811
    """In few rows and in tiles, with more experts than one step of the search holds (512) as well."""
    assert (gemmpath.path(pair, False, T, E, N, 64) > 4) == tile
    rng = np.random.default_rng(E + T)
    g = torch.Generator().manual_seed(T)
    K = 64
    xd, xv = operand(ex, torch.randn((T, K), generator=g), pair[0])
    wd, wv = operand(ex, torch.randn((E, N, K), generator=g) / 8, pair[1])
    for n, off in enumerate(tables(E, T, rng)):
        print(f"moe_gemm {pair} {E} experts, {T} rows, table {n}", flush=True)
        od = torch.from_numpy(np.ascontiguousarray(off, np.int32)).cuda()
        got = []
        for _ in range(2):
            y = torch.full((T + 3, N), float("nan"), device="cuda")
            assert ex.moe_gemm(ex.make_gemm(xd, wd, None, od, y[:T])) == 0
            got.append(y.cpu())
        want, tol = mx4ref.gemm(xv, wv, None, disjoint(off, T), T, 1, False)
        assert mx4ref.close(got[0][:T], want, tol)
        assert torch.equal(got[0][:T], got[1][:T]) and torch.isnan(got[0][T:]).all()
