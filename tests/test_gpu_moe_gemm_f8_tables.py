"""moe_gemm with F8 weights and expert_offset tables that are no routing: every row of y against the contract, which clamps the offsets to [0, T], counts one below
an earlier one as that one and leaves the rows that no run holds as zeros; on the kernel of few rows and on every tile."""
import numpy as np
import pytest

from test_gpu_moe_gemm_f8 import SIZES, XS, check, ex, path

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def tables(T, E):
    """Offsets that fall, that begin behind row 0 and end before T, that lie outside [0, T], all past it, all zero, at the ends of 32 bits."""
    up = [T * (e + 1) // (E + 2) for e in range(E + 1)]
    fall = list(up)
    fall[1], fall[2] = up[2] + 3, up[1] - 2
    low, high = -2 ** 31, 2 ** 31 - 1
    return {"within": up, "falling": fall, "reversed": up[::-1], "outside": [-5, T // 3] + [T // 3 + 900 * e for e in range(E - 1)],
            "past": [T + 6] * (E + 1), "zeros": [0] * (E + 1), "ends": [low, high] + [low] * (E - 1)}


@pytest.mark.parametrize("xt", XS)
@pytest.mark.parametrize("name", list(tables(64, 6)))
def test_few_rows(ex, xt, name):
    E, T, K, N = 6, 64, 64, 40
    assert path(ex, xt, "f32", False, T, E, N, K) == 2
    off = np.array(tables(T, E)[name], np.int64).astype(np.int32)
    check(ex, xt, "f32", False, T, 1, E, N, K, route=(np.random.default_rng(1).permutation(T).astype(np.int32), off))


@pytest.mark.parametrize("xt,yt,p", [("f16", "f32", 32), ("bf16", "f32", 64), ("f8", "f32", 32), ("f8", "f32", 64), ("f8", "f16", 32), ("f8", "bf16", 64), ("f8", "bf16", 128)])
@pytest.mark.parametrize("name", list(tables(64, 6)))
def test_tiles(ex, xt, yt, p, name):
    T, E, N, K = SIZES[p]
    assert path(ex, xt, yt, False, T, E, N, K) == p
    off = np.array(tables(T, E)[name], np.int64).astype(np.int32)
    check(ex, xt, yt, False, T, 1, E, N, K, route=(np.random.default_rng(1).permutation(T).astype(np.int32), off))
