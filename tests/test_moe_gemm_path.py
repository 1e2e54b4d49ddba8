"""The rule by which moe_gemm takes its kernels, as the library states it (CPU): the sizes that the device tests use do take the
kernels that they are named for, and each kernel of each pair of types has such a size."""
import pytest

import exl3c4  # noqa: F401
import gemmpath

PAIRS = [("f16", "f16"), ("bf16", "bf16"), ("f16", "mx4"), ("bf16", "mx4"), ("mx4", "mx4")]


@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
@pytest.mark.parametrize("swiglu", [False, True])
def test_the_sizes_of_the_tests_take_their_kernels(pair, swiglu):
    for p in gemmpath.paths(pair):
        T, E, n = gemmpath.SIZES[p]
        K = 2080 if p == 256 else 416
        assert gemmpath.path(pair, swiglu, T, E, n, K) == p


def test_the_rule():
    f = gemmpath.path
    one = ("bf16", "bf16")
    assert f(one, True, 10, 512, 512, 2048) == 2 and f(one, True, 320, 512, 512, 2048) == 4         # one token, 32 tokens of top-10
    assert f(one, True, 6130, 512, 640, 2560) == 64 and f(one, True, 16384, 8, 1408, 2048) == 256
    assert f(one, False, 77, 1, 512, 2048) == 2
    mixed, both = ("f16", "mx4"), ("mx4", "mx4")
    assert f(mixed, True, 640, 512, 512, 2048) == 4 and f(mixed, True, 40960, 512, 512, 2048) == 64
    assert f(both, True, 20480, 512, 512, 2048) == 64 and f(both, False, 16384, 8, 2048, 1408) == 128
    assert f(both, True, 16384, 8, 1408, 2048) == 256
