"""gemmpath.py -- which kernel a moe_gemm takes (the library's own rule), sizes that take each, and experts that share weights: what the
device tests of the product use to run every kernel on purpose."""
import ctypes as C

import torch

import exl3c4
import mx4ref

CODE = {"f16": exl3c4.F16, "bf16": exl3c4.BF16, "mx4": exl3c4.MX4}
# (T, experts, columns of y): few rows an expert by 2 and by 4 strips of weight rows, tiles of 32 to 256 rows; the last column tile is not whole
SIZES = {2: (40, 3, 200), 4: (40, 40, 1650), 32: (150, 2, 1450), 64: (250, 4, 3700), 128: (260, 2, 5510), 256: (3000, 2, 4400)}


def path(pair, swiglu, T, E, n_out, K):
    f = exl3c4.lib().exl3c4_dev_gemm_path
    f.restype, f.argtypes = C.c_int, [C.c_int32] * 3 + [C.c_int64] * 4
    return f(CODE[pair[0]], CODE[pair[1]], exl3c4.ACT_SWIGLU if swiglu else exl3c4.ACT_NONE, T, E, 2 * n_out if swiglu else n_out, K)


def paths(pair):
    """The paths that a pair of types has."""
    return [2, 4, 32, 64] if pair[1] == "mx4" and pair[0] != "mx4" else [2, 4, 32, 64, 128, 256]


class Shared:
    """Experts e = 0 .. E - 1 whose weights are w64[e % n] (as mx4ref.gemm takes them)."""
    def __init__(self, w64, E):
        self.w64, self.shape = w64, (E,) + tuple(w64.shape[1:])

    def __getitem__(self, e):
        return self.w64[e % self.w64.shape[0]]


def share(gm, wd, E):
    """gm, made for wd's n experts, over E: expert e's weights are wd's e % n, by pointer tables."""
    def table(t):
        return torch.tensor([t[e % t.shape[0]].data_ptr() for e in range(E)], dtype=torch.int64, device=t.device)
    gm.n_expert, gm.w_stride = E, 0
    if isinstance(wd, exl3c4.Mx4):
        tw, ts = table(wd.codes), table(wd.scales)
        gm.w, gm.w_scales, gm.ws_stride, gm.shared = tw.data_ptr(), ts.data_ptr(), 0, (wd, tw, ts)
    else:
        tw = table(wd)
        gm.w, gm.shared = tw.data_ptr(), (wd, tw)
    return gm


def mx4_weights(g, n, N, K, scale):
    """Random codes of n experts with the scale bytes `scale` ([n, N, K / 32] or one that spreads to it): (operand, values in f64)."""
    codes = torch.randint(0, 256, (n, N, K // 2), dtype=torch.uint8, generator=g)
    s = torch.full((n, N, (K // 32 + 3) // 4 * 4), 255, dtype=torch.uint8)
    s[..., :K // 32] = scale
    return exl3c4.Mx4(codes.cuda(), s.cuda(), K), mx4ref.dequant(codes, s, K)
