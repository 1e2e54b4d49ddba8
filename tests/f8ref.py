"""f8ref.py -- 8-bit floats with a scale for each block of 128 columns (include/exl3c4.h), on the CPU, written from the format: what the device
tests compare with. The product in 64 bits is mx4ref.gemm's, on the values."""
import numpy as np
import torch

# the values of codes 0 .. 126 (127 is NaN), in order: the magnitudes' bits are their order
GRID = np.array([(m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)) for e in range(16) for m in range(8)][:127])
LEAST = np.float32(2.0 ** -96)


def up(n, m):
    return (n + m - 1) // m * m


def encode(v):
    """Code bytes of f32 values (finite, of magnitude up to 448 and what rounds to it): nearest, ties to the even code."""
    a = np.abs(v.astype(np.float64))
    hi = np.clip(np.searchsorted(GRID, a), 1, 126)
    lo = hi - 1
    dl, dh = a - GRID[lo], GRID[hi] - a
    c = np.where(dl < dh, lo, np.where(dh < dl, hi, np.where(lo % 2 == 0, lo, hi)))
    return (c | (np.signbit(v).astype(np.int64) << 7)).astype(np.uint8)


def decode(codes):
    """f64 values of code bytes."""
    q = codes.astype(np.int64)
    v = np.append(GRID, np.nan)[q & 127]
    return np.where(q >> 7, -v, v)


def quant(x, block):
    """(codes uint8 [mats, rows, cols up to 16], scales f32 [mats, ceil(rows / block), ceil(cols / 128)]) of x [mats, rows, cols]."""
    m, R, C = x.shape
    v = np.zeros((m, up(R, block), up(C, 128)), np.float32)
    v[:, :R, :C] = x.float().numpy()
    b = v.reshape(m, -1, block, v.shape[2] // 128, 128)
    bad = ~np.isfinite(b).all((2, 4), keepdims=True)
    b = np.where(bad, np.float32(0), b)
    top = np.maximum(np.abs(b).max((2, 4), keepdims=True), LEAST)
    scales = np.where(bad, np.float32(np.nan), top / np.float32(448))
    prod = b * (np.float32(448) / top)
    assert prod.dtype == np.float32 and scales.dtype == np.float32
    codes = np.where(bad, 0, encode(prod)).astype(np.uint8).reshape(v.shape)[:, :R, :up(C, 16)]
    return torch.from_numpy(codes.copy()), torch.from_numpy(scales[:, :, 0, :, 0].copy())


def values(codes, scales, cols, block):
    """f64 values [mats, rows, cols] of the planes (scales' blocks block x 128)."""
    v = torch.from_numpy(decode(codes.numpy()))[..., :cols]
    s = scales.double().repeat_interleave(block, 1)[:, :v.shape[1]].repeat_interleave(128, 2)[..., :cols]
    return v * s


def weights(codes, scales, halves):
    """f64 values of weights' codes [E, N, K] and scales, each expert's rows `halves` matrices one behind the other."""
    E, N, K = codes.shape
    return values(codes.reshape(E * halves, N // halves, K), scales.reshape(E * halves, -1, scales.shape[-1]), K, 128).view(E, N, K)


def peaks(codes, spread):
    """What the largest product of each eight neighbouring columns is bounded by, an operand's part of it: the largest magnitude of the eight codes,
    at least 2^-6 (where the exponents end), times the scale (spread [.., columns], f64: the scale that each code has). Columns in 8s."""
    v = torch.from_numpy(np.maximum(np.nan_to_num(np.abs(decode(codes.numpy())), nan=448.0), 2.0 ** -6)) * spread
    return v.unflatten(-1, (-1, 8)).amax(-1)


def gemm(x, w, sorted_tok, offset, T, top_k, swiglu, cut=None):
    """(y, bound) in f64: the product by the definition over the clamped runs, x and w [E, N, K] in f64, and how far the device's may be off before
    its one rounding. Sums in f32 lose at most a step, 2^-23 of sum |w x|, for each product but a block's first, half of one for each block's
    multiply-add and its scales' product, and two in all where the parts of k meet: less than K + 4. cut (peaks of x, peaks of w): products as
    codes, of which each of seven of eight may lose 2^-13 of the largest. SwiGLU: |silu'| <= 1.1 and |silu(g)| carry the sums' errors on, and silu(g) u
    itself is within 17 steps of 2^-24."""
    E, N, K = w.shape
    n_out = N // 2 if swiglu else N
    y, tol = torch.zeros(T, n_out, dtype=torch.float64), torch.zeros(T, n_out, dtype=torch.float64)
    off = np.maximum.accumulate(np.clip(np.asarray(offset, dtype=np.int64), 0, T))
    for e in range(E):
        i = torch.arange(off[e], off[e + 1])
        st = i * top_k if sorted_tok is None else torch.as_tensor(sorted_tok)[i].long()
        r = torch.div(st, top_k, rounding_mode="floor")
        ok = (st >= 0) & (r < x.shape[0])
        i, r = i[ok], r[ok]
        if len(i) == 0:
            continue
        p = x[r] @ w[e].T
        t = (K + 4) * 2.0 ** -23 * (x[r].abs() @ w[e].abs().T)
        if cut is not None:
            t = t + 7 * 2.0 ** -13 * (cut[0][r] @ cut[1][e].T)
        if swiglu:
            g, u, tg, tu = p[:, :n_out], p[:, n_out:], t[:, :n_out], t[:, n_out:]
            s = torch.nn.functional.silu(g)
            p = s * u
            t = 1.1 * tg * (u.abs() + tu) + s.abs() * tu + 17 * 2.0 ** -24 * p.abs()
        y[i], tol[i] = p, t
    return y, tol
