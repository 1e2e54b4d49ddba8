"""mx4ref.py -- microscaled 4-bit floats (include/exl3c4.h) and the grouped product in 64 bits on the CPU, written from the
format: what the device tests compare with."""
import torch

GRID = torch.tensor([0.0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
EPS = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}      # half a step, relative
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}  # half the smallest step


def quant(x):
    """codes uint8 [rows, 16 nb] and scale bytes uint8 [rows, nb] of x [rows, cols]."""
    rows, cols = x.shape
    b = torch.nn.functional.pad(x.double(), (0, -cols % 32)).view(rows, -1, 32)
    bad = ~torch.isfinite(b).all(-1)
    b = torch.where(bad[..., None], 0.0, b)
    top = b.abs().amax(-1)
    e = torch.where(top > 0, torch.frexp(top).exponent - 3, -127).clamp(min=-127)
    a = torch.ldexp(b.abs(), -e[..., None].double())
    d = (a[..., None] - GRID).abs()                                # nearest, ties to the even code
    near = d == d.amin(-1, keepdim=True)
    even = near & (torch.arange(8) % 2 == 0)
    c = torch.where(even.any(-1), even.to(torch.uint8).argmax(-1), near.to(torch.uint8).argmax(-1))
    c = torch.where(a >= 6, 7, c)
    c = (c | (torch.signbit(b).long() << 3)) * ~bad[..., None]
    c = c.view(rows, -1)
    return (c[:, 0::2] | (c[:, 1::2] << 4)).to(torch.uint8), torch.where(bad, 255, e + 127).to(torch.uint8)


def dequant(codes, scales, cols):
    """f64 values [..., cols] of codes [..., >= 16 nb] and scale bytes [..., >= nb]."""
    nb = (cols + 31) // 32
    q = torch.stack([codes[..., :16 * nb] & 15, codes[..., :16 * nb] >> 4], -1).reshape(*codes.shape[:-1], nb, 32).long()
    v = GRID[q & 7] * (1 - 2.0 * (q >> 3))
    s = scales[..., :nb].double()
    s = torch.where(s == 255, torch.nan, torch.exp2(s - 127))
    return (v * s[..., None]).reshape(*codes.shape[:-1], 32 * nb)[..., :cols]


def gemm(x, w, sorted_tok, offset, T, top_k, swiglu):
    """(y, bound) in f64: the product by the definition over the clamped runs, and how far f32 sums may be off: each of the
    K additions loses at most a step of the running sum, so K 2^-23 sum |w x|; SwiGLU: |silu'| <= 1.1 and |silu(g)| carry
    the sums' errors on, and silu itself is within 8 + |g| steps of 2^-24 (the exponent's argument is rounded once)."""
    E, N, K = w.shape
    n_out = N // 2 if swiglu else N
    y, tol = torch.zeros(T, n_out, dtype=torch.float64), torch.zeros(T, n_out, dtype=torch.float64)
    off = [min(max(int(o), 0), T) for o in offset]
    for e in range(E):
        i = torch.arange(off[e], max(off[e], off[e + 1]))
        st = i * top_k if sorted_tok is None else torch.as_tensor(sorted_tok)[i].long()
        r = torch.div(st, top_k, rounding_mode="floor")
        ok = (st >= 0) & (r < x.shape[0])
        i, r = i[ok], r[ok]
        p = x[r] @ w[e].T
        t = K * 2.0 ** -23 * (x[r].abs() @ w[e].abs().T)
        if swiglu:
            g, u, tg, tu = p[:, :n_out], p[:, n_out:], t[:, :n_out], t[:, n_out:]
            s = torch.nn.functional.silu(g)
            p = s * u
            t = 1.1 * tg * (u.abs() + tu) + s.abs() * tu + (8 + g.abs()) * 2.0 ** -24 * p.abs()
        y[i], tol[i] = p, t
    return y, tol


def close(got, want, tol):
    """got (any float type) within tol and half a step of its own type of want, element for element; NaN where want is."""
    g, w = got.double(), want
    if not torch.equal(torch.isnan(g), torch.isnan(w)):
        return False
    ok = (g - w).abs() <= tol * (1 + EPS[got.dtype]) + EPS[got.dtype] * w.abs() + TINY[got.dtype]
    return bool((ok | torch.isnan(w) | (g == w)).all())
