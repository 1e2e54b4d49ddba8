"""operators.py -- the products of routed experts whose weights are not trellis codes, and the quantisation that makes
their 4-bit operands: what a layer kept in 16 bits or in microscaled 4-bit floats asks of this library.

  quant   mx4_quant of activation or weight rows (e2m1 codes, one e8m0 scale each 32 columns), and mx4_dequant of the
          result: the values that the codes stand for
  gemm    moe_gemm over the sorted rows of a routing: y[i] = W[expert of i] x[row of i], x gathered by token (gate and up,
          with SwiGLU) or given by sorted row (down). Weights and x in 16 bits; weights MX4 and x in 16 bits; or both
          MX4, x quantised in the pass. One expert makes it a plain linear layer (the router's logits).

A case's `tokens` x `top_k` sorted rows are spread over `n_expert` experts evenly or, with `zipf`, by a Zipf(1.1)
popularity; `n` and `k` are an expert's weight rows and columns.
"""
import math
import os
import sys

import torch

own = False
ZIPF_S = 1.1


def _gemm(name, tokens, **kw):
    c = {"name": name, "kind": "gemm", "tokens": tokens, "n": 1024, "k": 2048, "n_expert": 512, "top_k": 10, "x": "bf16",
         "w": "16", "y": "bf16", "swiglu": True, "gather": True, "zipf": False}
    c.update(kw)
    return c


def listed():
    return [
        # the hidden states of a decode batch, before the experts' products: latency
        {"name": "quant-8", "kind": "quant", "rows": 8, "cols": 2048, "type": "bf16"},
        # the experts' hidden rows of a prefill, a width that is not whole blocks
        {"name": "quant-rows", "kind": "quant", "rows": 20480, "cols": 650, "type": "f16"},
        # a loader quantises the experts of a layer from full precision
        {"name": "quant-weights", "kind": "quant", "rows": 131072, "cols": 2048, "type": "f32"},
        # gate and up of one sequence's decode step, a layer kept in 16 bits
        _gemm("bf16-gu-1", 1),
        # down of a speculative batch: sorted rows in
        _gemm("f16-down-8", 8, n=2048, k=512, x="f16", y="f16", swiglu=False, gather=False),
        # a prompt over many experts, uneven
        _gemm("bf16-gu-613-zipf", 613, n=1280, k=2560, zipf=True),
        # a large batch over few experts: bound by the matrix units
        _gemm("bf16-gu-8192", 8192, n=2816, n_expert=8, top_k=2),
        # the router's logits: one "expert", f32 out, an odd count of rows
        _gemm("router-77", 77, n=512, n_expert=1, top_k=1, y="f32", swiglu=False),
        # MX4 weights, activations in 16 bits: a decode step of one sequence, and of a batch
        _gemm("mx4w-gu-1", 1, x="f16", y="f16", w="mx4"),
        _gemm("mx4w-gu-32", 32, w="mx4"),
        # MX4 on both sides: a prompt over many experts, and a large batch over few
        _gemm("mx4-gu-2048-zipf", 2048, x="mx4", w="mx4", zipf=True),
        _gemm("mx4-down-8192", 8192, n=2048, k=1408, n_expert=8, top_k=2, x="mx4", w="mx4", swiglu=False, gather=False),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.25:
        cols = rng.choice([log(17, 5000), 32 * log(1, 160)])
        return {"kind": "quant", "rows": max(1, log(1, 3e8) // cols), "cols": cols, "type": rng.choice(["f16", "bf16", "f32"])}
    w = rng.choice(["16", "mx4", "mx4"])
    x = rng.choice(["f16", "bf16"] if w == "16" else ["f16", "bf16", "mx4", "mx4"])
    hidden, width = rng.choice([(2048, 512), (2560, 640), (1024, 256), (2048, 768), (2048, 1408), (992, 330), (1504, 200)])
    e, top_k = rng.choice([(512, 10), (512, 8), (128, 8), (64, 6), (16, 4), (8, 2), (1, 1)])
    gather = rng.random() < 0.6
    c = {"kind": "gemm", "n": 2 * width if gather else hidden - rng.choice([0, 0, 0, 3]), "k": hidden if gather else width // 32 * 32,
         "n_expert": e, "top_k": top_k, "x": x, "w": w, "y": rng.choice(["f16", "bf16", "f32"]), "swiglu": gather, "gather": gather,
         "zipf": rng.random() < 0.4, "tokens": log(1, 8192)}
    while _cost(c) > _cost(_gemm("", 8192, n=2816, n_expert=8, top_k=2)):
        c["tokens"] = c["tokens"] * 2 // 3
    return c


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 2, w["flops"] / 100)


# ------------------------------------------------------------------------------------------ inputs
_TYPE = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _up(n, m):
    return (n + m - 1) // m * m


def _mx4_buffers(rows, cols):
    """Codes (two a byte, the lower column in the low half; 16 bytes a block) and scales (a byte a block) of rows x cols."""
    nb = (cols + 31) // 32
    return (torch.zeros((rows, 16 * nb), dtype=torch.uint8, device="cuda"),
            torch.zeros((rows, _up(nb, 4)), dtype=torch.uint8, device="cuda"))


def _mx4_of(x):
    """Codes and scales of f32 rows whose columns are whole blocks."""
    b = x.view(x.shape[0], -1, 32)
    e = _block_exponent(b)
    q = _e2m1_index(torch.ldexp(b.abs(), -e[..., None])) | ((b < 0).to(torch.uint8) << 3)
    q = q.view(x.shape[0], -1)
    s = torch.zeros((x.shape[0], _up(e.shape[1], 4)), dtype=torch.uint8, device=x.device)
    s[:, :e.shape[1]] = e + 127
    return q[:, 0::2] | (q[:, 1::2] << 4), s


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    s = {"case": case, "stream": torch.cuda.current_stream()}
    if case["kind"] == "quant":
        R, C, t = case["rows"], case["cols"], _TYPE[case["type"]]
        x = torch.randn((R, C), device="cuda", generator=g)
        x *= torch.rand((R, 1), device="cuda", generator=g) * 2 + 0.05             # rows of unlike magnitude
        s["x"] = x.to(t)
        s["codes"], s["scales"] = _mx4_buffers(R, C)
        s["out"] = torch.zeros((R, C), dtype=torch.float32 if t == torch.float32 else torch.bfloat16, device="cuda")
        return s
    M, k, E, N, K = case["tokens"], case["top_k"], case["n_expert"], case["n"], case["k"]
    T = M * k
    # the routing: distinct experts a token, the pairs sorted by expert
    score = -torch.log(-torch.log(torch.rand((M, E), device="cuda", generator=g).clamp_(1e-12, 1 - 1e-7)))
    if case["zipf"]:
        score -= ZIPF_S * torch.log(torch.randperm(E, device="cuda", generator=g).float() + 1.0)
    ids = torch.topk(score, k, dim=1).indices.reshape(-1)
    s["sorted_tok"] = torch.argsort(ids, stable=True).to(torch.int32)
    s["offset"] = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    s["offset"][1:] = torch.cumsum(torch.bincount(ids, minlength=E), 0)
    rows = M if case["gather"] else T
    x = torch.randn((rows, K), device="cuda", generator=g)
    if not case["gather"]:
        x *= torch.randn((rows, K), device="cuda", generator=g)                    # what SwiGLU leaves
    s["x"] = x.to(_TYPE["bf16" if case["x"] == "mx4" else case["x"]])
    if case["x"] == "mx4":
        s["x_codes"], s["x_scales"] = _mx4_buffers(rows, K)
    if case["w"] == "16":
        s["w"] = torch.randn((E, N, K), dtype=s["x"].dtype, device="cuda", generator=g)
        s["w"] *= 1 / math.sqrt(K)
    else:
        codes, scales = _mx4_buffers(E * N, K)
        step = max(1, (1 << 26) // K)
        for r in range(0, E * N, step):
            w = torch.randn((min(step, E * N - r), K), device="cuda", generator=g) / math.sqrt(K)
            w *= torch.rand((w.shape[0], 1), device="cuda", generator=g) + 0.5
            codes[r:r + step], scales[r:r + step] = _mx4_of(w)
        s["w_codes"], s["w_scales"] = codes.view(E, N, -1), scales.view(E, N, -1)
    s["y"] = torch.zeros((T, N // 2 if case["swiglu"] else N), dtype=_TYPE[case["y"]], device="cuda")
    return s


# ------------------------------------------------------------------------------------------ one pass
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _ok(rc):
    if rc:
        raise RuntimeError(f"status {rc}")


def _run_own(s):
    pkg = os.path.join(os.getcwd(), "radiance-exl3_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import exl3c4
    case, st = s["case"], s["stream"]
    if case["kind"] == "quant":
        if "q" not in s:                                                           # views that a program keeps
            s["q"] = exl3c4.Mx4(s["codes"], s["scales"], case["cols"])
        _ok(exl3c4.mx4_quant(s["x"], s["q"], st))
        _ok(exl3c4.mx4_dequant(s["q"], s["out"], st))
        return s["out"]
    if "gemm" not in s:                                                            # the descriptor that a program keeps
        x = s["x"]
        if case["x"] == "mx4":
            x = s["xq"] = exl3c4.Mx4(s["x_codes"], s["x_scales"], case["k"])
        w = s["w"] if case["w"] == "16" else exl3c4.Mx4(s["w_codes"], s["w_scales"], case["k"])
        s["gemm"] = exl3c4.make_gemm(x, w, s["sorted_tok"] if case["gather"] else None, s["offset"], s["y"],
                                     top_k=case["top_k"], act=exl3c4.ACT_SWIGLU if case["swiglu"] else exl3c4.ACT_NONE)
    if case["x"] == "mx4":
        _ok(exl3c4.mx4_quant(s["x"], s["xq"], st))
    _ok(exl3c4.moe_gemm(s["gemm"], st))
    return s["y"]


def _block_exponent(b):
    """The scale's exponent of each block (the last dimension): floor(log2(max |x|)) - 2, at least -127."""
    e = torch.frexp(b.abs().amax(-1)).exponent - 3                                  # frexp's mantissa is in [1/2, 1)
    return torch.where(b.abs().amax(-1) > 0, e, -127).clamp(min=-127)


def _e2m1_index(a):
    """The code (0 .. 7) nearest to a >= 0 among 0, 1/2, 1, 3/2, 2, 3, 4, 6; ties to the even code."""
    n = (a > 0.25).to(torch.uint8)
    n += a >= 0.75
    n += a > 1.25
    n += a >= 1.75
    n += a > 2.5
    n += a >= 3.5
    n += a > 5
    return n


def _values(device):
    return torch.tensor([0.0, 0.5, 1, 1.5, 2, 3, 4, 6], device=device)


def _rounded(x):
    """The values in f32 that x's codes and scales stand for."""
    R, C = x.shape
    b = torch.nn.functional.pad(x.float(), (0, -C % 32)).view(R, -1, 32)
    e = _block_exponent(b)[..., None]
    v = _values(x.device)[_e2m1_index(torch.ldexp(b.abs(), -e)).to(torch.int32)]
    return torch.ldexp(torch.copysign(v, b), e).view(R, -1)[:, :C]


def _decoded(codes, scales, K):
    """f32 values of codes [..., K / 2] and scales [..., at least K / 32]."""
    v = _values(codes.device)
    v = torch.cat([v, -v])
    pair = torch.stack([v.repeat(16), v.repeat_interleave(16)], 1)                  # a byte's two values
    w = pair[codes.to(torch.int32)].view(*codes.shape[:-1], K // 32, 32)
    return (w * torch.exp2(scales[..., :K // 32, None].float() - 127)).view(*codes.shape[:-1], K)


def _run_plain(s):
    case = s["case"]
    if case["kind"] == "quant":
        return _rounded(s["x"]).to(s["out"].dtype)
    T, E, K = s["y"].shape[0], case["n_expert"], case["k"]
    x = _rounded(s["x"]) if case["x"] == "mx4" else s["x"].float()
    # the sorted rows in blocks of R rows of one expert each (the last of an expert padded), one batched product
    R = 1 << max(0, min(8, int(math.log2(max(1, T / min(E, T))))))
    off = s["offset"].long()
    blocks = (off[1:] - off[:-1] + R - 1) // R
    ends = torch.cumsum(blocks, 0)
    b = torch.arange(T // R + min(E, T), device=x.device)
    e = torch.searchsorted(ends, b, right=True).clamp(max=E - 1)
    row = (off[e] + (b - (ends - blocks)[e]) * R)[:, None] + torch.arange(R, device=x.device)
    live = (row < off[e + 1][:, None]) & (b < ends[-1])[:, None]
    row = torch.where(live, row, 0)
    xb = x[s["sorted_tok"].long()[row] // case["top_k"]] if case["gather"] else x[row]
    w = s["w"][e].float() if case["w"] == "16" else _decoded(s["w_codes"][e], s["w_scales"][e], K)
    y = torch.bmm(w, xb.transpose(1, 2).contiguous()).transpose(1, 2)               # [blocks, R, N] in f32
    if case["swiglu"]:
        gate, up = y[..., :case["n"] // 2], y[..., case["n"] // 2:]
        y = gate / (1 + torch.exp(-gate)) * up
    out = torch.zeros((T + 1, y.shape[-1]), dtype=s["y"].dtype, device=x.device)    # row T takes the padding
    out[torch.where(live, row, T).reshape(-1)] = y.reshape(-1, y.shape[-1]).to(out.dtype)
    return out[:T]


# ------------------------------------------------------------------------------------------ what it cannot do without
def _live(case):
    """Experts that hold a row, by expectation."""
    E, M, k = case["n_expert"], case["tokens"], case["top_k"]
    if not case["zipf"]:
        return E * (1.0 - (1.0 - k / E) ** M)
    pop = [1.0 / (i + 1) ** ZIPF_S for i in range(E)]
    return sum(1.0 - math.exp(-M * k * p / sum(pop)) for p in pop) if E > 1 else 1.0


def work(case):
    if case["kind"] == "quant":
        n = case["rows"] * case["cols"]
        size = 4 if case["type"] == "f32" else 2
        return {"bytes": n * (2 * size + 2 * 17 / 32), "flops": 0}                  # x; codes and scales both ways; values
    T, N, K = case["tokens"] * case["top_k"], case["n"], case["k"]
    rows = case["tokens"] if case["gather"] else T
    weights = _live(case) * N * K * (2 if case["w"] == "16" else 17 / 32)
    y = T * (N // 2 if case["swiglu"] else N) * (4 if case["y"] == "f32" else 2)
    return {"bytes": weights + rows * K * 2 + y + 4 * (T + case["n_expert"]), "flops": 2.0 * T * N * K}


# ------------------------------------------------------------------------------------------ in 64 bits
def _grid64(x):
    """x rounded to MX4 in 64 bits: steps of 1/2 below 2, of 1 below 4, of 2 from there, torch.round's ties to even."""
    R, C = x.shape
    b = torch.nn.functional.pad(x.double(), (0, -C % 32)).view(R, -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    scale = torch.where(top > 0, torch.exp2(torch.floor(torch.log2(top)) - 2), 1.0).clamp(min=2.0 ** -127)
    a = b.abs() / scale
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return (torch.sign(b) * torch.clamp(torch.round(a / step) * step, max=6.0) * scale).view(R, -1)[:, :C]


def _weights64(s, e):
    if "w" in s:
        return s["w"][e].double()
    codes, K = s["w_codes"][e], s["case"]["k"]
    q = torch.stack([codes & 15, codes >> 4], -1).view(codes.shape[0], K).long()
    exp, man = (q >> 1) & 3, (q & 1).double()
    mag = torch.where(exp == 0, man / 2, (1 + man / 2) * torch.exp2(exp.double() - 1))
    scale = torch.exp2(s["w_scales"][e][:, :K // 32].double() - 127).repeat_interleave(32, dim=1)
    return mag * (1 - 2.0 * (q >> 3)) * scale


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "quant":
        return torch.cat([_grid64(p) for p in torch.split(s["x"], max(1, (1 << 26) // case["cols"]))])
    y = torch.zeros(s["y"].shape, dtype=torch.float64, device="cuda")
    off = s["offset"].tolist()
    for e in range(case["n_expert"]):
        if off[e + 1] == off[e]:
            continue
        rows = torch.arange(off[e], off[e + 1], device="cuda")
        x = s["x"][s["sorted_tok"][rows].long() // case["top_k"] if case["gather"] else rows]
        p = (_grid64(x) if case["x"] == "mx4" else x.double()) @ _weights64(s, e).T
        if case["swiglu"]:
            p = torch.nn.functional.silu(p[:, :case["n"] // 2]) * p[:, case["n"] // 2:]
        y[rows] = p
    return y
