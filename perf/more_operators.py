"""more_operators.py -- what a routed layer asks of this library whose router scores by sigmoid or softmax with a bias and groups, and whose
experts are kept in 8-bit floats (F8: e4m3 codes, an f32 scale for each block of 128).

  route   moe_route: scores, the choice of groups and of experts, the weights, and the scatter of the pairs by expert
  quant   f8_quant of activation rows (blocks of 1 x 128) or of weights (128 x 128), and f8_dequant of the result: the values that the
          codes stand for
  gemm    moe_gemm over the sorted rows of a routing with F8 weights: y[i] = W[expert of i] x[row of i], x gathered by token (gate and up,
          with SwiGLU) or given by sorted row (down), in 16 bits or in F8, quantised in the pass. One expert makes it a linear layer.

A gemm case's `tokens` x `top_k` sorted rows are spread over `n_expert` experts evenly or, with `zipf`, by a Zipf(1.1) popularity; `n` and
`k` are an expert's weight rows and columns.
"""
import math
import os
import sys

import torch

own = False
ZIPF_S = 1.1
TINY = 2.0 ** -96                                                                   # the least magnitude that sets a block's scale


def _route(name, tokens, **kw):
    c = {"name": name, "kind": "route", "tokens": tokens, "n_expert": 256, "top_k": 8, "n_group": 8, "top_group": 4, "score": "sigmoid",
         "group": "top2", "bias": True, "renorm": True, "scale": 2.5, "type": "f32", "scatter": True}
    c.update(kw)
    return c


def _gemm(name, tokens, **kw):
    c = {"name": name, "kind": "gemm", "tokens": tokens, "n": 1024, "k": 2048, "n_expert": 512, "top_k": 10, "x": "bf16", "y": "bf16",
         "swiglu": True, "gather": True, "zipf": False}
    c.update(kw)
    return c


def listed():
    return [
        # the router of one sequence's decode step: latency
        _route("route-1", 1),
        # a batch just past what one workgroup routes: softmax with a bias over many experts, no groups
        _route("route-33", 33, n_expert=512, top_k=10, n_group=1, top_group=1, score="softmax", scale=1.0),
        # a prompt: groups by their best expert, weights as they are, logits in 16 bits (equal ones are common)
        _route("route-613", 613, n_expert=160, top_k=6, top_group=3, score="softmax", group="max", bias=False, renorm=False, scale=16.0,
               type="bf16"),
        # the largest prompt
        _route("route-8192", 8192, n_expert=512, top_k=10),
        # the hidden states of a decode batch, before the experts' products: latency
        {"name": "quant-8", "kind": "quant", "mats": 1, "rows": 8, "cols": 2048, "block": 1, "type": "bf16"},
        # the experts' hidden rows of a prefill, a width that is not whole blocks
        {"name": "quant-rows", "kind": "quant", "mats": 1, "rows": 20480, "cols": 650, "block": 1, "type": "f16"},
        # a loader quantises the gate and up halves of some of a layer's experts from full precision
        {"name": "quant-weights", "kind": "quant", "mats": 64, "rows": 1000, "cols": 2048, "block": 128, "type": "f32"},
        # gate and up of one sequence's decode step, activations in 16 bits
        _gemm("f8w-gu-1", 1, x="f16", y="f16"),
        # the same of a decode batch
        _gemm("f8w-gu-32", 32),
        # down of a prompt over many experts, uneven; sorted rows in, quantised in the pass
        _gemm("f8-down-613-zipf", 613, n=2560, k=640, x="f8", swiglu=False, gather=False, zipf=True),
        # a large batch over few experts: bound by the matrix units
        _gemm("f8-gu-8192", 8192, n=2816, n_expert=8, top_k=2, x="f8"),
        # a shared projection: one "expert", f32 out, odd sizes
        _gemm("f8-linear-77", 77, n=517, k=1040, n_expert=1, top_k=1, x="f8", y="f32", swiglu=False),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    kind = rng.random()
    if kind < 0.3:
        e = rng.choice([8, 16, 64, 128, 160, 256, 384, 512, log(8, 1024)])
        n_group = rng.choice([g for g in (1, 1, 2, 4, 5, 8, 16) if e % g == 0 and g <= e // 2])
        top_group = rng.randint(max(1, n_group // 3), n_group)
        top_k = min(rng.choice([1, 2, 4, 6, 8, 10, log(1, 64)]), top_group * (e // n_group))
        return {"kind": "route", "tokens": log(1, 8192), "n_expert": e, "top_k": top_k, "n_group": n_group, "top_group": top_group,
                "score": rng.choice(["sigmoid", "softmax"]), "group": rng.choice(["top2", "max"]), "bias": rng.random() < 0.6,
                "renorm": rng.random() < 0.7, "scale": rng.choice([1.0, 2.5, 16.0]), "type": rng.choice(["f32", "f32", "bf16", "f16"]),
                "scatter": rng.random() < 0.7}
    if kind < 0.5:
        block = rng.choice([1, 1, 128])
        cols = rng.choice([log(17, 5000), 128 * log(1, 40)])
        rows = max(1, log(1, 1e8) // cols)
        mats = rng.choice([1, 3, 16]) if block == 128 else 1
        return {"kind": "quant", "mats": mats, "rows": max(1, rows // mats), "cols": cols, "block": block,
                "type": rng.choice(["f16", "bf16", "f32"])}
    hidden, width = rng.choice([(2048, 512), (2560, 640), (1024, 256), (2048, 768), (2048, 1408), (992, 336), (1504, 208)])
    e, top_k = rng.choice([(512, 10), (512, 8), (128, 8), (64, 6), (16, 4), (8, 2), (1, 1)])
    gather = rng.random() < 0.6
    c = {"kind": "gemm", "n": 2 * width if gather else hidden - rng.choice([0, 0, 0, 3]), "k": hidden if gather else width, "n_expert": e,
         "top_k": top_k, "x": rng.choice(["f16", "bf16", "f8", "f8"]), "y": rng.choice(["f16", "bf16", "f32"]), "swiglu": gather,
         "gather": gather, "zipf": rng.random() < 0.4, "tokens": log(1, 8192)}
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


def _f8_buffers(mats, rows, cols, block):
    """Codes (a byte a column, rows of whole 16 bytes) and scales of `mats` matrices of rows x cols."""
    return (torch.zeros((mats, rows, _up(cols, 16)), dtype=torch.uint8, device="cuda"),
            torch.zeros((mats, _up(rows, block) // block, _up(cols, 128) // 128), dtype=torch.float32, device="cuda"))


def _by_448(top):
    """448 / top and top / 448, each rounded once: as quotients of tensors, for torch takes a number's reciprocal first."""
    most = torch.full_like(top, 448)
    return most / top, top / most


def _f8_weights(w):
    """Codes and scales of weights [mats, rows, cols] in f32, cols a multiple of 16."""
    m, R, C = w.shape
    codes, scales = _f8_buffers(m, R, C, 128)
    b = torch.nn.functional.pad(w, (0, -C % 128, 0, -R % 128)).view(m, scales.shape[1], 128, scales.shape[2], 128)
    inv, scales[:] = _by_448(b.abs().amax((2, 4)).clamp_(min=TINY))
    q = (b * inv[:, :, None, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    codes[:] = q.view(m, _up(R, 128), _up(C, 128))[:, :R, :C]
    return codes, scales


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    s = {"case": case, "stream": torch.cuda.current_stream()}
    if case["kind"] == "route":
        M, E, k = case["tokens"], case["n_expert"], case["top_k"]
        s["logits"] = (torch.randn((M, E), device="cuda", generator=g) * 1.5).to(_TYPE[case["type"]])
        if case["bias"]:                                                           # on the scores' scale
            s["bias"] = torch.randn(E, device="cuda", generator=g) * (0.1 if case["score"] == "sigmoid" else 1 / E)
        for name, shape, t in (("ids", (M, k), torch.int32), ("w", (M, k), torch.float32), ("sorted_tok", (M * k,), torch.int32),
                               ("offset", (E + 1,), torch.int32), ("count", (E,), torch.int32), ("row_of", (M * k,), torch.int32)):
            s[name] = torch.zeros(shape, dtype=t, device="cuda")
        return s
    if case["kind"] == "quant":
        m, R, C, t = case["mats"], case["rows"], case["cols"], _TYPE[case["type"]]
        x = torch.randn((m, R, C), device="cuda", generator=g)
        x *= torch.rand((m, R, 1), device="cuda", generator=g) * 2 + 0.05          # rows of unlike magnitude
        s["x"] = x.to(t)
        s["codes"], s["scales"] = _f8_buffers(m, R, C, case["block"])
        s["out"] = torch.zeros((m, R, C), dtype=t, device="cuda")
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
    s["x"] = x.to(_TYPE["bf16" if case["x"] == "f8" else case["x"]])
    if case["x"] == "f8":
        s["x_codes"], s["x_scales"] = (t[0] for t in _f8_buffers(1, rows, K, 1))
    # gate and up are matrices of their own, one behind the other in an expert's rows
    half = 2 if case["swiglu"] else 1
    s["w_codes"], s["w_scales"] = _f8_buffers(E * half, N // half, K, 128)
    step = max(1, (1 << 27) // (N // half * K))
    for i in range(0, E * half, step):
        w = torch.randn((min(step, E * half - i), N // half, K), device="cuda", generator=g) / math.sqrt(K)
        w *= torch.rand((w.shape[0], N // half, 1), device="cuda", generator=g) + 0.5
        s["w_codes"][i:i + step], s["w_scales"][i:i + step] = _f8_weights(w)
    s["w_codes"] = s["w_codes"].view(E, N, K)
    s["w_scales"] = s["w_scales"].view(E, -1, s["w_scales"].shape[-1])
    s["y"] = torch.zeros((T, N // 2 if case["swiglu"] else N), dtype=_TYPE[case["y"]], device="cuda")
    return s


# ------------------------------------------------------------------------------------------ one pass
def run(s):
    return _run_own(s) if own else _PLAIN[s["case"]["kind"]](s)


def _ok(rc):
    if rc:
        raise RuntimeError(f"status {rc}")


def _routed(s, ids, w, sorted_tok, offset, count, row_of):
    return (ids, w, sorted_tok, offset, count, row_of) if s["case"]["scatter"] else (ids, w)


def _run_own(s):
    pkg = os.path.join(os.getcwd(), "radiance-exl3_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import exl3c4
    case, st = s["case"], s["stream"]
    if case["kind"] == "route":
        if "route" not in s:                                                       # the descriptor that a program keeps
            scatter = dict(sorted_tok=s["sorted_tok"], expert_offset=s["offset"], expert_count=s["count"], row_of=s["row_of"])
            s["route"] = exl3c4.make_route(
                s["logits"], case["top_k"], s["ids"], s["w"], score=exl3c4.SCORE_SIGMOID if case["score"] == "sigmoid" else exl3c4.SCORE_SOFTMAX,
                bias=s.get("bias"), n_group=case["n_group"], top_group=case["top_group"],
                group_score=exl3c4.GROUP_TOP2 if case["group"] == "top2" else exl3c4.GROUP_MAX, renorm=case["renorm"], scale=case["scale"],
                **(scatter if case["scatter"] else {}))
        _ok(exl3c4.moe_route(s["route"], st))
        return _routed(s, s["ids"], s["w"], s["sorted_tok"], s["offset"], s["count"], s["row_of"])
    if case["kind"] == "quant":
        if "q" not in s:                                                           # views that a program keeps
            s["q"] = exl3c4.F8(s["codes"], s["scales"], case["cols"], case["block"])
        _ok(exl3c4.f8_quant(s["x"], s["q"], st))
        _ok(exl3c4.f8_dequant(s["q"], s["out"], st))
        return s["out"]
    if "gemm" not in s:
        x = s["x"]
        if case["x"] == "f8":
            x = s["xq"] = exl3c4.F8(s["x_codes"], s["x_scales"], case["k"], 1)
        s["gemm"] = exl3c4.make_gemm(x, exl3c4.F8(s["w_codes"], s["w_scales"], case["k"], 128), s["sorted_tok"] if case["gather"] else None,
                                     s["offset"], s["y"], top_k=case["top_k"], act=exl3c4.ACT_SWIGLU if case["swiglu"] else exl3c4.ACT_NONE)
    if case["x"] == "f8":
        _ok(exl3c4.f8_quant(s["x"], s["xq"], st))
    _ok(exl3c4.moe_gemm(s["gemm"], st))
    return s["y"]


def _plain_route(s):
    """In 64 bits: experts and groups are ranked, and the values next to a rank's border may be close."""
    case = s["case"]
    M, E, k, G = case["tokens"], case["n_expert"], case["top_k"], case["n_group"]
    l = s["logits"].double()
    if case["score"] == "sigmoid":
        score = 1 / (1 + torch.exp(-l))
    else:
        score = torch.exp(l - l.amax(1, keepdim=True))
        score = score / score.sum(1, keepdim=True)
    value = score + s["bias"].double() if case["bias"] else score
    choice = value if case["bias"] else l                                          # the scores' own order is the logits'
    if G > 1:
        by_group = value.view(M, G, E // G).sort(2, descending=True).values
        top = by_group[..., :2].sum(2) if case["group"] == "top2" else by_group[..., 0]
        kept = torch.sort(top, dim=1, descending=True, stable=True).indices[:, :case["top_group"]]
        off = torch.ones((M, G), dtype=torch.bool, device=l.device).scatter_(1, kept, False)
        choice = torch.where(off.repeat_interleave(E // G, dim=1), -math.inf, choice)
    ids = torch.sort(choice, dim=1, descending=True, stable=True).indices[:, :k]
    w = torch.gather(score, 1, ids)
    if case["renorm"]:
        w = w / w.sum(1, keepdim=True)
    w = (w * case["scale"]).float()
    if not case["scatter"]:
        return ids.to(torch.int32), w
    order = torch.argsort(ids.reshape(-1), stable=True)
    row_of = torch.empty_like(order)
    row_of[order] = torch.arange(M * k, device=l.device)
    count = torch.bincount(ids.reshape(-1), minlength=E)
    offset = torch.cat([count.new_zeros(1), torch.cumsum(count, 0)])
    return tuple(t.to(torch.int32) if t is not w else t for t in (ids, w, order, offset, count, row_of))


def _rounded(x, block):
    """The values in f32 that the codes of x [mats, rows, cols] stand for, and each block's scale spread over them."""
    m, R, C = x.shape
    b = torch.nn.functional.pad(x.float(), (0, -C % 128, 0, -R % block)).view(m, -1, block, _up(C, 128) // 128, 128)
    inv, scale = _by_448(b.abs().amax((2, 4), keepdim=True).clamp(min=TINY))
    a = b * inv
    e = (torch.frexp(a).exponent - 1).clamp(min=-6) - 3                             # e4m3's step is 2^e
    a = torch.ldexp(torch.round(torch.ldexp(a, -e)), e)
    return (a * scale).view(m, -1, _up(C, 128))[:, :R, :C]


def _plain_quant(s):
    return _rounded(s["x"], s["case"]["block"]).to(s["out"].dtype)


def _decoded(codes, scales, halves):
    """f32 values of weights' codes [e, N, K] and scales [e, rows of blocks, blocks a row]."""
    e, N, K = codes.shape
    v = codes.view(torch.float8_e4m3fn).float().view(e, halves, N // halves, K)
    sc = scales.view(e, halves, -1, scales.shape[-1]).repeat_interleave(128, 2)[:, :, :N // halves].repeat_interleave(128, 3)[..., :K]
    return (v * sc).view(e, N, K)


def _plain_gemm(s):
    case = s["case"]
    T, E, K = s["y"].shape[0], case["n_expert"], case["k"]
    x = _rounded(s["x"][None], 1)[0] if case["x"] == "f8" else s["x"].float()
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
    w = _decoded(s["w_codes"][e], s["w_scales"][e], 2 if case["swiglu"] else 1)
    y = torch.bmm(w, xb.transpose(1, 2).contiguous()).transpose(1, 2)               # [blocks, R, N] in f32
    if case["swiglu"]:
        gate, up = y[..., :case["n"] // 2], y[..., case["n"] // 2:]
        y = gate / (1 + torch.exp(-gate)) * up
    out = torch.zeros((T + 1, y.shape[-1]), dtype=s["y"].dtype, device=x.device)    # row T takes the padding
    out[torch.where(live, row, T).reshape(-1)] = y.reshape(-1, y.shape[-1]).to(out.dtype)
    return out[:T]


_PLAIN = {"route": _plain_route, "quant": _plain_quant, "gemm": _plain_gemm}


# ------------------------------------------------------------------------------------------ what it cannot do without
def _live(case):
    """Experts that hold a row, by expectation."""
    E, M, k = case["n_expert"], case["tokens"], case["top_k"]
    if not case["zipf"]:
        return E * (1.0 - (1.0 - k / E) ** M)
    pop = [1.0 / (i + 1) ** ZIPF_S for i in range(E)]
    return sum(1.0 - math.exp(-M * k * p / sum(pop)) for p in pop) if E > 1 else 1.0


def work(case):
    if case["kind"] == "route":
        M, E, T = case["tokens"], case["n_expert"], case["tokens"] * case["top_k"]
        out = 8 * T + (8 * T + 4 * (2 * E + 1) if case["scatter"] else 0)
        return {"bytes": M * E * (4 if case["type"] == "f32" else 2) + (4 * E if case["bias"] else 0) + out, "flops": 10.0 * M * E}
    if case["kind"] == "quant":
        n = case["mats"] * case["rows"] * case["cols"]
        size = 4 if case["type"] == "f32" else 2
        scales = 4 / 128 if case["block"] == 1 else 4 / 16384
        return {"bytes": n * (2 * size + 2 * (1 + scales)), "flops": 0}             # x; codes and scales both ways; values
    T, N, K = case["tokens"] * case["top_k"], case["n"], case["k"]
    rows = case["tokens"] if case["gather"] else T
    y = T * (N // 2 if case["swiglu"] else N) * (4 if case["y"] == "f32" else 2)
    return {"bytes": _live(case) * N * K + rows * K * 2 + y + 4 * (T + case["n_expert"]), "flops": 2.0 * T * N * K}


# ------------------------------------------------------------------------------------------ in 64 bits
def _exact_route(s):
    """Row by row from the definition, in numpy."""
    import numpy as np
    case = s["case"]
    E, k, G = case["n_expert"], case["top_k"], case["n_group"]
    l = s["logits"].double().cpu().numpy()
    bias = s["bias"].double().cpu().numpy() if case["bias"] else None
    ids, w = [], []
    for row in l:
        if case["score"] == "sigmoid":
            p = np.where(row >= 0, 1 / (1 + np.exp(-np.abs(row))), np.exp(-np.abs(row)) / (1 + np.exp(-np.abs(row))))
        else:
            p = np.exp(row - row.max())
            p /= p.sum()
        v = p if bias is None else p + bias
        c = row if bias is None else v
        if G > 1:
            gv = v.reshape(G, -1)
            if case["group"] == "max":
                gs = gv.max(1)
            else:
                gs = np.partition(gv, gv.shape[1] - 2, 1)[:, -2:].sum(1)
            keep = np.zeros(G, bool)
            keep[np.lexsort((np.arange(G), -gs))[:case["top_group"]]] = True
            c = np.where(np.repeat(keep, E // G), c, -np.inf)
        i = np.lexsort((np.arange(E), -c))[:k]
        q = p[i] / p[i].sum() if case["renorm"] else p[i]
        ids.append(i)
        w.append(q * case["scale"])
    ids, w = np.array(ids), torch.from_numpy(np.array(w)).cuda()
    flat = ids.reshape(-1)
    order = np.argsort(flat, kind="stable")
    count = np.bincount(flat, minlength=E)
    row_of = np.empty(len(flat), np.int64)
    row_of[order] = np.arange(len(flat))
    i32 = [torch.from_numpy(a.astype(np.int32)).cuda() for a in (ids, order, np.concatenate([[0], np.cumsum(count)]), count, row_of)]
    return _routed(s, i32[0], w, *i32[1:])


def _grid64(x, block):
    """x [mats, rows, cols] rounded to F8: the scales and the products with their inverses in f32, as the definition has them, each
    from its value in 64 bits; the codes' grid by its steps."""
    m, R, C = x.shape
    b = torch.nn.functional.pad(x.double(), (0, -C % 128, 0, -R % block)).view(m, -1, block, _up(C, 128) // 128, 128)
    top = b.abs().amax((2, 4), keepdim=True).clamp(min=TINY)
    inv, scale = (t.float().double() for t in _by_448(top))
    a = (b * inv).float().double()
    step = torch.exp2(torch.floor(torch.log2(a.abs().clamp(min=2.0 ** -6))) - 3)
    q = torch.clamp(torch.round(a / step) * step, -448, 448)
    return (q * scale).view(m, -1, _up(C, 128))[:, :R, :C]


def _weights64(s, e):
    q = s["w_codes"][e].int()
    exp, man = (q >> 3) & 15, (q & 7).double()
    v = torch.where(exp == 0, man / 8 * 2.0 ** -6, (1 + man / 8) * torch.exp2(exp.double() - 7)) * (1 - 2.0 * (q >> 7))
    n = torch.arange(q.shape[0], device=q.device)
    per = q.shape[0] // 2 if s["case"]["swiglu"] else q.shape[0]
    rows = n // per * ((per + 127) // 128) + n % per // 128
    return v * s["w_scales"][e].double()[rows][:, torch.arange(q.shape[1], device=q.device) // 128]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "route":
        return _exact_route(s)
    if case["kind"] == "quant":
        step = max(1, (1 << 26) // (case["rows"] * case["cols"]))
        if case["block"] == 1:                                                     # rows are apart: in parts of them
            x = s["x"].view(-1, case["cols"])
            return torch.cat([_grid64(p[None], 1)[0] for p in torch.split(x, max(1, (1 << 26) // case["cols"]))])[None].view(s["x"].shape)
        return torch.cat([_grid64(p, 128) for p in torch.split(s["x"], step)])
    y = torch.zeros(s["y"].shape, dtype=torch.float64, device="cuda")
    off = s["offset"].tolist()
    for e in range(case["n_expert"]):
        if off[e + 1] == off[e]:
            continue
        rows = torch.arange(off[e], off[e + 1], device="cuda")
        x = s["x"][s["sorted_tok"][rows].long() // case["top_k"] if case["gather"] else rows]
        p = (_grid64(x[None], 1)[0] if case["x"] == "f8" else x.double()) @ _weights64(s, e).T
        if case["swiglu"]:
            p = torch.nn.functional.silu(p[:, :case["n"] // 2]) * p[:, case["n"] // 2:]
        y[rows] = p
    return y
