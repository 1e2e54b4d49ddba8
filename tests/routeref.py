"""routeref.py -- moe_route by its definition (include/exl3c4.h), row by row in float64 on the CPU: what the device tests compare with."""
import numpy as np


def route(logits, top_k, score, bias=None, n_group=1, top_group=1, group="max", renorm=True, scale=1.0):
    """(ids int32, w float64) [n_tok, top_k] of logits [n_tok, n_expert] (any float array)."""
    n_tok, E = logits.shape
    ids, w = np.full((n_tok, top_k), -1, np.int32), np.zeros((n_tok, top_k))
    for t in range(n_tok):
        l = logits[t].astype(np.float64)
        ok = l > -np.inf                                             # False for NaN
        s = np.zeros(E)
        if score == "sigmoid":
            e = np.exp(-np.abs(l[ok]))
            s[ok] = np.where(l[ok] >= 0, 1 / (1 + e), e / (1 + e))
        elif ok.any():
            m = l[ok].max()
            with np.errstate(invalid="ignore"):
                e = np.exp(np.where(l[ok] == m, 0.0, l[ok] - m))
            s[ok] = e / e.sum()
        b = np.zeros(E) if bias is None else bias.astype(np.float64)
        out = ~ok | ~(b > -np.inf)
        value = s + b
        choice = np.where(out, -np.inf, l if bias is None else value)
        if n_group > 1:
            gv = np.full(n_group, -np.inf)
            for g in range(n_group):
                live = [i for i in range(g * E // n_group, (g + 1) * E // n_group) if not out[i]]
                v = sorted((value[i] if group == "top2" else choice[i] for i in live), reverse=True)
                if v:
                    gv[g] = v[0] if group == "max" or len(v) == 1 else v[0] + v[1]
            keep = sorted(range(n_group), key=lambda g: (-gv[g], g))[:top_group]
            for g in range(n_group):
                if g not in keep:
                    out[g * E // n_group:(g + 1) * E // n_group] = True
        live = [i for i in range(E) if not out[i]]
        chosen = sorted(live, key=lambda i: (-choice[i], i))[:top_k]
        p = s[chosen]
        if renorm:
            p = p / p.sum() if p.sum() > 0 else np.zeros(len(p))
        ids[t, :len(chosen)], w[t, :len(chosen)] = chosen, p * scale
    return ids, w


def scatter(ids, E):
    """(sorted_tok, expert_offset, expert_count, row_of) of ids [n_tok, top_k], pairs of -1 dropped."""
    f = ids.reshape(-1)
    live = np.flatnonzero(f >= 0)
    order = live[np.argsort(f[live], kind="stable")]
    sorted_tok, row_of = np.full(len(f), -1, np.int32), np.full(len(f), -1, np.int32)
    sorted_tok[:len(order)] = order
    row_of[order] = np.arange(len(order))
    count = np.bincount(f[live], minlength=E).astype(np.int32)
    return sorted_tok, np.concatenate([[0], np.cumsum(count)]).astype(np.int32), count, row_of
