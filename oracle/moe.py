"""CPU restatement of the expert network's operators in float64, one token at a time (routing and experts of the
reference: ``oracle/decode_engine.py:122-133`` of it; packed weights: ``ref_torch/quant.py:19-45``)."""
import math

import torch

F64 = torch.float64
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def unpack(codes, scales):
    """float64 [..., K] of codes [..., K/2] and scale bytes [..., K/32] (255: NaN)."""
    table = torch.tensor(GRID + tuple(-v for v in GRID), dtype=F64)
    v = torch.stack([table[(codes % 16).long()], table[(codes // 16).long()]], dim=-1).flatten(-2)
    s = torch.pow(2.0, scales.to(F64) - 127)
    s[scales == 255] = math.nan
    return v * s.repeat_interleave(32, dim=-1)


def pack(w):
    """The nearest e2m1 values (ties to the even code) under a power of two per 32, from amax / 6 up."""
    x = w.to(F64).unflatten(-1, (-1, 32))
    e = torch.ceil(torch.log2(x.abs().amax(-1, keepdim=True).clamp(min=6 * 2.0 ** -126) / 6))
    z = x / torch.pow(2.0, e)
    grid = torch.tensor(GRID, dtype=F64)
    d = (z.abs()[..., None] - grid).abs()
    best = d.amin(-1, keepdim=True)
    code = torch.zeros_like(z, dtype=torch.long)
    for c in (7, 5, 3, 1, 6, 4, 2, 0):      # the even ones last: they win a tie
        code[(d[..., c:c + 1] == best).squeeze(-1)] = c
    code += 8 * torch.signbit(z).long()
    code = code.flatten(-2)
    return (code[..., ::2] + 16 * code[..., 1::2]).to(torch.uint8), (e.squeeze(-1) + 127).to(torch.uint8)


def scores(row, kind):
    """Scores of one token's logits (a list of floats)."""
    if kind == "softmax":
        if any(math.isnan(v) for v in row):
            return [math.nan] * len(row)
        m = max(row)
        if m == -math.inf:
            return [0.0] * len(row)
        p = [math.exp(v - m) if m < math.inf else math.nan for v in row]
        t = math.fsum(p)
        return [v / t for v in p]
    out = []
    for v in row:
        if math.isnan(v):
            out.append(v)
        elif kind == "sigmoid":
            out.append(1 / (1 + math.exp(-v)) if v > -700 else 0.0)
        else:
            out.append(math.sqrt(max(v, 0.0) + math.log1p(math.exp(-abs(v)))))
    return out


def _order(ids, value):
    """ids by value, largest first, the lower id first among equals; NaN as -inf."""
    return sorted(ids, key=lambda e: (-(-math.inf if math.isnan(value[e]) else value[e]), e))


def route(logits, k, score, bias=None, groups=1, topk_groups=1, renorm=True, scale=1.0, shared=0, ids=None):
    T, E = logits.shape
    out_i, out_w = [], []
    for t in range(T):
        row = logits[t].to(F64).tolist()
        s = scores(row, score)
        if ids is not None:
            pick = ids[t].tolist()
        else:
            r = s if bias is None else [a + b for a, b in zip(s, bias.to(F64).tolist())]
            allowed = range(E)
            if groups > 1:
                per = E // groups
                best = [sorted((-math.inf if math.isnan(v) else v for v in r[g * per:(g + 1) * per]), reverse=True)[:2]
                        for g in range(groups)]
                kept = _order(range(groups), [sum(b) for b in best])[:topk_groups]
                allowed = [e for e in range(E) if e // per in kept]
            pick = _order(allowed, row if bias is None else r)[:k]
        w = [s[e] if 0 <= e < E else 0.0 for e in pick]
        if renorm:
            total = math.fsum(w) if not any(math.isnan(v) for v in w) else math.nan
            w = [v / total if total > 0 else total for v in w]
        out_i.append(list(pick) + [E + i for i in range(shared)])
        out_w.append([v * scale for v in w] + [1.0] * shared)
    return torch.tensor(out_i, dtype=torch.int32).view(T, -1), torch.tensor(out_w, dtype=F64).view(T, -1)


def experts(x, ids, weights, gate, up, down, limit=math.inf):
    """(y, error bound): x [T, K], dense float64 weights.  The bound holds for kernels that sum in fp32 in any order,
    round the hidden row to bf16 once and y to bf16 (2^-8 each: half a step)."""
    T, k = ids.shape
    E, inner, K = gate.shape
    y, bound = torch.zeros(T, K, dtype=F64), torch.zeros(T, K, dtype=F64)
    eps = 2.0 ** -24
    for t in range(T):
        a = x[t].to(F64)
        for j in range(k):
            e, w = int(ids[t, j]), float(weights[t, j])
            if not 0 <= e < E:
                continue
            g, u = gate[e] @ a, up[e] @ a
            dg, du = (K + 1) * eps * (gate[e].abs() @ a.abs()), (K + 1) * eps * (up[e].abs() @ a.abs())
            g, u = g.clamp(max=limit), u.clamp(-limit, limit)
            s = g * torch.sigmoid(g)
            h = w * s * u
            # |silu'| <= 1.1; the exponential, the quotient and two products: 8 roundings of the value
            dh = abs(w) * (1.1 * dg * u.abs() + s.abs() * du + 1.1 * dg * du) + (2.0 ** -8 + 8 * eps) * h.abs()
            y[t] += down[e] @ h
            bound[t] += down[e].abs() @ dh + (inner + k + 1) * eps * (down[e].abs() @ (h.abs() + dh))
    return y, bound + 2.0 ** -8 * (y.abs() + bound)
