"""Timed and checked cases of a layer's expert network: routing, products with 4-bit weights, the experts.

The kinds:

* ``route``    ``moe.route``: router scores, a balance bias, expert groups, the top-k and its weights.
* ``linear``   ``mla.linear_fp4``: y = x W^T, W held as e2m1 codes with a power-of-two scale per 32.
* ``experts``  ``moe.experts``: every token through the gated feed-forward networks of its experts
               (weights e2m1 or bf16), their outputs weighted and summed.

``run`` computes them in plain torch where ``own`` is false, through the framework where it is true;
``exact`` restates the computed values in float64.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _own_modules():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "deepseek-v4-flash-mlx_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from smla import mla, moe
    return mla, moe


def listed():
    return [
        # one token's choice of 6 of 256 experts and the shared one: the smallest call, where latency counts
        {"name": "route_token", "kind": "route", "T": 1, "E": 256, "k": 6, "x": "f32", "score": "sqrtsoftplus", "bias": True,
         "groups": 1, "topk_groups": 1, "renorm": True, "scale": 1.5, "shared": 1},
        # a long prompt with the experts in 8 groups, of which a token may use 4
        {"name": "route_prompt", "kind": "route", "T": 16384, "E": 256, "k": 8, "x": "f32", "score": "sigmoid", "bias": True,
         "groups": 8, "topk_groups": 4, "renorm": True, "scale": 2.5, "shared": 0},
        # softmax over a number of experts that is no power of two, bf16 logits with many ties
        {"name": "route_softmax", "kind": "route", "T": 1031, "E": 100, "k": 4, "x": "bf16", "score": "softmax", "bias": False,
         "groups": 1, "topk_groups": 1, "renorm": False, "scale": 1.0, "shared": 0},
        # one token through the layer's second output projection
        {"name": "linear_token", "kind": "linear", "T": 1, "N": 4096, "K": 8192, "y": "bf16"},
        # the q up projection of 24 tokens in flight, for an epilogue that takes fp32
        {"name": "linear_batch", "kind": "linear", "T": 24, "N": 32768, "K": 1024, "y": "f32"},
        # sizes that are multiples of nothing but the scales' 32
        {"name": "linear_odd", "kind": "linear", "T": 77, "N": 1000, "K": 4128, "y": "f32"},
        # a prompt's output projection
        {"name": "linear_prompt", "kind": "linear", "T": 4096, "N": 4096, "K": 8192, "y": "bf16"},
        # a decode step of one sequence and of eight: 6 of 256 experts of [2048, 4096] each
        {"name": "experts_token", "kind": "experts", "T": 1, "E": 256, "of": 256, "k": 6, "K": 4096, "I": 2048, "w": "fp4", "limit": 10.0},
        {"name": "experts_step", "kind": "experts", "T": 8, "E": 256, "of": 256, "k": 6, "K": 4096, "I": 2048, "w": "fp4", "limit": 10.0},
        # a server's batch: most experts get a few tokens
        {"name": "experts_batch", "kind": "experts", "T": 100, "E": 256, "of": 256, "k": 6, "K": 4096, "I": 2048, "w": "fp4",
         "limit": 10.0},
        # bf16 experts, half of the model's on this device
        {"name": "experts_bf16", "kind": "experts", "T": 500, "E": 24, "of": 48, "k": 4, "K": 2048, "I": 1408, "w": "bf16", "limit": 0.0},
        # a prompt of 4096 tokens: the largest
        {"name": "experts_prompt", "kind": "experts", "T": 4096, "E": 256, "of": 256, "k": 6, "K": 4096, "I": 2048, "w": "fp4",
         "limit": 10.0},
    ]


def _logint(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["route", "linear", "linear", "experts", "experts"])
    if kind == "route":
        score = rng.choice(["softmax", "sigmoid", "sqrtsoftplus"])
        groups = rng.choice([1, 1, 1, 4, 8])
        E = groups * _logint(rng, 4 if groups > 1 else 8, 512 // groups)
        top = rng.randint(1, groups)
        return {"kind": kind, "T": _logint(rng, 1, 16384), "E": E, "k": rng.randint(1, min(16, top * (E // groups))),
                "x": rng.choice(["f32", "bf16"]), "score": score, "bias": rng.random() < 0.6, "groups": groups, "topk_groups": top,
                "renorm": rng.random() < 0.7, "scale": rng.choice([1.0, 1.5, 2.5]), "shared": rng.choice([0, 0, 1])}
    if kind == "linear":
        K = 32 * _logint(rng, 2, 512)
        N = _logint(rng, 16, 1 << 15)
        N = max(16, min(N, (1 << 26) // K))
        T = _logint(rng, 1, 8192)
        return {"kind": kind, "T": max(1, min(T, (1 << 37) // (N * K))), "N": N, "K": K, "y": rng.choice(["bf16", "f32"])}
    w = rng.choice(["fp4", "fp4", "fp4", "bf16"])
    K, inner = 32 * _logint(rng, 8, 128), 32 * _logint(rng, 8, 64)
    E = _logint(rng, 2, min(256, (1 << 31) // (K * inner) if w == "fp4" else (1 << 29) // (K * inner)))
    of = E * rng.choice([1, 1, 2])
    return {"kind": kind, "T": _logint(rng, 1, 4096), "E": E, "of": of, "k": rng.randint(1, min(6, of)), "K": K, "I": inner, "w": w,
            "limit": rng.choice([0.0, 7.0, 10.0])}


# ---------------------------------------------------------------------------------------------
# inputs

class _Draw:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(int(seed))

    def normal(self, *shape, std=1.0, dtype=torch.float32):
        x = torch.randn(*shape, generator=self.g, device=DEV, dtype=dtype)
        return x if std == 1.0 else x.mul_(std)

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.g, device=DEV)


def _quantised(r, *shape):
    """Codes [.., K/2] and scale bytes [.., K/32] of normal weights [.., K] of deviation K^-0.5: per 32 the
    power of two from amax / 6 up, the nearest e2m1 value, element 2i in the low half of byte i."""
    K = shape[-1]
    rows = math.prod(shape[:-1])
    codes = torch.empty(rows, K // 2, dtype=torch.uint8, device=DEV)
    scales = torch.empty(rows, K // 32, dtype=torch.uint8, device=DEV)
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=DEV)
    step = max(1, (1 << 27) // K)
    for a in range(0, rows, step):
        x = r.normal(min(step, rows - a), K // 32, 32, std=K ** -0.5)
        e = torch.ceil(torch.log2(x.abs().amax(-1, keepdim=True) / 6.0))
        z = x * torch.exp2(-e)
        c = torch.bucketize(z.abs(), edges, out_int32=True).to(torch.uint8) | ((z < 0).to(torch.uint8) << 3)
        codes[a:a + step] = (c[..., ::2] | (c[..., 1::2] << 4)).flatten(-2)
        scales[a:a + step] = (e.squeeze(-1) + 127).to(torch.uint8)
    return codes.view(*shape[:-1], K // 2), scales.view(*shape[:-1], K // 32)


def _weights(r, kind, *shape):
    return _quantised(r, *shape) if kind == "fp4" else r.normal(*shape, std=shape[-1] ** -0.5, dtype=torch.bfloat16)


def prepare(case, seed):
    c, r = case, _Draw(seed)
    st = {"case": dict(c)}
    T = c["T"]
    if c["kind"] == "route":
        x = r.normal(T, c["E"], std=1.5) + r.normal(c["E"], std=0.5)  # some experts are liked more
        st["logits"] = x.to(torch.bfloat16) if c["x"] == "bf16" else x
        st["bias"] = r.normal(c["E"], std=0.1) if c["bias"] else None
        return st
    st["x"] = r.normal(T, c["K"], dtype=torch.bfloat16)
    if c["kind"] == "linear":
        st["codes"], st["scales"] = _quantised(r, c["N"], c["K"])
        return st
    for name, n, k in (("gate", c["I"], c["K"]), ("up", c["I"], c["K"]), ("down", c["K"], c["I"])):
        st[name] = _weights(r, c["w"], c["E"], n, k)
    # k different experts a token, some more popular than others
    like = r.normal(c["of"], std=0.5) - torch.log(-torch.log(r.uniform(T, c["of"]).clamp(1e-9, 1 - 1e-7)))
    st["ids"] = like.topk(c["k"], dim=-1).indices.to(torch.int32)
    w = r.uniform(T, c["k"]) + 0.1
    st["weights"] = 1.5 * w / w.sum(-1, keepdim=True)
    return st


# ---------------------------------------------------------------------------------------------
# the plain forms

def _route_plain(st):
    c = st["case"]
    T, E, k = c["T"], c["E"], c["k"]
    x = st["logits"].double()  # values next to a border
    if c["score"] == "softmax":
        s = torch.exp(x - x.amax(-1, keepdim=True))
        s = s / s.sum(-1, keepdim=True)
    elif c["score"] == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-x))
    else:
        s = torch.sqrt(x.clamp(min=0) + torch.log1p(torch.exp(-x.abs())))
    r = s if st["bias"] is None else s + st["bias"].double()
    rank = x if st["bias"] is None else r  # without a bias the scores' order is the logits'
    if c["groups"] > 1:
        g = r.view(T, c["groups"], -1)
        best = g.sort(dim=-1, descending=True).values[..., :2].sum(-1)
        keep = best.sort(dim=-1, descending=True, stable=True).indices[:, :c["topk_groups"]]
        inside = torch.zeros(T, c["groups"], dtype=torch.bool, device=DEV).scatter_(1, keep, True)
        rank = rank.masked_fill(~inside.repeat_interleave(E // c["groups"], dim=1), -math.inf)
    ids = rank.sort(dim=-1, descending=True, stable=True).indices[:, :k]
    w = s.gather(1, ids)
    if c["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    w = (w * c["scale"]).float()
    n = c["shared"]
    more = torch.arange(E, E + n, device=DEV).expand(T, n)
    return {"ids": torch.cat([ids, more], 1).to(torch.int32), "weights": torch.cat([w, torch.ones(T, n, device=DEV)], 1)}


def _full(w):
    """fp32 weights from bf16 ones, or from codes and scale bytes."""
    if not isinstance(w, tuple):
        return w.float()
    codes, scales = w
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=DEV)
    v = torch.stack([table[(codes & 15).int()], table[(codes >> 4).int()]], dim=-1).flatten(-2)
    s = torch.exp2(scales.float() - 127.0)
    return (v.unflatten(-1, (-1, 32)) * s.unsqueeze(-1)).flatten(-2)


def _pick(w, e):
    """Expert e's weights; e a number or a tensor of one."""
    if isinstance(w, tuple):
        return tuple(_pick(p, e) for p in w)
    return w[e] if isinstance(e, int) else w.index_select(0, e)[0]


def _network_plain(st, x, e):
    lim = st["case"]["limit"]
    g, u = x @ _full(_pick(st["gate"], e)).t(), x @ _full(_pick(st["up"], e)).t()
    if lim:
        g, u = g.clamp(max=lim), u.clamp(-lim, lim)
    return (g / (1.0 + torch.exp(-g)) * u) @ _full(_pick(st["down"], e)).t()


def _experts_plain(st):
    c = st["case"]
    T, E, k = c["T"], c["E"], c["k"]
    x, ids, w = st["x"].float(), st["ids"], st["weights"]
    flat = ids.flatten()
    y = torch.zeros(T, c["K"], device=DEV)
    if T * k <= 16 and c["of"] == E:  # a few rows: one at a time, without a look at the ids on the host
        for p in range(T * k):
            t = p // k
            y[t] += w[t, p % k] * _network_plain(st, x[t:t + 1], flat[p:p + 1])[0]
        return y.to(torch.bfloat16)
    order = torch.argsort(flat, stable=True)
    counts = torch.bincount(flat, minlength=c["of"])[:E].tolist()
    at = 0
    for e, n in enumerate(counts):
        if n:
            p = order[at:at + n]
            t = torch.div(p, k, rounding_mode="floor")
            y.index_add_(0, t, w.flatten()[p][:, None] * _network_plain(st, x[t], e))
            at += n
    return y.to(torch.bfloat16)


def run(state):
    st, c = state, state["case"]
    if not own:
        if c["kind"] == "route":
            return _route_plain(st)
        if c["kind"] == "experts":
            return _experts_plain(st)
        y = st["x"].float() @ _full((st["codes"], st["scales"])).t()
        return y.to(torch.bfloat16) if c["y"] == "bf16" else y
    mla, moe = _own_modules()
    if c["kind"] == "route":
        ids, w = moe.route(st["logits"], c["k"], score=c["score"], bias=st["bias"], groups=c["groups"],
                           topk_groups=c["topk_groups"], renorm=c["renorm"], scale=c["scale"], shared=c["shared"])
        return {"ids": ids, "weights": w}
    if c["kind"] == "linear":
        return mla.linear_fp4(st["x"], st["codes"], st["scales"],
                              out_dtype=torch.bfloat16 if c["y"] == "bf16" else torch.float32)
    return moe.experts(st["x"], st["ids"], st["weights"], st["gate"], st["up"], st["down"], limit=c["limit"] or None)


# ---------------------------------------------------------------------------------------------

def work(case):
    c = case
    T = c["T"]
    if c["kind"] == "route":
        size = 4 if c["x"] == "f32" else 2
        return {"bytes": T * (c["E"] * size + 8 * (c["k"] + c["shared"])) + (4 * c["E"] if c["bias"] else 0), "flops": 10 * T * c["E"]}
    if c["kind"] == "linear":
        N, K = c["N"], c["K"]
        return {"bytes": N * K * 17 // 32 + 2 * T * K + T * N * (2 if c["y"] == "bf16" else 4), "flops": 2 * T * N * K}
    per = 17 / 32 if c["w"] == "fp4" else 2
    used = c["E"] * (1.0 - (1.0 - c["k"] / c["of"]) ** T)  # experts that some token has chosen
    pairs = T * c["k"] * c["E"] / c["of"]
    return {"bytes": int(used * 3 * c["K"] * c["I"] * per) + 4 * T * c["K"] + 8 * T * c["k"],
            "flops": int(6 * pairs * c["K"] * c["I"])}


def _decoded(w):
    """float64 weights: sign, exponent and mantissa of every code, times 2^(byte - 127)."""
    if not isinstance(w, tuple):
        return w.double()
    codes, scales = w
    n = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.int32, device=DEV)
    n[..., ::2], n[..., 1::2] = codes.int() % 16, codes.int() // 16
    e, m = n // 2 % 4, n % 2
    v = torch.where(e == 0, 0.5 * m, (1.0 + 0.5 * m) * 2.0 ** (e - 1)).double()
    v = torch.where(n >= 8, -v, v)
    return v * torch.pow(torch.tensor(2.0, dtype=torch.float64, device=DEV), scales.double() - 127).repeat_interleave(32, -1)


def exact(case, seed):
    c, dd = case, torch.float64
    st = prepare(case, seed)
    if c["kind"] == "linear":
        return st["x"].to(dd) @ _decoded((st["codes"], st["scales"])).mT
    if c["kind"] == "route":
        x = st["logits"].to(dd)
        s = {"softmax": lambda: torch.softmax(x, -1), "sigmoid": lambda: torch.sigmoid(x),
             "sqrtsoftplus": lambda: torch.logaddexp(x, torch.zeros_like(x)).sqrt()}[c["score"]]()
        v = s if st["bias"] is None else s + st["bias"].to(dd)
        if c["groups"] > 1:
            per = c["E"] // c["groups"]
            two = v.unflatten(1, (-1, per)).topk(min(2, per), -1).values.sum(-1)
            place = torch.argsort(torch.argsort(-two, dim=1, stable=True), dim=1)
            v = torch.where((place < c["topk_groups"]).repeat_interleave(per, 1), v, -math.inf)
        w = s.gather(1, v.topk(c["k"], -1).indices)  # largest first
        if c["renorm"]:
            w = w / w.sum(1, keepdim=True)
        return {"ids": None, "weights": torch.cat([w * c["scale"], torch.ones(c["T"], c["shared"], dtype=dd, device=DEV)], 1)}
    out = torch.zeros(c["T"], c["K"], dtype=dd, device=DEV)
    x, cap = st["x"].to(dd), c["limit"] or math.inf
    for e in range(c["E"]):
        mine = (st["ids"] == e)
        t = mine.any(1).nonzero()[:, 0]
        if not len(t):
            continue
        share = (st["weights"].to(dd) * mine).sum(1)[t, None]
        a = torch.minimum(x[t] @ _decoded(_pick(st["gate"], e)).mT, torch.tensor(cap, dtype=dd, device=DEV))
        b = (x[t] @ _decoded(_pick(st["up"], e)).mT).clamp(-cap, cap)
        out[t] += share * ((a * torch.sigmoid(a) * b) @ _decoded(_pick(st["down"], e)).mT)
    return out
