"""The expert network of a layer (``oracle/decode_engine.py:122-133``), what follows the attention layer.

* ``route``    the router's scores, the choice of each token's experts and their weights;
* ``experts``  the tokens through their experts' gated networks, the outputs weighted and summed;
* ``pack_fp4`` weights to e2m1 codes with a power-of-two scale per 32, the form both ``experts`` and
  ``mla.linear_fp4`` multiply with as it is;
* ``ExpertLayer`` the three products of a layer in one call, with the shared expert as one more of the experts.

Which experts a token goes to stays on the GPU: the calls are stream-ordered, read nothing back and can be captured
into a graph that is replayed with other tokens.
"""
from dataclasses import dataclass
from typing import Optional, Union

import torch

from . import _lib, ops, qat


def route(logits, k, score="softmax", bias=None, groups=1, topk_groups=1, renorm=True, scale=1.0, shared=0, ids=None):
    """Each token's k experts: logits [T, E] fp32 or bf16 (rows may lie apart) -> ids [T, k + shared] int32 and weights
    of the same shape, fp32.

    ``score``: "softmax" of the row, "sigmoid" or "sqrtsoftplus" of each logit.  Experts are ranked by score + ``bias``
    [E] (which the weights do not see).  With ``groups`` > 1 only the experts of the ``topk_groups`` groups whose two
    largest values sum highest take part.  Ids come best first; ties go to the lower id, and the order is that of the exact
    values.  The weights are the scores of the ids, divided by their sum (``renorm``; 0 where it is 0), times
    ``scale``.  ``shared`` columns E, E + 1, .. of weight 1 follow: experts that every token uses, stored behind the E.
    ``ids`` [T, k] int32 are taken instead of a choice (a layer whose table gives every token its experts): those and
    their weights are returned, 0 for one outside 0 .. E-1.  Logits of -inf and NaN rank last.  E up to 1024, k + ``shared`` up to
    64."""
    if score not in _lib.SCORES:
        raise ValueError(f"score must be one of {sorted(_lib.SCORES)}, got {score!r}")
    return ops.route_op(logits, bias, int(k), _lib.SCORES[score], int(groups), int(topk_groups), bool(renorm), float(scale),
                        int(shared), ids)


def experts(x, ids, weights, gate, up, down, limit=None):
    """y [T, K] bf16 with y[t] = sum_j weights[t, j] down_e(silu(min(g, limit)) * clamp(u, -limit, limit)), g = gate_e(x[t]),
    u = up_e(x[t]), e = ids[t, j] (``limit`` None: no clamp).  x [T, K] bf16 (rows may lie apart), ids [T, k] int32,
    weights [T, k].  gate, up [E, I, K] and down [E, K, I]: dense bf16 tensors, or (codes, scales) pairs of ``pack_fp4``.
    An id outside 0 .. E-1 adds nothing: a device that holds some of the experts passes ids less its first one's.  The same
    id twice counts twice.  Sums are fp32, the hidden row (its weight in it) and y are rounded to bf16.  The same call gives the same
    bits; in a batch of up to 16 tokens the ids of the others may change the order of a token's fp32 sums.  E up to 1024, k up to 64;
    any number of tokens."""
    (gate, gs), (up, us), (down, ds) = (w if isinstance(w, (tuple, list)) else (w, None) for w in (gate, up, down))
    return ops.experts_op(x, ids, weights, gate, up, down, gs, us, ds, float("inf") if limit is None else float(limit))


def pack_fp4(w):
    """(codes [..., K/2], scales [..., K/32]) of weights [..., K] (fp32 or bf16, K a multiple of 32): the nearest e2m1
    values under a power of two per 32 (``v4mlx/qat.py:23-31`` without the rotation).  32 weights with one that is not finite are
    NaN, all of them."""
    if w.shape[-1] % 32:
        raise ValueError(f"rows of a multiple of 32 weights are packed, got {w.shape[-1]}")
    codes, scales = qat.fp4_pack(w.reshape(-1, 32), rotate=False)
    return codes.view(*w.shape[:-1], w.shape[-1] // 2), scales.view(*w.shape[:-1], w.shape[-1] // 32)


Weight = Union[torch.Tensor, tuple]


@dataclass
class ExpertWeights:
    """One layer's expert network (``blk.{L}.ffn_*``): router [E, K] bf16 or fp32; gate, up [E + shared, I, K] and down
    [E + shared, K, I], bf16 or ``pack_fp4`` pairs, the shared experts behind the E routed ones; bias [E] (layers that choose
    by score) or table [vocabulary, k] int32 (layers that choose by token)."""
    router: torch.Tensor
    gate: Weight
    up: Weight
    down: Weight
    bias: Optional[torch.Tensor] = None
    table: Optional[torch.Tensor] = None


class ExpertLayer:
    """The expert network of one layer: y = layer(xn) for xn [..., K] bf16, the normed input; 6 of the routed experts and the
    shared one by default, sqrt-softplus scores, weights summing to 1.5, the gate and up products clamped at 10
    (``oracle/decode_engine.py:46,122-133``).  Any number of tokens; a decode step and a prompt are the same call."""

    def __init__(self, w: ExpertWeights, k=6, score="sqrtsoftplus", groups=1, topk_groups=1, renorm=True, scale=1.5, limit=10.0):
        gate = w.gate[0] if isinstance(w.gate, (tuple, list)) else w.gate
        shared = gate.shape[0] - w.router.shape[0]
        if shared < 0:
            raise ValueError(f"{w.router.shape[0]} routed experts, but weights of {gate.shape[0]}")
        self.w, self.k, self.limit, self.shared = w, k, limit, shared
        self.choice = dict(score=score, groups=groups, topk_groups=topk_groups, renorm=renorm, scale=scale)

    def logits(self, xn):
        """The router's product [T, E], fp32."""
        r = self.w.router
        return ops.linear_op(xn if r.dtype == xn.dtype else xn.to(r.dtype), r, 1, torch.float32)

    def __call__(self, xn, tokens=None):
        """xn [..., K] bf16 -> [..., K] bf16.  ``tokens`` [...]: the token ids, which a layer with a table chooses by; one outside
        the table (a padded batch's) has the shared experts alone."""
        x = xn.reshape(-1, xn.shape[-1])
        if x.shape[0] == 0:
            return torch.empty_like(xn)
        ids = None
        if self.w.table is not None:
            if tokens is None:
                raise ValueError("this layer chooses its experts by token: tokens are needed")
            table = self.w.table
            at = tokens.reshape(-1).to(table.device, torch.long)
            row = at.clamp(0, table.shape[0] - 1)       # (no row is read that is not there)
            ids = table[row].masked_fill_((row != at)[:, None], -1)
        ids, weights = route(self.logits(x), self.k, bias=self.w.bias, shared=self.shared, ids=ids, **self.choice)
        return experts(x, ids, weights, self.w.gate, self.w.up, self.w.down, self.limit).view(xn.shape)
