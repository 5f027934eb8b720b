"""A mixture-of-experts layer for a few tokens (b200spmm_moe of the C ABI).

    layer = MoeLayer(router, gate_up, down, top_k=8)
    y = layer.forward(x)                                       # x [tokens, hidden] float16 or bfloat16
    y, ids, shares = layer.forward(x, return_routing=True)
    y = layer.experts(x, ids, shares)                          # with a routing of the caller's own

Experts in 16 bits, or in 4 as ``Int4Matrix``: of all experts, one after the other.  Each chosen expert is read once for all of its tokens (once for every
16, or for as many as there is room for in a block's shared memory where those are fewer: 8 at a hidden size of 8,192).
The reference has no such operator.
"""
from __future__ import annotations

from . import _capi as capi
from .fp4 import _lib, _on
from .int4 import Int4Matrix


class MoeLayer:
    """y = sum over a token's ``top_k`` experts of share * down(silu(gate x) * up x).

    ``router`` [experts, hidden], float16 or bfloat16: shares are the softmax of x routerᵀ, of the largest (of equal ones the first), divided by their sum where
    ``renormalize``.  None: for ``experts`` alone, whose number is then given where the matrices are Int4Matrix.
    ``gate_up``: [experts, 2 inner, hidden], the gate's rows before up's, and ``down`` [experts, hidden, inner], of the router's type, rows starting on 16
    bytes; or Int4Matrix of experts * 2 * inner rows and of experts * hidden rows.  All are kept, not copied: their
    values may change, and a call refuses them once they have another storage, type or shape."""

    __slots__ = ("top_k", "renormalize", "_parts", "_m")

    def __init__(self, router, gate_up, down, *, top_k: int, renormalize: bool = True, experts: int | None = None):
        codes = type(gate_up) is Int4Matrix, type(down) is Int4Matrix
        if codes[0] != codes[1]:
            raise ValueError("gate_up and down must both be Int4Matrix, or both 16-bit tensors")
        if not codes[0] and not all(getattr(w, "dim", lambda: 0)() == 3 for w in (gate_up, down)):
            raise ValueError("gate_up must be [experts, 2 inner, hidden] and down [experts, hidden, inner], float16 or bfloat16, or both Int4Matrix")
        n = router.shape[0] if router is not None else experts if codes[0] else gate_up.shape[0]
        if n is None:
            raise ValueError("without a router, the number of experts must be given")
        if experts is not None and experts != n:
            raise ValueError("the router has another number of experts")
        hidden, inner = (gate_up.cols, down.cols) if codes[0] else (gate_up.shape[2], down.shape[2])
        self._m = _lib().moe_layer(router, gate_up._m if codes[0] else gate_up, down._m if codes[1] else down, n, hidden, inner, top_k, bool(renormalize))
        self._parts = (router, gate_up, down)
        self.top_k, self.renormalize = top_k, bool(renormalize)

    router = property(lambda self: self._parts[0])
    gate_up = property(lambda self: self._parts[1])
    down = property(lambda self: self._parts[2])

    def _tensors(self):
        for p in self._parts:
            yield from (t for t in p._arrays if t is not None) if type(p) is Int4Matrix else () if p is None else (p,)

    def _run(self, X, out, routing, ids, shares, stream):
        if stream is not None:
            with _on(stream, *self._tensors(), *(t for t in (X, out, ids, shares) if t is not None)):
                return self._run(X, out, routing, ids, shares, None)
        y, i, s = _lib().moe(self._m, X, out, routing, ids, shares)
        if type(y) is int:
            raise capi.SpmmError(y, "b200spmm_moe" if ids is None else "b200spmm_moe_experts")
        return (y, i, s) if routing else y

    def forward(self, X, out=None, return_routing: bool = False, stream=None):
        """The layer for X [tokens, hidden], up to 256 tokens, in its type; with ``return_routing`` also ids [tokens, top_k] int32 and shares float32.
        Asynchronous.  There is no gradient: nothing may require one while gradients are recorded, nor have a tangent."""
        return self._run(X, out, bool(return_routing), None, None, stream)

    def experts(self, X, ids, shares, out=None, stream=None):
        """The experts alone, for a routing that is given: ids [tokens, top_k] int32 or int64, shares [tokens, top_k] float32.  Ids that are no
        expert's (-1, say, of a padded token) are left out; a token without any gets zeros; an expert may come twice."""
        if ids is None or shares is None:
            raise ValueError("ids and shares are given together")
        return self._run(X, out, False, ids, shares, stream)
