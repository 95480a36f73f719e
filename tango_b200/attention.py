"""Dot-product attention over the edges of a graph on 8-bit rows, forward, backward, and for a few nodes at a time.

In place of the chain sddmm_u_dot_v -> edge_softmax -> spmm_u_mul_e of the reference's transformer layer
(evaluation/test_HGT.py:58-62): one kernel per direction, no array of edges, one scale per node and head instead of one per
tensor, probabilities in fp32.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _native
from .rows8 import Packed8


def edge_attention(g, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: Optional[float] = None) -> torch.Tensor:
    """out[v] = sum over the incoming edges u -> v of softmax_u(scale * <q[v], k[u]>) * v[u], per head; a node without incoming
    edges gets zeros.  q, k, v: [N, H, D] of one type (fp32, bf16 or fp16), D up to 512; scale: 1 / sqrt(D) by default.

    All three are rounded to 8 bits with one scale per node and head (`rows8.pack8` with groups of D); scores, softmax and
    sums are fp32.  The backward pass computes the probabilities anew from the 8-bit tensors and two floats per node and head
    -- all that is kept -- with the incoming gradient rounded to 8 bits in the same way, and takes the rounding as the
    identity, as the other operators of this package do.  A score above fp32's range makes a node
    NaN; one below it weighs nothing, and a node without others gets NaN."""
    backward = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    return _native.call(_native.ops.edge_attention, _native.edge_graph(g, backward), q, k, v, _scale(q, scale))


def edge_attention_rows(g, rows: torch.Tensor, q: torch.Tensor, k8: Packed8, v8: Packed8, scale: Optional[float] = None) -> torch.Tensor:
    """edge_attention of the nodes `rows` ([R], int32 or int64; any order, repeats allowed) whose queries are q [R, H, D], over
    keys and values of all nodes that are kept in 8 bits: `pack8(k, D)` and `pack8(v, D)` of [N, H, D].  For serving: no
    gradient.  A row id outside the graph gives a row of NaN (checking it here would wait for the GPU).  A long row is shared out
    over more blocks when few rows are asked for, so that the last bits of a node's result may depend on how many are."""
    for name, t in (("k8", k8), ("v8", v8)):
        if not isinstance(t, Packed8):
            raise TypeError(f"edge_attention_rows: {name} must come from pack8, not {type(t).__name__}")
        if q.dim() != 3 or tuple(t.shape) != (g.num_nodes(), *q.shape[1:]) or t.group != q.shape[2]:
            raise ValueError(f"edge_attention_rows: {name} must be pack8(x, {q.shape[-1]}) of an x [{g.num_nodes()}, "
                             f"{', '.join(map(str, q.shape[1:]))}], not of {tuple(t.shape)} in groups of {t.group}")
    return _native.call(_native.ops.edge_attention_rows, _native.rows_graph(g), rows, q, k8.codes, k8.scales, v8.codes, v8.scales,
                        _scale(q, scale))


def _scale(q, scale) -> float:
    return 1.0 / math.sqrt(max(q.shape[-1], 1)) if scale is None else float(scale)
