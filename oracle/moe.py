"""The steps between a router's choices and the rows of a grouped layout, restated in loops and 64 bits (test infrastructure, never
shipped). Written from the definitions: the reference has no stand-alone counterpart to pin them to."""

from __future__ import annotations

import torch

from .sf_layout import align


def moe_rows(choices: int, experts: int, alignment: int) -> int:
    """The most rows that `choices` choices of `experts` experts can need."""
    used = min(choices, experts)
    return alignment * (used + (choices - used) // alignment) if used else 0


def moe_sort_ref(idx: torch.Tensor, experts: int, alignment: int = 256, max_m=None):
    """(layout, token_rows, row_choices) as int32 tensors on the CPU."""
    flat = [int(e) for e in idx.reshape(-1).tolist()]
    members = [[i for i, e in enumerate(flat) if e == g] for g in range(experts)] if len(flat) * experts < 1 << 22 else None
    if members is None:
        members = [[] for _ in range(experts)]
        for i, e in enumerate(flat):
            if 0 <= e < experts:
                members[e].append(i)
    rows = experts * max_m if max_m else moe_rows(len(flat), experts, alignment)
    layout, token_rows, row_choices, start = [], [-1] * len(flat), [-1] * rows, 0
    for g, choices in enumerate(members):
        if max_m:
            start, choices = g * max_m, choices[:max_m]
        for r, i in enumerate(choices):
            token_rows[i] = start + r
            row_choices[start + r] = i
        layout.append(len(choices) if max_m else start + len(choices))
        start = align(start + len(choices), alignment)
    as_int = lambda v, *shape: torch.tensor(v, dtype=torch.int32).view(*shape)  # noqa: E731
    return as_int(layout, -1), as_int(token_rows, *idx.shape), as_int(row_choices, experts, max_m) if max_m else as_int(row_choices, -1)


def moe_padding(layout: torch.Tensor, rows: int, alignment: int, max_m=None) -> torch.Tensor:
    """bool [rows]: the rows that `zero_padding` writes."""
    out = torch.zeros(rows, dtype=torch.bool)
    for g, p in enumerate(layout.tolist()):
        if max_m:
            out[g * max_m + p:(g + 1) * max_m] = True
        else:
            out[p:align(p, alignment)] = True
    return out


def moe_combine_ref(rows: torch.Tensor, token_rows: torch.Tensor, weights=None):
    """float64 (sum, sum of the terms' magnitudes) of `rows` [R, H] on the CPU."""
    tokens, topk = token_rows.shape
    out = torch.zeros(tokens, rows.size(-1), dtype=torch.float64)
    size = torch.zeros_like(out)
    for t in range(tokens):
        for j in range(topk):
            r = int(token_rows[t, j])
            if 0 <= r < rows.size(0):
                term = rows[r].double() * (1.0 if weights is None else weights[t, j].double())
                out[t] += term
                size[t] += term.abs()
    return out, size


def moe_combine_grad_ref(grad_out: torch.Tensor, rows: torch.Tensor, token_rows: torch.Tensor, weights: torch.Tensor):
    """float64 (grad_rows, grad_weights, sums of the magnitudes of grad_weights' terms); rows without a choice are NaN."""
    grad_rows = torch.full(rows.shape, float('nan'), dtype=torch.float64)
    grad_weights = torch.zeros(token_rows.shape, dtype=torch.float64)
    size = torch.zeros_like(grad_weights)
    for t in range(token_rows.size(0)):
        for j in range(token_rows.size(1)):
            r = int(token_rows[t, j])
            if 0 <= r < rows.size(0):
                grad_rows[r] = weights[t, j].double() * grad_out[t].double()
                terms = rows[r].double() * grad_out[t].double()
                grad_weights[t, j], size[t, j] = terms.sum(), terms.abs().sum()
    return grad_rows, grad_weights, size
