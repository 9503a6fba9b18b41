"""Beam search in plain 64-bit torch and Python: selection over beams and vocabulary, rows that follow their beams,
attention of one token per sequence from pages."""

from __future__ import annotations

import math

import torch

LARGEST = torch.finfo(torch.float32).max


def candidate_scores(logits: torch.Tensor, scores: torch.Tensor) -> torch.Tensor:
    """``[rows, vocab]`` in 64 bits: score of the beam plus log-softmax; -inf for what is no candidate."""
    x = logits.detach().cpu().float().double()
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x).clamp(max=LARGEST)
    out = torch.full_like(x, -math.inf)
    for row in range(x.shape[0]):
        s = float(scores[row])
        m = x[row].max()
        if math.isfinite(s) and m > -math.inf:
            out[row] = s + ((x[row] - m) - (x[row] - m).exp().sum().log())
    return out


def select(logits, scores, cu_beams, count):
    """Per request the candidates ``(score, beam, token)``, best first, ties by beam, logit, token; at most ``count``.  (A
    beam's scores are in the order of its logits; next to a score of 2^127 64 bits do not tell logits apart that differ by
    less than 2^74, so the logits themselves are asked.)"""
    total = candidate_scores(logits, scores)
    x = logits.detach().cpu().float()
    out = []
    for lo, hi in zip(cu_beams, cu_beams[1:]):
        best = []
        for row in range(lo, hi):
            order = torch.sort(torch.nan_to_num(x[row], nan=-math.inf, posinf=LARGEST, neginf=-math.inf), descending=True, stable=True).indices[:count].tolist()
            best += [(float(total[row, t]), row - lo, t) for t in order if float(total[row, t]) > -math.inf]
        best.sort(key=lambda c: (-c[0], c[1]))      # stable: a beam's own stay in their order
        out.append(best[:count])
    return out


def reorder(tensor: torch.Tensor, slots, parents) -> torch.Tensor:
    """The tensor after the rows have followed their beams."""
    out = tensor.clone()
    for s, p in zip(slots, parents):
        for b, parent in enumerate(p):
            if 0 <= parent < len(s) and 0 <= s[b] < tensor.shape[0] and 0 <= s[parent] < tensor.shape[0]:
                out[s[b]] = tensor[s[parent]]
    return out


def attend(q, k_pages, v_pages, tables, ctx_lens, heads, kv_heads, dim, scale, sinks=None):
    """(outputs, sum of |probability * value|) ``[rows, heads * dim]`` in 64 bits; keys on pages that are not there do not
    count."""
    q, k_pages, v_pages = (t.detach().cpu().double() for t in (q, k_pages, v_pages))
    nb, _, page, _ = k_pages.shape
    out = torch.zeros(q.shape[0], heads * dim, dtype=torch.float64)
    weight = torch.zeros_like(out)
    for i, n in enumerate(ctx_lens):
        keys = [j for j in range(min(n, len(tables[i]) * page)) if 0 <= tables[i][j // page] < nb]
        if not keys:
            continue
        blocks = torch.tensor([tables[i][j // page] for j in keys])
        at = torch.tensor([j % page for j in keys])
        for h in range(heads):
            kv = h // (heads // kv_heads)
            s = (k_pages[blocks, kv, at] @ q[i, h * dim:(h + 1) * dim]) * scale
            if sinks is not None:
                s = torch.cat([s, sinks[h:h + 1].detach().cpu().double()])
            p = torch.softmax(s, dim=0)[:len(keys)]
            v = v_pages[blocks, kv, :, at]
            out[i, h * dim:(h + 1) * dim] = p @ v
            weight[i, h * dim:(h + 1) * dim] = p @ v.abs()
    return out, weight
