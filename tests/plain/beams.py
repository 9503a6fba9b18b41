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


def search(next_logits, prompt, width, max_tokens, length_penalty=1.0, early_stopping=False, stops=()):
    """Beam search by its definition: ``next_logits(tokens)`` are the logits behind a whole sequence.  Returns the ended
    sequences ``(output tokens, log-probability, score, reason)``, best first, and the smallest difference that a choice went
    by: of the last candidate that was taken and the first that was not, of scores that were ranked, of the best living
    score and the worst ended one (what a search with other rounding may choose otherwise)."""
    beams, ended, gap = [((), 0.0)], [], math.inf
    for step in range(1, max_tokens + 1):
        everyone = []
        for b, (tokens, log_prob) in enumerate(beams):
            lp = torch.log_softmax(next_logits(list(prompt) + list(tokens)).double(), dim=0)
            best = torch.sort(lp, descending=True, stable=True).indices[:2 * width + 1].tolist()
            everyone += [(log_prob + float(lp[t]), b, t) for t in best]
        everyone.sort(key=lambda c: (-c[0], c[1], c[2]))
        following, left = [], None
        for rank, (log_prob, b, token) in enumerate(everyone[:2 * width]):
            tokens = beams[b][0] + (token,)
            if token in stops:
                if rank < width:
                    ended.append((list(tokens), log_prob, log_prob / step ** length_penalty, "stop"))
            elif len(following) < width:
                following.append((tokens, log_prob))
            elif left is None:
                left = log_prob
        if left is not None:
            gap = min(gap, following[-1][1] - left)
        for at in (width, 2 * width):         # what may end is cut off there, and what is looked at
            if len(everyone) > at and (at == width and (everyone[at - 1][2] in stops or everyone[at][2] in stops) or at > width and left is None):
                gap = min(gap, everyone[at - 1][0] - everyone[at][0])
        if step == max_tokens:
            ended += [(list(t), p, p / step ** length_penalty, "length") for t, p in following]
        ended = sorted(ended, key=lambda e: -e[2])
        gap = min([gap] + [a[2] - b[2] for a, b in zip(ended, ended[1:width + 1])])
        ended = ended[:width]
        if step == max_tokens or not following:
            break
        if len(ended) == width:
            best = max(p for _, p in following) / step ** length_penalty
            if not early_stopping:
                gap = min(gap, abs(best - ended[-1][2]))
            if early_stopping or best <= ended[-1][2]:
                break
        beams = following
    return ended, gap
