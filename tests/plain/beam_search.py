"""Beam search from what its parameters say, looking at every continuation of every beam."""

from __future__ import annotations

import torch


def search(next_logits, prompt, width, max_tokens, length_penalty=1.0, early_stopping=False, stops=(), gaps=None):
    """The ended sequences ``(output tokens, log-probability, score, reason)``, best first.  ``next_logits(tokens)``: the logits behind a
    whole sequence.  Of all continuations of the beams those that end and are among the ``width`` best have ended; the
    ``width`` best that do not end are followed.  ``gaps`` (a list) gets every difference that a choice went by: of what is followed
    or ended and what is not, of scores that are ranked, of the best living score and the worst ended one."""
    beams, ended, gaps = [((), 0.0)], [], gaps if gaps is not None else []
    for step in range(1, max_tokens + 1):
        everyone = []
        for b, (tokens, log_prob) in enumerate(beams):
            lp = torch.log_softmax(next_logits(list(prompt) + list(tokens)).double(), dim=0)
            everyone += [(log_prob + x, b, t) for t, x in enumerate(lp.tolist())]
        everyone.sort(key=lambda c: (-c[0], c[1], c[2]))
        going_on = [c for c in everyone if c[2] not in stops]
        if any(t in stops for _, _, t in everyone[:width + 1]):
            gaps += [a[0] - b[0] for a, b in zip(everyone[:width], everyone[1:])]
        gaps += [a[0] - b[0] for a, b in zip(going_on[width - 1:width], going_on[width:width + 1])]
        for log_prob, b, t in everyone[:width]:
            if t in stops:
                ended.append(([*beams[b][0], t], log_prob, log_prob / step ** length_penalty, "stop"))
        beams = [((*beams[b][0], t), log_prob) for log_prob, b, t in going_on[:width]]
        if step == max_tokens:
            ended += [(list(t), p, p / step ** length_penalty, "length") for t, p in beams]
        ended.sort(key=lambda e: -e[2])
        gaps += [a[2] - b[2] for a, b in zip(ended, ended[1:width + 1])]
        del ended[width:]
        if step == max_tokens or not beams:
            break
        if len(ended) == width:
            best = max(p for _, p in beams) / step ** length_penalty
            if not early_stopping:
                gaps.append(abs(best - ended[-1][2]))
            if early_stopping or best <= ended[-1][2]:
                break
    return ended
