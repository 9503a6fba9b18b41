"""What beam search adds to the engine's work on the device, by itself: the operators, their plain form in
elementary torch operations, and their definition in 64 bits.

* ``select``: the best continuations of every request over its beams and the vocabulary.  With logits ``l`` and
  running scores ``S`` of the beams, the candidate (beam, token) scores ``S + l - log sum exp l``; the ``count`` best
  of a request are wanted, best first, equal scores by the lower beam, then the lower token.
* ``reorder``: what beams own (their last cache page, their recurrent state, in every layer) follows the
  beams that were selected: row ``slots[b]`` of every tensor becomes what row ``slots[parents[b]]`` was.
* ``attend``: one token of every beam attends over the paged cache; the beams of a request share the pages of
  their first keys (the prompt) and have pages of their own behind them.
"""

from __future__ import annotations

import math

import torch

own = False          # whether ``run`` makes the framework's calls or computes the plain form

DEV = "cuda"
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
PAGE = 16            # tokens of a cache page, the engine's default


# ------------------------------------------------------------------------------------- cases
def _select(requests, beams, vocab, count, dtype="float32", ragged=False):
    """``beams`` of every request (``ragged``: from none to so many), ``count`` candidates wanted of each."""
    return {"op": "select", "requests": requests, "beams": beams, "vocab": vocab, "count": count, "dtype": dtype,
            "ragged": ragged}


def _reorder(requests, beams, layers, row, tensors, dtype="bfloat16", spare=0):
    """``layers`` times ``tensors`` tensors, rows of ``row`` elements, ``spare`` further elements between rows."""
    return {"op": "reorder", "requests": requests, "beams": beams, "layers": layers, "row": row, "tensors": tensors,
            "dtype": dtype, "spare": spare}


def _attend(groups, beams, shared, tail, heads, kv_heads, dim, dtype="bfloat16", ragged=False, sinks=False, page=PAGE):
    """``beams`` of every request behind ``shared`` common keys, with up to ``tail`` keys of their own each
    (``ragged``: from one beam, and from a sixteenth of the common keys, on)."""
    return {"op": "attend", "groups": groups, "beams": beams, "shared": shared, "tail": tail, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "ragged": ragged, "sinks": sinks, "page": page}


def listed():
    return [dict(c, name=n) for n, c in (
        # one user of a small model: what counts is the latency of a step
        ("select_small", _select(1, 4, 8192, 8)),
        # a handful of requests translated at once, the vocabulary of the 1B and 8B models
        ("select_served", _select(8, 4, 128256, 8)),
        # a loaded batch server
        ("select_loaded", _select(64, 8, 128256, 16)),
        # requests with beams of their own number each, logits as a bf16 head leaves them, an odd vocabulary
        ("select_ragged_bf16", _select(23, 12, 50001, 24, "bfloat16", ragged=True)),
        # the last pages (K and V) of one request's beams, 16 layers of 8 heads of 64
        ("reorder_pages_small", _reorder(1, 4, 16, 8 * PAGE * 64, 2)),
        # and of a loaded server's, 32 layers of 8 heads of 128
        ("reorder_pages_loaded", _reorder(32, 8, 32, 8 * PAGE * 128, 2)),
        # matrix memories of a recurrent model: 8 heads of 128 by 256 and as many normalisers, in 32 bits
        ("reorder_states", _reorder(8, 4, 8, 8 * (128 * 256 + 128 + 1), 1, "float32")),
        # one user, a question of 300 tokens
        ("attend_small", _attend(1, 4, 300, 20, 32, 8, 64)),
        # eight requests of uneven prompts and beams, a sink in the softmax
        ("attend_served", _attend(8, 5, 2900, 90, 32, 8, 64, ragged=True, sinks=True)),
        # long documents behind wide heads
        ("attend_long", _attend(4, 8, 32768, 250, 32, 8, 128)),
        # 24 heads over 8, wider searches of middling prompts
        ("attend_wide", _attend(12, 16, 1777, 130, 24, 8, 128)),
        # the 32-bit engine
        ("attend_fp32", _attend(3, 4, 1500, 61, 32, 8, 64, "float32")),
    )]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["select", "reorder", "attend"])
    beams = _log_int(rng, 1, 16)
    if op == "select":
        vocab = _log_int(rng, 500, 128256)
        requests = _log_int(rng, 1, max(1, min(64, 64 * 8 // beams)))
        return _select(requests, beams, vocab, rng.choice([beams, 2 * beams, 2 * beams]),
                       "bfloat16" if rng.random() < 0.3 else "float32", ragged=rng.random() < 0.4)
    if op == "reorder":
        beams = max(beams, 2)
        requests = _log_int(rng, 1, max(1, 32 * 8 // beams))
        most = 32 * 8 * 32 * 2 * 8 * PAGE * 128 * 2 // (requests * beams)       # bytes of a beam, by the largest listed case
        if rng.random() < 0.6:
            row = rng.choice([1, 2, 4, 8]) * rng.choice([8, 16, 32]) * rng.choice([16, 32, 64, 80, 128])
            dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
            size = 2 if dtype == "bfloat16" else 4
            return _reorder(requests, beams, _log_int(rng, 1, max(1, min(32, most // (2 * row * size)))), row, 2, dtype)
        row = _log_int(rng, 33, 264200)
        return _reorder(requests, beams, _log_int(rng, 1, max(1, min(32, most // (row * 4)))), row, 1, "float32",
                        spare=rng.choice([0, 0, 1, 7, 12]))
    dtype = "float32" if rng.random() < 0.25 else "bfloat16"
    heads, kv_heads, dim = rng.choice([(32, 8, 64), (32, 8, 128), (24, 8, 128), (8, 4, 64), (16, 1, 256), (6, 2, 80),
                                       (4, 4, 32), (4, 2, 16)])
    size = 2 if dtype == "bfloat16" else 4
    groups = _log_int(rng, 1, 16)
    shared = _log_int(rng, 1, min(32768, 4 * 32768 * 8 * 128 * 2 // (groups * kv_heads * dim * size)))
    tail = _log_int(rng, 1, min(512, max(1, 32 * 250 * 8 * 128 * 2 // (groups * beams * kv_heads * dim * size))))
    return _attend(groups, beams, shared, tail, heads, kv_heads, dim, dtype, ragged=rng.random() < 0.5,
                   sinks=rng.random() < 0.2, page=rng.choice([8, 16, 16, 32]))


# ------------------------------------------------------------------------------------- layouts, from the case alone
def _counts(case):
    """Beams of every request (``select``)."""
    r, w = case["requests"], case["beams"]
    return [(7 * i + w) % (w + 1) for i in range(r)] if case["ragged"] else [w] * r


def _groups(case):
    """(beams, shared keys, own keys of every beam) of every group (``attend``)."""
    out = []
    for g in range(case["groups"]):
        w, n = case["beams"], case["shared"]
        if case["ragged"] and g:
            w, n = 1 + (5 * g + 2) % w, max(1, n * (1 + (11 * g) % 16) // 16)
        out.append((w, n, [1 + (37 * g + 13 * b + case["tail"] - 1) % case["tail"] for b in range(w)]))
    return out


def _parents(case, seed):
    """Beam ``b`` of a request goes on from beam ``parents[b]``: those that have descendants keep one in their own
    place, so that what is moved is never moved on."""
    gen = torch.Generator().manual_seed(seed + 1)
    r, w = case["requests"], case["beams"]
    out = torch.empty(r, w, dtype=torch.int64)
    for i in range(r):
        kept = torch.randperm(w, generator=gen)[: 1 + int(torch.randint(0, w, (1,), generator=gen))]
        out[i] = kept[torch.randint(0, len(kept), (w,), generator=gen)]
        out[i, kept] = kept
    return out


# ------------------------------------------------------------------------------------- inputs
def _inputs(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    state = {"case": case}
    if case["op"] == "select":
        counts = _counts(case)
        rows, vocab = sum(counts), case["vocab"]
        # a head's logits: broad, with a handful of likely tokens, some tokens ruled out
        logits = torch.randn(rows, vocab, generator=gen, device=DEV) * 2.0
        likely = torch.randint(0, vocab, (rows, 24), generator=gen, device=DEV)
        logits.scatter_add_(1, likely, torch.rand(rows, 24, generator=gen, device=DEV) * 9.0)
        logits[:, torch.randint(0, vocab, (3,), generator=gen, device=DEV)] = -math.inf
        scores = -torch.rand(rows, generator=gen, device=DEV) * 8.0 - 4.0
        scores[torch.rand(rows, generator=gen, device=DEV) < 0.05] = -math.inf      # beams that have ended
        cu = torch.tensor([0] + counts).cumsum(0)
        state.update(logits=logits.to(DTYPES[case["dtype"]]), scores=scores, counts=counts,
                     cu=cu.to(torch.int32).to(DEV),
                     where=torch.tensor([i * case["beams"] + b for i, c in enumerate(counts) for b in range(c)], device=DEV))
    elif case["op"] == "reorder":
        r, w = case["requests"], case["beams"]
        rows = r * w + 3
        held = [torch.randn(rows, case["row"] + case["spare"], generator=gen, device=DEV).to(DTYPES[case["dtype"]])[:, :case["row"]]
                for _ in range(case["layers"] * case["tensors"])]
        slots = torch.randperm(rows, generator=torch.Generator().manual_seed(seed))[:r * w].view(r, w)
        parents = _parents(case, seed)
        state.update(held=held, slots=slots.to(torch.int32).to(DEV), parents=parents.to(torch.int32).to(DEV))
    else:
        heads, kv, d, page, dtype = case["heads"], case["kv_heads"], case["dim"], case["page"], DTYPES[case["dtype"]]
        groups = _groups(case)
        n = sum(w for w, _, _ in groups)
        ctx = [m + t for w, m, own_keys in groups for t in own_keys]
        width = -(-max(ctx) // page)
        # whole pages of the shared keys are held once; every beam has its own from there on
        used = sum(m // page + sum(-(-(m + t) // page) - m // page for t in tails) for _, m, tails in groups)
        free = torch.randperm(used + 5, generator=torch.Generator().manual_seed(seed)).tolist()
        table = torch.full((n, width), -1, dtype=torch.int32)
        i = 0
        for w, m, tails in groups:
            common = [free.pop() for _ in range(m // page)]
            for t in tails:
                mine = [free.pop() for _ in range(-(-(m + t) // page) - m // page)]
                table[i, :len(common) + len(mine)] = torch.tensor(common + mine, dtype=torch.int32)
                i += 1
        k_pages = torch.randn(used + 5, kv, page, d, generator=gen, device=DEV).to(dtype)
        v_pages = torch.randn(used + 5, kv, d, page, generator=gen, device=DEV).to(dtype)
        q = (torch.randn(n, heads * d, generator=gen, device=DEV) * 1.5).to(dtype)
        sinks = torch.randn(heads, generator=gen, device=DEV) if case["sinks"] else None
        cu = [0]
        for w, _, _ in groups:
            cu.append(cu[-1] + w)
        shared = [m // page * page for _, m, _ in groups]
        state.update(q=q, k=k_pages, v=v_pages, table=table.to(DEV), sinks=sinks, cu=cu, shared=shared, ctx=ctx,
                     cu_dev=torch.tensor(cu, dtype=torch.int32, device=DEV),
                     shared_dev=torch.tensor(shared, dtype=torch.int32, device=DEV),
                     ctx_dev=torch.tensor(ctx, dtype=torch.int32, device=DEV))
    return state


def prepare(case, seed):
    state = _inputs(case, seed)
    if not own:
        return state
    # what a program that searches keeps from step to step: outputs, workspaces, the list of what beams own
    from kvforge_amd.kernels import ops
    if case["op"] == "select":
        r, k = case["requests"], case["count"]
        state["out"] = (torch.empty(r, k, device=DEV), torch.empty(r, k, dtype=torch.int32, device=DEV),
                        torch.empty(r, k, dtype=torch.int32, device=DEV))
        state["work"] = ops.beam_select_workspace(state["logits"].shape[0], case["vocab"], k, DEV)
    elif case["op"] == "reorder":
        state["rows"] = ops.CacheRows(state["held"])
    else:
        cu, ctx, shared = state["cu"], state["ctx"], state["shared"]
        state["widest"] = max(hi - lo for lo, hi in zip(cu, cu[1:]))
        behind = max(c - m for m, lo, hi in zip(shared, cu, cu[1:]) for c in ctx[lo:hi])
        heads, d = case["heads"], case["dim"]
        state["cuts"] = ops.attn_beams_cuts(state["q"], state["k"], heads, case["kv_heads"], d, len(shared), len(ctx),
                                            state["widest"], max(shared), behind)
        state["work"] = ops.attn_beams_workspace(len(ctx), heads, d, state["cuts"], DEV)
        state["out"] = torch.empty_like(state["q"])
    return state


# ------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    return {"select": _run_select, "reorder": _run_reorder, "attend": _run_attend}[case["op"]](case, state)


def _best(flat, count):
    """The ``count`` largest of every row of ``flat`` in order, equal ones by the lower index: (values, indices)."""
    n = flat.shape[1]
    least = flat.topk(count, dim=1).values[:, -1:]
    place = n - torch.arange(n, device=flat.device)
    rank = torch.where(flat > least, place + n, torch.where(flat == least, place, torch.zeros_like(place)))
    index = rank.topk(count, dim=1).indices.sort(dim=1).values
    values, by = flat.gather(1, index).sort(dim=1, descending=True, stable=True)
    return values, index.gather(1, by)


def _run_select(case, state):
    if own:
        from kvforge_amd.kernels import ops
        ops.beam_select(state["logits"], state["scores"], state["cu"], *state["out"], state["work"])
        return state["out"]
    # candidates of several beams may lie closer than 32 bits tell apart
    logits, vocab, count = state["logits"].double(), case["vocab"], case["count"]
    best = logits.amax(1, keepdim=True)
    total = state["scores"].double()[:, None] + (logits - best) - (logits - best).exp().sum(1, keepdim=True).log()
    most = case["beams"]
    if case["ragged"]:
        padded = torch.full((case["requests"] * most, vocab), -math.inf, dtype=torch.float64, device=DEV)
        padded[state["where"]] = total
        total = padded
    flat = total.view(case["requests"], most * vocab)
    values, index = _best(flat, min(count, most * vocab))
    there = values > -math.inf
    beams = torch.where(there, index // vocab, torch.full_like(index, -1))
    tokens = torch.where(there, index % vocab, torch.full_like(index, -1))
    return values.float(), beams.to(torch.int32), tokens.to(torch.int32)


def _run_reorder(case, state):
    if own:
        from kvforge_amd.kernels import ops
        ops.beam_reorder(state["rows"], state["slots"], state["parents"])
        return state["held"]
    to = state["slots"].long()
    source = to.gather(1, state["parents"].long())
    for t in state["held"]:
        t[to.view(-1)] = t[source.view(-1)]
    return state["held"]


def _run_attend(case, state):
    heads, kv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    scale = d ** -0.5
    if own:
        from kvforge_amd.kernels import ops
        ops.attn_beams(state["q"], state["k"], state["v"], state["table"], state["cu_dev"], state["shared_dev"],
                       state["ctx_dev"], state["out"], heads, kv, d, scale, state["widest"], state["cuts"], state["work"],
                       sinks=state["sinks"])
        return state["out"]
    n, width = state["table"].shape
    pages = state["table"].long().clamp(min=0)
    k = state["k"][pages].float().permute(0, 2, 1, 3, 4).reshape(n, kv, width * page, d)
    v = state["v"][pages].float().permute(0, 2, 1, 4, 3).reshape(n, kv, width * page, d)
    s = torch.matmul(state["q"].float().view(n, kv, heads // kv, d) * scale, k.transpose(2, 3).contiguous())
    behind = torch.arange(width * page, device=DEV)[None, :] >= state["ctx_dev"].long()[:, None]
    s = s.masked_fill(behind[:, None, None, :], -math.inf)
    most = s.amax(3, keepdim=True)
    if state["sinks"] is not None:
        sink = state["sinks"].view(1, kv, -1, 1)
        most = torch.maximum(most, sink)
    p = (s - most).exp()
    total = p.sum(3, keepdim=True)
    if state["sinks"] is not None:
        total = total + (sink - most).exp()
    return (torch.matmul(p, v) / total).reshape(n, heads * d).to(state["q"].dtype)


# ------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    size = 2 if case["dtype"] == "bfloat16" else 4
    if case["op"] == "select":
        rows = sum(_counts(case))
        n = rows * case["vocab"]
        # a maximum, an exponential and a sum for every logit
        return {"bytes": n * size + rows * 4 + case["requests"] * case["count"] * 12, "flops": 4 * n}
    if case["op"] == "reorder":
        # the layout's seed decides what is moved; this is the mean over many: every parent that has more than
        # one descendant is read once, every row that changes is written once
        w = case["beams"]
        moved = sum(w - kept for kept in range(1, w + 1)) / w
        read = sum(kept * (1 - (1 - 1 / kept) ** (w - kept)) for kept in range(1, w + 1)) / w
        row = case["row"] * size * case["layers"] * case["tensors"] * case["requests"]
        return {"bytes": row * (moved + read) + 8 * case["requests"] * w, "flops": 0}
    heads, kv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    held = pairs = beams = 0
    for w, m, tails in _groups(case):
        m_whole = m // page * page
        held += m_whole + sum(m + t - m_whole for t in tails)
        pairs += sum(m + t for t in tails)
        beams += w
    return {"bytes": 2 * held * kv * d * size + 2 * beams * heads * d * size, "flops": 4 * pairs * heads * d}


# ------------------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    if case["op"] == "reorder":
        return None          # nothing is computed: rows are copied
    state = _inputs(case, seed)
    if case["op"] == "select":
        first, out = 0, []
        for c in state["counts"]:
            rows = slice(first, first + c)
            first += c
            lp = torch.log_softmax(state["logits"][rows].double(), dim=1) + state["scores"][rows].double()[:, None]
            best = lp.reshape(-1).sort(descending=True).values[:case["count"]]
            out.append(torch.cat([best, best.new_full((case["count"] - best.shape[0],), -math.inf)]))
        return torch.stack(out), None, None
    heads, kv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    out = torch.empty(state["q"].shape, dtype=torch.float64, device=DEV)
    for b, n in enumerate(state["ctx"]):
        blocks = state["table"][b, :-(-n // page)].long()
        k = state["k"][blocks].double().transpose(0, 1).reshape(kv, -1, d)[:, :n]
        v = state["v"][blocks].double().permute(1, 2, 0, 3).reshape(kv, d, -1)[:, :, :n]
        for h in range(heads):
            s = k[h // (heads // kv)] @ state["q"][b, h * d:(h + 1) * d].double() / math.sqrt(d)
            if case["sinks"]:
                s = torch.cat([s, state["sinks"][h:h + 1].double()])
            p = torch.softmax(s, dim=0)[:n]
            out[b, h * d:(h + 1) * d] = v[h // (heads // kv)] @ p
    return out
