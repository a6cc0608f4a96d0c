"""Cases of the served selective attention's operators, in plain form and through the package.

The operators: ``plan`` (block tables and slot maps from request lengths), ``append`` (new keys
and values into a paged 8-bit cache, one scale for each page and key head, and the cache read back
as the values it stands for), ``decode`` (one query token for each request over that cache) and
``prefill`` (causal attention over packed prompts with grouped heads). Every case is a dict of plain values; ``prepare`` makes its inputs from a seed.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"int8": (torch.int8, 127.0), "fp8": (torch.float8_e4m3fn, 448.0)}
INF = float("inf")


# ---------------------------------------------------------------------------- cases
def listed():
    return [
        # a decode step's bookkeeping: every running request gets one token, one in 16 a new page
        {"name": "plan_step", "op": "plan", "requests": 256, "cached": 4096, "new": 1, "page": 16},
        # a wave of prompts enters next to running requests
        {"name": "plan_prompts", "op": "plan", "requests": 384, "cached": 2048, "new": 2048, "page": 64},
        # the keys and values of one decode step
        {"name": "append_step", "op": "append", "requests": 64, "cached": 15, "new": 1, "heads": 8, "dim": 128,
         "page": 16, "code": "int8", "dtype": "bf16", "gated": True},
        # the keys and values of a batch of prompts
        {"name": "append_prompts", "op": "append", "requests": 6, "cached": 0, "new": 4096, "heads": 8, "dim": 128,
         "page": 64, "code": "fp8", "dtype": "f16", "gated": False},
        # one user, a short conversation: latency
        {"name": "decode_one", "op": "decode", "requests": 1, "longest": 1000, "heads": 32, "groups": 8, "dim": 128,
         "page": 16, "code": "int8", "dtype": "bf16", "gated": False},
        # a full batch of ragged requests
        {"name": "decode_batch", "op": "decode", "requests": 64, "longest": 8192, "heads": 32, "groups": 8,
         "dim": 128, "page": 16, "code": "int8", "dtype": "bf16", "gated": False},
        # one very long context
        {"name": "decode_long", "op": "decode", "requests": 1, "longest": 131071, "heads": 32, "groups": 4,
         "dim": 128, "page": 64, "code": "fp8", "dtype": "f16", "gated": False},
        # the selective layer's own form: as many key heads as query heads, gates, fp32 queries
        {"name": "decode_gated", "op": "decode", "requests": 24, "longest": 4097, "heads": 24, "groups": 24,
         "dim": 64, "page": 32, "code": "int8", "dtype": "f32", "gated": True},
        # many short prompts at once
        {"name": "prefill_short", "op": "prefill", "requests": 32, "longest": 333, "heads": 32, "groups": 8,
         "dim": 128, "dtype": "bf16", "gated": False},
        # a batch of prompts of mixed lengths
        {"name": "prefill_mixed", "op": "prefill", "requests": 8, "longest": 4096, "heads": 32, "groups": 8,
         "dim": 128, "dtype": "f16", "gated": False},
        # one long prompt
        {"name": "prefill_long", "op": "prefill", "requests": 1, "longest": 8192, "heads": 32, "groups": 8,
         "dim": 128, "dtype": "bf16", "gated": False},
        # the selective layer's own form, with gates
        {"name": "prefill_gated", "op": "prefill", "requests": 4, "longest": 2047, "heads": 24, "groups": 24,
         "dim": 64, "dtype": "bf16", "gated": True},
    ]


def _log_int(rng, lo, hi):
    return min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    op = rng.choice(["plan", "append", "decode", "decode", "prefill", "prefill"])
    if op == "plan":
        return {"op": op, "requests": _log_int(rng, 1, 512), "cached": _log_int(rng, 1, 8192),
                "new": rng.choice([1, _log_int(rng, 1, 4096)]), "page": rng.choice([16, 32, 64, 128])}
    case = {"op": op, "dtype": rng.choice(["bf16", "f16", "bf16", "f16", "f32"]), "gated": rng.random() < 0.4}
    dim = rng.choice([64, 128])
    if op == "append":
        new = rng.choice([1, _log_int(rng, 1, 4096)])
        most = max(1, 16384 // new)
        return {**case, "requests": _log_int(rng, 1, min(256, most)), "cached": rng.randint(0, 40), "new": new,
                "heads": rng.randint(1, 16), "dim": dim, "page": rng.choice([16, 32, 64, 128]),
                "code": rng.choice(["int8", "fp8"])}
    groups = rng.choice([1, 2, 3, 4, 8, 8, 16])
    heads = groups * rng.choice([1, 2, 4, 5, 8] if groups < 16 else [1, 2, 4])
    case.update(heads=heads, groups=groups, dim=dim)
    if op == "decode":
        longest = _log_int(rng, 1, 65536)
        most = max(1, (1 << 22) // (longest * groups))  # of the cache's size at most that of the listed ones
        return {**case, "requests": _log_int(rng, 1, min(128, most)), "longest": longest,
                "page": rng.choice([16, 32, 64, 128]), "code": rng.choice(["int8", "fp8"])}
    longest = _log_int(rng, 1, 4096 if case["dtype"] != "f32" else 1024)
    most = max(1, (1 << 31) // (longest * longest * heads))
    return {**case, "requests": _log_int(rng, 1, min(64, most)), "longest": longest}


def _lengths(case, longest, seed=0, least=1):
    """Ragged lengths up to ``longest``, one of them just that: the same for every seed, as a case's work is."""
    r = case["requests"]
    step = 0.6180339887498949
    out = [max(least, min(longest, int(longest * ((0.37 + (i + seed) * step) % 1.0)) + 1)) for i in range(r)]
    out[r // 2] = longest
    return out


def _state_lengths(case):
    """(cached, new) tokens of each request of a plan or append case."""
    r = case["requests"]
    cached = [0] * r if not case["cached"] else [n - 1 for n in _lengths(case, case["cached"] + 1, 3)]
    new = [1] * r if case["new"] == 1 else _lengths(case, case["new"], 7, least=0)
    return cached, new


def work(case):
    op = case["op"]
    if op == "plan":
        cached, new = _state_lengths(case)
        pages = sum(-(-(c + n) // case["page"]) - -(-c // case["page"]) for c, n in zip(cached, new))
        return {"bytes": 20 * case["requests"] + 8 * pages + 12 * sum(new), "flops": 0}
    s = DTYPES[case["dtype"]].itemsize
    if op == "append":
        cached, new = _state_lengths(case)
        page, width = case["page"], 2 * case["heads"] * case["dim"]
        pages = sum(-(-(c + n) // page) for c, n in zip(cached, new))
        whole = pages * page * width  # the cache, which is read back as the values it stands for
        gates = 8 * sum(new) * case["heads"] if case["gated"] else 0
        return {"bytes": sum(new) * (width * (s + 1) + 8) + 5 * whole + 8 * pages * page + gates,
                "flops": 4 * sum(new) * width + whole}
    d, hq, hk = case["dim"], case["heads"], case["groups"]
    ns = _lengths(case, case["longest"])
    if op == "decode":
        pages = sum(-(-n // case["page"]) for n in ns)
        per = hk * (2 * d + (4 if case["gated"] else 0))
        return {"bytes": sum(ns) * per + pages * (8 * hk + 4) + 2 * len(ns) * hq * d * s,
                "flops": 4 * d * hq * sum(ns)}
    t = sum(ns)
    return {"bytes": t * d * s * (2 * hq + 2 * hk) + (4 * t * hk if case["gated"] else 0),
            "flops": 4 * d * hq * sum(n * (n + 1) // 2 for n in ns)}


# ---------------------------------------------------------------------------- inputs
def _gates(shape, g, dev):
    """Log-gates as a selective layer gives them: log of a sigmoid, one in 32 shut (-inf)."""
    x = torch.nn.functional.logsigmoid(torch.randn(shape, generator=g, device=dev) + 1.0)
    return x.masked_fill_(torch.rand(shape, generator=g, device=dev) < 1 / 32, -INF)


def _keys(shape, g, dev):
    """Keys with a few strong channels, as trained layers have them."""
    k = torch.randn(shape, generator=g, device=dev)
    return k.mul_(1.0 + 3.0 * (torch.rand(shape[-1], generator=g, device=dev) < 0.05))


def _tables(pages_of, num_pages, width, dev, g):
    order = torch.randperm(num_pages, generator=g, device=dev).to(torch.int32)
    counts = torch.tensor(pages_of, device=dev)
    first = counts.cumsum(0) - counts
    at = torch.arange(width, device=dev)[None, :]
    held = at < counts[:, None]
    index = (first[:, None] + at).clamp_(max=num_pages - 1)
    return torch.where(held, order[index], torch.full_like(index, -1, dtype=torch.int32)), order


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    op = case["op"]
    st = {"case": case}
    if op in ("plan", "append"):
        cached, new = _state_lengths(case)
        page = case["page"]
        before = [-(-c // page) for c in cached]
        after = [-(-(c + n) // page) for c, n in zip(cached, new)]
        width, held, total = max(max(after), 1), sum(before), max(sum(after), 1)
        table, order = _tables(before, total, width, dev, g)
        st.update(lengths=torch.tensor(cached, dtype=torch.int32, device=dev),
                  new=torch.tensor(new, dtype=torch.int32, device=dev), table=table, tokens=sum(new),
                  free=order.roll(-held).contiguous(),
                  free_state=torch.tensor([0, total - held], dtype=torch.int64, device=dev))
    if op == "append":
        # the slots of the new tokens, as the plan gives them
        slots = _plan_plain(st, page)[3]
        h, d, t = case["heads"], case["dim"], st["tokens"]
        kind, most = CODES[case["code"]]
        x = _keys((total, h, page, d), g, dev)
        y = torch.randn((total, h, page, d), generator=g, device=dev)
        st["slots"] = slots
        st["all_slots"] = torch.arange(total * page, device=dev)
        st["k"] = (_keys((t, h, d), g, dev) * 1.1).to(DTYPES[case["dtype"]])
        st["v"] = torch.randn((t, h, d), generator=g, device=dev).to(DTYPES[case["dtype"]])
        st["k_cache"], st["k_scale"] = _coded(x, kind, most)
        st["v_cache"], st["v_scale"] = _coded(y, kind, most)
        st["gate"] = _gates((t, h), g, dev) if case["gated"] else None
        st["gate_cache"] = _gates((total, h, page), g, dev) if case["gated"] else None
    elif op == "decode":
        ns, page = _lengths(case, case["longest"]), case["page"]
        pages = [-(-n // page) for n in ns]
        total, hk, d = sum(pages), case["groups"], case["dim"]
        kind, most = CODES[case["code"]]
        st["table"], _ = _tables(pages, total, max(pages), dev, g)
        st["lengths"] = torch.tensor(ns, dtype=torch.int32, device=dev)
        st["k_cache"], st["k_scale"] = _coded(_keys((total, hk, page, d), g, dev), kind, most)
        st["v_cache"], st["v_scale"] = _coded(torch.randn((total, hk, page, d), generator=g, device=dev), kind, most)
        st["gate_cache"] = _gates((total, hk, page), g, dev) if case["gated"] else None
        st["q"] = torch.randn((len(ns), case["heads"], d), generator=g, device=dev).to(DTYPES[case["dtype"]])
    elif op == "prefill":
        ns = _lengths(case, case["longest"])
        t, d, hq, hk = sum(ns), case["dim"], case["heads"], case["groups"]
        # one projection's output, of which queries, keys and values are slices
        qkv = torch.randn((t, hq + 2 * hk, d), generator=g, device=dev)
        qkv[:, hq:hq + hk] = _keys((t, hk, d), g, dev)
        qkv = qkv.to(DTYPES[case["dtype"]])
        st["q"], st["k"], st["v"] = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
        st["gate"] = _gates((t, hk), g, dev) if case["gated"] else None
        st["longest"] = max(ns)
        st["cu"] = torch.tensor([0] + ns, device=dev).cumsum(0).to(torch.int32)
    return st


def _coded(x, kind, most):
    """(codes, scales) of whole pages: scale = the page's largest magnitude over the code's."""
    scale = x.abs().amax(dim=(2, 3)) / most
    x = x.div_(scale[:, :, None, None])
    return (x.round_() if kind == torch.int8 else x).clamp_(-most, most).to(kind), scale


def _values(codes, scale):
    s = scale[:, :, None, None]
    return codes * s if codes.dtype == torch.int8 else codes.float() * s


# ---------------------------------------------------------------------------- plain forms
def _plan_plain(st, page):
    lengths, new, table, free = st["lengths"].long(), st["new"].long(), st["table"], st["free"].long()
    head, tail = st["free_state"][0], st["free_state"][1]
    r, width = table.shape
    has = (lengths + page - 1) // page
    end = (lengths + new + page - 1) // page
    fits = end <= width
    need = torch.where(fits, end - has, 0)
    upto = need.cumsum(0)
    served = fits & ((need == 0) | (upto <= tail - head))
    at = torch.arange(width, device=table.device)[None, :]
    fresh = served[:, None] & (at >= has[:, None]) & (at < end[:, None])
    index = (head + (upto - need)[:, None] + at - has[:, None]) % free.numel()
    table = torch.where(fresh, free[index].to(torch.int32), table)
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)])
    token = torch.arange(st["tokens"], device=table.device)
    of = torch.searchsorted(cu[1:], token, right=True).clamp_(max=r - 1)
    inside = token < cu[r]
    pos = torch.where(inside, lengths[of] + token - cu[of], 0)
    slot = table[of, (pos // page).clamp(max=width - 1)].long() * page + pos % page
    slot = torch.where(inside & served[of], slot, -1)
    given = torch.where(served, need, 0).sum()
    return (table, torch.where(served, lengths + new, lengths).to(torch.int32), cu.to(torch.int32), slot,
            pos.to(torch.int32), torch.stack([head + given, tail]))


def _append_plain(x, slots, cache, scale, most):
    """In place, as the operator is: pages that the slots touch get their scale, grown pages their new codes."""
    pages, _, page, _ = cache.shape
    block, row = slots // page, slots % page
    x = x.float()
    top = torch.zeros_like(scale).index_reduce_(0, block, x.abs().amax(dim=2), "amax")
    first = torch.full((pages,), page, device=scale.device).index_reduce_(0, block, row, "amin")
    old = torch.where(first[:, None] == 0, 0.0, scale)
    new = torch.maximum(old, top / most)
    ratio = torch.where(new > old, old / new, 1.0)[block][:, :, None, None]
    held = cache[block].float()
    moved = held * ratio
    y = x / new[block][:, :, None]
    y = torch.where(new[block][:, :, None] > 0, y, 0.0)
    if cache.dtype == torch.int8:
        moved, y = moved.round(), y.round()
    old_row = torch.arange(page, device=row.device)[None, :] < first[block][:, None]
    raw = cache.view(torch.uint8)
    raw[block] = torch.where(old_row[:, None, :, None], moved, held).to(cache.dtype).view(torch.uint8)
    raw[block, :, row] = y.clamp(-most, most).to(cache.dtype).view(torch.uint8)
    scale.copy_(torch.where(first[:, None] < page, new, scale))


def _read_plain(slots, cache, scale):
    block, row = slots // cache.shape[2], slots % cache.shape[2]
    return cache.view(torch.uint8)[block, :, row].view(cache.dtype).float() * scale[block][:, :, None]


def _decode_plain(st):
    case, q, n = st["case"], st["q"], st["lengths"].long()
    hk, d, page = case["groups"], case["dim"], case["page"]
    r, hq, _ = q.shape
    table = st["table"].long().clamp(min=0)
    span = table.shape[1] * page
    k = _values(st["k_cache"][table].flatten(0, 1), st["k_scale"][table].flatten(0, 1))
    k = k.view(r, -1, hk, page, d).transpose(1, 2).reshape(r, hk, span, d)
    s = q.float().view(r, hk, hq // hk, d) @ k.transpose(2, 3) * d ** -0.5
    del k
    at = torch.arange(span, device=q.device)[None, :]
    live = at < n[:, None]
    if st["gate_cache"] is not None:
        gate = st["gate_cache"][table].transpose(1, 2).reshape(r, hk, 1, span)
        s = s + torch.where((at < n[:, None] - 1)[:, None, None], gate, 0.0)
    s = torch.where(live[:, None, None], s, -INF)
    v = _values(st["v_cache"][table].flatten(0, 1), st["v_scale"][table].flatten(0, 1))
    v = v.view(r, -1, hk, page, d).transpose(1, 2).reshape(r, hk, span, d)
    p = (s - s.amax(dim=3, keepdim=True)).exp()
    return ((p @ v) / p.sum(dim=3, keepdim=True)).view(r, hq, d).to(q.dtype)


def _prefill_plain(st):
    q, k, v, cu, longest = st["q"], st["k"], st["v"], st["cu"].long(), st["longest"]
    t, hq, d = q.shape
    hk, r = k.shape[1], cu.numel() - 1
    at = torch.arange(longest, device=q.device)
    rows = (cu[:-1, None] + at[None, :]).clamp_(max=t - 1)
    qs = q[rows].float().view(r, longest, hk, hq // hk, d).permute(0, 2, 3, 1, 4)
    ks = k[rows].float().permute(0, 2, 3, 1)[:, :, None]
    vs = v[rows].float().permute(0, 2, 1, 3)[:, :, None]
    s = (qs * d ** -0.5) @ ks
    if st["gate"] is not None:
        its_own = s.diagonal(dim1=3, dim2=4).clone()
        s.add_(st["gate"][rows].permute(0, 2, 1)[:, :, None, None])
        s.diagonal(dim1=3, dim2=4).copy_(its_own)
    s.masked_fill_(at[None, :] > at[:, None], -INF)
    s.sub_(s.amax(dim=4, keepdim=True)).exp_()
    out = (s @ vs) / s.sum(dim=4, keepdim=True)
    out = out.permute(0, 3, 1, 2, 4).reshape(r, longest, hq, d)
    token = torch.arange(t, device=q.device)
    of = torch.searchsorted(cu[1:], token, right=True)
    return out[of, token - cu[of]].to(q.dtype)


# ---------------------------------------------------------------------------- one pass
PLAN_NAMES = ("table", "lengths", "cu", "slots", "positions", "free_state")


def run(state):
    case = state["case"]
    op = case["op"]
    if op == "plan":
        if own:
            import selective_attention_b200 as sab
            out = sab.sattn_paged_plan(state["lengths"], state["new"], state["table"], state["free"],
                                       state["free_state"], state["tokens"], case["page"])
            return dict(zip(PLAN_NAMES, (state["table"], *out)))
        return dict(zip(PLAN_NAMES, _plan_plain(state, case["page"])))
    if op == "append":
        if own:
            import selective_attention_b200 as sab
            sab.sattn_paged_append(state["k"], state["v"], state["slots"], state["k_cache"], state["v_cache"],
                                   state["k_scale"], state["v_scale"], state["gate"], state["gate_cache"])
        else:
            slots, page, most = state["slots"], case["page"], CODES[case["code"]][1]
            _append_plain(state["k"], slots, state["k_cache"], state["k_scale"], most)
            _append_plain(state["v"], slots, state["v_cache"], state["v_scale"], most)
            if state["gate"] is not None:
                state["gate_cache"][slots // page, :, slots % page] = state["gate"]
        # the cache is held in 8 bits: it is read back as the values it stands for
        if own:
            k, v = sab.sattn_paged_read(state["all_slots"], state["k_cache"], state["v_cache"], state["k_scale"],
                                        state["v_scale"], torch.float32)
        else:
            k, v = (_read_plain(state["all_slots"], state[c + "_cache"], state[c + "_scale"]) for c in "kv")
        return {"k": k, "v": v, "k_scale": state["k_scale"], "v_scale": state["v_scale"], "gate": state["gate_cache"]}
    if op == "decode":
        if own:
            import selective_attention_b200 as sab
            return sab.sattn_paged_decode(state["q"], state["k_cache"], state["v_cache"], state["k_scale"],
                                          state["v_scale"], state["table"], state["lengths"], state["gate_cache"])
        return _decode_plain(state)
    if own:
        import selective_attention_b200 as sab
        return sab.sattn_prefill_packed(state["q"], state["k"], state["v"], state["cu"], state["gate"])
    return _prefill_plain(state)


# ---------------------------------------------------------------------------- 64 bits
def _attend64(q, k, v, gate, causal):
    """Rows of one head group in 64 bits: q (g, n, d) against k, v (m, d); the last rows line up."""
    s = torch.einsum("gnd,md->gnm", q, k) / math.sqrt(q.shape[-1])
    n, m = s.shape[1:]
    i = torch.arange(n, device=q.device)[:, None] + (m - n)
    j = torch.arange(m, device=q.device)[None, :]
    if gate is not None:
        s = torch.where(j < i, s + gate[None, None, :], s)
    if causal:
        s = torch.where(j <= i, s, -INF)
    return torch.softmax(s, dim=-1) @ v


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "plan":
        return None
    if op == "append":
        page = case["page"]
        kind, most = CODES[case["code"]]
        slots = st["slots"].cpu()
        out = {"gate": None}
        if case["gated"]:
            gc = st["gate_cache"].double()
            gc[st["slots"] // page, :, st["slots"] % page] = st["gate"].double()
            out["gate"] = gc
        block, row = (slots // page), (slots % page)
        starts = [0] + (((block[1:] != block[:-1]).nonzero().flatten() + 1).tolist() if len(slots) else [])
        ends = starts[1:] + [len(slots)]
        for c in "kv":
            x, codes = st[c].double(), st[c + "_cache"].double()
            scale = st[c + "_scale"].double()
            for lo, hi in zip(starts, ends if len(slots) else []):
                b, o = int(block[lo]), int(row[lo])
                part = x[lo:hi].transpose(0, 1)  # (h, rows, d)
                was = scale[b] if o else torch.zeros_like(scale[b])
                now = torch.maximum(was, part.abs().amax(dim=(1, 2)) / most)
                grown = (now > was)[:, None, None]
                moved = codes[b, :, :o] * (was / now)[:, None, None]
                fresh = part / now[:, None, None]
                moved, fresh = ((moved.round(), fresh.round()) if kind == torch.int8 else
                                (moved.to(kind).double(), fresh.to(kind).double()))
                codes[b, :, :o] = torch.where(grown, moved, codes[b, :, :o])
                codes[b, :, o:o + hi - lo] = fresh
                scale[b] = now
            out[c] = (codes * scale[:, :, None, None]).transpose(1, 2).flatten(0, 1)
            out[c + "_scale"] = scale
        return out
    hk = case["groups"]
    g = case["heads"] // hk
    ns = _lengths(case, case["longest"])
    if op == "decode":
        out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
        for r, n in enumerate(ns):
            pages = st["table"][r, :-(-n // case["page"])].long()
            for h in range(hk):
                k, v = (((st[c + "_cache"][pages, h].double()) * st[c + "_scale"][pages, h].double()[:, None, None])
                        .flatten(0, 1)[:n] for c in "kv")
                gate = None if st["gate_cache"] is None else st["gate_cache"][pages, h].double().flatten()[:n]
                q = st["q"][r, h * g:(h + 1) * g].double()[:, None]
                out[r, h * g:(h + 1) * g] = _attend64(q, k, v, gate, False)[:, 0]
        return out
    if sum(n * n for n in ns) * case["heads"] > 1 << 33:
        return None
    out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
    lo = 0
    for n in ns:
        for h in range(hk):
            q = st["q"][lo:lo + n, h * g:(h + 1) * g].double().transpose(0, 1)
            k, v = st["k"][lo:lo + n, h].double(), st["v"][lo:lo + n, h].double()
            gate = None if st["gate"] is None else st["gate"][lo:lo + n, h].double()
            for at in range(0, n, 1024):  # of the rows, so many at once
                end = min(n, at + 1024)
                part = _attend64(q[:, at:end], k[:end], v[:end], None if gate is None else gate[:end], True)
                out[lo + at:lo + end, h * g:(h + 1) * g] = part.transpose(0, 1)
        lo += n
    return out
