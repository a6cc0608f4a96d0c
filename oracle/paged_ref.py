"""CPU restatements of the served selective attention's operators, request by request and row by
row in 64 bits (the 8-bit codes in the 32-bit arithmetic that defines them)."""
from __future__ import annotations

import math

import torch

INF = float("inf")
MOST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def plan(lengths, new_lengths, block_table, free_pages, free_state, num_tokens, page):
    """Returns (table, lengths_out, cu_new, slots, positions, free_state) as lists and tensors."""
    table = block_table.clone()
    head, tail = (int(x) for x in free_state)
    W = table.shape[1]
    out, cu, slots, pos = [], [0], [], []
    upto = 0
    given = 0
    for r, (n, add) in enumerate(zip(lengths.tolist(), new_lengths.tolist())):
        n0, n, add = n, max(n, 0), max(add, 0)
        has, end = -(-n // page), -(-(n + add) // page)
        served = end <= W
        if served:
            upto += end - has
            served = end == has or upto <= min(tail - head, free_pages.numel())
        served = served and (add == 0 or cu[-1] + add <= num_tokens)
        if served and end > has:
            for i in range(end - has):
                at = head + upto - (end - has) + i
                table[r, has + i] = free_pages[at % free_pages.numel()]
            given = upto
        for i in range(min(add, num_tokens - len(slots))):
            p = n + i
            slots.append(int(table[r, p // page]) * page + p % page if served else -1)
            pos.append(p)
        out.append(n + add if served else n0)
        cu.append(cu[-1] + add)
    slots = (slots + [-1] * num_tokens)[:num_tokens]
    pos = (pos + [0] * num_tokens)[:num_tokens]
    return (table, torch.tensor(out, dtype=torch.int32), torch.tensor(cu).clamp(max=2 ** 31 - 1).to(torch.int32),
            torch.tensor(slots, dtype=torch.int64), torch.tensor(pos, dtype=torch.int32),
            torch.tensor([head + given, tail], dtype=torch.int64))


def _encode(x, kind):
    if kind == torch.int8:
        x = torch.where(x.isnan(), torch.zeros_like(x), x.round().clamp(-127, 127))
        return x.to(torch.int8)
    return torch.where(x.isnan(), x, x.clamp(-448, 448)).to(kind)


def append(x, slots, codes, scale):
    """In place on codes (P, H, page, D) and scale (P, H), 32-bit arithmetic."""
    P, H, page, D = codes.shape
    most, kind = MOST[codes.dtype], codes.dtype
    x = x.float()
    runs = []
    for t, s in enumerate(slots.tolist()):
        if not 0 <= s < P * page:
            continue
        if runs and runs[-1][1] == t - 1 and slots[t - 1] == s - 1 and s % page:
            runs[-1][1] = t
        else:
            runs.append([t, t])
    for lo, hi in runs:
        b, o = divmod(int(slots[lo]), page)
        for h in range(H):
            part = x[lo:hi + 1, h]
            top = torch.where(part.isfinite(), part.abs(), torch.zeros_like(part)).max()
            was = scale[b, h].clone() if o else torch.tensor(0.0)
            now = torch.maximum(was, top * (torch.tensor(1.0) / torch.tensor(most)))
            if now > was and o:
                codes[b, h, :o] = _encode(codes[b, h, :o].float() * (was / now), kind)
            codes[b, h, o:o + hi + 1 - lo] = _encode(part / now if now > 0 else torch.zeros_like(part), kind)
            scale[b, h] = now


def read(slots, codes, scale):
    """(N, H, D) values in 32 bits."""
    P, H, page, D = codes.shape
    out = torch.zeros(len(slots), H, D)
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < P * page:
            out[i] = codes[s // page, :, s % page].float() * scale[s // page][:, None]
    return out


def attend(q, k, v, gate, own, scale):
    """One row in 64 bits: q (D,), keys (n, D); gate (n,) or None; ``own`` is the ungated key."""
    n = k.shape[0]
    if n == 0:
        return torch.zeros(v.shape[1], dtype=torch.float64)
    keep = torch.ones(n, dtype=torch.bool)
    add = torch.zeros(n, dtype=torch.float64)
    if gate is not None:
        add = gate.double().clone()
        add[own] = 0.0
        keep = add != -INF
    s = (k[keep].double() @ q.double()) * scale + add[keep]
    return torch.softmax(s, 0) @ v[keep].double()


def decode(q, k_codes, v_codes, k_scale, v_scale, table, lengths, gate=None, scale=None):
    R, Hq, D = q.shape
    P, Hk, page, _ = k_codes.shape
    scale = 1 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(R, Hq, D, dtype=torch.float64)
    for r in range(R):
        n = min(max(int(lengths[r]), 0), table.shape[1] * page)
        pages = table[r, :-(-n // page)].long()
        for h in range(Hk):
            k, v = ((c[pages, h].double() * s[pages, h].double()[:, None, None]).reshape(-1, D)[:n]
                    for c, s in ((k_codes, k_scale), (v_codes, v_scale)))
            g = None if gate is None else gate[pages, h].reshape(-1)[:n]
            for i in range(h * (Hq // Hk), (h + 1) * (Hq // Hk)):
                out[r, i] = attend(q[r, i], k, v, g, n - 1, scale)
    return out


def prefill_packed(q, k, v, cu, gate=None, scale=None):
    T, Hq, D = q.shape
    Hk = k.shape[1]
    scale = 1 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(T, Hq, D, dtype=torch.float64)
    for lo, hi in zip(cu.tolist()[:-1], cu.tolist()[1:]):
        for h in range(Hq):
            kh = h // (Hq // Hk)
            for i in range(lo, hi):
                g = None if gate is None else gate[lo:i + 1, kh]
                out[i, h] = attend(q[i, h], k[lo:i + 1, kh], v[lo:i + 1, kh], g, i - lo, scale)
    return out
