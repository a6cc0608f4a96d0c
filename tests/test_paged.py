"""The paged 8-bit cache of served selective attention: plan, append, read and decode against
``oracle/paged_ref.py``.

Tolerances. Plans and codes are whole numbers (or the results of named 32-bit roundings): equal.
Decode: q and the codes enter the products exactly; a probability is rounded to 16 bits
(2^-11 of itself) for 16-bit queries and to about 2^-21 for fp32 ones, so that the output is off
by at most that much of the largest |v| a row can see; scores are fp32 sums of D products
(below 1e-5 at the magnitudes here), and the result is rounded once to q's dtype. So
|err| <= round(dtype) * |out| + p(dtype) * max|v| with (round, p) = (2^-8, 2^-10) for bfloat16,
(2^-10, 2^-10) for float16 and (1e-5, 3e-5) for float32.
"""
import ctypes
import math

import pytest
import torch

from oracle import paged_ref

INF = float("inf")
TOL = {torch.bfloat16: (2 ** -8, 2 ** -10), torch.float16: (2 ** -10, 2 ** -10), torch.float32: (1e-5, 3e-5)}


def close(got, ref, vmax, what=""):
    rel, p = TOL[got.dtype]
    got, ref = got.double().cpu(), ref.double().cpu()
    assert torch.equal(got.isnan(), ref.isnan()), f"{what}: NaN in other places"
    fine = ~ref.isnan()
    err = (got - ref).abs()[fine]
    bound = rel * ref.abs()[fine] + p * vmax
    assert bool((err <= bound).all()), f"{what}: {int((err > bound).sum())} outside, max err {err.max().item():.3e}"


# ----------------------------------------------------------------------------- the oracle itself (CPU)
def test_plan_oracle_hands_out_pages_in_order():
    table = torch.full((3, 3), -1, dtype=torch.int32)
    table[0, 0] = 7
    t, n, cu, slots, pos, st = paged_ref.plan(torch.tensor([15, 0, 0]), torch.tensor([2, 17, 1]), table,
                                              torch.tensor([3, 4, 5, 6], dtype=torch.int32), torch.tensor([0, 4]), 22,
                                              16)
    assert t[0].tolist() == [7, 3, -1] and t[1].tolist() == [4, 5, -1] and t[2].tolist() == [6, -1, -1]
    assert slots[:2].tolist() == [7 * 16 + 15, 3 * 16] and slots[2].item() == 64 and slots[18].item() == 80
    assert slots[19].item() == 96 and slots[20:].tolist() == [-1, -1]
    assert cu.tolist() == [0, 2, 19, 20] and n.tolist() == [17, 17, 1] and st.tolist() == [4, 4]
    assert pos[:3].tolist() == [15, 16, 0]


def test_append_oracle_scale_grows_and_page_starts_anew():
    codes, scale = torch.zeros(1, 1, 16, 32, dtype=torch.int8), torch.full((1, 1), 9.0)
    x = torch.ones(1, 1, 32)
    paged_ref.append(x, torch.tensor([0]), codes, scale)  # a page's first token: the old scale is void
    assert scale.item() == pytest.approx(1 / 127) and bool((codes[0, 0, 0] == 127).all())
    paged_ref.append(2 * x, torch.tensor([1]), codes, scale)
    assert scale.item() == pytest.approx(2 / 127) and bool((codes[0, 0, 0] == 64).all())


# ----------------------------------------------------------------------------- refusals (CPU)
def _cache(pages=4, heads=2, page=16, D=64, kind=torch.int8, gated=True, device="cpu"):
    return dict(k_cache=torch.zeros(pages, heads, page, D, dtype=kind, device=device),
                v_cache=torch.zeros(pages, heads, page, D, dtype=kind, device=device),
                k_scale=torch.zeros(pages, heads, device=device), v_scale=torch.zeros(pages, heads, device=device),
                log_gate_cache=torch.zeros(pages, heads, page, device=device) if gated else None)


def test_structs_match_the_header():
    import os
    import shutil
    import subprocess
    import tempfile

    from conftest import ROOT
    from selective_attention_b200 import _lib

    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    from selective_attention_b200 import paged

    for cname, cls, packed in (("sattn_cache", _lib.SattnCache, paged._CACHE),
                               ("sattn_packed_params", _lib.SattnPackedParams, paged._PACKED)):
        # the bytes that the wrappers pass have every field in its place
        values = [(i + 1) / 2 if "f" == t._type_ else i + 1 for i, (_, t) in enumerate(cls._fields_)]
        got = cls.from_buffer_copy(packed.pack(*values))
        assert [getattr(got, f) for f, _ in cls._fields_] == values
        fields = [f[0] for f in cls._fields_]
        prog = ["#include <stdio.h>", "#include <stddef.h>",
                f'#include "{os.path.join(ROOT, "include", "ssd_b200.h")}"', "int main(void){",
                f'printf("%zu\\n", sizeof({cname}));']
        prog += [f'printf("%zu\\n", offsetof({cname}, {f}));' for f in fields] + ["return 0;}"]
        with tempfile.TemporaryDirectory() as d:
            src, exe = os.path.join(d, "p.c"), os.path.join(d, "p")
            open(src, "w").write("\n".join(prog))
            subprocess.run(["gcc", "-std=c99", src, "-o", exe], check=True)
            out = [int(x) for x in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
        assert out[0] == ctypes.sizeof(cls)
        for f, off in zip(fields, out[1:]):
            assert getattr(cls, f).offset == off, f


def test_widths_whose_product_with_the_page_wraps_are_refused():
    from selective_attention_b200 import _lib

    L, bad = _lib.lib(), _lib.SSD_ERR_INVALID_ARGUMENT
    c = ctypes.byref(_lib.SattnCache(num_pages=4, nkv=2, page_size=16, head_dim=64, code=0, k_codes=4096, v_codes=4096,
                                     k_scale=4096, v_scale=4096, log_gate=None))
    for width in (1 << 31, 1 << 60, (1 << 62) + 1):
        assert L.sattn_paged_plan(*[4096] * 10, 1, width, 4, 1, 16, None) == bad, width
        assert L.sattn_paged_decode(c, 4096, 4096, 4096, 4096, 1, width, 2, 1.0, 1, 4096, 1 << 40, None) == bad, width
        assert L.sattn_paged_decode_workspace_size(c, 1, width, 2) == 0, width


def test_cpu_tensors_are_refused():
    import selective_attention_b200 as sab

    i32 = dict(dtype=torch.int32)
    c = _cache()
    with pytest.raises(ValueError):
        sab.sattn_paged_plan(torch.zeros(1, **i32), torch.zeros(1, **i32), torch.zeros(1, 1, **i32),
                             torch.zeros(1, **i32), torch.zeros(2, dtype=torch.int64), 1, 16)
    with pytest.raises(ValueError):
        sab.sattn_paged_append(torch.zeros(1, 2, 64), torch.zeros(1, 2, 64), torch.zeros(1, dtype=torch.int64),
                               log_gate=torch.zeros(1, 2), **c)
    with pytest.raises(ValueError):
        sab.sattn_paged_decode(torch.zeros(1, 2, 64), block_table=torch.zeros(1, 1, **i32),
                               lengths=torch.zeros(1, **i32), **c)


def test_c_entries_refuse_without_launching():
    from selective_attention_b200 import _lib

    L = _lib.lib()
    bad = _lib.SSD_ERR_INVALID_ARGUMENT

    def cache(**kw):
        d = dict(num_pages=4, nkv=2, page_size=16, head_dim=64, code=0, k_codes=4096, v_codes=4096, k_scale=4096,
                 v_scale=4096, log_gate=None)
        d.update(kw)
        return ctypes.byref(_lib.SattnCache(**d))

    def decode(c, q=4096, R=1, W=1, H=2, dtype=1):
        return L.sattn_paged_decode(c, q, 4096, 4096, 4096, R, W, H, 1.0, dtype, None, 0, None)

    for kw in (dict(page_size=24), dict(head_dim=48), dict(num_pages=0), dict(nkv=0), dict(k_codes=None),
               dict(v_scale=None), dict(k_codes=4097)):
        assert decode(cache(**kw)) == bad, kw
        assert L.sattn_paged_read(cache(**kw), 4096, 1, 4096, 4096, 0, None) == bad, kw
        assert L.sattn_paged_append(cache(**kw), 4096, 4096, None, 4096, 1, 128, 64, 128, 64, 0, None) == bad, kw
    assert decode(cache(code=2)) == _lib.SSD_ERR_UNSUPPORTED_DTYPE
    assert decode(cache(), dtype=7) == _lib.SSD_ERR_UNSUPPORTED_DTYPE
    assert decode(cache(), H=3) == bad and decode(cache(), q=None) == bad and decode(cache(), R=0) == bad
    assert decode(cache(), q=4100) == bad
    # gates for a cache without them, and the other way round
    assert L.sattn_paged_append(cache(), 4096, 4096, 4096, 4096, 1, 128, 64, 128, 64, 0, None) == bad
    assert L.sattn_paged_append(cache(log_gate=4096), 4096, 4096, None, 4096, 1, 128, 64, 128, 64, 0, None) == bad
    assert L.sattn_paged_append(cache(), None, None, None, None, 0, 0, 0, 0, 0, 0, None) == 0  # no tokens
    assert L.sattn_paged_plan(*([None] * 10), 1, 1, 1, 1, 16, None) == bad
    assert L.sattn_paged_plan(*([4096] * 10), 1, 1, 1, 1, 20, None) == bad
    assert L.sattn_paged_plan(*([4096] * 10), -1, 1, 1, 1, 16, None) == bad


# ----------------------------------------------------------------------------- GPU: plan
def _plan_inputs(lengths, new, width, pages, page, head=0, free=None, spare=0):
    g = torch.Generator().manual_seed(len(lengths) + pages)
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(lengths):
        k = -(-max(n, 0) // page)
        table[r, :k] = order[at:at + k]
        at += k
    left = pages - at
    ring = torch.full((pages + spare,), -7, dtype=torch.int32)
    for i in range(left):
        ring[(head + i) % ring.numel()] = order[at + i]
    free = left if free is None else free
    return (torch.tensor(lengths, dtype=torch.int32), torch.tensor(new, dtype=torch.int32), table, ring,
            torch.tensor([head, head + free], dtype=torch.int64))


@pytest.mark.gpu
@pytest.mark.parametrize("case", [
    dict(lengths=[5], new=[1], width=1, pages=1, page=16),
    dict(lengths=[16, 0, 31, 15], new=[1, 1, 1, 1], width=3, pages=9, page=16),           # page boundaries
    dict(lengths=[0, 100, 0], new=[0, 0, 0], width=8, pages=8, page=16),                   # nothing new
    dict(lengths=[0, 3, 0, 7], new=[3000, 0, 1, 2100], width=200, pages=400, page=32),     # over several CTAs
    dict(lengths=[10] * 700, new=[i % 3 for i in range(700)], width=1, pages=700, page=16),  # more than one scan
    dict(lengths=[0, 0, 5, 0], new=[40, 40, 2, 1], width=4, pages=6, page=16, free=4),     # the ring runs short
    dict(lengths=[0, 0, 0], new=[70, 16, 16], width=4, pages=6, page=16),                  # wider than the table
    dict(lengths=[3, 0], new=[14, 33], width=4, pages=8, page=16, head=1000003, spare=5),  # the ring wraps
    dict(lengths=[-4, 2], new=[5, -3], width=2, pages=4, page=128),                        # negative: none
])
@pytest.mark.parametrize("extra", [0, 5])
def test_plan(case, extra):
    import selective_attention_b200 as sab

    page = case["page"]
    args = _plan_inputs(**case)
    T = sum(max(x, 0) for x in case["new"]) + extra
    ref = paged_ref.plan(*args, T, page)
    dev = [a.cuda() for a in args]
    got = sab.sattn_paged_plan(*dev, T, page)
    assert torch.equal(dev[2].cpu(), ref[0])
    for g, r, n in zip(got, ref[1:], ("lengths", "cu", "slots", "positions", "free_state")):
        assert g.dtype == r.dtype and torch.equal(g.cpu(), r), n
    for a, b in zip((0, 1, 3, 4), (0, 1, 3, 4)):
        assert torch.equal(dev[a].cpu(), args[b])


@pytest.mark.gpu
def test_plan_without_requests():
    import selective_attention_b200 as sab

    e = torch.empty(0, dtype=torch.int32, device="cuda")
    n, cu, slots, pos, st = sab.sattn_paged_plan(e, e, torch.empty(0, 4, dtype=torch.int32, device="cuda"), e,
                                                 torch.tensor([2, 2], device="cuda"), 3, 16)
    assert n.numel() == 0 and cu.tolist() == [0] and slots.tolist() == [-1] * 3 and st.tolist() == [2, 2]


# ----------------------------------------------------------------------------- GPU: append, read
def _tokens(T, H, D, dtype, seed=0, strided=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, 3 * H, D + (8 if strided else 0), generator=g) * (
        0.2 + 3 * torch.rand(T, 1, 1, generator=g))
    x = x.to(dtype)
    return x[:, :H, :D], x[:, H:2 * H, :D], torch.randn(T, H, generator=g)


def same(a, b):
    return a.dtype == b.dtype and torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


def _check_append(c, k, v, slots, gate):
    import selective_attention_b200 as sab

    want = {n: None if t is None else t.clone() for n, t in c.items()}
    paged_ref.append(k, slots, want["k_cache"], want["k_scale"])
    paged_ref.append(v, slots, want["v_cache"], want["v_scale"])
    if gate is not None:
        page = c["k_cache"].shape[2]
        for t, s in enumerate(slots.tolist()):
            if 0 <= s < c["k_cache"].shape[0] * page:
                want["log_gate_cache"][s // page, :, s % page] = gate[t]
    dev = {n: None if t is None else t.cuda() for n, t in c.items()}
    sab.sattn_paged_append(k.cuda(), v.cuda(), slots.cuda(), log_gate=None if gate is None else gate.cuda(), **dev)
    for n, t in want.items():
        if t is not None:
            raw = (lambda x: x.view(torch.uint8)) if t.dtype.itemsize == 1 else (lambda x: x)
            assert torch.equal(raw(dev[n].cpu()), raw(t)), n
    ids = torch.cat([slots, torch.tensor([-1, c["k_cache"].shape[0] * c["k_cache"].shape[2]])])
    dev.pop("log_gate_cache")
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        gk, gv = sab.sattn_paged_read(ids.cuda(), dtype=dtype, **dev)
        assert same(gk.cpu(), paged_ref.read(ids, want["k_cache"], want["k_scale"]).to(dtype))
        assert same(gv.cpu(), paged_ref.read(ids, want["v_cache"], want["v_scale"]).to(dtype))
    return {n: None if t is None else t.cpu() for n, t in {**dev, "log_gate_cache": want["log_gate_cache"]}.items()}


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page,D,H", [(16, 64, 3), (32, 128, 2), (64, 32, 1), (128, 256, 2)])
def test_append_prompts_then_single_tokens(kind, dtype, page, D, H):
    """Requests that end inside pages, then tokens one by one whose magnitudes rise and fall."""
    lens = [1, page - 1, page, page + 1, 2 * page + 3]
    pages = [-(-(n + 3) // page) for n in lens]
    order = torch.randperm(sum(pages), generator=torch.Generator().manual_seed(1)).tolist()
    tables, at = [], 0
    for p in pages:
        tables.append(order[at:at + p])
        at += p
    c = _cache(sum(pages), H, page, D, kind)
    c["k_scale"].fill_(5.0)  # of earlier owners: void
    c["k_cache"].view(torch.uint8).fill_(0x7f)
    slots = torch.tensor([tables[r][i // page] * page + i % page for r, n in enumerate(lens) for i in range(n)])
    k, v, g = _tokens(len(slots), H, D, dtype, strided=dtype != torch.float16)
    c = _check_append(c, k, v, slots, g)
    for step in range(3):
        slots = torch.tensor([tables[r][(n + step) // page] * page + (n + step) % page for r, n in enumerate(lens)])
        k, v, g = _tokens(len(lens), H, D, dtype, seed=step + 2)
        c = _check_append(c, k * (3.0 ** (step - 1)), v, slots, g)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.int8, torch.float8_e4m3fn])
def test_append_many_tokens_odd_slots_and_unaligned_rows(kind):
    page, H, D = 16, 5, 64
    c = _cache(80, H, page, D, kind, gated=False)
    slots = torch.arange(80 * page)
    slots = torch.cat([slots[:500], torch.tensor([-1, -1]), slots[528:], torch.tensor([80 * page, -5])])
    k, v, _ = _tokens(len(slots), H, D, torch.bfloat16)
    flat = torch.zeros(k.numel() + 1, dtype=k.dtype)
    flat[1:] = k.reshape(-1)
    _check_append(c, flat[1:].view(k.shape), v, slots, None)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.int8, torch.float8_e4m3fn])
def test_append_zeros_infinities_and_nan(kind):
    c = _cache(2, 2, 16, 32, kind)
    k, v, g = _tokens(6, 2, 32, torch.float32)
    k, v = k.clone(), v.clone()
    k[:, 0] = 0.0
    k[1, 1, 3], k[2, 1, 4], k[3, 1, 5] = INF, -INF, float("nan")
    v[:] = float("nan")
    v[:, 1, 7] = 1e-44
    _check_append(c, k, v, torch.arange(3, 9), g)


# ----------------------------------------------------------------------------- GPU: decode
def _filled(lens, Hk, D, page, kind, gated, width=None, seed=0):
    """A cache with ragged requests; what no request holds is filled with the worst codes and NaN."""
    g = torch.Generator().manual_seed(seed)
    pages = [-(-n // page) for n in lens]
    total = sum(pages) + 2
    order = torch.randperm(total, generator=g).to(torch.int32)
    width = max(max(pages), 1) if width is None else width
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    kc = torch.full((total, Hk, page, D), 0x7f, dtype=torch.uint8).view(kind)  # e4m3: NaN
    vc = kc.clone()
    ks, vs = torch.full((total, Hk), float("nan")), torch.full((total, Hk), float("nan"))
    gc = torch.full((total, Hk, page), float("nan")) if gated else None
    at = 0
    for r, n in enumerate(lens):
        for j in range(pages[r]):
            p = int(order[at])
            at += 1
            table[r, j] = p
            rows = min(page, n - j * page)
            slots = torch.arange(p * page, p * page + rows)
            paged_ref.append(torch.randn(rows, Hk, D, generator=g) * (0.3 + 2 * torch.rand(1, generator=g)),
                             slots - 0, kc[:], ks)
            paged_ref.append(torch.randn(rows, Hk, D, generator=g), slots, vc, vs)
            if gated:
                x = torch.nn.functional.logsigmoid(torch.randn(Hk, rows, generator=g))
                x[torch.rand(Hk, rows, generator=g) < 0.1] = -INF
                gc[p, :, :rows] = x
    return dict(k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, log_gate_cache=gc), table, \
        torch.tensor(lens, dtype=torch.int32)


def _check_decode(c, table, lens, q, scale=None, what="", **kw):
    import selective_attention_b200 as sab

    ref = paged_ref.decode(q, *(c[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")), table, lens,
                           c["log_gate_cache"], scale)
    dev = {n: None if t is None else t.cuda() for n, t in c.items()}
    got = sab.sattn_paged_decode(q.cuda(), block_table=table.cuda(), lengths=lens.cuda(), scale=scale, **dev, **kw)
    assert got.dtype == q.dtype and got.shape == q.shape
    k, live = c["v_cache"].float() * c["v_scale"][:, :, None, None], c["v_scale"].isfinite()
    vmax = k[live][k[live].isfinite()].abs().max().item() if bool(live.any()) else 1.0
    close(got, ref, vmax, what)
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("Hq,Hk,D,page,gated", [
    (4, 4, 64, 16, True), (8, 2, 128, 16, False), (7, 1, 128, 64, True), (16, 1, 64, 32, False),
    (10, 2, 32, 16, True), (4, 2, 256, 128, False), (40, 2, 128, 32, True),
])
def test_decode(kind, dtype, Hq, Hk, D, page, gated):
    lens = [0, 1, 2, page - 1, page, page + 1, 5 * page + 7, 700]
    c, table, n = _filled(lens, Hk, D, page, kind, gated)
    q = torch.randn(len(lens), Hq, D, generator=torch.Generator().manual_seed(3)).to(dtype)
    _check_decode(c, table, n, q)


@pytest.mark.gpu
@pytest.mark.parametrize("R,lens", [(1, [3000]), (1, [1]), (2, [2500, 31])])
def test_decode_few_requests_long_and_short(R, lens):
    c, table, n = _filled(lens, 1, 128, 16, torch.int8, True, width=220)
    q = torch.randn(R, 8, 128, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    got = _check_decode(c, table, n, q, scale=0.2)
    again = _check_decode(c, table, n, q, scale=0.2)
    assert torch.equal(got, again)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_decode_every_earlier_key_dropped_and_odd_values(dtype):
    """All gates -inf: the token's own value. Codes and scales of dropped keys do not matter; a NaN
    in a key that is seen, or in the query, makes its rows NaN and no others."""
    c, table, n = _filled([40, 40, 40], 2, 64, 16, torch.float8_e4m3fn, True)
    c["log_gate_cache"][:] = torch.where(c["log_gate_cache"].isnan(), c["log_gate_cache"], torch.tensor(-INF))
    p, q1 = int(table[1, 0]), int(table[2, 2])
    c["k_cache"].view(torch.uint8)[p, :, 3] = 0x7f
    c["v_cache"].view(torch.uint8)[p, :, 5] = 0xff
    c["v_cache"].view(torch.uint8)[q1, 1, 7, 9] = 0x7f  # the third request's own value
    q = torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(3)).to(dtype)
    q[0, 1, 5] = float("nan")
    _check_decode(c, table, n, q)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_decode_scales_and_queries_far_apart(dtype):
    """Pages whose scales differ by many orders, large and tiny queries, large scores."""
    c, table, n = _filled([130, 65], 2, 128, 16, torch.int8, False)
    f = 10.0 ** (torch.arange(c["v_scale"].shape[0]) % 7 - 5)[:, None]
    c["v_scale"] *= f
    q = torch.randn(2, 6, 128, generator=torch.Generator().manual_seed(3))
    q[0, 0] *= 100
    q[0, 1] *= 1e-4
    q[1, 2] = 0
    _check_decode(c, table, n, q.to(dtype))


@pytest.mark.gpu
def test_decode_table_entries_outside_the_cache_drop_out():
    import selective_attention_b200 as sab

    c, table, n = _filled([64], 1, 64, 16, torch.int8, False)
    dev = {k: None if t is None else t.cuda() for k, t in c.items()}
    q = torch.randn(1, 1, 64, generator=torch.Generator().manual_seed(3))
    for bad in (-1, 1 << 30):
        t2 = table.clone()
        t2[0, 1] = bad
        got = sab.sattn_paged_decode(q.cuda(), block_table=t2.cuda(), lengths=n.cuda(), **dev)
        keep = table[:, [0, 2, 3]]
        ref = paged_ref.decode(q, *(c[k] for k in ("k_cache", "v_cache", "k_scale", "v_scale")), keep,
                               torch.tensor([48]))
        close(got, ref, 5.0)


@pytest.mark.gpu
def test_decode_side_stream_out_and_empty_calls():
    import selective_attention_b200 as sab

    c, table, n = _filled([300, 20], 2, 64, 16, torch.int8, False, width=30)
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    dev = {k: None if t is None else t.cuda() for k, t in c.items()}
    t, nn, qq = table.cuda(), n.cuda(), q.cuda()
    out = torch.empty_like(qq)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = sab.sattn_paged_decode(qq, block_table=t, lengths=nn, out=out, **dev)
    s.synchronize()
    assert got.data_ptr() == out.data_ptr()
    assert torch.equal(out, sab.sattn_paged_decode(qq, block_table=t, lengths=nn, **dev))
    assert sab.sattn_paged_decode(qq[:0], block_table=t[:0], lengths=nn[:0], **dev).shape == (0, 4, 64)
    assert not sab.sattn_paged_decode(qq, block_table=t[:, :0].contiguous(), lengths=nn, **dev).any()


@pytest.mark.gpu
def test_gpu_refusals():
    import selective_attention_b200 as sab

    c = _cache(device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    q, t, n = torch.zeros(2, 4, 64, device="cuda"), torch.zeros(2, 3, **i32), torch.zeros(2, **i32)
    k, s, g = torch.zeros(1, 2, 64, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda"), \
        torch.zeros(1, 2, device="cuda")
    sab.sattn_paged_decode(q, block_table=t, lengths=n, **c)
    sab.sattn_paged_append(k, k, s, log_gate=g, **c)
    for bad in (dict(q=q[:, :3]), dict(q=q[..., :32]), dict(block_table=t.long()), dict(lengths=n[:1]),
                dict(k_cache=c["k_cache"].float()), dict(v_cache=c["v_cache"][:, :, :8]),
                dict(k_scale=c["k_scale"].half()), dict(v_scale=c["v_scale"].t()), dict(q=q.double()),
                dict(log_gate_cache=c["log_gate_cache"][:2]), dict(out=q.bfloat16())):
        with pytest.raises(ValueError):
            sab.sattn_paged_decode(**{**dict(q=q, block_table=t, lengths=n), **c, **bad})
    for bad in (dict(k=k[:, :1]), dict(v=k.half()), dict(slots=s.int()), dict(slots=s[:0]), dict(log_gate=None),
                dict(log_gate_cache=None), dict(k=k.double(), v=k.double()), dict(log_gate=g[:, :1])):
        with pytest.raises(ValueError):
            sab.sattn_paged_append(**{**dict(k=k, v=k, slots=s, log_gate=g), **c, **bad})
    with pytest.raises(ValueError):
        sab.sattn_paged_plan(n, n, t, n, s, 1, 16)  # free_state of one value
    with pytest.raises(ValueError):
        sab.sattn_paged_plan(n, n, t, n, torch.zeros(2, dtype=torch.int64, device="cuda"), 1, 17)
    with pytest.raises(ValueError):
        sab.sattn_paged_read(s.int(), *(c[x] for x in ("k_cache", "v_cache", "k_scale", "v_scale")))


# ----------------------------------------------------------------------------- GPU: all of it together
@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.int8, torch.float8_e4m3fn])
def test_cache_object_over_steps_with_requests_coming_and_going(kind):
    """Plans, appends, decodes and releases in turn: pages go round the ring, and each decode is that of
    the oracle on the cache as it stands."""
    import selective_attention_b200 as sab

    g = torch.Generator().manual_seed(5)
    c = sab.PagedSelectiveCache(2, 3, 64, 7, 2, 64, 16, kind)
    news = [[20, 0, 33], [1, 5, 1], [0, 1, 0], "release 0 2", [40, 1, 0], [1, 1, 16], "release 1", [0, 17, 1]]
    for new in news:
        if isinstance(new, str):
            rows = torch.tensor([int(x) for x in new.split()[1:]])
            c.release(rows.cuda())
            continue
        before = c.lengths.cpu()
        T = sum(new)
        cu, slots, pos = c.plan(torch.tensor(new, dtype=torch.int32, device="cuda"), T)
        n = c.lengths.cpu()
        assert n.tolist() == [b + a for b, a in zip(before.tolist(), new)], "every request is served"
        assert cu.tolist() == [0] + torch.tensor(new).cumsum(0).tolist()
        held = [p for r in range(3) for p in c.block_table[r, :-(-int(n[r]) // 16)].tolist()]
        assert len(set(held)) == len(held) and all(0 <= p < 7 for p in held), "no page has two owners"
        for layer in range(2):
            k, v = (torch.randn(T, 2, 64, generator=g).to(torch.bfloat16) for _ in range(2))
            gate = torch.nn.functional.logsigmoid(torch.randn(T, 2, generator=g))
            c.append(layer, k.cuda(), v.cuda(), slots, gate.cuda())
            q = torch.randn(3, 4, 64, generator=g).to(torch.bfloat16)
            at = {m: None if t is None else t.cpu() for m, t in c.layer(layer).items()}
            ref = paged_ref.decode(q, at["k_cache"], at["v_cache"], at["k_scale"], at["v_scale"], c.block_table.cpu(),
                                   n, at["log_gate_cache"])
            close(c.decode(layer, q.cuda()), ref, 5.0, f"{new} layer {layer}")
    assert c.free_state[0].item() - 7 <= c.free_state[1].item() - 7 <= c.free_state[0].item()


@pytest.mark.gpu
def test_cache_that_is_full_leaves_requests_waiting():
    import selective_attention_b200 as sab

    c = sab.PagedSelectiveCache(1, 2, 64, 2, 1, 64, 16)
    cu, slots, _ = c.plan(torch.tensor([30, 30], dtype=torch.int32, device="cuda"), 60)
    assert c.lengths.tolist() == [30, 0] and (slots[30:] == -1).all() and (slots[:30] >= 0).all()
    x = torch.randn(60, 1, 64, device="cuda")
    c.append(0, x, x, slots, torch.zeros(60, 1, device="cuda"))
    c.release(torch.tensor([0], device="cuda"))
    c.plan(torch.tensor([0, 30], dtype=torch.int32, device="cuda"), 30)
    assert c.lengths.tolist() == [0, 30]


@pytest.mark.gpu
def test_example_serves_every_request_and_returns_every_page():
    import importlib.util
    import os

    from conftest import ROOT

    spec = importlib.util.spec_from_file_location("serve_selective", os.path.join(ROOT, "examples", "serve_selective.py"))
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(512, (n,), generator=g).tolist() for n in (3, 40, 17, 1, 64)]
    budgets = [4, 2, 6, 5, 3]
    done, cache = ex.serve(prompts, budgets, rows=2)
    assert [len(done[i]) for i in range(5)] == [len(p) + b for p, b in zip(prompts, budgets)]
    assert all(done[i][:len(p)] == p for i, p in enumerate(prompts))
    head, tail = cache.free_state.tolist()
    assert tail - head == cache.free_pages.numel()  # every page is back
