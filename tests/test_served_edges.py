"""Served selective attention where values, weights or lengths are far from ordinary, against
``oracle/paged_ref.py``: page scales many orders apart, weights that underflow.

Tolerances are those of ``test_paged.py`` and ``test_sattn_packed.py``: a share of the result for its own rounding
and a share of the weighted magnitudes sum_j w_j |v_j| that the row adds up for the rounding of its weights, each of
which is relative. Where one group of keys holds all the weight, that sum is at most the group's largest |v|.
"""
import ctypes
import math

import pytest
import torch

from oracle import paged_ref

INF = float("inf")
NAN = float("nan")
PROMPT_TOL = {torch.bfloat16: (2 ** -8, 2 ** -8), torch.float16: (2 ** -10, 2 ** -10), torch.float32: (1e-5, 3e-5)}
DECODE_TOL = {torch.bfloat16: (2 ** -8, 2 ** -10), torch.float16: (2 ** -10, 2 ** -10), torch.float32: (1e-5, 3e-5)}


def close(got, ref, vmax, tol, what=""):
    rel, p = tol[got.dtype]
    got, ref = got.double().cpu(), ref.double().cpu()
    assert torch.equal(got.isnan(), ref.isnan()), f"{what}: NaN in other places"
    fine = ref.isfinite()
    assert torch.equal(got[ref.isinf()], ref[ref.isinf()]), f"{what}: infinities"
    err = (got - ref).abs()[fine]
    bound = rel * ref.abs()[fine] + p * vmax
    assert bool((err <= bound).all()), f"{what}: {int((err > bound).sum())} outside, max err {err.max().item():.3e}"


# ----------------------------------------------------------------------------- refusals (CPU)
def test_sizes_past_the_grids_are_invalid_arguments():
    from selective_attention_b200 import _lib

    L, bad = _lib.lib(), _lib.SSD_ERR_INVALID_ARGUMENT

    def cache(**kw):
        return ctypes.byref(_lib.SattnCache(**{**dict(num_pages=4, nkv=2, page_size=16, head_dim=64, code=0, k_codes=4096,
                                                      v_codes=4096, k_scale=4096, v_scale=4096, log_gate=None), **kw}))

    for c, requests in ((cache(), 65536), (cache(num_pages=2 ** 30), 1)):
        assert L.sattn_paged_decode(c, 4096, 4096, 4096, 4096, requests, 1, 2, 1.0, 1, 4096, 1 << 40, None) == bad
        assert L.sattn_paged_decode_workspace_size(c, requests, 1, 2) == 0
    for kw in (dict(num_seqs=65535), dict(num_tokens=256 * 65535, nkv=2), dict(num_tokens=128 * 65535),
               dict(num_tokens=64 * 65535, dtype=0), dict(num_tokens=64 * 65000, num_seqs=535, impl=_lib.IMPL_SIMT)):
        p = _lib.SattnPackedParams(**{**dict(
            num_tokens=4, num_seqs=1, nheads=2, nkv=1, head_dim=64, q_token_stride=128, q_head_stride=64,
            k_token_stride=64, k_head_stride=64, v_token_stride=64, v_head_stride=64, dtype=1, impl=0, scale=1.0, q=4096,
            k=4096, v=4096, log_gate=None, cu_seqlens=4096, out=4096), **kw})
        assert L.sattn_prefill_packed(ctypes.byref(p), None) == bad, kw


def test_an_impl_that_is_not_of_packed_prompts_is_refused():
    from selective_attention_b200 import _lib

    for impl in (_lib.IMPL_TC_STAGED, -1, 9):
        p = _lib.SattnPackedParams(num_tokens=0, num_seqs=1, nheads=2, nkv=1, head_dim=64, dtype=1, impl=impl)
        assert _lib.lib().sattn_prefill_packed(ctypes.byref(p), None) == _lib.SSD_ERR_INVALID_ARGUMENT


@pytest.mark.gpu
def test_tensors_of_other_ranks_are_refused():
    import selective_attention_b200 as sab

    c = {n: t.cuda() for n, t in _two_kinds_of_pages(torch.int8, 1.0)[0].items()}
    i32 = dict(dtype=torch.int32, device="cuda")
    q, k, slots = torch.zeros(2, 4, 64, device="cuda"), torch.zeros(3, 1, 64, device="cuda"), torch.arange(3, device="cuda")
    table, n, cu = torch.zeros(2, 3, **i32), torch.zeros(2, **i32), torch.zeros(2, **i32)
    state = torch.zeros(2, dtype=torch.int64, device="cuda")
    for bad in (dict(q=q[0, 0, 0]), dict(q=q[0, 0]), dict(q=q[0]), dict(q=q[None]), dict(block_table=table[0, 0]),
                dict(block_table=table[0]), dict(block_table=table[None]), dict(lengths=n[0]), dict(lengths=table)):
        with pytest.raises(ValueError):
            sab.sattn_paged_decode(**{**dict(q=q, block_table=table, lengths=n), **c, **bad})
    for bad in (dict(k=k[0, 0, 0]), dict(k=k[0]), dict(v=k[0, 0]), dict(slots=slots[0]), dict(slots=slots[None])):
        with pytest.raises(ValueError):
            sab.sattn_paged_append(**{**dict(k=k, v=k, slots=slots), **c, **bad})
    for bad in (dict(q=k[0, 0, 0]), dict(k=k[0]), dict(v=k[0, 0]), dict(cu_seqlens=cu[0]), dict(cu_seqlens=cu[None])):
        with pytest.raises(ValueError):
            sab.sattn_prefill_packed(**{**dict(q=k, k=k, v=k, cu_seqlens=cu), **bad})
    for bad in (dict(lengths=n[0]), dict(new_lengths=n[None]), dict(block_table=table[0]), dict(free_pages=n[0]),
                dict(free_state=state[0])):
        with pytest.raises(ValueError):
            sab.sattn_paged_plan(**{**dict(lengths=n, new_lengths=n, block_table=table, free_pages=n, free_state=state,
                                           num_tokens=0, page_size=16), **bad})
    with pytest.raises(ValueError):
        sab.sattn_paged_read(slots[0], *(c[x] for x in ("k_cache", "v_cache", "k_scale", "v_scale")))


# ----------------------------------------------------------------------------- decode: page scales
def _two_kinds_of_pages(kind, high, pages=24, page=16, D=64, seed=0):
    """A request whose pages are of two kinds in mixed order: first element of every key +1 or -1 (so that a
    query along it weighs one kind e^(2 |q|) times the other), values of scale ``high`` where it is -1."""
    g = torch.Generator().manual_seed(seed)
    minus = torch.arange(pages) % 3 == 1
    kc = torch.zeros(pages, 1, page, D)
    kc[..., 0] = torch.where(minus, -64.0, 64.0)[:, None, None]
    vc = (torch.rand(pages, 1, page, D, generator=g) * 2 - 1) * 96
    if kind == torch.int8:
        vc = vc.round()
    vs = torch.where(minus, high, 1.0 / 96)[:, None].float()
    c = dict(k_cache=kc.to(kind), v_cache=vc.to(kind), k_scale=torch.full((pages, 1), 1.0 / 64), v_scale=vs)
    return c, torch.arange(pages, dtype=torch.int32)[None], minus


def _decode(c, q, table, lengths, gate, scale):
    import selective_attention_b200 as sab

    dev = {n: t.cuda() for n, t in c.items()}
    got = sab.sattn_paged_decode(q.cuda(), block_table=table.cuda(), lengths=lengths.cuda(), scale=scale,
                                 log_gate_cache=None if gate is None else gate.cuda(), **dev)
    ref = paged_ref.decode(q, c["k_cache"], c["v_cache"], c["k_scale"], c["v_scale"], table, lengths, gate, scale)
    return got, ref


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("high", [1e4, 1e9, 1e20, INF, NAN])
def test_scales_of_dropped_pages_do_not_matter(kind, dtype, high):
    c, table, minus = _two_kinds_of_pages(kind, high)
    gate = torch.zeros(len(minus), 1, 16)
    gate[minus] = -INF
    q = torch.randn(1, 3, 64, generator=torch.Generator().manual_seed(3)).to(dtype)
    got, ref = _decode(c, q, table, torch.tensor([len(minus) * 16 - 3], dtype=torch.int32), gate, 0.5)
    close(got, ref, 1.0, DECODE_TOL)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("high", [1e4, 1e9, 1e15])
@pytest.mark.parametrize("heads", [2, 12])
def test_scales_of_pages_without_weight_do_not_matter_to_a_head(kind, dtype, high, heads):
    """Every second head weighs the other kind of pages: each has the bits that its own pages' values need."""
    c, table, minus = _two_kinds_of_pages(kind, high)
    q = torch.zeros(1, heads, 64)
    q[0, :, 0] = torch.where(torch.arange(heads) % 2 == 0, 40.0, -40.0)  # weights e^-80 of the other kind
    got, ref = _decode(c, q.to(dtype), table, torch.tensor([len(minus) * 16], dtype=torch.int32), None, 1.0)
    close(got[:, ::2], ref[:, ::2], 1.0 + math.exp(-80) * 96 * high, DECODE_TOL, "ordinary pages")
    if dtype != torch.float16:  # (whose range ends before these values)
        close(got[:, 1::2], ref[:, 1::2], 96.0 * high, DECODE_TOL, "pages of large values")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scale", [0.0, 1e-38, 1e-30, 1e30])
def test_values_near_the_ends_of_the_range(dtype, scale):
    c, table, minus = _two_kinds_of_pages(torch.int8, scale)
    c["v_scale"][:] = scale
    q = torch.randn(1, 2, 64, generator=torch.Generator().manual_seed(3)).to(dtype)
    got, ref = _decode(c, q, table, torch.tensor([len(minus) * 16], dtype=torch.int32), None, 0.5)
    close(got, ref, 96.0 * scale + 1e-38, DECODE_TOL)


# ----------------------------------------------------------------------------- decode: workspace
@pytest.mark.gpu
@pytest.mark.parametrize("how", ["expanded", "strided", "short", "unaligned"])
def test_a_workspace_that_is_not_one_piece_of_memory_is_not_written(how):
    """Its numel says nothing of the bytes behind it: the call takes one of its own."""
    import selective_attention_b200 as sab

    c, table, _ = _two_kinds_of_pages(torch.int8, 0.01, pages=120)
    dev = {n: t.cuda() for n, t in c.items()}
    args = dict(block_table=table.cuda(), lengths=torch.tensor([1900], dtype=torch.int32, device="cuda"), **dev)
    q = torch.randn(1, 2, 64, generator=torch.Generator().manual_seed(3)).cuda()
    want = sab.sattn_paged_decode(q, **args)
    held = torch.zeros(1 << 23, dtype=torch.uint8, device="cuda")
    work = {"expanded": held[:1].expand(1 << 22), "strided": held[::2], "short": held[:64],
            "unaligned": held[8:]}[how]
    assert torch.equal(sab.sattn_paged_decode(q, workspace=work, **args), want) and not held.any()
    good = held[:1 << 22]
    assert torch.equal(sab.sattn_paged_decode(q, workspace=good, **args), want) and bool(held.any())


# ----------------------------------------------------------------------------- packed prompts
def _prompt(q, k, v, gate=None, scale=None, impl="auto"):
    import selective_attention_b200 as sab

    cu = torch.tensor([0, q.shape[0]], dtype=torch.int32)
    got = sab.sattn_prefill_packed(q.cuda(), k.cuda(), v.cuda(), cu.cuda(), None if gate is None else gate.cuda(), scale,
                                   impl=impl)
    sab.check_device_error()
    return got, paged_ref.prefill_packed(q, k, v, cu, gate, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("T", [20, 150])
def test_a_nan_under_a_weight_that_underflows_is_seen(dtype, D, T):
    """A key's value is NaN and its score 400 below the others: rows from its position on see it."""
    g = torch.Generator().manual_seed(T + D)
    q, k, v = (torch.randn(T, 1, D, generator=g) * 0.1 for _ in range(3))
    q[..., 0], k[..., 0] = 20.0, 10.0
    at = T - 9
    k[at, 0, 0] = -10.0
    v[at, 0, 3] = NAN
    q, k, v = (x.to(dtype) for x in (q, k, v))
    got, ref = _prompt(q, k, v, scale=1.0)
    assert bool(ref[at:, 0, 3].isnan().all()) and not bool(ref[:at].isnan().any())
    close(got, ref, v[v.isfinite()].float().abs().max().item(), PROMPT_TOL)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
def test_many_keys_of_small_weight_add_up(dtype, D):
    """One key of weight 1 and value 0, and 131000 keys of weight e^-16.2 (1.55 steps of fp16's smallest number) and value 1:
    together they are 1 % of the sum. The last rows are compared; q and k are exact, so the oracle is their sum."""
    import selective_attention_b200 as sab

    T, gap = 131000, 16.2
    q, k, v = (torch.zeros(T, 1, D, dtype=dtype) for _ in range(3))
    q[:, 0, 0] = 1.0
    k[0, 0, 0] = 8.0
    k[1:, 0, 0] = 8.0 - 16.0
    v[1:] = 1.0
    scale = gap / 16
    cu = torch.tensor([0, T], dtype=torch.int32)
    got = sab.sattn_prefill_packed(q.cuda(), k.cuda(), v.cuda(), cu.cuda(), None, scale)[-300:]
    sab.check_device_error()
    n = torch.arange(T - 300, T, dtype=torch.float64)
    w = n * math.exp(-gap)
    ref = (w / (1 + w))[:, None, None].expand(-1, 1, D)
    # a weight's rounding is relative (the weighted magnitudes are the result itself), but half a step of 2^-31 of the
    # largest weight where float16 has no exponent left; the scores' own roundings in 32 bits move a weight by 1e-4 at most
    rel, least = {torch.bfloat16: (2 ** -7, 0.0), torch.float16: (2 ** -9, 2 ** -32)}[dtype]
    err = (got.double().cpu() - ref).abs()
    bound = (rel + 1e-4) * ref + T * least
    assert bool((err <= bound).all()), f"max relative err {(err / ref).max().item():.3e}"


# ----------------------------------------------------------------------------- plan: tokens past the planned ones
MANY = 2 ** 31 - 1


def _plan(lengths, new, width, num_tokens, page=16, free=64):
    args = (torch.tensor(lengths, dtype=torch.int32), torch.tensor(new, dtype=torch.int32),
            torch.full((len(lengths), width), -1, dtype=torch.int32), torch.arange(free, dtype=torch.int32).flip(0).contiguous(),
            torch.tensor([0, free]))
    for r, n in enumerate(lengths):
        args[2][r, :-(-n // page)] = 100 + r
    return args, num_tokens, page


PAST = [_plan([0, 0, 0], [20, 30, 5], 4, 54), _plan([0, 0, 0], [20, 30, 5], 4, 20), _plan([0, 0], [20, 30], 4, 19),
        _plan([3, 40, 0, 9], [2, 0, 60, 0], 4, 10), _plan([5], [3], 2, 0), _plan([0] * 300, [7] * 300, 1, 1500, free=300),
        _plan([0, 0, 0, 0], [5, MANY, MANY, 6], 4, 12), _plan([0] * 600, [9] + [MANY] * 598 + [5], 4, 1100),
        # sums that pass 2^32 by a little
        _plan([0, 0, 0, 0], [MANY, MANY, 2, 9], 4, 100), _plan([0] * 34, [5] + [MANY] * 32 + [50], 4, 60)]


@pytest.mark.parametrize("case", PAST)
def test_plan_oracle_serves_no_request_past_the_planned_tokens(case):
    (lengths, new, table, free, state), T, page = case
    got, n, cu, slots, _, st = paged_ref.plan(lengths, new, table, free, state, T, page)
    assert slots.numel() == T and st[0] - state[0] == ((got >= 0) & (table < 0)).sum()
    for r in range(len(n)):
        pages = -(-int(n[r]) // page)
        assert bool((got[r, :pages] >= 0).all()) and bool((got[r, pages:] == -1).all())


@pytest.mark.gpu
@pytest.mark.parametrize("case", PAST)
def test_plan_serves_no_request_past_the_planned_tokens(case):
    """Every request holds just the pages that its table names, whatever its new length."""
    import selective_attention_b200 as sab

    args, T, page = case
    ref = paged_ref.plan(*args, T, page)
    dev = [a.cuda() for a in args]
    got = sab.sattn_paged_plan(*dev, T, page)
    assert torch.equal(dev[2].cpu(), ref[0])
    for g, r, n in zip(got, ref[1:], ("lengths", "cu", "slots", "positions", "free_state")):
        assert torch.equal(g.cpu(), r), n


@pytest.mark.gpu
def test_pages_come_back_whole_after_a_plan_for_too_few_tokens():
    import selective_attention_b200 as sab

    c = sab.PagedSelectiveCache(1, 2, 64, 6, 1, 64, 16)
    c.plan(torch.tensor([20, 20], dtype=torch.int32, device="cuda"), 39)
    assert c.lengths.tolist() == [20, 0]
    c.release(torch.tensor([0, 1], device="cuda"))
    head, tail = c.free_state.tolist()
    ring = c.free_pages.tolist()
    assert sorted(ring[i % 6] for i in range(head, tail)) == list(range(6))


# ----------------------------------------------------------------------------- gates of the type's lowest value
LOWEST = torch.finfo(torch.float32).min


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
def test_a_gate_of_the_lowest_value_does_not_drop_its_key_from_prompts(dtype, D):
    """Only -inf drops a key. One with the lowest finite gate has no weight, but a NaN there is seen."""
    g = torch.Generator().manual_seed(D)
    T = 300
    q, k, v = (torch.randn(T, 2, D, generator=g).to(dtype) for _ in range(3))
    gate = torch.nn.functional.logsigmoid(torch.randn(T, 2, generator=g))
    gate[torch.rand(T, 2, generator=g) < 0.5] = LOWEST
    vmax = v.float().abs().max().item()
    got, ref = _prompt(q, k, v, gate)
    close(got, ref, vmax, PROMPT_TOL, "no weight")
    gate[:, 1] = LOWEST
    got, ref = _prompt(q, k, v, gate)
    close(got, ref, vmax, PROMPT_TOL, "no weight for any earlier key")
    gate[[5, 270]], v[5, 0, 2], v[270, 1, 7] = LOWEST, NAN, NAN
    gate[[9, 280]], v[9, 0, 3], v[280, 1, 4] = -INF, NAN, NAN  # these rows alone
    got, ref = _prompt(q, k, v, gate)
    assert bool(ref[5:, 0, 2].isnan().all()) and bool(ref[270:, 1, 7].isnan().all())
    assert int(ref[:, 0, 3].isnan().sum()) == 1 and int(ref[:, 1, 4].isnan().sum()) == 1
    close(got, ref, vmax, PROMPT_TOL, "NaN")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_gate_of_the_lowest_value_does_not_drop_its_key_from_a_decode(dtype):
    c, table, _ = _two_kinds_of_pages(torch.float8_e4m3fn, 1.0 / 96)
    gate = torch.full((24, 1, 16), LOWEST)
    gate[7] = -INF
    c["v_cache"].view(torch.uint8)[4, 0, 3, 5] = 0x7f  # seen
    c["v_cache"].view(torch.uint8)[7, 0, 3, 6] = 0x7f  # dropped
    q = torch.randn(1, 2, 64, generator=torch.Generator().manual_seed(3)).to(dtype)
    got, ref = _decode(c, q, table, torch.tensor([24 * 16], dtype=torch.int32), gate, 0.5)
    assert bool(ref[..., 5].isnan().all()) and not bool(ref[..., 6].isnan().any())
    close(got, ref, 1.0, DECODE_TOL)


# ----------------------------------------------------------------------------- decode: many rows to join
@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hk,D,gated", [(16, 2, 64, True), (20, 2, 128, False), (16, 4, 256, False), (16, 1, 32, True)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_rows_that_several_ctas_share(Hq, Hk, D, gated, dtype):
    """From 592 requests x query heads on a row's parts are joined by four warps instead of sixteen."""
    from test_paged import _check_decode, _filled

    lens = [(97 * i) % 331 for i in range(39)] + [620]
    c, table, n = _filled(lens, Hk, D, 16, torch.int8, gated)
    q = torch.randn(len(lens), Hq, D, generator=torch.Generator().manual_seed(3)).to(dtype)
    got = _check_decode(c, table, n, q)
    assert torch.equal(got, _check_decode(c, table, n, q))


# ----------------------------------------------------------------------------- captured calls
@pytest.mark.gpu
def test_captured_append_decode_and_prompts_replay():
    """The functions' launches in a graph, on inputs that change between replays; the calls' own tensors are the state."""
    import selective_attention_b200 as sab

    g = torch.Generator().manual_seed(1)
    c = sab.PagedSelectiveCache(1, 3, 1024, 200, 2, 64)
    lens = [700, 33, 300]
    cu, slots, _ = c.plan(torch.tensor(lens, dtype=torch.int32, device="cuda"), sum(lens))
    k, v = (torch.randn(sum(lens), 2, 64, generator=g).bfloat16().cuda() for _ in range(2))
    q = torch.randn(sum(lens), 4, 64, generator=g).bfloat16().cuda()
    gate = torch.nn.functional.logsigmoid(torch.randn(sum(lens), 2, generator=g)).cuda()

    def step():
        c.append(0, k, v, slots, gate)
        return sab.sattn_prefill_packed(q, k, v, cu, gate), c.decode(0, q[:3])

    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = step()
    for _ in range(2):
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=g).bfloat16())
        graph.replay()
        got = [o.clone() for o in outs]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)
