"""Selective attention over packed prompts against ``oracle/paged_ref.py`` in 64 bits.

Tolerances. fp32: fp32 sums and expf, 1e-5 of the result and 3e-5 of the largest |v|. 16-bit: the
products' inputs are exact, a probability is rounded to the dtype before its product (2^-9
of itself in bfloat16, 2^-11 in float16; the exponential itself is good to 2^-12), so the
output is off by at most that much of the largest |v| a row can see, and it is rounded once:
|err| <= 2^-8 |out| + 2^-8 max|v| in bfloat16, 2^-10 |out| + 2^-10 max|v| in float16.
"""
import ctypes

import pytest
import torch

from oracle import paged_ref

INF = float("inf")
TOL = {torch.bfloat16: (2 ** -8, 2 ** -8), torch.float16: (2 ** -10, 2 ** -10), torch.float32: (1e-5, 3e-5)}


def close(got, ref, vmax, what=""):
    rel, p = TOL[got.dtype]
    got, ref = got.double().cpu(), ref.double().cpu()
    assert torch.equal(got.isnan(), ref.isnan()), f"{what}: NaN in other places"
    inf = ref.isinf()
    assert torch.equal(got[inf], ref[inf]), f"{what}: infinities"
    fine = ref.isfinite()
    err = (got - ref).abs()[fine]
    bound = rel * ref.abs()[fine] + p * vmax
    assert bool((err <= bound).all()), f"{what}: {int((err > bound).sum())} outside, max err {err.max().item():.3e}"


def make(lens, Hq, Hk, D, dtype, gated, seed=0, extra=0):
    g = torch.Generator().manual_seed(seed)
    T = sum(lens) + extra
    qkv = torch.randn(T, Hq + 2 * Hk, D, generator=g).to(dtype)
    gate = None
    if gated:
        gate = torch.nn.functional.logsigmoid(torch.randn(T, Hk, generator=g) + 1)
        gate[torch.rand(T, Hk, generator=g) < 0.1] = -INF
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    return qkv, gate, cu


def check(qkv, gate, cu, Hq, Hk, scale=None, impl="auto", what="", split=True):
    import selective_attention_b200 as sab

    parts = (slice(0, Hq), slice(Hq, Hq + Hk), slice(Hq + Hk, Hq + 2 * Hk))
    ref = paged_ref.prefill_packed(*(qkv[:, p] for p in parts), cu, gate, scale)
    d = qkv.cuda()
    args = [d[:, p] if split else d[:, p].contiguous() for p in parts]
    got = sab.sattn_prefill_packed(*args, cu.cuda(), None if gate is None else gate.cuda(), scale, impl=impl)
    sab.check_device_error()
    v = qkv[:, parts[2]].float()
    close(got, ref, v[v.isfinite()].abs().max().item() if v.numel() else 1.0, what)
    return got


def test_refusals_on_the_cpu():
    import selective_attention_b200 as sab
    from selective_attention_b200 import _lib

    x = torch.zeros(4, 2, 64)
    with pytest.raises(ValueError):
        sab.sattn_prefill_packed(x, x, x, torch.tensor([0, 4], dtype=torch.int32))
    L = _lib.lib()

    def call(**kw):
        d = dict(num_tokens=4, num_seqs=1, nheads=2, nkv=1, head_dim=64, q_token_stride=128, q_head_stride=64,
                 k_token_stride=64, k_head_stride=64, v_token_stride=64, v_head_stride=64, dtype=1, impl=0, scale=1.0,
                 q=4096, k=4096, v=4096, log_gate=None, cu_seqlens=4096, out=4096)
        d.update(kw)
        return L.sattn_prefill_packed(ctypes.byref(_lib.SattnPackedParams(**d)), None)

    bad = _lib.SSD_ERR_INVALID_ARGUMENT
    for kw in (dict(nheads=3, nkv=2), dict(head_dim=48), dict(q=None), dict(out=4098), dict(k_token_stride=65),
               dict(v_head_stride=-64), dict(num_tokens=-1), dict(num_seqs=-1), dict(nkv=0), dict(cu_seqlens=None),
               dict(impl=_lib.IMPL_TC, dtype=0), dict(impl=_lib.IMPL_TC, head_dim=32)):
        assert call(**kw) == bad, kw
    assert call(dtype=9) == _lib.SSD_ERR_UNSUPPORTED_DTYPE
    assert call(num_tokens=0, q=None) == 0
    assert L.sattn_prefill_packed(None, None) == bad


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("Hq,Hk,D,gated", [(4, 1, 64, False), (2, 2, 64, True), (6, 2, 128, False), (4, 4, 128, True),
                                           (3, 1, 32, True), (2, 1, 16, False)])
def test_ragged(dtype, Hq, Hk, D, gated):
    lens = [1, 63, 64, 65, 0, 127, 128, 129, 200, 300]
    check(*make(lens, Hq, Hk, D, dtype, gated), Hq, Hk)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("lens", [[1], [2], [255], [256], [257], [700, 1], [1, 385], [0, 0, 5], [0], [129, 0, 513]])
@pytest.mark.parametrize("D", [64, 128])
def test_lengths(dtype, lens, D):
    check(*make(lens, 2, 1, D, dtype, True), 2, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("D", [64, 128])
def test_long_and_short_works_follow_one_another(D, gated):
    """Heads that cannot be paired: works of two, one and no second tile, several for each CTA, checked
    against the CUDA-core kernel (fp32 sums over the same 16-bit inputs), twice with the same result."""
    import selective_attention_b200 as sab

    lens = [2047, 1, 758, 1266, 300, 129, 1900, 17, 640, 1024, 385]
    qkv, gate, cu = make(lens, 24, 24, D, torch.bfloat16, gated, seed=9)
    d, g = qkv.cuda(), None if gate is None else gate.cuda()
    args = (d[:, :24], d[:, 24:48], d[:, 48:], cu.cuda(), g)
    ref = sab.sattn_prefill_packed(*args, impl="simt")
    got = sab.sattn_prefill_packed(*args, impl="tc")
    sab.check_device_error()
    vmax = d[:, 48:].float().abs().max().item()
    close(got, ref.float(), 2 * vmax, "against the CUDA cores")  # (both sides round)
    for _ in range(3):
        assert torch.equal(got, sab.sattn_prefill_packed(*args, impl="tc"))


@pytest.mark.gpu
@pytest.mark.parametrize("impl", ["auto", "simt"])
def test_many_short_sequences_and_padding_rows(impl):
    lens = [(7 * i) % 41 for i in range(150)]
    got = check(*make(lens, 3, 3, 64, torch.bfloat16, False, extra=600), 3, 3, impl=impl)
    assert not got[sum(lens):].any()
    qkv, gate, cu = make([], 2, 1, 128, torch.bfloat16, False, extra=70)  # no sequence at all
    assert not check(qkv, gate, cu, 2, 1, impl=impl).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
def test_what_is_not_seen_changes_nothing(dtype, D):
    """NaN and infinities in the keys and values of other sequences, of later positions and of dropped
    keys stay out; where a row sees one, that row has it."""
    lens = [100, 130, 300, 40]
    qkv, gate, cu = make(lens, 2, 1, D, dtype, True)
    k, v = qkv[:, 2], qkv[:, 3]
    nan = float("nan")
    v[0:100, 3] = nan            # a whole sequence next to others
    k[230 + 60] = nan            # rows from 60 on of the third
    v[230 + 200, 5] = INF        # rows from 200 on, one column
    gate[230 + 60:] = gate[230 + 60:].clamp(min=-3.0)
    v[100 + 20, 7], k[100 + 30] = nan, nan
    gate[100 + 20], gate[100 + 30] = -INF, -INF  # only their own rows
    v[100 + 128, 1] = -INF
    v[-1, 2] = nan               # the last row of the last sequence only
    qkv[530 + 7, 1, 0] = nan     # one query of one head
    check(qkv, gate, cu, 2, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
def test_all_keys_dropped_and_large_scores(dtype, D):
    qkv, gate, cu = make([300, 150], 2, 2, D, dtype, True)
    gate[:] = -INF
    check(qkv, gate, cu, 2, 2, what="every earlier key dropped")
    qkv, gate, cu = make([300, 150], 2, 2, D, dtype, False, seed=4)
    qkv[:, :4] *= 8
    check(qkv, gate, cu, 2, 2, scale=0.5, what="large scores")
    qkv[:, 0] = 0
    check(qkv, gate, cu, 2, 2, what="even weights")


@pytest.mark.gpu
def test_layouts_streams_and_refusals():
    import selective_attention_b200 as sab

    qkv, gate, cu = make([90, 170], 4, 2, 64, torch.bfloat16, True)
    got = check(qkv, gate, cu, 4, 2)
    assert torch.equal(got, check(qkv, gate, cu, 4, 2, split=False))
    d, cud, gd = qkv.cuda(), cu.cuda(), gate.cuda()
    q, k, v = d[:, :4], d[:, 4:6], d[:, 6:]
    # heads first in memory, an odd start, rows apart
    hf = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    assert torch.equal(got, sab.sattn_prefill_packed(*hf, cud, gd))
    flat = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")
    flat[1:] = q.reshape(-1)
    assert torch.equal(got, sab.sattn_prefill_packed(flat[1:].view(q.shape), k, v, cud, gd))
    wide = torch.zeros(260, 4, 67, dtype=q.dtype, device="cuda")
    wide[..., :64] = q
    assert torch.equal(got, sab.sattn_prefill_packed(wide[..., :64], k, v, cud, gd))
    # one key head spread over both
    one = k[:, :1].expand(-1, 2, -1)
    assert torch.equal(sab.sattn_prefill_packed(q, one, v, cud), sab.sattn_prefill_packed(q, one.contiguous(), v, cud))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    out = torch.empty(260, 4, 64, dtype=q.dtype, device="cuda")
    with torch.cuda.stream(s):
        sab.sattn_prefill_packed(q, k, v, cud, gd, out=out)
    s.synchronize()
    assert torch.equal(out, got)
    assert sab.sattn_prefill_packed(q[:0], k[:0], v[:0], cud[:1]).shape == (0, 4, 64)
    for bad in (dict(q=q[:, :3]), dict(k=k.half()), dict(v=v[:1]), dict(cu_seqlens=cud.long()), dict(log_gate=gd[:, :1]),
                dict(cu_seqlens=cud[:0]), dict(out=out[:1]), dict(q=q.double(), k=k.double(), v=v.double()),
                dict(q=q[..., :48], k=k[..., :48], v=v[..., :48])):
        with pytest.raises(ValueError):
            sab.sattn_prefill_packed(**{**dict(q=q, k=k, v=v, cu_seqlens=cud, log_gate=gd), **bad})
