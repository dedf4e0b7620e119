"""Attention over long rows and the norm + rotation of queries and keys (``mmt::long_attention``, ``mmt::qk_norm_rope``) against 64-bit
restatements, element by element within the bound that rounding allows (oracle/long_rows.py derives it), and their refusals."""
import ctypes
import math

import pytest
import torch

from multimodal_transformer_amd import _lib, ops, torch_ops
from multimodal_transformer_amd._lib import MmtError
from oracle import long_rows

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
TYPES = [BF16, F16, F32]
IDS = {BF16: "bf16", F16: "fp16", F32: "fp32"}
DEV = "cuda:0"


# ---------------------------------------------------------------------------------------------------------------- CPU: refusals
def _desc(**kw):
    a = _lib.LongAttention()
    a.q = a.k = a.v = 0x1000
    a.dtype, a.B, a.Lq, a.Lk, a.H, a.Hk, a.dh, a.scale = _lib.MMT_BF16, 2, 5, 7, 4, 2, 64, 0.125
    a.q_bs, a.q_rs, a.q_hs = 5 * 256, 256, 64
    a.k_bs = a.v_bs = 7 * 128
    a.k_rs = a.v_rs = 128
    a.k_hs = a.v_hs = 64
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad,word", [
    (dict(q=0), b"null"), (dict(dtype=7), b"type"), (dict(B=0), b"positive"), (dict(Lq=0), b"positive"), (dict(Lk=-3), b"positive"),
    (dict(Hk=3), b"multiple"), (dict(dh=60), b"head size"), (dict(dh=136), b"head size"), (dict(scale=0.0), b"scale"),
    (dict(scale=math.nan), b"scale"), (dict(scale=-1.0), b"scale"), (dict(softcap=-1.0), b"cap"), (dict(softcap=math.inf), b"cap"),
    (dict(prefix=0x1000), b"prefix"), (dict(q_doc=0x1000), b"documents"), (dict(rel_bias=0x1000), b"bias"),
    (dict(rel_bias=0x1000, rel_buckets=0x1000, n_buckets=65, reach=8), b"buckets"),
    (dict(rel_bias=0x1000, rel_buckets=0x1000, n_buckets=8, reach=0), b"reach"),
    (dict(rel_bias=0x1000, rel_buckets=0x1000, n_buckets=64, reach=1025), b"reach"),
    (dict(q=0x1008), b"16 bytes"), (dict(k_rs=129), b"16 bytes"), (dict(B=1 << 30, Lq=1 << 20), b"too many")])
def test_attention_refuses_on_the_host(bad, word):
    """Every argument the kernels could not run with is an error of the call, before anything is launched."""
    lib = _lib.load()
    a = _desc(**bad)
    assert lib.mmt_long_attention_workspace_bytes(ctypes.byref(a), 1) == 0
    rc = lib.mmt_long_attention_fwd(ctypes.byref(a), 0x1000, None, None, 0x1000, 1 << 40, None)
    assert rc == -1 and word in lib.mmt_last_error()
    rc = lib.mmt_long_attention_bwd(ctypes.byref(a), 0x1000, None, 0x1000, 0x1000, 0, 0, 0, None, 0x1000, 0x1000, 0x1000, 0x1000, 0x1000, 1 << 40,
                                    None)
    assert rc == -1 and word in lib.mmt_last_error()


def test_attention_refuses_missing_outputs_and_small_workspaces():
    lib = _lib.load()
    a = _desc(rel_bias=0x1000, rel_buckets=0x1000, n_buckets=8, reach=8)
    need = lib.mmt_long_attention_workspace_bytes(ctypes.byref(a), 1)
    assert need > 0
    fwd = lambda out, ws, n: lib.mmt_long_attention_fwd(ctypes.byref(a), out, None, None, ws, n, None)
    bwd = lambda dq, bias, ws, n, dout=0x1000: lib.mmt_long_attention_bwd(ctypes.byref(a), 0x1000, None, 0x1000, dout, 0, 0, 0, None, dq, 0x1000,
                                                                          0x1000, bias, ws, n, None)
    assert fwd(None, 0x1000, 1 << 40) == -1 and fwd(0x1004, 0x1000, 1 << 40) == -1
    assert bwd(None, 0x1000, 0x1000, need) == -1 and bwd(0x1000, None, 0x1000, need) == -1
    assert bwd(0x1000, 0x1000, 0x1000, need - 1) == -1 and b"workspace" in lib.mmt_last_error()
    assert bwd(0x1000, 0x1000, None, need) == -1 and bwd(0x1000, 0x1000, 0x1004, need) == -1
    assert bwd(0x1000, 0x1000, 0x1000, need, dout=0x1002) == -1
    assert lib.mmt_long_attention_fwd(None, 0x1000, None, None, None, 0, None) == -1
    long = _desc(Lq=1, Lk=4096, B=1)                      # split over the keys: needs somewhere to put the parts
    need = lib.mmt_long_attention_workspace_bytes(ctypes.byref(long), 0)
    assert need > 0
    assert lib.mmt_long_attention_fwd(ctypes.byref(long), 0x1000, None, None, None, 0, None) == -1 and b"workspace" in lib.mmt_last_error()


@pytest.mark.parametrize("bad,word", [
    (dict(q=0), b"null"), (dict(inv_freq=0), b"null"), (dict(dtype=5), b"type"), (dict(w_dtype=_lib.MMT_F16), b"weights"),
    (dict(L=0), b"positive"), (dict(Hk=0), b"positive"), (dict(dh=12), b"head size"), (dict(dh=264), b"head size"),
    (dict(rot=7), b"even"), (dict(rot=72), b"even"), (dict(rot=0), b"even"), (dict(eps=-1.0), b"eps"), (dict(eps=math.nan), b"eps"),
    (dict(k=0x1004), b"16 bytes"), (dict(q_hs=60), b"16 bytes"), (dict(H=70000), b"too many")])
def test_norm_rope_refuses_on_the_host(bad, word):
    lib = _lib.load()
    a = _lib.QkNormRope()
    a.q = a.k = a.q_weight = a.k_weight = a.inv_freq = 0x1000
    a.dtype = a.w_dtype = _lib.MMT_BF16
    a.B, a.L, a.H, a.Hk, a.dh, a.rot, a.eps = 2, 3, 4, 2, 64, 64, 1e-6
    a.q_bs, a.q_rs, a.q_hs, a.k_bs, a.k_rs, a.k_hs = 768, 256, 64, 384, 128, 64
    for k, v in bad.items():
        setattr(a, k, v)
    assert lib.mmt_qk_norm_rope_workspace_bytes(ctypes.byref(a)) == 0
    assert lib.mmt_qk_norm_rope_fwd(ctypes.byref(a), 0x1000, 0x1000, None) == -1 and word in lib.mmt_last_error()
    rc = lib.mmt_qk_norm_rope_bwd(ctypes.byref(a), 0x1000, 0, 0, 0, 0x1000, 0, 0, 0, 0x1000, 0x1000, 0x1000, 0x1000, 0x1000, 1 << 40, None)
    assert rc == -1 and word in lib.mmt_last_error()


def test_host_tensors_are_refused_and_shapes_propagate():
    q, k = torch.zeros(2, 3, 4, 16), torch.zeros(2, 5, 2, 16)
    with pytest.raises(MmtError):
        torch_ops.long_attention(q, k, k)
    with pytest.raises(MmtError):
        ops.long_attention(q, k, k)
    with pytest.raises(MmtError):
        torch_ops.qk_norm_rope(q, q, torch.ones(16), torch.ones(16), ops.rotary_frequencies(16))
    with pytest.raises(NotImplementedError):
        torch.ops.mmt.long_attention(q, k, k, None, False, None, None, None, None, 0.0, None, None, None)
    with torch.device("meta"):
        q, k, w = torch.empty(2, 3, 4, 16, dtype=BF16), torch.empty(2, 5, 2, 16, dtype=BF16), torch.empty(16)
        out, lse, low = torch.ops.mmt.long_attention(q, k, k, None, False, None, None, None, None, 0.0, None, None, None)
        assert low.shape == q.shape and out.shape == q.shape and out.dtype == BF16 and lse.shape == (2, 4, 3) and lse.dtype == F32
        a, b = torch.ops.mmt.qk_norm_rope(q, q[:, :, :2], w, w, torch.empty(8, dtype=torch.float64), None, 1e-6, False)
        assert a.shape == q.shape and b.shape == (2, 3, 2, 16)


def test_relative_buckets():
    """Exact at the borders: with 8 logarithmic steps from 8 to 128 a step is half an octave, so 16, 32 and 64 start a bucket."""
    t = ops.relative_buckets(16, 128, False).tolist()
    of = {d: t[128 - d] for d in range(129)}
    assert [of[d] for d in range(8)] == list(range(8))
    assert of[8] == 8 and of[15] == 9 and of[16] == 10 and of[31] == 11 and of[32] == 12 and of[63] == 13 and of[64] == 14 and of[128] == 15
    assert all(t[128 + d] == 0 for d in range(1, 129))
    t = ops.relative_buckets(32, 128, True).tolist()
    assert len(t) == 257 and t[128] == 0 and t[129] == 17 and t[127] == 1 and t[0] == 15 and t[256] == 31
    assert all(t[128 + d] == 16 + t[128 - d] for d in range(1, 129))
    for n, reach, both in ((1, 8, False), (3, 8, True), (2, 8, True), (66, 128, False), (32, 8, False)):
        with pytest.raises(MmtError):
            ops.relative_buckets(n, reach, both)
    with pytest.raises(MmtError):
        ops.rotary_frequencies(7)
    assert ops.rotary_frequencies(8, 100.0).tolist() == pytest.approx([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], rel=1e-15)


# ------------------------------------------------------------------------------------------------------------------------- GPU
def _near(got, want, tol, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, what
    same = (got == want) | (torch.isinf(want) & (got == want))
    bad = ~same & ~((got - want).abs() <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} elements off, worst {float((got - want).abs()[bad].max()):.3e} "
                           f"where {float(tol[bad].min()):.3e} is allowed, first at {bad.nonzero()[0].tolist()}")


def _case(dtype, B, Lq, Lk, H, Hk, dh, seed=0, docs=None, prefix=False, cache=False, slopes=False, buckets=0, reach=0, both=False, spread=1.0):
    """Inputs of a case on the GPU; ``docs``: per batch row a list of (id, length)."""
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: (torch.randn(*s, generator=g) * spread).to(dtype).to(DEV)
    t = {"q": rnd(B, Lq, H, dh), "k": rnd(B, Lk, Hk, dh), "v": rnd(B, Lk, Hk, dh), "go": rnd(B, Lq, H, dh)}
    kw = {}
    if docs is not None:
        ids = torch.tensor([[i for i, n in row for _ in range(n)] for row in docs], dtype=torch.int32)
        assert ids.shape == (B, Lk)
        kw["k_doc"] = ids.to(DEV)
        kw["q_doc"] = ids[:, Lk - Lq:].contiguous().to(DEV)
    if prefix:
        kw["prefix"] = torch.tensor([(7 * b + 3) % (Lk + 2) for b in range(B)], dtype=torch.int32, device=DEV)
    if cache:
        kw["kv_len"] = torch.tensor([(Lk, 0, 1, Lq, Lk - 1, (Lk + Lq) // 2)[b % 6] for b in range(B)], dtype=torch.int32, device=DEV)
    if slopes:
        kw["slopes"] = torch.tensor([2.0 ** -(h + 1) for h in range(H)], device=DEV)
    if buckets:
        kw["rel_buckets"] = ops.relative_buckets(buckets, reach, both, DEV)
        kw["rel_bias"] = torch.randn(H, buckets, generator=g).to(DEV)
    return t, kw


def _check(t, kw, dtype, with_lse_grad=False, **plain):
    q, k, v = (t[n].clone().requires_grad_() for n in "qkv")
    kw = dict(kw)
    if "rel_bias" in kw:
        kw["rel_bias"] = kw["rel_bias"].clone().requires_grad_()
    out, lse = torch_ops.long_attention(q, k, v, return_lse=True, **kw, **plain)
    outs, grads = [out], [t["go"]]
    dlse = None
    if with_lse_grad:
        dlse = torch.randn(lse.shape, generator=torch.Generator().manual_seed(5)).to(DEV)
        outs.append(lse), grads.append(dlse)
    leaves = [q, k, v] + ([kw["rel_bias"]] if "rel_bias" in kw else [])
    got = torch.autograd.grad(outs, leaves, grads)
    val, tol = long_rows.attention(t["q"], t["k"], t["v"], dout=t["go"], dlse=dlse, dtype=dtype, **kw, **plain)
    _near(out, val["out"], tol["out"], "out")
    _near(lse, val["lse"], tol["lse"], "lse")
    for name, x in zip(("dq", "dk", "dv", "dbias"), got):
        _near(x, val[name], tol[name], name)


SHAPES = [  # B, Lq, Lk, H, Hk, dh
    (1, 1, 1, 1, 1, 8), (2, 21, 21, 8, 8, 32), (1, 64, 64, 2, 2, 64), (1, 65, 65, 2, 1, 64), (1, 129, 129, 2, 2, 128), (2, 33, 200, 4, 2, 80),
    (1, 200, 33, 2, 1, 96), (3, 1, 70, 6, 2, 16), (1, 257, 257, 1, 1, 40), (1, 3, 600, 4, 1, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_attention_shapes(dtype, shape, causal):
    t, kw = _case(dtype, *shape, seed=sum(shape))
    _check(t, kw, dtype, causal=causal)


FEATURES = {
    "cap": dict(plain=dict(softcap=1.5)), "cap_wide": dict(plain=dict(softcap=50.0, causal=True)), "slopes": dict(slopes=True),
    "slopes_causal": dict(slopes=True, plain=dict(causal=True)),
    "prefix": dict(prefix=True, plain=dict(causal=True)), "cache": dict(cache=True, plain=dict(causal=True)),
    "cache_all": dict(cache=True), "cache_prefix": dict(cache=True, prefix=True, plain=dict(causal=True)),
    "buckets": dict(buckets=32, reach=24, both=True), "buckets_causal": dict(buckets=16, reach=100, plain=dict(causal=True)),
    "buckets_far": dict(buckets=4, reach=3, both=True, plain=dict(causal=True)),
    "buckets_cache": dict(buckets=8, reach=40, both=True, cache=True),
    "everything": dict(buckets=32, reach=64, both=True, slopes=True, prefix=True, cache=True, plain=dict(causal=True, softcap=3.0)),
    "lse": dict(plain=dict(with_lse_grad=True)), "lse_buckets": dict(buckets=8, reach=20, plain=dict(with_lse_grad=True, causal=True)),
    "scale": dict(plain=dict(scale=0.37), spread=0.7),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", sorted(FEATURES))
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_attention_features(dtype, name):
    f = dict(FEATURES[name])
    plain = f.pop("plain", {})
    t, kw = _case(dtype, 6 if f.get("cache") else 2, 150, 150, 4, 2, 64, seed=len(name), **f)
    _check(t, kw, dtype, **plain)


@pytest.mark.gpu
@pytest.mark.parametrize("dh", [32, 96, 128])
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_attention_everything_at_other_head_sizes(dtype, dh):
    t, kw = _case(dtype, 3, 70, 140, 4, 1, dh, seed=dh, buckets=32, reach=64, both=True, slopes=True, cache=True,
                  docs=[[(4, 50), (1, 70), (-1, 20)], [(0, 140)], [(2, 64), (3, 64), (-1, 12)]])
    _check(t, kw, dtype, causal=True, softcap=3.0)


DOCS = {
    "packed": [[(0, 40), (1, 7), (2, 90), (-1, 13)], [(5, 64), (9, 64), (-1, 22)]],
    "all_padding": [[(-1, 150)], [(0, 150)]],
    "unsorted": [[(3, 30), (0, 50), (3, 40), (1, 30)], [(7, 1), (2, 148), (7, 1)]],
    "padding_first": [[(-1, 70), (0, 80)], [(-1, 1), (4, 148), (-1, 1)]],
}


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
@pytest.mark.parametrize("name", sorted(DOCS))
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_attention_documents(dtype, name, causal):
    """Rows that see nothing (padding; with unsorted ids also none) give exact zeros, forward and backward."""
    t, kw = _case(dtype, 2, 150, 150, 2, 1, 64, seed=3, docs=DOCS[name], buckets=8, reach=16, both=True)
    _check(t, kw, dtype, causal=causal)
    out, lse = torch_ops.long_attention(t["q"], t["k"], t["v"], causal=causal, return_lse=True, **kw)
    dead = kw["q_doc"] < 0
    assert (out[dead] == 0).all() and (lse.transpose(1, 2)[dead] == -math.inf).all()
    # fewer queries than keys, and a mask that leaves live rows nothing: every query is of a document without keys
    kw["q_doc"] = torch.full_like(kw["q_doc"], 77)
    q, k, v = (t[n].clone().requires_grad_() for n in "qkv")
    out, lse = torch_ops.long_attention(q, k, v, causal=causal, return_lse=True, **kw)
    assert (out == 0).all() and (lse == -math.inf).all()
    assert all((g == 0).all() for g in torch.autograd.grad(out, (q, k, v), t["go"]))


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_what_padding_and_cache_tails_hold_does_not_matter(dtype, bad):
    docs = [[(0, 70), (-1, 10), (1, 70)], [(-1, 3), (2, 100), (-1, 47)]]
    for f, plain in ((dict(docs=docs), dict(causal=True)), (dict(docs=docs), {}), (dict(cache=True), {}), (dict(cache=True), dict(causal=True))):
        t, kw = _case(dtype, 2, 150, 150, 4, 2, 64, seed=8, **f)
        if f.get("cache"):
            kw["kv_len"] = torch.tensor([150, 77], dtype=torch.int32, device=DEV)
            dead = torch.arange(150, device=DEV)[None] >= kw["kv_len"][:, None]
            dead_q = torch.zeros_like(dead)
        else:
            dead, dead_q = kw["k_doc"] < 0, kw["q_doc"] < 0
        t["k"][dead], t["v"][dead] = bad, bad
        t["q"][dead_q], t["go"][dead_q] = bad, bad
        _check(t, kw, dtype, **plain)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_hidden_buckets_and_large_scores(dtype):
    """A bias entry of -inf or of a type's lowest value hides its bucket, forward and backward; scores of hundreds."""
    t, kw = _case(dtype, 1, 130, 130, 2, 2, 64, seed=4, buckets=8, reach=16, both=True, spread=4.0)
    kw["rel_bias"][0, 0] = -math.inf
    kw["rel_bias"][1, 2] = torch.finfo(F32).min
    kw["rel_bias"][1, 5] = -math.inf
    _check(t, kw, dtype)
    for lowest in (-math.inf, torch.finfo(F32).min, torch.finfo(BF16).min):
        kw["rel_bias"].fill_(lowest)
        q, k, v = (t[n].clone().requires_grad_() for n in "qkv")
        out, lse = torch_ops.long_attention(q, k, v, return_lse=True, **kw)
        assert (out == 0).all() and (lse == -math.inf).all()
        assert all((g == 0).all() for g in torch.autograd.grad(out, (q, k, v), t["go"]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_small_and_large_gradients(dtype):
    """Gradients a million times smaller or larger than one come out as exactly: fp16 has 5 exponent bits for the score gradients."""
    for factor in (2.0 ** -20, 2.0 ** 10):
        if dtype == F16 and factor < 1:
            factor = 2.0 ** -8
        t, kw = _case(dtype, 1, 140, 140, 2, 1, 64, seed=6, buckets=8, reach=16)
        t["go"] = (t["go"].float() * factor).to(dtype)
        _check(t, kw, dtype, causal=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_layouts(dtype):
    """Views of one projection, (batch, head, token) order, broadcast heads, a transposed head axis, an odd offset, an expanded
    gradient: the same bits as from contiguous copies."""
    g = torch.Generator().manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=g).to(dtype).to(DEV)
    B, L, H, Hk, dh = 2, 90, 4, 2, 64
    qkv = rnd(B, L, H + 2 * Hk, dh)
    bhld = rnd(B, H, L, dh).transpose(1, 2)
    flat = rnd(B * L * H * dh + 1)
    odd = flat[1:].view(B, L, H, dh)
    last = rnd(B, L, dh, H).transpose(2, 3)
    one_head = rnd(B, L, 1, dh).expand(B, L, Hk, dh)
    k, v = qkv[:, :, H:H + Hk], qkv[:, :, H + Hk:]
    for q in (qkv[:, :, :H], bhld, odd, last):
        for kk in (k, one_head):
            for go in (rnd(B, L, H, dh), rnd(1, 1, 1, dh).expand(B, L, H, dh), rnd(B, H, L, dh).transpose(1, 2),
                       torch.ones((), dtype=dtype, device=DEV).expand(B, L, H, dh)):
                got, want = [], []
                for fresh, res in ((lambda x: x.detach().requires_grad_(), got), (lambda x: x.detach().contiguous().clone().requires_grad_(), want)):
                    a, b, c = fresh(q), fresh(kk), fresh(v)
                    o = torch_ops.long_attention(a, b, c, causal=True)
                    res += [o] + list(torch.autograd.grad(o, (a, b, c), go if res is got else go.contiguous()))
                assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_broadcast_keys_get_the_summed_gradient(dtype):
    t, _ = _case(dtype, 2, 40, 40, 4, 1, 32)
    k = t["k"].clone().requires_grad_()
    out = torch_ops.long_attention(t["q"], k.expand(2, 40, 4, 32), t["v"].expand(2, 40, 4, 32))
    dk, = torch.autograd.grad(out, k, t["go"])
    k4 = t["k"].expand(2, 40, 4, 32).contiguous().requires_grad_()
    out4 = torch_ops.long_attention(t["q"], k4, t["v"].expand(2, 40, 4, 32).contiguous())
    assert torch.equal(out, out4)
    assert torch.equal(dk, torch.autograd.grad(out4, k4, t["go"])[0].sum(2, keepdim=True))


@pytest.mark.gpu
def test_empty_calls():
    for B, Lq, Lk in ((0, 4, 4), (2, 0, 5), (2, 4, 0)):
        q, k, v = (torch.randn(B, n, 2, 32, device=DEV, requires_grad=True) for n in (Lq, Lk, Lk))
        bias = torch.randn(2, 8, device=DEV, requires_grad=True)
        out, lse = torch_ops.long_attention(q, k, v, return_lse=True, rel_bias=bias, rel_buckets=ops.relative_buckets(8, 16, True, DEV))
        assert out.shape == q.shape and lse.shape == (B, 2, Lq) and (out == 0).all() and (lse == -math.inf).all()
        assert all((g == 0).all() for g in torch.autograd.grad(out.sum(), (q, k, v, bias)))
    q, w = torch.randn(2, 0, 4, 32, device=DEV, requires_grad=True), torch.ones(32, device=DEV, requires_grad=True)
    a, b = torch_ops.qk_norm_rope(q, q, w, w, ops.rotary_frequencies(32, device=DEV))
    assert a.shape == q.shape and all((g == 0).all() for g in torch.autograd.grad(a.sum() + b.sum(), (q, w)))


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    t, _ = _case(BF16, 1, 8, 8, 4, 2, 32)
    q, k, v = t["q"], t["k"], t["v"]
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    lut = ops.relative_buckets(8, 16, True, DEV)
    for args, kw in (((q, k.float(), v), {}), ((q, k, v[:, :4]), {}), ((q[..., :24], k, v), {}), ((q[:, :, :3], k, v), {}),
                     ((q.double(), k.double(), v.double()), {}), ((q, k, v), dict(prefix=i32(2))), ((q, k, v), dict(q_doc=i32(*[0] * 8)[None])),
                     ((q, k, v), dict(kv_len=i32(2, 3))), ((q, k, v), dict(kv_len=torch.tensor([2], device=DEV))), ((q, k, v), dict(softcap=-1.0)),
                     ((q, k, v), dict(scale=0.0)), ((q, k, v), dict(slopes=torch.ones(2, device=DEV))), ((q, k, v), dict(rel_bias=torch.ones(4, 8, device=DEV))),
                     ((q, k, v), dict(rel_bias=torch.ones(4, 8, device=DEV), rel_buckets=lut[:-1].contiguous())),
                     ((q, k, v), dict(rel_bias=torch.ones(4, 8, device=DEV), rel_buckets=lut.cpu())),
                     ((q, k, v), dict(rel_bias=torch.ones(4, 65, device=DEV), rel_buckets=lut)), ((q[0], k[0], v[0]), {})):
        with pytest.raises((MmtError, RuntimeError)):
            torch_ops.long_attention(*args, **kw)
    with pytest.raises(MmtError):
        torch_ops.long_attention(q, k, v, slopes=torch.ones(4, device=DEV, requires_grad=True))
    w = torch.ones(32, dtype=BF16, device=DEV)
    f = ops.rotary_frequencies(32, device=DEV)
    for a in ((q, k[:, :4], w, w, f), (q, k, w[:16], w, f), (q, k, w.half(), w, f), (q, k, w, w.float(), f), (q, k, w, w, f.float()),
              (q, k, w, w, ops.rotary_frequencies(64, device=DEV)), (q, k, w, w, f, torch.zeros(1, 8, device=DEV)), (q, k, w, w, f, torch.zeros(8, dtype=torch.int64, device=DEV))):
        with pytest.raises((MmtError, RuntimeError)):
            torch_ops.qk_norm_rope(*a)
    # no second derivative: an error, not a silent zero
    q = q.clone().requires_grad_()
    for fn in (lambda: torch_ops.long_attention(q, k, v), lambda: torch.ops.mmt.long_attention(q, k, v, None, False, None, None, None, None, 0.0, None, None, None)[0]):
        g, = torch.autograd.grad(fn().float().sum(), q, create_graph=True)
        with pytest.raises((MmtError, RuntimeError)):
            g.float().sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_dispatcher_calls_equal_the_wrappers(dtype):
    """torch.ops.mmt.* (what tracing sees) and the torch_ops wrappers (straight to the kernels): the same bits, gradients included."""
    t, kw = _case(dtype, 2, 70, 70, 4, 2, 64, buckets=8, reach=16)
    w, f = torch.ones(64, dtype=dtype, device=DEV), ops.rotary_frequencies(64, device=DEV)
    res = []
    for way in (0, 1):
        q, k, v, b, ww = (x.clone().requires_grad_() for x in (t["q"], t["k"], t["v"], kw["rel_bias"], w))
        if way:
            x, y = torch.ops.mmt.qk_norm_rope(q, k, ww, w, f, None, 1e-6, False)
            o, lse, _ = torch.ops.mmt.long_attention(x, y, v, None, True, None, None, None, None, 0.0, None, b, kw["rel_buckets"])
        else:
            x, y = torch_ops.qk_norm_rope(q, k, ww, w, f)
            o, lse = torch_ops.long_attention(x, y, v, causal=True, rel_bias=b, rel_buckets=kw["rel_buckets"], return_lse=True)
        res.append([o, lse] + list(torch.autograd.grad((o, lse), (q, k, v, b, ww), (t["go"], torch.ones_like(lse)))))
    assert all(torch.equal(x, y) for x, y in zip(*res))
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():                                # tracing: shapes without a kernel
        q = torch.empty(2, 5, 4, 64, dtype=dtype, device=DEV)
        assert torch_ops.long_attention(q, q[:, :, :2], q[:, :, 2:]).shape == q.shape


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_same_bits_every_call_and_on_any_stream(dtype):
    t, kw = _case(dtype, 2, 300, 300, 4, 2, 64, seed=2, buckets=32, reach=64, both=True)

    def step():
        q, k, v, b = (x.clone().requires_grad_() for x in (t["q"], t["k"], t["v"], kw["rel_bias"]))
        o = torch_ops.long_attention(q, k, v, rel_bias=b, rel_buckets=kw["rel_buckets"])
        return [o] + list(torch.autograd.grad(o, (q, k, v, b), t["go"]))
    first = step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    res = []
    for s in streams:                                     # two calls at once
        with torch.cuda.stream(s):
            res.append(step())
    torch.cuda.synchronize()
    for r in res + [step()]:
        assert all(torch.equal(a, b) for a, b in zip(first, r))
    one = torch_ops.long_attention(t["q"][1:], t["k"][1:], t["v"][1:], **{k: v for k, v in kw.items()})
    assert torch.equal(one, first[0][1:])                 # a row does not depend on the batch it is in


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
def test_captured_calls_replay(dtype):
    """Forward (split over the keys) and backward captured through the plain entry points; every replay equals the eager result on the
    inputs of its turn, with eager work between the replays.  Two graphs captured side by side do not share a workspace."""
    t, kw = _case(dtype, 1, 200, 200, 2, 1, 64, seed=7, buckets=8, reach=30, docs=[[(0, 80), (1, 100), (-1, 20)]])
    d, dkw = _case(dtype, 2, 1, 3000, 4, 1, 64, seed=9, cache=True)
    dkw["kv_len"] = torch.tensor([3000, 1777], dtype=torch.int32, device=DEV)
    w = torch.ones(64, dtype=dtype, device=DEV)
    f = ops.rotary_frequencies(64, device=DEV)

    def train():
        a, b = ops.qk_norm_rope(t["q"], t["k"], w, w, f)
        o, lse, low = ops.long_attention(a, b, t["v"], causal=True, keep_low=True, **kw)
        g = ops.long_attention_backward(t["go"], None, o, lse, low, a, b, t["v"], causal=True, **kw)
        return (o, lse) + tuple(g) + tuple(ops.qk_norm_rope_backward(g[0], g[1], t["q"], t["k"], w, w, f))

    def serve():
        return ops.long_attention(d["q"], d["k"], d["v"], causal=True, **dkw)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        train(), serve()
    torch.cuda.synchronize()
    graphs = []
    for fn in (train, serve, train):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = fn()
        graphs.append((g, fn, out))
    for turn in range(4):
        for x in (t["q"], t["v"], t["go"], d["q"], d["v"]):
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(100 + turn)).to(dtype))
        dkw["kv_len"].copy_(torch.tensor([3000 - 900 * turn, 5 + turn], dtype=torch.int32))
        want = [[x.clone() for x in fn()] for _, fn, _ in graphs]
        for g, _, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (_, _, out), ref in zip(graphs, want):
            assert all(torch.equal(a, b) for a, b in zip(out, ref)), turn


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_single_tokens_equal_the_row(dtype):
    """Decoding a row token by token over a cache gives what the whole row gives, each within its bound."""
    B, L, H, Hk, dh = 2, 40, 4, 2, 64
    t, kw = _case(dtype, B, L, L, H, Hk, dh, seed=12, slopes=True, buckets=8, reach=16)
    val, tol = long_rows.attention(t["q"], t["k"], t["v"], causal=True, softcap=5.0, dtype=dtype, **kw)
    cache_k = torch.full((B, 64, Hk, dh), math.nan, dtype=dtype, device=DEV)
    cache_v = cache_k.clone()
    for i in range(L):
        cache_k[:, i], cache_v[:, i] = t["k"][:, i], t["v"][:, i]
        n = torch.full((B,), i + 1, dtype=torch.int32, device=DEV)
        o = torch_ops.long_attention(t["q"][:, i:i + 1], cache_k, cache_v, causal=True, softcap=5.0, kv_len=n, **kw)
        _near(o[:, 0], val["out"][:, i], tol["out"][:, i], f"token {i}")


@pytest.mark.gpu
def test_a_cache_beyond_32_bit_offsets():
    """Byte offsets inside one cache pass 2^32: the last request's keys lie beyond."""
    B, Lk, Hk, dh = 9, 262144, 8, 128                     # 9 x 512 MiB
    k = torch.zeros(B, Lk, Hk, dh, dtype=BF16, device=DEV)
    v = torch.zeros_like(k)
    q = torch.randn(B, 1, 8, dh, generator=torch.Generator().manual_seed(0)).to(BF16).to(DEV)
    k[:, -600:] = torch.randn(600, Hk, dh, generator=torch.Generator().manual_seed(1)).to(BF16).to(DEV)
    v[:, -600:] = torch.randn(600, Hk, dh, generator=torch.Generator().manual_seed(2)).to(BF16).to(DEV)
    slopes = torch.full((8,), 0.25, device=DEV)
    out = torch_ops.long_attention(q, k, v, causal=True, slopes=slopes)
    near = torch_ops.long_attention(q, k[:, -600:].contiguous(), v[:, -600:].contiguous(), causal=True, slopes=slopes)
    val, tol = long_rows.attention(q, k[:, -600:], v[:, -600:], causal=True, slopes=slopes, dtype=BF16)
    _near(near, val["out"], tol["out"], "near")
    _near(out, val["out"], tol["out"], "out")             # what is 600 tokens away weighs e^-150


@pytest.mark.gpu
def test_gradients_against_differences():
    """fp32 gradients along a random direction against central differences of the operator's own (fp32) outputs, summed in 64 bits.  The
    step h = 2^-6 leaves a relative curvature error of about h^2 and a rounding error of about 2^-24 * sqrt(terms) / h: 1e-2 covers both."""
    t, kw = _case(F32, 1, 50, 50, 2, 1, 32, seed=21, buckets=8, reach=16, both=True, slopes=True)
    names = ["q", "k", "v"]
    leaves = {n: t[n].clone().requires_grad_() for n in names}
    bias = kw.pop("rel_bias").clone().requires_grad_()

    def f(q, k, v, b):
        a, kk = torch_ops.qk_norm_rope(q, k, torch.ones(32, device=DEV), torch.ones(32, device=DEV), ops.rotary_frequencies(16, device=DEV))
        return torch_ops.long_attention(a, kk, v, causal=True, softcap=4.0, rel_bias=b, **kw)
    xs = [leaves[n] for n in names] + [bias]
    grads = torch.autograd.grad(f(*xs), xs, t["go"])
    h = 2.0 ** -6
    for n, (x, g) in enumerate(zip(xs, grads)):
        d = torch.randn(x.shape, generator=torch.Generator().manual_seed(n)).to(DEV)
        at = lambda s: [y.detach() + s * d if y is x else y.detach() for y in xs]
        num = ((f(*at(h)) - f(*at(-h))).double() * t["go"].double()).sum() / (2 * h)
        ana = (g.double() * d.double()).sum()
        assert abs(float(num - ana)) <= 1e-2 * float((g.double() * d.double()).norm()) * 4, (n, float(num), float(ana))


ROPE = [  # B, L, H, Hk, dh, rot, interleaved, positions
    (2, 5, 4, 2, 64, 64, False, "far"), (1, 1, 1, 1, 8, 8, False, None), (3, 37, 8, 8, 32, 16, True, None), (2, 19, 3, 1, 80, 40, False, "far"),
    (1, 130, 2, 2, 96, 96, True, "back"), (2, 9, 4, 4, 128, 128, False, "far"), (1, 33, 2, 1, 256, 128, False, "far"), (1, 7, 2, 2, 24, 2, False, None),
    (5, 1, 16, 4, 128, 64, True, "far"), (1, 4500, 2, 1, 64, 64, False, None), (1, 2, 1, 1, 200, 200, False, "far")]


@pytest.mark.gpu
@pytest.mark.parametrize("case", ROPE, ids=lambda c: "x".join(map(str, c[:6])) + ("i" if c[6] else ""))
@pytest.mark.parametrize("w_fp32", [False, True], ids=["w", "w32"])
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_norm_rope(dtype, w_fp32, case):
    B, L, H, Hk, dh, rot, inter, where = case
    g = torch.Generator().manual_seed(L + dh)
    qkv = torch.randn(B, L, H + 2 * Hk, dh, generator=g).to(dtype).to(DEV)
    q, k = qkv[:, :, :H].detach().requires_grad_(), qkv[:, :, H:H + Hk].detach().requires_grad_()
    wt = F32 if w_fp32 else dtype
    qw, kw = ((1 + 0.3 * torch.randn(dh, generator=g)).to(wt).to(DEV).requires_grad_() for _ in range(2))
    pos = None
    if where == "far":
        pos = torch.randint(0, 1 << 20, (B, L), generator=g).to(DEV)
    elif where == "back":
        pos = -torch.arange(L).expand(B, L).contiguous().to(DEV)
    f = ops.rotary_frequencies(rot, 10000.0, DEV)
    gq, gk = torch.randn(B, L, H, dh, generator=g).to(dtype).to(DEV), torch.randn(B, L, Hk, dh, generator=g).to(dtype).to(DEV)
    yq, yk = torch_ops.qk_norm_rope(q, k, qw, kw, f, pos, eps=1e-5, interleaved=inter)
    dq, dk, dqw, dkw = torch.autograd.grad((yq, yk), (q, k, qw, kw), (gq, gk))
    for x, w, gy, y, dx, dw, what in ((q, qw, gq, yq, dq, dqw, "q"), (k, kw, gk, yk, dk, dkw, "k")):
        val, tol = long_rows.norm_rope(x, w, f, pos, 1e-5, inter, gy)
        _near(y, val["y"], tol["y"], what)
        _near(dx, val["dx"], tol["dx"], "d" + what)
        _near(dw, val["dw"], tol["dw"], f"d{what}_weight")


@pytest.mark.gpu
def test_norm_rope_zero_rows_and_one_gradient():
    """A row of zeros stays zero (eps keeps its norm finite); only one of the two outputs may have a gradient."""
    q = torch.zeros(1, 3, 2, 32, device=DEV, requires_grad=True)
    k = torch.randn(1, 3, 1, 32, device=DEV, requires_grad=True)
    w = torch.ones(32, device=DEV, requires_grad=True)
    a, b = torch_ops.qk_norm_rope(q, k, w, w.detach(), ops.rotary_frequencies(32, device=DEV))
    assert (a == 0).all()
    dq, dk = torch.autograd.grad(a.sum(), (q, k))
    assert torch.isfinite(dq).all() and (dk == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_a_block_of_scene_attention(dtype):
    """The operators as they are used together: projections of packed scenes, norm + rotation with positions that start again in every
    scene, capped attention with document mask, history prefix and learned bias; results and every gradient against the same block
    in 64 bits with torch's autograd.  The bound on a deviation is statistical: errors of the element type's half step u enter at four
    places of the chain (q/k, p, out, gradients), so the relative L2 error of a tensor stays under 16 u."""
    B, L, H, Hk, dh, dm = 2, 120, 4, 2, 32, 64
    g = torch.Generator().manual_seed(31)
    x = torch.randn(B, L, dm, generator=g)
    wqkv = torch.randn(dm, (H + 2 * Hk) * dh, generator=g) / 8
    bias = torch.randn(H, 16, generator=g) * 0.5
    qw, kw = 1 + 0.1 * torch.randn(dh, generator=g), 1 + 0.1 * torch.randn(dh, generator=g)
    go = torch.randn(B, L, H * dh, generator=g)
    lens = [50, 40, 25]
    doc = torch.tensor([i for i, n in enumerate(lens) for _ in range(n)] + [-1] * (L - sum(lens)), dtype=torch.int32).expand(B, L).contiguous()
    pos = torch.tensor([j for n in lens for j in range(n)] + list(range(L - sum(lens)))).expand(B, L).contiguous()
    lut = ops.relative_buckets(16, 32, True)
    prefix = torch.tensor([20, 60], dtype=torch.int32)
    freq = ops.rotary_frequencies(dh)
    qkv = (x @ wqkv).view(B, L, H + 2 * Hk, dh).to(dtype)
    leaves = [t.to(DEV).requires_grad_() for t in (qkv, qw.to(dtype), kw.to(dtype), bias)]
    a, w1, w2, table = leaves
    q, k = torch_ops.qk_norm_rope(a[:, :, :H], a[:, :, H:H + Hk], w1, w2, freq.to(DEV), pos.to(DEV))
    o = torch_ops.long_attention(q, k, a[:, :, H + Hk:], causal=True, prefix=prefix.to(DEV), q_doc=doc.to(DEV), k_doc=doc.to(DEV), softcap=5.0,
                                 rel_bias=table, rel_buckets=lut.to(DEV))
    got = [o] + list(torch.autograd.grad(o, leaves, go.view(B, L, H, dh).to(dtype).to(DEV)))
    # the same in 64 bits
    ref = [t.detach().cpu().double().requires_grad_() for t in leaves]
    a, w1, w2, table = ref
    ang = (pos.double()[..., None] * freq)[:, :, None]

    def turn(z, w):
        n = z * (z.pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt() * w
        p, r = n[..., :dh // 2], n[..., dh // 2:]
        return torch.cat((p * ang.cos() - r * ang.sin(), r * ang.cos() + p * ang.sin()), -1)
    q, k, v = turn(a[:, :, :H], w1), turn(a[:, :, H:H + Hk], w2), a[:, :, H + Hk:]
    k, v = (t.repeat_interleave(H // Hk, 2) for t in (k, v))
    s = torch.einsum("bihd,bjhd->bhij", q, k) * dh ** -0.5
    s = 5.0 * torch.tanh(s / 5.0)
    i = torch.arange(L)
    apart = i[None] - i[:, None]
    s = s + table[:, lut.long()[apart.clamp(-32, 32) + 32]]
    see = (doc[:, :, None] == doc[:, None]) & (doc >= 0)[:, :, None] & ((apart <= 0)[None] | (i < prefix[:, None])[:, None])
    p = torch.softmax(s.masked_fill(~see[:, None], -1e300), -1) * see[:, None]
    o = torch.einsum("bhij,bjhd->bihd", p, v)
    want = [o] + list(torch.autograd.grad(o, ref, go.view(B, L, H, dh).to(dtype).double()))
    for n, x, y in zip(("out", "dqkv", "dq_weight", "dk_weight", "dbias"), got, want):
        rel = float((x.detach().cpu().double() - y).norm() / y.norm())
        assert rel <= 16 * long_rows.unit(dtype) + 2e-6, (n, rel)


# ----------------------------------------------------------------------------------------------------------- further CPU checks
@pytest.mark.parametrize("bad,word", [
    (dict(scale=3e38), b"scale"), (dict(softcap=3e38), b"cap"), (dict(scale=1.0, softcap=1e-39), b"cap"),
    (dict(B=9000, Lq=128000, Lk=128), b"too many"), (dict(Lk=(1 << 30) + 1), b"2^30"), (dict(k_rs=1 << 24), b"2^25"),
    (dict(dtype=_lib.MMT_F32, v_rs=1 << 23), b"2^25")])
def test_attention_refuses_what_would_overflow(bad, word):
    lib = _lib.load()
    a = _desc(**bad)
    assert lib.mmt_long_attention_workspace_bytes(ctypes.byref(a), 0) == 0
    assert lib.mmt_long_attention_fwd(ctypes.byref(a), 0x1000, None, None, 0x1000, 1 << 40, None) == -1 and word in lib.mmt_last_error()


def test_native_nodes_refuse_another_library():
    """The nodes are bound to entry points by address: another number of them, or structs of other sizes, is an error."""
    n = _lib.native()
    sizes = ctypes.sizeof(_lib.LongAttention), ctypes.sizeof(_lib.QkNormRope)
    for entries, s in (([0] * 6, sizes), ([0] * 7, (sizes[0] + 8, sizes[1])), ([0] * 7, (sizes[0], sizes[1] - 8))):
        with pytest.raises(RuntimeError):
            n.bind(entries, s, MmtError)


# ----------------------------------------------------------------------------------------------------------- further GPU checks
PACKED = {   # Lq, Lk, H, Hk, dh: rows of all heads of a key head fill fewer tiles of 128 together, and are more than 32
    "slopes": ((20, 300, 8, 2, 64), dict(slopes=True)), "cap": ((40, 700, 4, 1, 128), dict()), "three": ((33, 90, 6, 2, 80), dict(slopes=True, cache=True)),
    "docs": ((33, 150, 6, 2, 32), dict(docs=[[(4, 50), (1, 80), (-1, 20)], [(0, 150)]])), "prefix": ((15, 64, 8, 2, 96), dict(prefix=True, slopes=True))}


@pytest.mark.gpu
@pytest.mark.parametrize("name", sorted(PACKED))
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_rows_of_several_heads_in_a_tile(dtype, name):
    shape, f = PACKED[name]
    t, kw = _case(dtype, 2, *shape, seed=17, **f)
    _check(t, kw, dtype, causal=True, softcap=2.0 if name == "cap" else 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("case", [(BF16, 64), (F16, 128), (F32, 64)], ids=lambda c: f"{IDS[c[0]]}x{c[1]}")
def test_gradients_in_parts_over_heads_and_queries(case):
    """Few key tiles: dK and dV in parts over the four query heads of a key head and over the queries; with a gradient of the log-sum."""
    dtype, dh = case
    t, kw = _case(dtype, 1, 1100, 200, 4, 1, dh, seed=23, slopes=True)
    _check(t, kw, dtype, with_lse_grad=True)
    t, kw = _case(dtype, 1, 1100, 1100, 4, 1, dh, seed=24, buckets=8, reach=70)
    _check(t, kw, dtype, causal=True)


@pytest.mark.gpu
@pytest.mark.parametrize("Lk", [192, 256, 257, 320, 512, 513])
@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
def test_around_the_longest_row_of_two_passes(dtype, Lk):
    t, kw = _case(dtype, 1, 130, Lk, 2, 1, 64, seed=Lk, docs=[[(0, Lk - 90), (1, 80), (-1, 10)]])
    _check(t, kw, dtype, causal=True)


def _run(t, kw, **plain):
    q, k, v = (t[n].clone().requires_grad_() for n in "qkv")
    kw = dict(kw)
    leaves = [q, k, v]
    if "rel_bias" in kw:
        kw["rel_bias"] = kw["rel_bias"].clone().requires_grad_()
        leaves.append(kw["rel_bias"])
    out, lse = torch_ops.long_attention(q, k, v, return_lse=True, **kw, **plain)
    return [out, lse] + list(torch.autograd.grad(out, leaves, t["go"]))


@pytest.mark.gpu
@pytest.mark.parametrize("Lq", [1, 40])
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_numbers_out_of_range_are_clamped(dtype, Lq):
    """Cache lengths below 0 and above Lk, bucket numbers outside the table, prefixes beyond the row: as the nearest that is inside."""
    t, kw = _case(dtype, 4, Lq, 90, 4, 2, 64, seed=29, buckets=8, reach=16, both=True)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    lut = kw["rel_buckets"].clone()
    lut[3], lut[20] = -7, 1000
    far = _run(t, dict(kw, kv_len=i32([-5, 1 << 30, 3, 90]), rel_buckets=lut, prefix=i32([-(1 << 30), 1 << 30, 200, 5])), causal=True)
    near = _run(t, dict(kw, kv_len=i32([0, 90, 3, 90]), rel_buckets=lut.clamp(0, 7), prefix=i32([0, 90, 90, 5])), causal=True)
    assert all(torch.equal(a, b) for a, b in zip(far, near))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_any_document_ids(dtype):
    """Ids are only compared: the largest ones, in alternation within a tile, give the bits of small ones; so do queries whose ids
    are in another order than the keys'."""
    t, kw = _case(dtype, 2, 140, 140, 2, 1, 64, seed=33)
    small = (torch.arange(140, dtype=torch.int32, device=DEV) % 3).expand(2, 140).contiguous()
    large = small * ((1 << 30) - 1) + 1                     # 1, 2^30, 2^31 - 1
    _check(t, dict(q_doc=small, k_doc=small), dtype, causal=True)
    for q_small in (small, small.flip(1).contiguous()):
        a = _run(t, dict(q_doc=q_small, k_doc=small), causal=True)
        b = _run(t, dict(q_doc=q_small * ((1 << 30) - 1) + 1, k_doc=large), causal=True)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32], ids=IDS.get)
def test_tokens_far_apart(dtype):
    """Token strides at and beyond 2^25 bytes are copied, below it read in place; head and batch strides may be of any size."""
    far = (1 << 25) // dtype.itemsize
    flat = torch.zeros(3 * far + 64, dtype=dtype, device=DEV)
    g = torch.Generator().manual_seed(2)
    for stride in (far - 64, far):                        # (2 x 2 heads at distinct multiples of the stride)
        for st in ((0, stride, 16, 1), (2 * stride, 32, stride, 1)):
            k = torch.as_strided(flat, (1, 3, 2, 16) if st[0] == 0 else (2, 1, 2, 16), st)
            x = torch.randn(k.shape, generator=g).to(dtype).to(DEV)
            k.copy_(x)
            q = torch.randn(k.shape, generator=g).to(dtype).to(DEV)
            a = _run({"q": k, "k": q, "v": q, "go": q}, {})
            b = _run({"q": x, "k": q, "v": q, "go": q}, {})
            assert all(torch.equal(u, w) for u, w in zip(a, b))
            out = [torch_ops.long_attention(q, kk, kk) for kk in (k, x)]
            assert torch.equal(*out)
    with pytest.raises(MmtError):
        torch_ops.long_attention(q, q.new_zeros(2, 1, 2, 16).expand(2, (1 << 30) + 1, 2, 16), q.new_zeros(2, 1, 2, 16).expand(2, (1 << 30) + 1, 2, 16))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_the_graph_keeps_autograds_rules(dtype):
    """Saved tensors that come back from elsewhere, a graph kept and walked twice, recomputation, some leaves only; inputs changed in
    place, a graph walked after its end, forward-mode and functional transforms are errors."""
    t, kw = _case(dtype, 2, 50, 50, 4, 2, 32, seed=41, buckets=8, reach=16)
    w, f = torch.ones(32, dtype=dtype, device=DEV), ops.rotary_frequencies(32, device=DEV)
    leaves = [x.clone().requires_grad_() for x in (t["q"], t["k"], t["v"], kw["rel_bias"], w)]

    def call(q, k, v, b, ww):
        x, y = torch_ops.qk_norm_rope(q, k, ww, w, f)
        return torch_ops.long_attention(x, y, v.transpose(1, 2).contiguous().transpose(1, 2), causal=True, rel_bias=b, rel_buckets=kw["rel_buckets"])
    out = call(*leaves)
    want = torch.autograd.grad(out, leaves, t["go"], retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(out, leaves, t["go"])))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out, leaves, t["go"])
    with torch.autograd.graph.save_on_cpu():
        out = call(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(out, leaves, t["go"])))
    out = torch.utils.checkpoint.checkpoint(call, *leaves, use_reentrant=False)
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(out, leaves, t["go"])))
    for n in range(5):
        some = [x if i == n else x.detach() for i, x in enumerate(leaves)]
        assert torch.equal(torch.autograd.grad(call(*some), leaves[n], t["go"])[0], want[n])
    assert not call(*[x.detach() for x in leaves]).requires_grad
    with torch.no_grad():
        assert not call(*leaves).requires_grad
    with torch.inference_mode():
        assert torch.equal(call(*leaves), out)
    q = leaves[0] * 1
    o = torch_ops.long_attention(q, leaves[1], leaves[2])
    q.zero_()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(o, leaves[1], t["go"])
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(t["q"], t["go"])
        for fn in (lambda: torch_ops.long_attention(dual, t["k"], t["v"]), lambda: torch_ops.qk_norm_rope(dual, t["k"], w, w, f)):
            with pytest.raises((MmtError, RuntimeError)):
                fn()
    with pytest.raises((MmtError, RuntimeError)):
        torch.func.grad(lambda q: torch_ops.long_attention(q, t["k"], t["v"]).float().sum())(t["q"])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
def test_a_training_step_in_a_graph(dtype):
    """Forward and backward through the differentiable entry points, captured together on leaves of their own; every replay equals the
    eager step on the inputs of its turn."""
    t, kw = _case(dtype, 2, 140, 140, 4, 2, 64, seed=43, buckets=8, reach=30)
    w, f = torch.ones(64, dtype=dtype, device=DEV), ops.rotary_frequencies(64, device=DEV)

    def step():
        q, k, v, b, ww = (x.detach().requires_grad_() for x in (t["q"], t["k"], t["v"], kw["rel_bias"], w))
        x, y = torch_ops.qk_norm_rope(q, k, ww, w, f)
        o = torch_ops.long_attention(x, y, v, causal=True, rel_bias=b, rel_buckets=kw["rel_buckets"])
        return [o.detach()] + list(torch.autograd.grad(o, (q, k, v, b, ww), t["go"]))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for turn in range(3):
        for x in (t["q"], t["k"], t["go"]):
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(200 + turn)).to(dtype))
        want = [x.clone() for x in step()]
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), turn


@pytest.mark.gpu
@pytest.mark.parametrize("dh,rot", [(256, 256), (128, 32), (96, 48), (256, 80), (32, 32), (16, 16), (64, 24), (64, 6)])
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_norm_rope_pairs(dtype, dh, rot):
    """Every distance between the two of a pair: 1, 2, 4, 8, 16 lanes, other numbers of whole lanes, halves that end inside a lane."""
    g = torch.Generator().manual_seed(dh + rot)
    q, k = (torch.randn(2, 11, n, dh, generator=g).to(dtype).to(DEV).requires_grad_() for n in (3, 1))
    w = (1 + 0.3 * torch.randn(dh, generator=g)).to(dtype).to(DEV).requires_grad_()
    f = ops.rotary_frequencies(rot, 100.0, DEV)
    gq, gk = (torch.randn(x.shape, generator=g).to(dtype).to(DEV) for x in (q, k))
    for inter in (False, True):
        yq, yk = torch_ops.qk_norm_rope(q, k, w, w.detach(), f, interleaved=inter)
        dq, dk, dw = torch.autograd.grad((yq, yk), (q, k, w), (gq, gk))
        for x, gy, y, dx, dwx in ((q, gq, yq, dq, dw), (k, gk, yk, dk, None)):
            val, tol = long_rows.norm_rope(x, w, f, None, 1e-6, inter, gy)
            _near(y, val["y"], tol["y"], "y")
            _near(dx, val["dx"], tol["dx"], "dx")
            if dwx is not None:
                _near(dwx, val["dw"], tol["dw"], "dw")


@pytest.mark.gpu
@pytest.mark.parametrize("name", sorted(FEATURES))
@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
def test_features_of_rows_that_two_teams_share(dtype, name):
    """16-bit calls of few workgroups and more than three tiles of keys: an odd number of tiles, tiles that only one team has."""
    f = dict(FEATURES[name])
    plain = f.pop("plain", {})
    t, kw = _case(dtype, 6 if f.get("cache") else 1, 70, 290, 2, 1, 64, seed=len(name), **f)
    _check(t, kw, dtype, **plain)


@pytest.mark.gpu
@pytest.mark.parametrize("dh", [32, 96, 128])
@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
def test_documents_of_rows_that_two_teams_share(dtype, dh):
    docs = [[(0, 70), (-1, 3), (1, 130), (2, 40), (-1, 77), (3, 280)], [(-1, 200), (5, 1), (4, 399)], [(0, 600)]]
    t, kw = _case(dtype, 3, 600, 600, 2, 1, dh, seed=dh, docs=docs, buckets=8, reach=40, both=True, slopes=True)
    _check(t, kw, dtype, causal=True, softcap=4.0)
    _check(t, kw, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_many_short_rows(dtype):
    """A batch beyond 2^16: first, middle and last rows, forward and backward, within the bounds of 64 bits (dK and dV of shared heads are
    added in parts that depend on the size of the call: not the bits of a batch of one)."""
    B, L, H, dh = 70000, 3, 2, 8
    g = torch.Generator().manual_seed(47)
    q, k, v, go = (torch.randn(B, L, n, dh, generator=g).to(dtype).to(DEV) for n in (H, 1, 1, H))
    got = _run({"q": q, "k": k, "v": v, "go": go}, {}, causal=True)
    rot = torch_ops.qk_norm_rope(q, k, torch.ones(dh, dtype=dtype, device=DEV), torch.ones(dh, dtype=dtype, device=DEV), ops.rotary_frequencies(dh, device=DEV))
    for b in (0, 34999, 65536, B - 1):
        s = slice(b, b + 1)
        val, tol = long_rows.attention(q[s], k[s], v[s], dout=go[s], causal=True, dtype=dtype)
        for n, x in zip(("out", "lse", "dq", "dk", "dv"), got):
            _near(x[s], val[n], tol[n], f"{n} of batch row {b}")
        r = torch_ops.qk_norm_rope(q[s], k[s], torch.ones(dh, dtype=dtype, device=DEV), torch.ones(dh, dtype=dtype, device=DEV), ops.rotary_frequencies(dh, device=DEV))
        assert all(torch.equal(x[s], y) for x, y in zip(rot, r)), b


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_a_row_of_forty_thousand_tokens(dtype):
    """Single rows of a long causal call against 64 bits, and its gradients against a call of the last tokens alone over the same keys:
    a gradient of zero in all other rows makes the two the same sums."""
    L, H, dh = 40000, 2, 32
    t, kw = _case(dtype, 1, L, L, H, 1, dh, seed=53, slopes=True, buckets=16, reach=200)
    t["go"][:, :-70] = 0
    got = _run(t, kw, causal=True)
    for i in (0, 12345, 33333, L - 1):
        val, tol = long_rows.attention(t["q"][:, i:i + 1], t["k"][:, :i + 1], t["v"][:, :i + 1], causal=True, dtype=dtype, **kw)
        _near(got[0][:, i:i + 1], val["out"], tol["out"], f"row {i}")
        _near(got[1][:, :, i:i + 1], val["lse"], tol["lse"], f"lse of row {i}")
    val, tol = long_rows.attention(t["q"][:, -70:], t["k"], t["v"], dout=t["go"][:, -70:], causal=True, dtype=dtype, **kw)
    _near(got[2][:, -70:], val["dq"], tol["dq"], "dq")
    assert (got[2][:, :-70] == 0).all()
    # keys so far away that their probability is under 2^-126 get none at all (fp32 holds no smaller normal number): each of the 70 x 2 rows
    # then misses at most 2^-126 |dP - delta| scale |q| of a dK and 2^-126 |dO| of a dV, with |dP|, |delta| <= 32 max|dO| max|v| < 2^10 and
    # scale |q|, |dO| < 2^3: less than 140 * 2^-126 * 2^11 * 2^3 < 2^-104 together
    for n, x in zip(("dk", "dv", "dbias"), got[3:]):
        _near(x, val[n], tol[n] + (2.0 ** -104 if n != "dbias" else 0.0), n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_plain_calls_equal_the_checked_ones(dtype, monkeypatch):
    """Calls that need no copy are filled in natively: the same bits as through the checks, with every option; what the native call does
    not take (a list for a tensor, a view to copy) goes through them."""
    t, kw = _case(dtype, 3, 60, 200, 4, 2, 64, seed=59, docs=[[(0, 150), (-1, 50)], [(1, 80), (2, 120)], [(3, 200)]], prefix=True, cache=True,
                  slopes=True, buckets=16, reach=40)
    w, f = torch.ones(64, dtype=dtype, device=DEV, requires_grad=True), ops.rotary_frequencies(64, device=DEV)
    pos = torch.arange(60, device=DEV).expand(3, 60).contiguous() * 3

    def both():
        x, y = torch_ops.qk_norm_rope(t["q"], t["k"][:, :60], w, w, f, pos, eps=1e-5, interleaved=True)
        return _run(t, kw, causal=True, softcap=6.0, scale=0.3) + [x, y] + list(torch.autograd.grad(x.float().sum() + y.float().sum(), w))
    plain = both()
    monkeypatch.setattr(torch_ops, "_plain", lambda *a: None)
    assert all(torch.equal(a, b) for a, b in zip(plain, both()))
    monkeypatch.undo()
    seen = []
    take = torch_ops._plain
    monkeypatch.setattr(torch_ops, "_plain", lambda *a: seen.append(take(*a)) or seen[-1])
    torch_ops.long_attention(t["q"], t["k"], t["v"])
    torch_ops.long_attention(t["q"].transpose(2, 3).contiguous().transpose(2, 3), t["k"], t["v"])
    assert seen[0] is not None and seen[1] is None
    for bad in (dict(kv_len=[1, 2, 3]), dict(q_doc=3, k_doc=3), dict(rel_bias=1.0, rel_buckets=kw["rel_buckets"])):
        with pytest.raises(MmtError):
            torch_ops.long_attention(t["q"], t["k"], t["v"], **bad)
    for bad in ((None, t["k"], w, w, f), (t["q"], t["k"][:, :60], w, None, f), (t["q"], t["k"][:, :60], w, w, [1.0])):
        with pytest.raises(MmtError):
            torch_ops.qk_norm_rope(*bad)


@pytest.mark.gpu
def test_two_threads_at_once():
    """Training steps of two Python threads (the calls let go of the interpreter), each on a stream of its own: the bits of one alone."""
    import threading
    cases = [_case(BF16, 2, 150, 150, 4, 2, 64, seed=n, buckets=8, reach=20) for n in (61, 62)]
    want = [_run(t, kw, causal=True) for t, kw in cases]
    torch.cuda.synchronize()
    got, failed = [[], []], []

    def work(n):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[n].append(_run(*cases[n], causal=True))
                with pytest.raises(MmtError):
                    torch_ops.long_attention(cases[n][0]["q"], cases[n][0]["k"], cases[n][0]["v"], scale=-1.0)
        except BaseException as e:
            failed.append(e)
    threads = [threading.Thread(target=work, args=(n,)) for n in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    torch.cuda.synchronize()
    assert not failed, failed
    for n in range(2):
        assert len(got[n]) == 20 and all(torch.equal(a, b) for run in got[n] for a, b in zip(want[n], run))
