"""Edges of attention over long rows and of the norm + rotation in front of it: calls under torch's tracer, tensors that are not plain
memory, rows that see nothing, lowest-value biases, head sizes inside a tile, precision of the corrected backward pass."""
import ctypes
import math

import pytest
import torch

from multimodal_transformer_amd import _lib, ops, torch_ops
from multimodal_transformer_amd._lib import MmtError
from oracle import long_rows
from test_long_attention import BF16, DEV, F16, F32, IDS, TYPES, _case, _check, _desc, _near, _run


# ------------------------------------------------------------------------------------------------------------------ under the tracer
def _host_attention(q, k, v, *rest):
    """Stands in for the kernels on the CPU: the operator's results in elementary operations."""
    s = torch.matmul(q.transpose(1, 2), k.permute(0, 2, 3, 1)) * q.shape[-1] ** -0.5
    return torch.matmul(s.softmax(-1), v.transpose(1, 2)).transpose(1, 2).contiguous(), s.logsumexp(-1), q.new_empty(0)


def test_a_traced_call_is_recorded_as_the_operator():
    """torch.jit.trace records the operators themselves: the traced function computes on new inputs."""
    with torch.library._scoped_library("mmt", "IMPL") as lib:
        lib.impl("long_attention", _host_attention, "CPU")
        lib.impl("qk_norm_rope", lambda q, k, *rest: (q * 2, k * 3), "CPU")

        def block(q, k, v, w, f):
            a, b = torch_ops.qk_norm_rope(q, k, w, w, f)
            return torch_ops.long_attention(a, b, v)
        g = torch.Generator().manual_seed(0)
        w, f = torch.ones(8), ops.rotary_frequencies(8)
        draw = lambda: [torch.randn(1, 5, 2, 8, generator=g) for _ in range(3)]
        q, k, v = draw()
        traced = torch.jit.trace(block, (q, k, v, w, f), check_trace=False)
        assert "mmt::long_attention" in str(traced.graph) and "mmt::qk_norm_rope" in str(traced.graph)
        for q, k, v in (draw(), draw()):
            assert torch.equal(traced(q, k, v, w, f), _host_attention(q * 2, k * 3, v)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_a_traced_call_computes_on_new_inputs(dtype):
    w, f = torch.ones(32, dtype=dtype, device=DEV), ops.rotary_frequencies(32, device=DEV)

    def block(q, k, v):
        a, b = torch_ops.qk_norm_rope(q, k, w, w, f)
        return torch_ops.long_attention(a, b, v, causal=True, softcap=4.0, return_lse=True)
    first, then = (_case(dtype, 2, 40, 40, 4, 2, 32, seed=s)[0] for s in (1, 2))
    traced = torch.jit.trace(block, tuple(first[n] for n in "qkv"), check_trace=False)
    for t in (then, first):
        assert all(torch.equal(a, b) for a, b in zip(traced(*(t[n] for n in "qkv")), block(*(t[n] for n in "qkv"))))


# ------------------------------------------------------------------------------------------- tensors that are not plain memory
class _Held(torch.Tensor):
    """A subclass without memory of its own: every operator that meets it gets the tensor it holds."""

    @staticmethod
    def __new__(cls, held):
        return torch.Tensor._make_wrapper_subclass(cls, held.shape, strides=held.stride(), dtype=held.dtype, device=held.device)

    def __init__(self, held):
        self.held = held

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        give = lambda x: x.held if isinstance(x, _Held) else x
        return func(*(give(x) for x in args), **{n: give(x) for n, x in (kwargs or {}).items()})


def test_tensors_without_memory_are_refused_by_the_plain_calls():
    """ops.* reads addresses: a tensor that has none is an error, not an argument that was left out."""
    held = _Held(torch.empty(4, device="meta"))
    assert held.data_ptr() == 0
    on = torch.Tensor._make_wrapper_subclass(_Held, (1, 3, 4, 8), dtype=F32, device="cuda:0")
    for call in (lambda: ops._side(on, "slopes", on.shape, F32, on.device),
                 lambda: ops._head_rows(on, "q", None, F32, on.device)):
        with pytest.raises(MmtError, match="memory"):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_subclasses_and_lazy_views_count_like_what_they_stand_for(dtype):
    """A tensor subclass, a lazily negated view, a lazy zero in place of any argument: the bits of the plain tensor."""
    t, kw = _case(dtype, 2, 50, 90, 4, 2, 32, seed=71, prefix=True, cache=True, slopes=True, buckets=8, reach=16,
                  docs=[[(0, 60), (1, 30)], [(0, 90)]])
    args = dict(kw, **{n: t[n] for n in "qkv"})
    call = lambda **a: torch_ops.long_attention(a.pop("q"), a.pop("k"), a.pop("v"), causal=True, return_lse=True, **a)
    want = call(**args)
    for name, x in args.items():
        ways = [_Held(x)]
        if x.is_floating_point():
            ways.append(torch._neg_view(-x))
        for way in ways:
            assert all(torch.equal(a, b) for a, b in zip(call(**dict(args, **{name: way})), want)), name
    zero = torch._efficientzerotensor((4,), dtype=F32, device=DEV)
    got = call(**dict(args, slopes=zero)), call(**dict(args, slopes=torch.zeros(4, device=DEV)))
    assert all(torch.equal(a, b) for a, b in zip(*got))
    w, f = torch.linspace(0.5, 2, 32, device=DEV), ops.rotary_frequencies(32, device=DEV)
    pos = torch.arange(50, device=DEV).expand(2, 50).contiguous() * 7
    args = dict(q=t["q"], k=t["k"][:, :50].contiguous(), q_weight=w, k_weight=2 * w, inv_freq=f, positions=pos)
    want = torch_ops.qk_norm_rope(**args)
    for name, x in args.items():
        for way in [_Held(x)] + ([torch._neg_view(-x)] if x.is_floating_point() else []):
            assert all(torch.equal(a, b) for a, b in zip(torch_ops.qk_norm_rope(**dict(args, **{name: way})), want)), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_gradients_that_come_as_lazy_views(dtype):
    t, _ = _case(dtype, 2, 40, 40, 4, 2, 32, seed=73)
    w, f = torch.ones(32, dtype=dtype, device=DEV), ops.rotary_frequencies(32, device=DEV)
    q, k, v = (t[n].clone().requires_grad_() for n in "qkv")
    dlse = torch.randn(2, 4, 40, generator=torch.Generator().manual_seed(1)).to(DEV)
    lazy = lambda x: torch._neg_view(-x)
    zeros = lambda x: torch._efficientzerotensor(x.shape, dtype=x.dtype, device=x.device)

    def grads(how_out, how_lse):
        x, y = torch_ops.qk_norm_rope(q, k, w, w, f)
        both = torch_ops.long_attention(x, y, v, causal=True, return_lse=True)
        first = torch.autograd.grad(both, (x, y, v), (how_out(t["go"]), how_lse(dlse)), retain_graph=True)
        return list(first) + list(torch.autograd.grad((x, y), (q, k), (how_out(first[0]), how_out(first[1]))))
    plain = grads(lambda x: x, lambda x: x)
    assert all(torch.equal(a, b) for a, b in zip(plain, grads(lazy, lazy)))
    assert all(torch.equal(a, b) for a, b in zip(grads(lambda x: x, torch.zeros_like), grads(lambda x: x, zeros)))
    assert all(torch.equal(a, b) for a, b in zip(grads(torch.zeros_like, lambda x: x), grads(zeros, lambda x: x)))


# --------------------------------------------------------------------------------------------------------- rows that see nothing
def _blind(case, dtype, dh):
    """A case in which some rows see no key: (tensors, masks, plain arguments)."""
    f = {"cache": dict(cache=True), "docs": dict(docs=[[(0, 60), (1, 140)], [(2, 200)]]), "bias": dict(buckets=8, reach=16, both=True),
         "table": dict(buckets=8, reach=16, both=True, docs=[[(0, 60), (1, 140)], [(2, 200)]])}[case]
    t, kw = _case(dtype, 2, 150, 200, 4, 2, dh, seed=81, **f)
    if case == "cache":                                   # positions before the first key; a cache that holds nothing
        kw["kv_len"] = torch.tensor([61, 0], dtype=torch.int32, device=DEV)
    elif case == "bias":                                  # what lies ahead, and the row itself, are hidden: the first row sees nothing
        t, kw = _case(dtype, 2, 150, 150, 4, 2, dh, seed=81, **f)
        kw["rel_bias"][:, 4:] = -math.inf
        kw["rel_bias"][:, 0] = -math.inf
    else:                                                 # ids without keys, in the middle and at the end of a tile
        kw["q_doc"][0, 37:90:3] = 77
        kw["q_doc"][1, 120:] = 78
    return t, kw, dict(causal=case != "bias", softcap=3.0 if case == "table" else 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf], ids=str)
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("case", ["cache", "docs", "bias", "table"])
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_gradients_of_rows_that_see_nothing_reach_nothing(dtype, case, dh, bad):
    """A row that sees nothing has an output of 0 and a log-sum of -inf whatever the inputs are: gradients that arrive there, such as the
    -inf of a squared log-sum, count as none."""
    t, kw, plain = _blind(case, dtype, dh)
    q, k, v = (t[n].clone().requires_grad_() for n in "qkv")
    kw = dict(kw)
    leaves = [q, k, v]
    if "rel_bias" in kw:
        leaves.append(kw["rel_bias"].requires_grad_())
    out, lse = torch_ops.long_attention(q, k, v, return_lse=True, **kw, **plain)
    none = (lse == -math.inf).transpose(1, 2)
    assert none.any() and not none.all() and (out[none] == 0).all()
    dlse = torch.randn(lse.shape, generator=torch.Generator().manual_seed(5)).to(DEV)
    clean_o, clean_l = t["go"].masked_fill(none[..., None], 0), dlse.masked_fill(none.transpose(1, 2), 0)
    val, tol = long_rows.attention(t["q"], t["k"], t["v"], dout=clean_o, dlse=clean_l, dtype=dtype, **kw, **plain)
    for go, dl in ((clean_o, clean_l.masked_fill(none.transpose(1, 2), bad)), (clean_o.masked_fill(none[..., None], bad), clean_l)):
        got = torch.autograd.grad((out, lse), leaves, (go, dl), retain_graph=True)
        assert (got[0][none] == 0).all()
        for name, x in zip(("dq", "dk", "dv", "dbias"), got):
            _near(x, val[name], tol[name], name)


# ------------------------------------------------------------------------------------------------- masks' constants in the bias table
LOWEST = {"-1e4": -1e4, "fp16": -65504.0, "-1e9": -1e9, "-2^99": -2.0 ** 99, "bf16": torch.finfo(BF16).min, "fp32": torch.finfo(F32).min,
          "-inf": -math.inf, "1e9": 1e9}


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 130, 130, 2, 2), (2, 1, 70, 4, 1), (1, 40, 300, 4, 2)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("name", list(LOWEST))
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_mask_constants_in_the_bias_table(dtype, name, shape):
    """The constants that serve as masks, in some buckets and in all of a head's: buckets they hide next to other keys, rows that see
    nothing else (the first token of a causal row, whose own bucket is masked; a head with all buckets masked)."""
    t, kw = _case(dtype, *shape, 64, seed=4, buckets=8, reach=16)
    kw["rel_bias"][0, 0] = kw["rel_bias"][0, 3] = LOWEST[name]
    kw["rel_bias"][1, :] = LOWEST[name]
    _check(t, kw, dtype, causal=True)
    _check(t, kw, dtype, causal=True, softcap=5.0)


# ------------------------------------------------------------------------------------------- head sizes inside a tile's padded one
@pytest.mark.gpu
@pytest.mark.parametrize("bias", [False, True], ids=["plain", "bias"])
@pytest.mark.parametrize("shape", [(1, 1, 70, 2, 1), (2, 21, 21, 4, 2), (1, 150, 200, 2, 1), (1, 130, 600, 2, 2)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dh", [8, 24, 32, 40, 56, 72, 80, 88, 104, 120, 128])
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_infinite_keys_at_every_head_size(dtype, dh, shape, bias):
    """A key with an infinite element whose products are -inf weighs nothing, forward and in every gradient but the infinite element's
    own, at head sizes that fill a tile and at those that do not."""
    B, Lq, Lk, H, Hk = shape
    t, kw = _case(dtype, B, Lq, Lk, H, Hk, dh, seed=dh, **(dict(buckets=8, reach=20) if bias else {}))
    t["q"][..., 3] = t["q"][..., 3].abs() + 0.25
    t["k"][:, 5, :, 3] = -math.inf
    t["k"][:, Lk - 2, 0, 3] = -math.inf
    got = _run(t, kw, causal=bias)
    val, tol = long_rows.attention(t["q"], t["k"], t["v"], dout=t["go"], dtype=dtype, causal=bias, **kw)
    others = [d for d in range(dh) if d != 3]
    got[2], val["dq"], tol["dq"] = (x[..., others] for x in (got[2], val["dq"], tol["dq"]))
    for name, x in zip(("out", "lse", "dq", "dk", "dv", "dbias"), got):
        _near(x, val[name], tol[name], name)


# --------------------------------------------------------------------------------------------------------------- forward mode
def test_a_tangent_under_the_dispatcher_is_refused():
    """Below autograd the dispatcher's op still sees the tangent of an argument: an error, whatever else is wrong with the call."""
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(torch.ones(1, 2, 2, 8), torch.ones(1, 2, 2, 8))
        for fn in (torch_ops._long_attention, torch_ops._long_attention_bwd):
            with pytest.raises(MmtError, match="forward-mode"):
                fn(dual, dual, dual)


@pytest.mark.gpu
def test_tangents_of_constants_are_refused():
    """Forward-mode gradients are not supported, of the constants as little as of q, k and v: an error, not a tangent that vanishes."""
    t, kw = _case(F32, 1, 20, 20, 2, 2, 32, seed=91, slopes=True)
    w, f = torch.ones(32, device=DEV), ops.rotary_frequencies(32, device=DEV)
    with torch.autograd.forward_ad.dual_level():
        dual = lambda x: torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for fn in (lambda: torch_ops.long_attention(t["q"], t["k"], t["v"], slopes=dual(kw["slopes"])),
                   lambda: torch_ops.long_attention(t["q"].transpose(2, 3).contiguous().transpose(2, 3), t["k"], t["v"], slopes=dual(kw["slopes"])),
                   lambda: torch_ops.qk_norm_rope(t["q"], t["k"], w, w, dual(f)),
                   lambda: torch_ops.qk_norm_rope(t["q"], t["k"], dual(w), w, f),
                   lambda: torch.ops.mmt.qk_norm_rope(t["q"], t["k"], w, w, dual(f), None, 1e-6, False),
                   lambda: torch.ops.mmt.long_attention(dual(t["q"]), t["k"], t["v"], None, False, None, None, None, None, 0.0, None, None, None),
                   lambda: torch.ops.mmt.long_attention(t["q"], t["k"], t["v"], None, False, None, None, None, None, 0.0, dual(kw["slopes"]),
                                                        None, None)):
            with pytest.raises((MmtError, RuntimeError)):
                fn()


# ------------------------------------------------------------------------------------------------------------- the bounds themselves
@pytest.mark.parametrize("bad", [0.0, math.nan, math.inf, -math.inf], ids=str)
@pytest.mark.parametrize("cache", [False, True], ids=["docs", "cache"])
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_the_bounds_do_not_depend_on_what_padding_holds(dtype, cache, bad):
    """The oracle's bounds with anything in padding and behind the cache's end: those of zeros there, and finite."""
    g = torch.Generator().manual_seed(8)
    q, k, v, go = (torch.randn(2, 60, n, 16, generator=g).to(dtype) for n in (4, 2, 2, 4))
    if cache:
        kw = dict(kv_len=torch.tensor([60, 33], dtype=torch.int32))
        dead, dead_q = torch.arange(60)[None] >= kw["kv_len"][:, None], torch.zeros(2, 60, dtype=torch.bool)
    else:
        ids = torch.tensor([[0] * 30 + [-1] * 9 + [1] * 21, [-1] * 3 + [2] * 50 + [-1] * 7], dtype=torch.int32)
        kw = dict(q_doc=ids, k_doc=ids)
        dead = dead_q = ids < 0
    res = []
    for hold in (0.0, bad):
        k[dead], v[dead] = hold, hold
        q[dead_q], go[dead_q] = hold, hold
        res.append(long_rows.attention(q, k, v, dout=go, causal=True, dtype=dtype, **kw))
    for name, x in res[0][1].items():
        assert torch.isfinite(x).all(), name
        assert torch.equal(x, res[1][1][name]), name


def test_a_bound_that_would_pass_anything_is_an_error():
    x = torch.rand(1, 3, 1, 8) + 0.5
    with pytest.raises(AssertionError, match="bound"):
        long_rows.attention(x, torch.full_like(x, math.inf), x, softcap=1.0, dtype=F32)


# ------------------------------------------------------------------------------------- precision of the rows' correction (delta)
def _rounded_gradients(q, k, v, go, dtype, causal, delta):
    """dq and dk in 64 bits but for the roundings that the backward makes: of P and dS to the element type where they enter a product, and
    of the results.  ``delta`` = rowsum(dO o) comes from o itself ("exact"), from the rounded output and what its rounding took ("low": P was
    rounded on its way there), or from the rounded output alone ("out")."""
    scale = q.shape[-1] ** -0.5
    # powers of two ahead of the roundings keep fp16's exponent range out of this
    rnd = lambda x: ((x * (up := 2.0 ** (14 - math.ceil(math.log2(float(x.abs().max())))))).to(dtype).double() / up)
    heads = lambda x: x.double().transpose(1, 2)
    Q, K, V, D = map(heads, (q, k, v, go))
    s = scale * Q @ K.transpose(2, 3)
    if causal:
        s = s.masked_fill(~torch.ones(s.shape[-2:], dtype=torch.bool).tril(), -math.inf)
    P = s.softmax(-1)
    out = P @ V if delta == "exact" else rnd(P) @ V
    if delta != "exact":
        kept = out.to(dtype).double()
        out = kept + (out - kept).to(dtype).double() if delta == "low" else kept
    dS = rnd(P * (D @ V.transpose(2, 3) - (D * out).sum(-1, keepdim=True)))
    return (scale * dS @ K).transpose(1, 2), (scale * dS.transpose(2, 3) @ Q).transpose(1, 2)


def _offset_case(dtype, L, H=2, dh=64):
    """Values around a common offset: all of a row's dP lie near delta, of which little may be lost."""
    g = torch.Generator().manual_seed(L)
    q, k, v, go = (torch.randn(1, L, H, dh, generator=g) for _ in range(4))
    return [x.to(dtype) for x in (q, k, 4 + v / 4, go)]


def _off(x, y):
    return float((x.double().cpu() - y).norm() / y.norm())


# (length, causal): up to 512 keys every row of dQ sees its corrected delta, beyond that the one from the output and its low part; dK always
# the corrected one.  Bound: twice what the roundings of P and dS alone do, which the next worse delta exceeds.
PRECISION = [(140, True, "exact", "low"), (400, True, "exact", "low"), (2304, False, "low", "out")]


@pytest.mark.parametrize("L,causal,has,worse", PRECISION, ids=lambda x: str(x))
@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
def test_what_the_precision_of_delta_is_worth(dtype, L, causal, has, worse):
    """The next test's bounds fail without what it tests: with the next worse delta dQ, and with the rounded output's dK, are beyond them."""
    t = _offset_case(dtype, L)
    want = _rounded_gradients(*t, torch.float64, causal, "exact")
    got = {d: [_off(x.to(dtype), y) for x, y in zip(_rounded_gradients(*t, dtype, causal, d), want)] for d in ("exact", "low", "out")}
    assert got[worse][0] > 2 * got[has][0] and got["out"][1] > 2 * got["exact"][1]


@pytest.mark.gpu
@pytest.mark.parametrize("L,causal,has,worse", PRECISION, ids=lambda x: str(x))
@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
def test_precision_of_delta(dtype, L, causal, has, worse):
    t = _offset_case(dtype, L)
    want = _rounded_gradients(*t, torch.float64, causal, "exact")
    allowed = [2 * _off(_rounded_gradients(*t, dtype, causal, d)[n].to(dtype), want[n]) for n, d in enumerate((has, "exact"))]
    dev = dict(zip(("q", "k", "v", "go"), (x.to(DEV) for x in t)))
    got = _run(dev, {}, causal=causal)
    for name, x, y, most in zip(("dq", "dk"), got[2:], want, allowed):
        assert _off(x, y) <= most, (name, _off(x, y), most)
    if L > 512:
        return
    # the same as scenes of one row: what counts is how many keys a row sees
    row = {n: torch.cat((x, x.flip(1), x), 1) for n, x in dev.items()}
    ids = torch.arange(3, dtype=torch.int32, device=DEV).repeat_interleave(L)[None].contiguous()
    got = _run(row, dict(q_doc=ids, k_doc=ids), causal=causal)
    for name, x, y, most in zip(("dq", "dk"), got[2:], want, allowed):
        for at in (0, 2 * L):
            assert _off(x[:, at:at + L], y) <= most, (name, at, _off(x[:, at:at + L], y), most)


# ------------------------------------------------------------------------------------------------------------ two passes of dQ
@pytest.mark.gpu
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16], ids=IDS.get)
def test_a_scene_has_the_same_gradient_wherever_it_starts(dtype, dh):
    """A scene of 4352 tokens behind another one, across token 4096, and at the start of its row: the same tiles in the same order, so the
    same bits (what a workgroup does depends on all the tiles it sees, not on how they are looked up)."""
    L, n = 8704, 4352
    a, _ = _case(dtype, 1, L, L, 2, 1, dh, seed=97)
    ids = lambda *s: torch.tensor([i for i, m in s for _ in range(m)], dtype=torch.int32, device=DEV)[None]
    first, late = ids((0, n), (1, L - n)), ids((1, 3840), (0, n), (2, L - n - 3840))
    b = {x: torch.cat((y[:, n:n + 3840], y[:, :n], y[:, n + 3840:]), 1) for x, y in a.items()}
    res = [_run(t, dict(q_doc=d, k_doc=d), causal=True) for t, d in ((a, first), (b, late))]
    cut = lambda x, at: x[:, at:at + n] if x.dim() == 4 else x[:, :, at:at + n]
    for name, x, y in zip(("out", "lse", "dq"), *res):
        assert torch.equal(cut(x, 0), cut(y, 3840)), name


@pytest.mark.gpu
@pytest.mark.parametrize("factor", [2.0 ** -14, 2.0 ** -20], ids=["2^-14", "2^-20"])
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_gradients_of_very_different_size_in_one_call(dtype, factor):
    """One row's gradient a million times the others': each keeps what its own type keeps of it (fp16 scales the score gradients of a call
    by one power of two, and what that costs the small ones is in the bound: 2^-38 of the largest)."""
    t, kw = _case(dtype, 2, 140, 140, 4, 2, 64, seed=101, buckets=8, reach=16)
    small = torch.full((2, 140, 1, 1), factor, device=DEV)
    small[0, 77] = 1.0
    t["go"] = (t["go"].float() * small).to(dtype)
    _check(t, kw, dtype, causal=True)
    _check(t, kw, dtype)


# ------------------------------------------------------------------------------------------------- numbers that fp32 cannot hold
def test_a_cap_that_vanishes_in_fp32_is_refused(monkeypatch):
    """1e-50 is a cap, 0 is none: a cap that fp32 rounds to 0 must not switch the cap off."""
    monkeypatch.setattr(ops, "_head_rows", lambda t, *a: (t, 0x1000, 0, 16, 16))
    q = torch.zeros(1, 2, 1, 8)
    for cap in (1e-50, 5e-324):
        with pytest.raises(MmtError, match="cap"):
            ops._attention_args(q, q, q, None, False, None, None, None, None, cap, None, None, None)
    ops._attention_args(q, q, q, None, False, None, None, None, None, 0.0, None, None, None)


@pytest.mark.gpu
def test_a_cap_that_vanishes_in_fp32_is_refused_by_the_native_call():
    t, _ = _case(F32, 1, 8, 8, 2, 2, 32)
    for cap in (1e-50, 1e-42):
        with pytest.raises(MmtError, match="cap"):
            torch_ops.long_attention(t["q"], t["k"], t["v"], softcap=cap)


def test_a_table_of_too_many_entries_is_refused():
    """One wave sums each entry of the bias gradient: a launch has fewer than 2^32 threads."""
    lib = _lib.load()
    a = _desc(B=1, Lq=1, Lk=1, H=1 << 21, Hk=1 << 21, rel_bias=0x1000, rel_buckets=0x1000, n_buckets=32, reach=8)
    assert lib.mmt_long_attention_workspace_bytes(ctypes.byref(a), 1) == 0 and b"too many" in lib.mmt_last_error()
    a.n_buckets = 31
    assert lib.mmt_long_attention_workspace_bytes(ctypes.byref(a), 1) > 0


# ------------------------------------------------------------------------------------------------------------- captured training steps
@pytest.mark.gpu
def test_leaves_of_a_graph_that_lives_elsewhere_are_refused_while_capturing():
    """A leaf whose accumulator an eager graph of another stream holds: the forward call of a captured step is an error.  Without that graph,
    or on leaves made inside, the step is captured and replays."""
    t, kw = _case(BF16, 1, 70, 70, 2, 2, 64, seed=103, buckets=8, reach=16)
    w, f = torch.ones(64, device=DEV, requires_grad=True), ops.rotary_frequencies(64, device=DEV)
    table = kw["rel_bias"].requires_grad_()

    def step(table, w, v):
        a, b = torch_ops.qk_norm_rope(t["q"], t["k"], w, w.detach(), f)
        return torch_ops.long_attention(a, b, v, causal=True, rel_bias=table, rel_buckets=kw["rel_buckets"])
    for leaf in (dict(table=table, w=w.detach(), v=t["v"]), dict(table=table.detach(), w=w, v=t["v"]),
                 dict(table=table.detach(), w=w.detach(), v=t["v"].clone().requires_grad_())):
        alive = step(**leaf)                                # an eager graph of the leaf, on the eager stream
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with pytest.raises(MmtError, match="capture"):
            with torch.cuda.graph(g):
                step(**leaf)
        torch.cuda.synchronize()
        of = [x for x in leaf.values() if x.requires_grad]
        want, = torch.autograd.grad(alive, of, t["go"])     # the eager graph is as it was
        del alive

        def captured():
            own = {n: x.detach().requires_grad_(x.requires_grad) for n, x in leaf.items()}
            return torch.autograd.grad(step(**own), [x for x in own.values() if x.requires_grad], t["go"])[0]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = captured()
        for _ in range(3):
            got.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)
            assert torch.equal(captured(), want)


# ------------------------------------------------------------------------------------------------------------------ under the compiler
def test_a_compiled_call_is_one_graph():
    """torch.compile takes the wrappers into its graph as the operators, without a break."""
    with torch.library._scoped_library("mmt", "IMPL") as lib:
        lib.impl("long_attention", _host_attention, "CPU")
        lib.impl("qk_norm_rope", lambda q, k, *rest: (q * 2, k * 3), "CPU")

        def block(q, k, v, w, f):
            a, b = torch_ops.qk_norm_rope(q, k, w, w, f)
            return torch_ops.long_attention(a, b, v, return_lse=True)
        g = torch.Generator().manual_seed(0)
        q, k, v = (torch.randn(1, 5, 2, 8, generator=g) for _ in range(3))
        got = torch.compile(block, backend="aot_eager", fullgraph=True)(q, k, v, torch.ones(8), ops.rotary_frequencies(8))
        assert all(torch.equal(x, y) for x, y in zip(got, _host_attention(q * 2, k * 3, v)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_a_compiled_step_has_the_same_bits(dtype):
    t, kw = _case(dtype, 2, 50, 50, 4, 2, 32, seed=107, buckets=8, reach=16, slopes=True, prefix=True)
    w, f = torch.ones(32, dtype=dtype, device=DEV), ops.rotary_frequencies(32, device=DEV)
    table = kw.pop("rel_bias")

    def block(q, k, v, table, w):
        a, b = torch_ops.qk_norm_rope(q, k, w, w, f)
        return torch_ops.long_attention(a, b, v, causal=True, softcap=5.0, rel_bias=table, **kw)
    res = []
    for fn in (block, torch.compile(block, backend="aot_eager", fullgraph=True)):
        leaves = [x.clone().requires_grad_() for x in (t["q"], t["k"], t["v"], table, w)]
        out = fn(*leaves)
        res.append([out] + list(torch.autograd.grad(out, leaves, t["go"])))
    assert all(torch.equal(x, y) for x, y in zip(*res))
