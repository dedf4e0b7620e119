"""The Level-2 operators as PyTorch custom ops (namespace ``mmt``), registered with ``torch.library`` on top of the C-ABI calls
of ``ops.py`` (SURVEY.md 8b "native op surface"): visible to the dispatcher (``torch.ops.mmt.*``), with Meta kernels so that
shape propagation / fake-tensor tracing works, CUDA (= HIP) implementations only - there is no CPU kernel to dispatch to.

Packed weight descriptors (``ops.PackedEncoder`` ...) are Python objects holding device pointers; an op receives one as an
integer handle (``handle_of``), which stays valid while the descriptor is alive.

    memory, pad = torch.ops.mmt.encoder_fwd(x_st, handle_of(enc.packed()))
    pred_st     = torch.ops.mmt.decoder_ar_fwd(memory, pad, start_pos, None, None, handle_of(packed), 12)
"""
from __future__ import annotations

import ctypes
import weakref

import torch
from torch.autograd import forward_ad

from . import ops
from ._lib import MmtError, native as _native

_HANDLES: "weakref.WeakValueDictionary[int, object]" = weakref.WeakValueDictionary()


def handle_of(packed) -> int:
    """Integer handle of a packed descriptor (valid while the descriptor object is alive)."""
    h = id(packed)
    _HANDLES[h] = packed
    return h


def _get(handle, kind):
    obj = _HANDLES.get(int(handle))
    if obj is None or not isinstance(obj, kind):
        raise MmtError(f"stale or foreign handle {handle}: expected a live {kind.__name__}")
    return obj


_lib = torch.library.Library("mmt", "DEF")
_lib.define("encoder_fwd(Tensor x_st, int handle) -> (Tensor, Tensor)")
_lib.define("decoder_ar_fwd(Tensor memory, Tensor? pad_mask, Tensor start_pos, Tensor? map_feat, Tensor? mem_feat, int handle, int ph) -> Tensor")
_lib.define("decoder_tf_fwd(Tensor memory, Tensor? pad_mask, Tensor tgt, Tensor? mem_feat, int handle) -> Tensor")
_lib.define("cnn_map_fwd(Tensor maps, int handle, bool input_affine) -> Tensor")
_lib.define("vit_map_fwd(Tensor maps, int handle, bool input_affine) -> Tensor")
_lib.define("lane_enc_fwd(Tensor lanes, int handle) -> Tensor")
_lib.define("unstandardize(Tensor pred_st, Tensor node_pos) -> Tensor")
_lib.define("ade_fde(Tensor pred, Tensor gt) -> (Tensor, Tensor)")
_ATTN = ("float? scale, bool causal, Tensor? prefix, Tensor? q_doc, Tensor? k_doc, Tensor? kv_len, float softcap, Tensor? slopes, "
         "Tensor? rel_bias, Tensor? rel_buckets")
_ROPE = "Tensor q, Tensor k, Tensor q_weight, Tensor k_weight, Tensor inv_freq, Tensor? positions, float eps, bool interleaved"
_lib.define(f"long_attention(Tensor q, Tensor k, Tensor v, {_ATTN}) -> (Tensor out, Tensor lse, Tensor low)")
_lib.define(f"long_attention_bwd(Tensor dout, Tensor? dlse, Tensor out, Tensor lse, Tensor? low, Tensor q, Tensor k, Tensor v, {_ATTN}) "
            "-> (Tensor, Tensor, Tensor, Tensor)")
_lib.define(f"qk_norm_rope({_ROPE}) -> (Tensor, Tensor)")
_lib.define(f"qk_norm_rope_bwd(Tensor dq_out, Tensor dk_out, {_ROPE}) -> (Tensor, Tensor, Tensor, Tensor)")


def _encoder_fwd(x_st, handle):
    return ops.encoder_forward(_get(handle, ops.PackedEncoder), x_st, want_mask=True)


def _encoder_fwd_meta(x_st, handle):
    enc = _get(handle, ops.PackedEncoder)
    B, T, _ = x_st.shape
    return x_st.new_empty(B, T, enc.d_model), x_st.new_empty(B, T, dtype=torch.uint8)


def _decoder_ar_fwd(memory, pad_mask, start_pos, map_feat, mem_feat, handle, ph):
    return ops.decoder_forward(_get(handle, ops.PackedDecoder), memory, pad_mask, start_pos, ph, map_feat=map_feat, mem_feat=mem_feat)[0]


def _decoder_ar_fwd_meta(memory, pad_mask, start_pos, map_feat, mem_feat, handle, ph):
    dec = _get(handle, ops.PackedDecoder)
    return memory.new_empty(memory.shape[0], ph, dec.n_in)


def _decoder_tf_fwd(memory, pad_mask, tgt, mem_feat, handle):
    return ops.decoder_forward(_get(handle, ops.PackedDecoder), memory, pad_mask, tgt=tgt, mem_feat=mem_feat)[1]


def _decoder_tf_fwd_meta(memory, pad_mask, tgt, mem_feat, handle):
    dec = _get(handle, ops.PackedDecoder)
    return memory.new_empty(memory.shape[0], tgt.shape[1], dec.n_out)


def _cnn_map_fwd(maps, handle, input_affine):
    return ops.cnn_forward(_get(handle, ops.PackedCnn), maps, input_affine=input_affine)


def _vit_map_fwd(maps, handle, input_affine):
    return ops.vit_forward(_get(handle, ops.PackedVit), maps, input_affine=input_affine)


def _lane_enc_fwd(lanes, handle):
    return ops.lane_forward(_get(handle, ops.PackedLane), lanes)


def _n_out_meta(kind):
    def meta(x, handle, *flags):
        return x.new_empty(x.shape[0], _get(handle, kind).desc.n_out)
    return meta


def _unstandardize(pred_st, node_pos):
    return ops.finalize(pred_st, node_pos)[0]


def _ade_fde(pred, gt):
    _, ade, fde, _ = ops.finalize(pred, None, gt, metres=False, want_pred=False, want_metrics=True)
    return ade, fde


# ---- attention over long rows, norm + rotation: differentiable ------------------------------------------------------------------
def _no_tangents(fn):
    """An operator without forward-mode gradients: a tangent that arrives is an error, it would vanish."""
    def call(*args):
        if forward_ad._current_level >= 0 and any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in args):
            raise MmtError("forward-mode gradients are not supported")
        return fn(*args)
    return call


@_no_tangents
def _long_attention(*args):
    out, lse, low = ops.long_attention(*args, keep_low=True)
    return out, lse, low if low is not None else out.new_empty(0)


@_no_tangents
def _long_attention_bwd(*args):
    dq, dk, dv, dbias = ops.long_attention_backward(*args)
    return dq, dk, dv, dbias if dbias is not None else dq.new_empty(0, dtype=torch.float32)


def _long_attention_meta(q, k, v, *rest):
    B, Lq, H, _ = q.shape
    return q.new_empty(q.shape), q.new_empty((B, H, Lq), dtype=torch.float32), q.new_empty(q.shape if q.dtype != torch.float32 else 0)


def _long_attention_bwd_meta(dout, dlse, out, lse, low, q, k, v, *rest):
    table = rest[-2]
    return q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape), \
        q.new_empty(table.shape if table is not None else 0, dtype=torch.float32)


def _qk_norm_rope_meta(q, k, *rest):
    return q.new_empty(q.shape), k.new_empty(k.shape)


def _qk_norm_rope_bwd_meta(dqo, dko, q, k, q_weight, k_weight, *rest):
    return q.new_empty(q.shape), k.new_empty(k.shape), q_weight.new_empty(q_weight.shape), k_weight.new_empty(k_weight.shape)


for _name, _fn, _meta in (
        ("long_attention", _long_attention, _long_attention_meta),
        ("long_attention_bwd", _long_attention_bwd, _long_attention_bwd_meta),
        ("qk_norm_rope", _no_tangents(ops.qk_norm_rope), _qk_norm_rope_meta),
        ("qk_norm_rope_bwd", _no_tangents(ops.qk_norm_rope_backward), _qk_norm_rope_bwd_meta),
        ("encoder_fwd", _encoder_fwd, _encoder_fwd_meta),
        ("decoder_ar_fwd", _decoder_ar_fwd, _decoder_ar_fwd_meta),
        ("decoder_tf_fwd", _decoder_tf_fwd, _decoder_tf_fwd_meta),
        ("cnn_map_fwd", _cnn_map_fwd, _n_out_meta(ops.PackedCnn)),
        ("vit_map_fwd", _vit_map_fwd, _n_out_meta(ops.PackedVit)),
        ("lane_enc_fwd", _lane_enc_fwd, _n_out_meta(ops.PackedLane)),
        ("unstandardize", _unstandardize, lambda p, n: torch.empty_like(p)),
        ("ade_fde", _ade_fde, lambda p, g: (p.new_empty(p.shape[0]), p.new_empty(p.shape[0])))):
    _lib.impl(_name, _fn, "CUDA")
    _lib.impl(_name, _meta, "Meta")


def _constant(t, what):
    if isinstance(t, torch.Tensor) and t.requires_grad:
        raise MmtError(f"{what} are constants, they get no gradient")


def _long_attention_grads(ctx, dout, dlse, bwd):
    out, lse, low, q, k, v, prefix, q_doc, k_doc, kv_len, slopes, rel_bias, rel_buckets = ctx.saved_tensors
    scale, causal, softcap = ctx.plain
    if dout is None and dlse is None:
        return (None,) * 13
    if dout is None:
        dout = torch.zeros_like(out)
    dq, dk, dv, dbias = bwd(dout, dlse, out, lse, low, q, k, v, scale, causal, prefix, q_doc, k_doc, kv_len, softcap, slopes, rel_bias,
                            rel_buckets)
    return (dq, dk, dv) + (None,) * 8 + (dbias if rel_bias is not None else None, None)


# gradients of the dispatcher's ops, for callers of torch.ops.mmt.* and for tracing
def _long_attention_ctx(ctx, inputs, output):
    q, k, v, scale, causal, prefix, q_doc, k_doc, kv_len, softcap, slopes, rel_bias, rel_buckets = inputs
    _constant(slopes, "long_attention: the slopes of the distance bias")
    out, lse, low = output
    ctx.set_materialize_grads(False)
    ctx.mark_non_differentiable(low)
    ctx.save_for_backward(out, lse, low if low.numel() == out.numel() else None, q, k, v, prefix, q_doc, k_doc, kv_len, slopes, rel_bias,
                          rel_buckets)
    ctx.plain = scale, causal, softcap


def _qk_norm_rope_ctx(ctx, inputs, output):
    q, k, q_weight, k_weight, inv_freq, positions, eps, interleaved = inputs
    _constant(inv_freq, "qk_norm_rope: the frequencies")
    ctx.save_for_backward(q, k, q_weight, k_weight, inv_freq, positions)
    ctx.plain = eps, interleaved


def _no_second(name):
    def refuse(ctx, *grads):
        raise MmtError(f"{name}: there is no second derivative")
    return refuse


torch.library.register_autograd("mmt::long_attention", lambda ctx, dout, dlse, _: _long_attention_grads(
    ctx, dout, dlse, torch.ops.mmt.long_attention_bwd), setup_context=_long_attention_ctx, lib=_lib)
torch.library.register_autograd("mmt::qk_norm_rope", lambda ctx, dqo, dko: tuple(torch.ops.mmt.qk_norm_rope_bwd(
    dqo, dko, *ctx.saved_tensors, *ctx.plain)) + (None,) * 4, setup_context=_qk_norm_rope_ctx, lib=_lib)
torch.library.register_autograd("mmt::long_attention_bwd", _no_second("long_attention"), lib=_lib)
torch.library.register_autograd("mmt::qk_norm_rope_bwd", _no_second("qk_norm_rope"), lib=_lib)


def _traced(t):
    """The call is being traced (fake tensors, a dispatch mode, torch.compile, torch.jit.trace): it has to go through the dispatcher.
    Otherwise the wrappers below go straight to the kernels."""
    return type(t) not in (torch.Tensor, torch.nn.Parameter) or torch.compiler.is_compiling() or torch._C._len_torch_dispatch_stack() > 0 or \
        torch._C._is_tracing()


def _lazy(*args):
    """Some argument is not the memory at its address (a tensor subclass, a lazily negated view, a lazy zero): the dispatcher turns it
    into what the kernels read."""
    return any(isinstance(t, torch.Tensor) and (type(t) not in (torch.Tensor, torch.nn.Parameter) or t.is_neg() or t._is_zerotensor())
               for t in args)


def _dispatched(op, *args):
    """(a lazy zero would become an expanded one, which the kernels' tables must not be: it is written out)"""
    return op(*(t.clone() if isinstance(t, torch.Tensor) and t._is_zerotensor() else t for t in args))


def _plain(fn, *args):
    """The native call that checks for itself; None where an argument is not what it expects."""
    try:
        return fn(*args)
    except TypeError:
        return None


# ---- what the module classes call: the same ops through the dispatcher, with this package's error for host tensors ------------
def _dev(*tensors):
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise MmtError(f"tensor is on {t.device}; the HIP kernels need device memory (no CPU fallback)")


def encoder_fwd(packed, x_st):
    _dev(x_st)
    return torch.ops.mmt.encoder_fwd(x_st, handle_of(packed))


def decoder_ar_fwd(packed, memory, pad_mask, start_pos, ph, map_feat=None, mem_feat=None):
    _dev(memory, pad_mask, start_pos, map_feat, mem_feat)
    return torch.ops.mmt.decoder_ar_fwd(memory, pad_mask, start_pos, map_feat, mem_feat, handle_of(packed), int(ph))


def decoder_tf_fwd(packed, memory, pad_mask, tgt, mem_feat=None):
    _dev(memory, pad_mask, tgt, mem_feat)
    return torch.ops.mmt.decoder_tf_fwd(memory, pad_mask, tgt, mem_feat, handle_of(packed))


def cnn_map_fwd(packed, maps, input_affine):
    _dev(maps)
    return torch.ops.mmt.cnn_map_fwd(maps, handle_of(packed), bool(input_affine))


def vit_map_fwd(packed, maps, input_affine):
    _dev(maps)
    return torch.ops.mmt.vit_map_fwd(maps, handle_of(packed), bool(input_affine))


def lane_enc_fwd(packed, lanes):
    _dev(lanes)
    return torch.ops.mmt.lane_enc_fwd(lanes, handle_of(packed))


def unstandardize(pred_st, node_pos):
    _dev(pred_st, node_pos)
    return torch.ops.mmt.unstandardize(pred_st, node_pos)


def long_attention(q, k, v, *, scale=None, causal=False, prefix=None, q_doc=None, k_doc=None, kv_len=None, softcap=0.0, slopes=None,
                   rel_bias=None, rel_buckets=None, return_lse=False):
    """Attention over rows of any length, differentiable in q, k, v and rel_bias.  q (B,Lq,H,dh), k and v (B,Lk,Hk,dh) in bfloat16,
    float16 or float32, H a multiple of Hk; query i of batch row b stands at position ``kv_len[b] - Lq + i`` (``Lk - Lq + i`` without
    cache lengths), so the same call serves training (Lq = Lk), a chunk of new tokens and a single one over a cache.

    scale      factor of the products, dh^-1/2 by default          softcap   > 0: scores become softcap * tanh(score / softcap)
    causal     keys behind the query's position are hidden ...     prefix    (B) int32: ... but the first prefix[b] are not
    kv_len     (B) int32: keys at and beyond it do not exist       q_doc, k_doc  (B,Lq), (B,Lk) int32: only equal ids see each other;
                                                                             negative: padding, sees and is seen by nothing
    slopes     (H) float32: -slopes[h] * distance is added         rel_bias  (H,n) float32, learned, at rel_buckets (2 reach + 1) int32 of
                                                                             the clamped distance (``ops.relative_buckets``);
               entries count as clamped to -2^14 .. 2^14, at or below -2^100 (-inf, a type's lowest value) they hide their bucket
    Rows that see nothing give zeros (and an lse of -inf).  Returns out (B,Lq,H,dh), with ``return_lse`` also the log-sums (B,H,Lq)."""
    if _traced(q):
        out, lse = torch.ops.mmt.long_attention(q, k, v, scale, bool(causal), prefix, q_doc, k_doc, kv_len, float(softcap), slopes,
                                                rel_bias, rel_buckets)[:2]
        return (out, lse) if return_lse else out
    both = _plain(_native().plain_long_attention, q, k, v, scale, causal, prefix, q_doc, k_doc, kv_len, softcap, slopes, rel_bias, rel_buckets)
    if both is None:                                      # something to copy, or to complain about
        if _lazy(q, k, v, prefix, q_doc, k_doc, kv_len, slopes, rel_bias, rel_buckets):
            both = _dispatched(torch.ops.mmt.long_attention, q, k, v, scale, bool(causal), prefix, q_doc, k_doc, kv_len, float(softcap),
                               slopes, rel_bias, rel_buckets)[:2]
        else:
            if torch.is_grad_enabled():
                _constant(slopes, "long_attention: the slopes of the distance bias")
            a, q, k, v = ops._attention_args(q, k, v, scale, causal, prefix, q_doc, k_doc, kv_len, softcap, slopes, rel_bias, rel_buckets)
            both = _native().long_attention(ctypes.addressof(a), q, k, v, prefix, q_doc, k_doc, kv_len, slopes, rel_bias, rel_buckets)
    out, lse = both
    return (out, lse) if return_lse else out


def qk_norm_rope(q, k, q_weight, k_weight, inv_freq, positions=None, *, eps=1e-6, interleaved=False):
    """RMS norm of queries (B,L,H,dh) and keys (B,L,Hk,dh) per head, times the weights (dh), and the rotation of their first
    2 * len(inv_freq) elements by position * inv_freq (float64, ``ops.rotary_frequencies``) in the same pass; differentiable in q, k
    and the weights.  ``positions`` (B,L) int64, None: 0..L-1.  Pairs are (m, m + rot/2), with ``interleaved`` (2m, 2m + 1)."""
    if _traced(q):
        return torch.ops.mmt.qk_norm_rope(q, k, q_weight, k_weight, inv_freq, positions, float(eps), bool(interleaved))
    both = _plain(_native().plain_qk_norm_rope, q, k, q_weight, k_weight, inv_freq, positions, eps, interleaved)
    if both is None:
        if _lazy(q, k, q_weight, k_weight, inv_freq, positions):
            return _dispatched(torch.ops.mmt.qk_norm_rope, q, k, q_weight, k_weight, inv_freq, positions, float(eps), bool(interleaved))
        if torch.is_grad_enabled():
            _constant(inv_freq, "qk_norm_rope: the frequencies")
        a, q, k = ops._rope_args(q, k, q_weight, k_weight, inv_freq, positions, eps, interleaved)
        both = _native().qk_norm_rope(ctypes.addressof(a), q, k, q_weight, k_weight, inv_freq, positions)
    return both
