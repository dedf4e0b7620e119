"""Edges of attention over long rows and of the norm + rotation in front of it: calls under torch's tracer, tensors that are not plain
memory, rows that see nothing, lowest-value biases, head sizes inside a tile, precision of the corrected backward pass."""
import math

import pytest
import torch

from multimodal_transformer_amd import ops, torch_ops
from multimodal_transformer_amd._lib import MmtError
from oracle import long_rows
from test_long_attention import BF16, DEV, F16, F32, IDS, TYPES, _case, _check, _near, _run


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
