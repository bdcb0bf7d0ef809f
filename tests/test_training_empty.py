"""Training operators' calls without tokens: whatever else they carry, they give empty outputs and zero gradients of the weights.
(The address of an empty tensor is null.)"""

import ctypes

import pytest
import torch

from kernel_opt_agent_b200 import _lib, qk_norm_rope, qk_norm_rope_bwd, training
from tests.test_training_capi import AXIS, INVALID, OK, _rope

ONE_AXIS = (ctypes.c_uint8 * 16)()
EMPTY = [
    # positions of several axes, of one axis beyond the tables' rows, none beyond them
    dict(axes=3, pair_axis=ctypes.addressof(AXIS)), dict(table_rows=1), dict(seqlen=500, table_rows=8),
    dict(seqlen=500, axes=2, pair_axis=ctypes.addressof(ONE_AXIS))]


@pytest.mark.parametrize("changes", EMPTY)
def test_no_tokens_without_positions_address(changes):
    lib = _lib.load()
    args = _rope(**{"batch": 0, "q": None, "k": None, "q_out": None, "k_out": None, **changes})
    assert lib.tokmix_qk_norm_rope_fwd(ctypes.byref(args), None, None) == OK, _lib.last_error()
    # the gradient of the weights needs a GPU: the refusals come before it is asked for
    assert lib.tokmix_qk_norm_rope_bwd(ctypes.byref(args), None, ctypes.c_void_p(16), None, 0, None, None) == INVALID
    assert b"weight gradient" in lib.tokmix_last_error()


@pytest.mark.parametrize("changes", [
    dict(batch=2, axes=3, pair_axis=ctypes.addressof(AXIS)), dict(batch=2, table_rows=4), dict(batch=0, axes=3),
    dict(batch=0, axes=5, pair_axis=ctypes.addressof(AXIS)), dict(batch=0, table_rows=0), dict(batch=0, eps=-1.0),
    dict(seqlen=0, axes=3)])
def test_what_stays_refused(changes):
    lib = _lib.load()
    assert lib.tokmix_qk_norm_rope_fwd(ctypes.byref(_rope(**changes)), None, None) == INVALID
    assert lib.tokmix_qk_norm_rope_bwd(ctypes.byref(_rope(**changes)), ctypes.c_void_p(16), ctypes.c_void_p(16),
                                       ctypes.c_void_p(16), 1 << 40, None, None) == INVALID


@pytest.mark.gpu
@pytest.mark.parametrize("b,s", [(0, 5), (3, 0), (0, 0), (0, 500)])
@pytest.mark.parametrize("sections,interleaved", [(None, False), ((3, 3, 2), True), ((4, 4), False), ((8,), False)])
def test_empty_calls_with_positions(cuda_device, b, s, sections, interleaved):
    dev = cuda_device
    q, k = (torch.empty(b, s, h, 64, dtype=torch.bfloat16, device=dev) for h in (3, 1))
    w = torch.ones(64, device=dev)
    cos, sin = qk_norm_rope.rotary_tables(8, 8, device=dev)
    pos = torch.empty((b, s) if sections is None else (len(sections), b, s), dtype=torch.int32, device=dev)
    kw = dict(sections=sections, interleaved=interleaved)
    out = qk_norm_rope.kernel_fn(q, k, w, w, cos, sin, pos, **kw)
    assert out[0].shape == q.shape and out[1].shape == k.shape
    grads = qk_norm_rope_bwd.kernel_fn(q, k, q, k, w, w, cos, sin, pos, **kw)
    assert grads[0].shape == q.shape and grads[1].shape == k.shape
    assert all(g.shape == w.shape and g.eq(0).all() for g in grads[2:])
    leaves = [t.clone().requires_grad_() for t in (q, k, w, w)]
    y = training.qk_norm_rope(*leaves, cos, sin, pos, **kw)
    torch.autograd.backward(y, [torch.empty_like(t) for t in y])
    assert all(x.grad.shape == x.shape for x in leaves) and leaves[2].grad.eq(0).all()
    qk_norm_rope.check_device_status(dev)


@pytest.mark.gpu
@pytest.mark.parametrize("b,s", [(0, 5), (2, 0)])
@pytest.mark.parametrize("layout", ["bhsd", "bshd"])
def test_empty_attention_trains(cuda_device, b, s, layout):
    """No tokens through the attention's autograd entry."""
    shape = (lambda h: (b, h, s, 64)) if layout == "bhsd" else (lambda h: (b, s, h, 64))
    q, k, v = (torch.empty(shape(h), dtype=torch.bfloat16, device=cuda_device).requires_grad_() for h in (4, 2, 2))
    o = training.attention(q, k, v, layout=layout)
    o.backward(torch.empty_like(o))
    assert o.shape == q.shape and all(t.grad.shape == t.shape for t in (q, k, v))
