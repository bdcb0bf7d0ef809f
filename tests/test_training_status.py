"""An error that a kernel met is reported by the operator that met it, under its name, and by no other."""

import ctypes

import pytest
import torch

from kernel_opt_agent_b200 import _lib, flash_attention_2, flash_attention_2_bwd, kv8_append, kv8_attention, qk_norm_rope
from kernel_opt_agent_b200 import qk_norm_rope_bwd, training

OPERATORS = ("kv8", "qk_norm_rope", "flash_attention_2_bwd")


class Word:
    """A host tensor in the place of the pinned word."""

    def __init__(self):
        self.tensor = torch.zeros(1, dtype=torch.int32)
        self.ptr = self.tensor.data_ptr()
        self.word = ctypes.c_uint32.from_address(self.ptr)


@pytest.fixture
def words(monkeypatch):
    monkeypatch.setattr(_lib, "_HostStatus", Word)
    monkeypatch.setattr(_lib, "_host_status", {})
    monkeypatch.setattr(_lib, "_STATUS_MODE", "async")
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return monkeypatch


@pytest.mark.parametrize("owner", OPERATORS)
def test_each_operator_has_its_word(words, owner):
    dev = torch.device("cuda", 0)
    ptrs = {name: _lib.host_status_ptr(dev, name) for name in OPERATORS}
    assert len(set(ptrs.values())) == len(OPERATORS) and _lib.host_status_ptr(torch.device("cuda", 1), owner) not in ptrs.values()
    ctypes.c_uint32.from_address(ptrs[owner]).value = 8
    for name in OPERATORS:
        if name != owner:  # neither raised there nor cleared
            assert _lib.host_status_ptr(dev, name) == ptrs[name]
            _lib.take_host_status(dev, name)
    with pytest.raises(_lib.TokmixDeviceError, match=f"^{owner}: "):
        _lib.host_status_ptr(dev, owner)
    assert _lib.host_status_ptr(dev, owner) == ptrs[owner]


def test_a_first_call_inside_a_capture_gets_its_word(words):
    """The words of a device are allocated by the first call of any operator on it."""
    dev = torch.device("cuda", 0)
    words.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    assert _lib.host_status_ptr(dev, "kv8") is None
    words.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    assert _lib.host_status_ptr(dev, "kv8") is not None
    words.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    for name in OPERATORS:
        assert _lib.host_status_ptr(dev, name) is not None
    assert _lib.host_status_ptr(torch.device("cuda", 1), "kv8") is None


@pytest.mark.gpu
def test_a_training_step_names_the_operator(cuda_device):
    """Positions outside the tables in a layer that is trained: the attention and its gradient say nothing."""
    dev = cuda_device
    q = torch.randn(1, 40, 4, 64, device=dev).to(torch.bfloat16).requires_grad_()
    w = torch.ones(64, device=dev)
    cos, sin = qk_norm_rope.rotary_tables(40, 32, device=dev)
    bad = torch.full((1, 40), 40, dtype=torch.int32, device=dev)
    qk_norm_rope.check_device_status(dev)
    with torch.no_grad():
        x, y = training.qk_norm_rope(q, q, w, w, cos, sin, bad)
    torch.cuda.synchronize()
    o, lse = flash_attention_2.kernel_fn(x, y, y, layout="bshd", return_lse=True)
    flash_attention_2_bwd.kernel_fn(o, x, y, y, o, lse, layout="bshd")
    flash_attention_2_bwd.check_device_status(dev)
    kv8_append.check_device_status(dev)
    with pytest.raises(_lib.TokmixDeviceError, match="^qk_norm_rope: "):
        qk_norm_rope.check_device_status(dev)
    qk_norm_rope.check_device_status(dev)
    # the gradient's own, raised by the next call of the forward
    qk_norm_rope_bwd.kernel_fn(q.detach(), q.detach(), q.detach(), q.detach(), w, w, cos, sin, bad)
    torch.cuda.synchronize()
    flash_attention_2_bwd.kernel_fn(o, x, y, y, o, lse, layout="bshd")
    with pytest.raises(_lib.TokmixDeviceError, match="^qk_norm_rope: "):
        qk_norm_rope.kernel_fn(q.detach(), q.detach(), w, w, cos, sin)
    qk_norm_rope.kernel_fn(q.detach(), q.detach(), w, w, cos, sin)
    qk_norm_rope.check_device_status(dev)


@pytest.mark.gpu
def test_the_caches_errors_stay_its_own(cuda_device):
    dev = cuda_device
    cache = kv8_append.make_cache(2, 1, 16, 64, device=dev)
    x = torch.ones(1, 1, 1, 64, dtype=torch.bfloat16, device=dev)
    bad, seq = (torch.tensor(v, dtype=torch.int32, device=dev) for v in ([[7, 0]], [1]))
    kv8_append.kernel_fn(x, x, *cache, bad, seq)
    torch.cuda.synchronize()
    w = torch.ones(64, device=dev)
    qk_norm_rope.kernel_fn(x, x, w, w, *qk_norm_rope.rotary_tables(4, 8, device=dev))
    qk_norm_rope.check_device_status(dev)
    flash_attention_2_bwd.check_device_status(dev)
    with pytest.raises(_lib.TokmixDeviceError, match="^kv8: "):
        kv8_attention.check_device_status(dev)
    kv8_append.check_device_status(dev)
