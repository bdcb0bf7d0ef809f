"""Status words of the 8-bit cache's calls: when they are looked at, and what they keep."""

import ctypes

import pytest
import torch

from kernel_opt_agent_b200 import _kv8, _lib
from kernel_opt_agent_b200 import kv8_append as append
from kernel_opt_agent_b200 import kv8_attention as attention


def _i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def test_without_checks_the_word_is_passed_but_not_looked_at(monkeypatch):
    """TOKMIX_CHECK_STATUS=0: launches still get the word's address, so that an explicit look finds what they stored; they
    do not raise for it themselves.  (A host tensor stands for the pinned word.)"""

    class Word:
        def __init__(self):
            self.tensor = torch.zeros(1, dtype=torch.int32)
            self.ptr = self.tensor.data_ptr()
            self.word = ctypes.c_uint32.from_address(self.ptr)

    monkeypatch.setattr(_lib, "_HostStatus", Word)
    monkeypatch.setattr(_lib, "_host_status", {})
    monkeypatch.setattr(_lib, "_STATUS_MODE", "off")
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    dev = torch.device("cuda", 0)
    ptr = _lib.host_status_ptr(dev, "kv8")
    assert ptr is not None
    ctypes.c_uint32.from_address(ptr).value = 8
    assert _lib.host_status_ptr(dev, "kv8") == ptr
    with pytest.raises(_lib.TokmixDeviceError, match="argument"):
        _lib.take_host_status(dev, "kv8")
    _lib.take_host_status(dev, "kv8")
    ctypes.c_uint32.from_address(ptr).value = 8
    monkeypatch.setattr(_lib, "_STATUS_MODE", "async")
    with pytest.raises(_lib.TokmixDeviceError):
        _lib.host_status_ptr(dev, "kv8")
    assert _lib.host_status_ptr(dev, "kv8") == ptr


@pytest.mark.gpu
def test_an_explicit_look_finds_errors_without_checks(cuda_device, monkeypatch):
    dev = cuda_device
    append.check_device_status(dev)
    monkeypatch.setattr(_lib, "_STATUS_MODE", "off")
    cache = append.make_cache(2, 1, 16, 64, device=dev)
    x = torch.ones(1, 1, 1, 64, dtype=torch.bfloat16, device=dev)
    bad, seq = _i32([[7, 0]], dev), _i32([1], dev)
    for call in (lambda: append.kernel_fn(x, x, *cache, bad, seq), lambda: attention.kernel_fn(x, *cache, bad, seq)):
        call()
        call()  # does not look
        with pytest.raises(_lib.TokmixDeviceError, match="argument"):
            append.check_device_status(dev)
        append.check_device_status(dev)


@pytest.mark.gpu
@pytest.mark.parametrize("before", [0, 0x1, 0x6])
def test_a_status_word_keeps_its_other_bits(cuda_device, before):
    """One device word for several kinds of call: a bad table entry adds its bit to those that are there."""
    dev, lib = cuda_device, _lib.load()
    cache = append.make_cache(2, 1, 16, 64, device=dev)
    x, out = torch.ones(1, 1, 1, 64, dtype=torch.bfloat16, device=dev), torch.empty(1, 1, 1, 64, dtype=torch.bfloat16, device=dev)
    ws = torch.empty(lib.tokmix_kv8_attention_workspace_bytes(1, 1, 1, 64), dtype=torch.uint8, device=dev)
    seq = _i32([1], dev)  # (the description holds addresses only)
    for table, want in ((_i32([[7, 0]], dev), before | 8), (_i32([[1, 0]], dev), before)):
        desc = _kv8.cache_args(x, *cache, table, seq, None)
        st, stream = x.stride()[:3], _lib.stream_ptr(dev)
        for call in (lambda w: lib.tokmix_kv8_append(x.data_ptr(), *st, x.data_ptr(), *st, 1, 0, _kv8.byref(desc), w, stream),
                     lambda w: lib.tokmix_kv8_attention(x.data_ptr(), *st, out.data_ptr(), None, 1, 1, 0, 0.125, _kv8.byref(desc),
                                                        ws.data_ptr(), ws.numel(), w, stream)):
            word = torch.tensor([before], dtype=torch.int32, device=dev)
            assert call(word.data_ptr()) == 0
            assert int(word) == want
