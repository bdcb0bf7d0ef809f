"""Status words of the 8-bit cache's calls: when they are looked at, and what they keep."""

import ctypes

import pytest
import torch

from kernel_opt_agent_b200 import _lib
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
