"""The serving step's kernels start while their predecessors drain: captured behind copies, fills and other streams' work, and
in graphs that share a pool, they still wait for all of it."""

import pytest
import torch

from kernel_opt_agent_b200 import add_rms_norm_quant as norm
from kernel_opt_agent_b200 import kv8_append as append
from kernel_opt_agent_b200 import kv8_attention as attention
from tests.test_kv8_gpu import E4M3, INT8, _i32

pytestmark = pytest.mark.gpu


def _step(dev, cache_dtype, seed, b=3, hq=8, hkv=2, d=128, page=16, room=256):
    """A step's state: pinned and device sources, what it copies them to, and the calls."""
    gen = torch.Generator().manual_seed(seed)
    n = -(-(100 + b) // page)
    cache = append.make_cache(b * n, hkv, page, d, cache_dtype, dev)
    table = torch.full((b, room), 0, dtype=torch.int32, device=dev)
    table[:, :n] = torch.randperm(b * n, generator=gen).view(b, n).int().to(dev)
    start = [99, 15, 48]
    old = [torch.randn(b, max(start), hkv, d, generator=gen).to(torch.bfloat16).to(dev) for _ in range(2)]
    append.kernel_fn(*old, *cache, table, _i32(start, dev), _i32(start, dev))
    src = torch.randn(4, b, 1, hq + 2 * hkv, d, generator=gen).to(torch.bfloat16)
    return dict(cache=cache, table=table, start=_i32(start, dev), seq=_i32(start, dev), src=src.to(dev), host=src.pin_memory(),
                qkv=torch.zeros(b, 1, hq + 2 * hkv, d, dtype=torch.bfloat16, device=dev), x=torch.zeros(b, 256, dtype=torch.bfloat16, device=dev),
                w=torch.ones(256, dtype=torch.bfloat16, device=dev), hq=hq, hkv=hkv)


def _run(s, i, side=None):
    """Copies (device to device, host to device), a fill and, on a side stream, the lengths; then the three operators."""
    main, hq, hkv = torch.cuda.current_stream(), s["hq"], s["hkv"]
    if side is not None:
        side.wait_stream(main)
    with torch.cuda.stream(side or main):
        s["seq"].copy_(s["start"])
        s["seq"].add_(1)
    s["qkv"].copy_(s["host"][i], non_blocking=True)
    if i % 2:
        s["qkv"].copy_(s["src"][i])
    s["x"].fill_(0.5 + i)
    y, scale, h = norm.kernel_fn(s["x"], None, s["w"])
    s["x"].copy_(s["qkv"].view(s["x"].shape[0], -1)[:, :256])
    if side is not None:
        main.wait_stream(side)
    append.kernel_fn(s["qkv"][:, :, hq:hq + hkv], s["qkv"][:, :, hq + hkv:], *s["cache"], s["table"], s["seq"])
    out, lse = attention.kernel_fn(s["qkv"][:, :, :hq], *s["cache"], s["table"], s["seq"], return_lse=True)
    y2, scale2, _ = norm.kernel_fn(s["x"], out.view(out.shape[0], -1)[:, :256].contiguous(), s["w"])
    s["qkv"].zero_()
    return [y.view(torch.uint8), scale, out, lse, y2.view(torch.uint8), scale2]


@pytest.mark.parametrize("room", [8, 256])
@pytest.mark.parametrize("cache_dtype", [E4M3, INT8])
def test_captured_behind_copies_and_other_streams(cuda_device, cache_dtype, room):
    dev = cuda_device
    s = _step(dev, cache_dtype, 5, room=room)
    want, side = [], torch.cuda.Stream()
    for i in range(4):
        got = _run(s, i)
        torch.cuda.synchronize()
        want.append([g.clone() for g in got])
    graphs = []
    for i in range(4):  # one pool: the graphs are replayed in any order, one after the other
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0][0].pool() if graphs else None):
            out = _run(s, i, side)
        graphs.append((g, out))
    for _ in range(20):
        for i in (2, 0, 3, 1, 1, 0):
            graphs[i][0].replay()
            got = [o.clone() for o in graphs[i][1]]
            assert all(torch.equal(a, b) for a, b in zip(got, want[i])), i
    append.check_device_status(dev)
