"""The attention's gradients on a B200 against the formula in 64 bits.

Tolerances.  Operands are bf16; P and dS are rounded to bf16 once more (at most half a step, 2^-8 of
the value), products are accumulated in fp32 and the results rounded to bf16 (2^-8 of the value).  An
output is a sum of terms t_i, each off by at most 2^-8 |t_i| (its P or dS rounding), so it is off by at most
2^-8 sum |t_i| plus its own rounding: the test compares against that bound, formed in 64 bits from the
absolute values.  dS is P (dP - delta), where dP and delta carry fp32 errors of at most (d + 8) 2^-24 of
their absolute sums, which the bound adds, as it does P's: the exponent c s - lse in fp32 is off by a few
2^-24 of its parts and of the absolute sum behind s.
"""

import math
import threading

import pytest
import torch

from kernel_opt_agent_b200 import flash_attention_2 as fa2
from kernel_opt_agent_b200 import flash_attention_2_bwd as bwd

pytestmark = pytest.mark.gpu


def formula(do, q, k, v, o, lse, causal, sm_scale, layout):
    """(dq, dk, dv) and bounds of their errors, float64, in the inputs' layout."""
    if layout == "bshd":
        do, q, k, v, o = (t.transpose(1, 2) for t in (do, q, k, v, o))
    do, q, k, v, o, lse = (t.double() for t in (do, q, k, v, o, lse))
    g = q.shape[1] // k.shape[1]
    kx, vx = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    s = q @ kx.transpose(2, 3) * sm_scale
    seen = torch.ones(s.shape[2:], dtype=torch.bool, device=s.device)
    if causal:
        seen = seen.tril()
    p = torch.where(seen, torch.exp(s - lse[..., None]), 0.0)
    dp = do @ vx.transpose(2, 3)
    delta = (do * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    d = q.shape[-1]
    # relative error of P before its rounding: the exponent's, in fp32
    s_abs = (q.abs() @ kx.abs().transpose(2, 3)) * sm_scale
    rel_p = (s_abs + s.abs() + lse.abs()[..., None]) * (d / 16 + 8) * 2.0 ** -24 + 2.0 ** -21
    dp_err = ((do.abs() @ vx.abs().transpose(2, 3)) + (do.abs() * o.abs()).sum(-1, keepdim=True)) * (d + 8) * 2.0 ** -24
    p_err = p * (rel_p + 2.0 ** -8)
    ds_err = ds.abs() * (rel_p + 2.0 ** -8) + p * dp_err

    def shared(x):
        return x.unflatten(1, (-1, g)).sum(2)

    n = p.shape[-1] + p.shape[-2] * g  # terms of the longest fp32 sums
    acc = n * 2.0 ** -24
    dv, dv_b = shared(p.transpose(2, 3) @ do), shared((p_err + acc * p).transpose(2, 3) @ do.abs())
    dk, dk_b = shared(ds.transpose(2, 3) @ q) * sm_scale, shared((ds_err + acc * ds.abs()).transpose(2, 3) @ q.abs()) * sm_scale
    dq, dq_b = ds @ kx * sm_scale, (ds_err + acc * ds.abs()) @ kx.abs() * sm_scale
    outs = []
    for x, b in ((dq, dq_b), (dk, dk_b), (dv, dv_b)):
        b = b + x.abs() * 2.0 ** -8 + 2.0 ** -133
        outs.append((x, b) if layout == "bhsd" else (x.transpose(1, 2), b.transpose(1, 2)))
    return outs


def make(b, hq, hkv, sq, skv, d, layout, seed=0, q_scale=1.0):
    gen = torch.Generator().manual_seed(seed)

    def t(h, s):
        return torch.randn((b, h, s, d) if layout == "bhsd" else (b, s, h, d), generator=gen)

    q, k, v, do = t(hq, sq) * q_scale, t(hkv, skv), t(hkv, skv), t(hq, sq)
    return [x.to(torch.bfloat16).cuda() for x in (q, k, v, do)]


def check(b, hq, hkv, sq, skv, d, causal, layout, seed=0, scale=None, q_scale=1.0):
    q, k, v, do = make(b, hq, hkv, sq, skv, d, layout, seed, q_scale)
    scale = d ** -0.5 if scale is None else scale
    o, lse = fa2.kernel_fn(q, k, v, causal, scale, layout=layout, return_lse=True)
    got = bwd.kernel_fn(do, q, k, v, o, lse, causal, scale, layout=layout)
    bwd.check_device_status(q.device)
    worst = []
    for name, x, (ref, bound) in zip(("dq", "dk", "dv"), got, formula(do, q, k, v, o, lse, causal, scale, layout)):
        assert x.shape == ref.shape and x.dtype == torch.bfloat16 and x.is_contiguous()
        used = ((x.double() - ref).abs() / bound).max().item()
        worst.append((name, used))
    assert all(w <= 1.0 for _, w in worst), worst


CASES = [
    # b, hq, hkv, sq, skv, d, causal, layout
    (1, 1, 1, 128, 128, 128, False, "bhsd"),
    (1, 1, 1, 128, 128, 128, True, "bhsd"),
    (1, 1, 1, 256, 256, 128, True, "bhsd"),
    (1, 1, 1, 64, 64, 256, True, "bhsd"),
    (1, 1, 1, 128, 128, 64, True, "bhsd"),
    (1, 2, 2, 1, 1, 128, True, "bhsd"),
    (1, 2, 1, 1, 1, 256, True, "bshd"),
    (1, 2, 2, 1, 1, 64, False, "bshd"),
    (1, 4, 2, 129, 129, 128, True, "bhsd"),
    (2, 4, 4, 257, 257, 128, True, "bhsd"),
    (1, 4, 2, 200, 200, 64, True, "bshd"),
    (1, 2, 1, 100, 100, 128, False, "bhsd"),
    (1, 8, 8, 512, 512, 64, True, "bshd"),
    (1, 4, 4, 1031, 1031, 128, True, "bhsd"),
    (2, 6, 3, 300, 300, 128, True, "bshd"),
    (1, 3, 1, 256, 256, 128, True, "bhsd"),
    (1, 10, 2, 333, 333, 64, False, "bhsd"),
    (3, 4, 1, 333, 333, 256, True, "bhsd"),
    (2, 8, 1, 200, 200, 256, True, "bshd"),
    (1, 2, 2, 65, 65, 256, False, "bhsd"),
    (1, 2, 2, 70, 500, 128, False, "bhsd"),    # more keys than queries
    (1, 2, 2, 500, 70, 128, False, "bshd"),    # more queries than keys
    (1, 2, 2, 70, 500, 128, True, "bhsd"),     # keys that no query sees
    (1, 2, 1, 500, 70, 64, True, "bhsd"),      # causal, queries behind the last key
    (1, 2, 1, 500, 70, 256, True, "bshd"),
    (1, 2, 1, 70, 500, 256, True, "bshd"),
    (1, 1, 1, 1, 1000, 128, False, "bhsd"),    # one query
    (1, 1, 1, 1000, 1, 64, False, "bhsd"),     # one key
]


@pytest.mark.parametrize("b,hq,hkv,sq,skv,d,causal,layout", CASES)
def test_gradients_match_the_formula(cuda_device, b, hq, hkv, sq, skv, d, causal, layout):
    check(b, hq, hkv, sq, skv, d, causal, layout, seed=sq + skv + hq)


@pytest.mark.parametrize("d,group", [(64, 3), (128, 4), (256, 8)])
def test_many_tiles_and_waves(cuda_device, d, group):
    """More units than SMs: every CTA takes several, rows of several waves."""
    check(3, 4 * group, 4, 1700, 1700, d, True, "bhsd", seed=d)


@pytest.mark.parametrize("b,hq,hkv,sq,skv,d,causal", [
    (1, 8, 1, 2048, 2048, 64, True), (1, 4, 2, 1500, 1100, 128, False), (1, 8, 1, 1024, 1024, 256, True),
    (1, 1, 1, 4096, 512, 64, False), (1, 2, 1, 2000, 130, 128, True), (1, 3, 3, 1100, 2500, 128, True), (2, 2, 1, 700, 700, 256, False)])
def test_few_key_tiles(cuda_device, b, hq, hkv, sq, skv, d, causal):
    """Too few key tiles to fill the GPU: they come in parts that are joined, and dQ in several sums.  The same bits beside
    other work on the GPU, which changes the order in which the CTAs get on."""
    check(b, hq, hkv, sq, skv, d, causal, "bhsd", seed=sq)
    q, k, v, do = make(b, hq, hkv, sq, skv, d, "bhsd", seed=sq)
    o, lse = fa2.kernel_fn(q, k, v, causal, return_lse=True)
    want = bwd.kernel_fn(do, q, k, v, o, lse, causal)
    side, x = torch.cuda.Stream(), torch.randn(2048, 2048, device="cuda")
    torch.cuda.synchronize()
    for _ in range(4):
        with torch.cuda.stream(side):
            x @ x
        got = bwd.kernel_fn(do, q, k, v, o, lse, causal)
        assert all(torch.equal(a, c) for a, c in zip(got, want))
    torch.cuda.synchronize()


def test_custom_scale_and_sharp_rows(cuda_device):
    check(1, 4, 2, 300, 300, 128, True, "bhsd", seed=3, scale=0.3)
    check(1, 2, 1, 300, 333, 64, False, "bshd", seed=4, q_scale=6.0)   # weights of nearly one key
    check(1, 2, 1, 200, 200, 256, True, "bshd", seed=5, q_scale=0.01)  # nearly flat


def test_gradient_against_differences(cuda_device):
    """The formula that the kernel is tested against is the forward's derivative (float64, central differences)."""
    q, k, v, do = (t.double() for t in make(1, 2, 1, 9, 9, 64, "bhsd", seed=1))

    def forward(q, k, v):
        s = q @ k.repeat_interleave(2, 1).transpose(2, 3) * 0.1
        s = s.masked_fill(~torch.ones(9, 9, dtype=torch.bool, device=s.device).tril(), -math.inf)
        return torch.softmax(s, -1) @ v.repeat_interleave(2, 1), torch.logsumexp(s, -1)

    o, lse = forward(q, k, v)
    grads = [x for x, _ in formula(do, q, k, v, o, lse, True, 0.1, "bhsd")]
    h = 2.0 ** -14
    for n, at in [(0, (0, 0, 0, 0)), (0, (0, 1, 8, 63)), (1, (0, 0, 0, 5)), (1, (0, 0, 8, 1)), (2, (0, 0, 3, 7))]:
        args = [q, k, v]
        step = torch.zeros_like(args[n])
        step[at] = h
        up, down = ([a + f * step if i == n else a for i, a in enumerate(args)] for f in (1, -1))
        diff = ((forward(*up)[0] - forward(*down)[0]) * do).sum() / (2 * h)
        assert abs(diff - grads[n][at]).item() < 1e-6


@pytest.mark.parametrize("d,s,hq,hkv,causal,layout", [(64, 200, 4, 2, True, "bshd"), (128, 333, 2, 2, False, "bhsd"),
                                                      (128, 1, 2, 1, True, "bhsd"), (256, 130, 4, 1, True, "bhsd"),
                                                      (128, 300, 3, 1, True, "bhsd")])
def test_forward_lse(cuda_device, d, s, hq, hkv, causal, layout):
    """lse against 64 bits: the exponents are fp32 (their parts' 2^-24, d / 16 + 8 roundings), each exponential and sum adds
    at most (s + 8) 2^-23; the output is the one of the call without lse."""
    q, k, v, _ = make(2, hq, hkv, s, s, d, layout, seed=s)
    o, lse = fa2.kernel_fn(q, k, v, causal, layout=layout, return_lse=True)
    assert lse.shape == (2, hq, s) and lse.dtype == torch.float32
    assert torch.equal(o, fa2.kernel_fn(q, k, v, causal, layout=layout))
    if layout == "bshd":
        q, k = q.transpose(1, 2), k.transpose(1, 2)
    kx = k.double().repeat_interleave(hq // hkv, 1).transpose(2, 3)
    x = q.double() @ kx * d ** -0.5
    size = (q.double().abs() @ kx.abs() * d ** -0.5).amax(-1)
    if causal:
        x = x.masked_fill(~torch.ones(s, s, dtype=torch.bool, device=x.device).tril(), -math.inf)
    ref = torch.logsumexp(x, -1)
    assert ((lse.double() - ref).abs() <= (size + ref.abs()) * (d / 16 + 8) * 2.0 ** -24 + (s + 8) * 2.0 ** -23).all()


def test_same_bits_every_time(cuda_device):
    for b, hq, hkv, s, d, causal in [(2, 8, 2, 1500, 128, True), (1, 8, 8, 1000, 64, False), (1, 8, 2, 700, 256, True)]:
        q, k, v, do = make(b, hq, hkv, s, s, d, "bhsd", seed=d)
        o, lse = fa2.kernel_fn(q, k, v, causal, return_lse=True)
        first = bwd.kernel_fn(do, q, k, v, o, lse, causal)
        for _ in range(4):
            assert all(torch.equal(x, y) for x, y in zip(first, bwd.kernel_fn(do, q, k, v, o, lse, causal)))


def test_heads_that_share_keys_are_summed(cuda_device):
    """dk and dv of a shared key head are those of the heads apart, added; dq is each head's own."""
    q, k, v, do = make(1, 4, 1, 260, 260, 128, "bhsd", seed=2)
    kx, vx = k.expand(1, 4, 260, 128).contiguous(), v.expand(1, 4, 260, 128).contiguous()
    o, lse = fa2.kernel_fn(q, k, v, return_lse=True)
    dq, dk, dv = bwd.kernel_fn(do, q, k, v, o, lse)
    dq4, dk4, dv4 = bwd.kernel_fn(do, q, kx, vx, o, lse)
    assert torch.equal(dq, dq4)
    for a, b in ((dk, dk4), (dv, dv4)):
        b = b.double()
        # four values rounded to bf16 and their sum rounded once; and the fp32 sums' order
        assert ((a.double() - b.sum(1, keepdim=True)).abs() <= 2.0 ** -8 * (b.abs().sum(1, keepdim=True) + a.double().abs())
                + 2.0 ** -16 * b.abs().sum(1, keepdim=True) + 2.0 ** -12).all()


@pytest.mark.parametrize("sq,skv,b", [(0, 5, 2), (5, 5, 0), (0, 0, 1)])
def test_empty(cuda_device, sq, skv, b):
    q, k, v, do = make(b, 4, 2, sq, skv, 64, "bhsd")
    dq, dk, dv = bwd.kernel_fn(do, q, k, v, q.clone(), torch.zeros(b, 4, sq, device=q.device))
    assert dq.shape == q.shape and dk.shape == k.shape and dk.eq(0).all() and dv.eq(0).all()


def test_refusals(cuda_device):
    q, k, v, do = make(1, 4, 2, 20, 20, 64, "bhsd")
    o, lse = fa2.kernel_fn(q, k, v, return_lse=True)
    ok = dict(do=do, q=q, k=k, v=v, o=o, lse=lse)
    for bad in (dict(do=do[:, :2]), dict(do=do.float()), dict(o=o[:, :, :3]), dict(lse=lse[..., :3]), dict(lse=lse.double()),
                dict(lse=lse.cpu()), dict(do=do.cpu()), dict(sm_scale=-1.0), dict(sm_scale=float("nan")),
                dict(k=k[:, :, :0], v=v[:, :, :0]), dict(layout="bshd")):
        with pytest.raises(ValueError):
            bwd.kernel_fn(**{**ok, **bad})


def test_views_and_expanded_gradients(cuda_device):
    q, k, v, do = make(2, 4, 2, 150, 150, 128, "bhsd", seed=7)
    o, lse = fa2.kernel_fn(q, k, v, return_lse=True)
    want = bwd.kernel_fn(do, q, k, v, o, lse)
    t = lambda x: x.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    odd = torch.zeros(do.numel() + 1, dtype=do.dtype, device=do.device)[1:].view(do.shape).copy_(do)
    for args in ((t(do), t(q), t(k), t(v), t(o), lse), (odd, q, k, v, o, lse), (do, q, k, v, o, lse.double().float())):
        assert all(torch.equal(a, b) for a, b in zip(bwd.kernel_fn(*args), want))
    one = torch.ones((), dtype=do.dtype, device=do.device).expand(do.shape)
    assert all(torch.equal(a, b) for a, b in zip(bwd.kernel_fn(one, q, k, v, o, lse), bwd.kernel_fn(one.contiguous(), q, k, v, o, lse)))


def test_calls_on_two_streams_and_in_graphs(cuda_device):
    """Two calls at once, and two graphs replayed at once: neither shares the other's sums."""
    cases = [make(2, 8, 2, 900, 900, 128, "bhsd", seed=1), make(2, 8, 2, 900, 900, 128, "bhsd", seed=2)]
    states = []
    for q, k, v, do in cases:
        states.append((do, q, k, v, *fa2.kernel_fn(q, k, v, return_lse=True)))
    want = [bwd.kernel_fn(*s) for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    for _ in range(3):
        got = []
        for s, st in zip(states, streams):
            with torch.cuda.stream(st):
                got.append([bwd.kernel_fn(*s) for _ in range(3)])
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(a, b) for r in g for a, b in zip(r, w))
    graphs, outs = [], []
    held = [tuple(t.clone() for t in s) for s in states]
    for s in held:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(bwd.kernel_fn(*s))
        graphs.append(g)
    for pick in ((0, 1), (1, 0)):
        for h, i in zip(held, pick):
            for a, b in zip(h, states[i]):
                a.copy_(b)
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for o, i in zip(outs, pick):
            assert all(torch.equal(a, b) for a, b in zip(o, want[i]))


def test_first_call_of_a_thread(cuda_device):
    """A thread that has made no CUDA call yet, as autograd's may be when all its memory comes from the allocator's cache."""
    q, k, v, do = make(1, 4, 2, 300, 300, 128, "bhsd", seed=12)

    def both():
        o, lse = fa2.kernel_fn(q, k, v, True, return_lse=True)
        return (o, *bwd.kernel_fn(do, q, k, v, o, lse, True))

    want = both()
    both()  # leaves its blocks in the cache
    got = []

    def run():
        try:
            got.extend(both())
        except Exception as e:  # shown by the assertions
            got.append(e)

    thread = threading.Thread(target=run)
    thread.start()
    thread.join()
    assert len(got) == 4, got
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_masked_infinities_stay_out(cuda_device):
    """A value row of infinities that no query up to some row sees: those rows' dq are what they were."""
    q, k, v, do = make(1, 1, 1, 256, 256, 128, "bhsd", seed=9)
    o, lse = fa2.kernel_fn(q, k, v, return_lse=True)
    want = bwd.kernel_fn(do, q, k, v, o, lse)
    v2 = v.clone()
    v2[0, 0, 200] = float("inf")
    got = bwd.kernel_fn(do, q, k, v2, o, lse)
    assert torch.equal(got[0][0, 0, :200], want[0][0, 0, :200])   # dS is replaced, not multiplied, where masked
    assert not torch.isfinite(got[0][0, 0, 200:].float()).all()
