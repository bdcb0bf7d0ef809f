"""The training operators as a layer uses them: norm and rotation, attention, and back, through autograd and captured."""

import pytest
import torch

from kernel_opt_agent_b200 import flash_attention_2 as fa2
from kernel_opt_agent_b200 import flash_attention_2_bwd as fa2_bwd
from kernel_opt_agent_b200 import kv8_append, kv8_attention, qk_norm_rope, qk_norm_rope_bwd, training

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def layer_inputs(b=2, s=300, hq=8, hkv=2, d=128, seed=0):
    gen = torch.Generator().manual_seed(seed)
    qkv = torch.randn(b, s, hq + 2 * hkv, d, generator=gen).to(BF16).cuda()
    w = [(1 + 0.2 * torch.randn(d, generator=gen)).cuda() for _ in range(2)]
    cos, sin = qk_norm_rope.rotary_tables(s + 50, d // 4)
    pos = torch.stack([torch.arange(s) + torch.randint(0, 50, (b, 1), generator=gen) for _ in range(3)]).int().cuda()
    do = (torch.randn(b, s, hq, d, generator=gen) / 16).to(BF16).cuda()
    return qkv, w, cos, sin, pos, do


def layer(qkv, qw, kw, cos, sin, pos, hq, hkv, d):
    q, k = training.qk_norm_rope(qkv[:, :, :hq], qkv[:, :, hq:hq + hkv], qw, kw, cos, sin, pos, nope_dim=0,
                                 sections=(d // 4 - 2 * (d // 12), d // 12, d // 12), interleaved=True)
    return training.attention(q, k, qkv[:, :, hq + hkv:], causal=True, layout="bshd")


def exact_layer(qkv, qw, kw, cos, sin, pos, hq, hkv, d):
    """The layer in 64 bits, with the roundings of the tensors between the operators."""
    half, third = d // 4, d // 12
    axis = torch.tensor([j % 3 if j < 3 * (half - 2 * third, third, third)[j % 3] else 0 for j in range(half)], device=qkv.device)
    rows = pos.long()[axis].permute(1, 2, 0)
    pair = torch.arange(half, device=qkv.device)
    c, s = (t.double()[rows, pair][:, :, None] for t in (cos, sin))

    def norm_rope(x, w):
        n = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
        a, b = n[..., :half], n[..., half:2 * half]
        return torch.cat((a * c - b * s, a * s + b * c, n[..., 2 * half:]), -1)

    q, k, v = norm_rope(qkv[:, :, :hq], qw), norm_rope(qkv[:, :, hq:hq + hkv], kw), qkv[:, :, hq + hkv:]
    q, k, v = (t.transpose(1, 2) for t in (q, k, v))
    g = hq // hkv
    x = q @ k.repeat_interleave(g, 1).transpose(2, 3) * d ** -0.5
    x = x.masked_fill(~torch.ones(x.shape[2:], dtype=torch.bool, device=x.device).tril(), float("-inf"))
    return (torch.softmax(x, -1) @ v.repeat_interleave(g, 1)).transpose(1, 2)


@pytest.mark.parametrize("d,hq,hkv", [(64, 4, 4), (128, 8, 2), (256, 8, 1)])
def test_layer_gradients(cuda_device, d, hq, hkv):
    """Gradients of the whole layer against 64 bits.  q, k, o, P, dS and every gradient between the operators are rounded to
    bf16, each off by at most 2^-8 of itself and independently of each other.  A score is a sum of d terms whose root square sum
    is about 1 (q and k are normalised), each off by 2^-7 of itself at most, so it is off by about 2^-8 and P by as much of
    itself.  In the 2-norm over a gradient the ten roundings on the way of any value add up to less than 10 * 2^-8 of it (they
    would, if all pulled one way)."""
    qkv, w, cos, sin, pos, do = layer_inputs(hq=hq, hkv=hkv, d=d, seed=d)
    leaves = [t.clone().requires_grad_() for t in (qkv, *w)]
    out = layer(*leaves, cos, sin, pos, hq, hkv, d)
    out.backward(do)
    exact = [t.double().requires_grad_() for t in (qkv, *w)]
    ref = exact_layer(*exact, cos, sin, pos, hq, hkv, d)
    ref.backward(do.double())
    assert ((out.double() - ref).norm() / ref.norm()).item() <= 4 * 2.0 ** -8  # q, k, P and the output itself
    for x, y in zip(leaves, exact):
        assert x.grad.dtype == x.dtype and x.grad.shape == x.shape
        assert ((x.grad.double() - y.grad).norm() / y.grad.norm()).item() <= 10 * 2.0 ** -8
    fa2_bwd.check_device_status(cuda_device)
    qk_norm_rope.check_device_status(cuda_device)


def test_autograd_attention_is_the_modules(cuda_device):
    qkv, w, cos, sin, pos, do = layer_inputs(seed=3)
    q, k, v = (t.contiguous() for t in (qkv[:, :, :8], qkv[:, :, 8:10], qkv[:, :, 10:]))
    o, lse = fa2.kernel_fn(q, k, v, layout="bshd", return_lse=True)
    want = fa2_bwd.kernel_fn(do, q, k, v, o, lse, layout="bshd")
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = training.attention(*leaves, layout="bshd")
    assert torch.equal(out, o)
    out.backward(do)
    assert all(torch.equal(x.grad, g) for x, g in zip(leaves, want))
    # frozen keys, heads first (a transposed view), gradient of a sum (expanded)
    q2 = q.clone().requires_grad_()
    training.attention(q2.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2)).sum().backward()
    one = torch.ones_like(o)
    assert torch.equal(q2.grad, fa2_bwd.kernel_fn(one, q, k, v, o, lse, layout="bshd")[0])
    with torch.no_grad():
        assert not training.attention(*leaves, layout="bshd").requires_grad


def test_second_order_is_refused(cuda_device):
    qkv, *_ = layer_inputs(s=20)
    q = qkv[:, :, :8].clone().requires_grad_()
    out = training.attention(q, qkv[:, :, 8:10], qkv[:, :, 10:], layout="bshd")
    (g,) = torch.autograd.grad(out.float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_captured_training_step(cuda_device):
    """The four kernels' calls captured together, replayed on changed inputs."""
    def step(qkv, w, cos, sin, pos, do):
        kw = dict(nope_dim=0)
        q, k = qk_norm_rope.kernel_fn(qkv[:, :, :8], qkv[:, :, 8:10], *w, cos, sin, pos[0], **kw)
        v = qkv[:, :, 10:]
        o, lse = fa2.kernel_fn(q, k, v, layout="bshd", return_lse=True)
        dq, dk, dv = fa2_bwd.kernel_fn(do, q, k, v, o, lse, layout="bshd")
        return [o, dv, *qk_norm_rope_bwd.kernel_fn(dq, dk, qkv[:, :, :8], qkv[:, :, 8:10], *w, cos, sin, pos[0], **kw)]

    states = [layer_inputs(seed=i) for i in range(3)]
    want = [step(*s) for s in states]
    held = layer_inputs(seed=0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*held)
    for s, ref in zip(states, want):
        for a, b in zip((held[0], *held[1], *held[2:]), (s[0], *s[1], *s[2:])):
            a.copy_(b)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(outs, ref))


def test_captured_autograd_step(cuda_device):
    """A step whose autograd graph is built inside the capture, on leaves that no other graph holds."""
    qkv, w, cos, sin, pos, do = layer_inputs(seed=1)
    leaves = [t.clone().requires_grad_() for t in (qkv, *w)]
    layer(*leaves, cos, sin, pos, 8, 2, 128).backward(do)
    want = [x.grad.clone() for x in leaves]
    leaves = [t.clone().requires_grad_() for t in (qkv, *w)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = torch.autograd.grad(layer(*leaves, cos, sin, pos, 8, 2, 128), leaves, do)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(grads, want))


def test_decode_step_with_norm_and_rotation(cuda_device):
    """One new token per sequence: norm and rotation at its position, into the 8-bit cache, attention over it.  Against the same
    step with the norm and rotation in 64 bits: both round q and k to bf16 once (2^-8), the cache to e4m3 (2^-4), the same
    values but where a bf16 rounding falls on the other side."""
    b, hq, hkv, d, page = 3, 8, 2, 128, 16
    gen = torch.Generator().manual_seed(4)
    lens = torch.tensor([37, 1, 64], dtype=torch.int32).cuda()
    qkv = torch.randn(b, 1, hq + 2 * hkv, d, generator=gen).to(BF16).cuda()
    w = [(1 + 0.2 * torch.randn(d, generator=gen)).to(BF16).cuda() for _ in range(2)]
    cos, sin = qk_norm_rope.rotary_tables(128, 32)
    table = torch.arange(b * 5, dtype=torch.int32).view(b, 5).cuda()
    old = torch.randn(b, 64, hkv, d, generator=gen).to(BF16).cuda()
    pos = (lens - 1).view(b, 1)
    outs = []
    q, k = qk_norm_rope.kernel_fn(qkv[:, :, :hq], qkv[:, :, hq:hq + hkv], *w, cos, sin, pos)
    x = [t.double() / (t.double().square().mean(-1, keepdim=True) + 1e-6).sqrt() * u.double()
         for t, u in ((qkv[:, :, :hq], w[0]), (qkv[:, :, hq:hq + hkv], w[1]))]
    c, s = (t.double()[pos.long()][:, :, None] for t in (cos, sin))
    x = [torch.cat((n[..., :64], n[..., 64:96] * c - n[..., 96:] * s, n[..., 64:96] * s + n[..., 96:] * c), -1).to(BF16) for n in x]
    for qq, kk in ((q, k), x):
        cache = kv8_append.make_cache(b * 5, hkv, page, d)
        kv8_append.kernel_fn(old, old, *cache, table, lens - 1, lens - 1)
        kv8_append.kernel_fn(kk, qkv[:, :, hq + hkv:], *cache, table, lens)
        outs.append(kv8_attention.kernel_fn(qq, *cache, table, lens).float())
    kv8_append.check_device_status(cuda_device)
    # q off by 2^-7 of itself at most, one key of the sequence by a step of e4m3 besides: the scores move by a few
    # hundredths, the output by as much of the values' spread
    assert (outs[0] - outs[1]).abs().max().item() <= 0.1
    assert (outs[0] - outs[1]).norm().item() <= 2.0 ** -6 * outs[1].norm().item()
