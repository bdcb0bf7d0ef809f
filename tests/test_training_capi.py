"""The training operators' C entry points and plugin modules refuse bad arguments without touching a GPU (CPU only)."""

import ctypes
import math

import pytest
import torch

from kernel_opt_agent_b200 import _lib, flash_attention_2_bwd, qk_norm_rope, qk_norm_rope_bwd

P = ctypes.c_void_p(16)
ODD = ctypes.c_void_p(24)
INVALID, UNSUPPORTED, OK = _lib.TOKMIX_ERR_INVALID_ARGUMENT, _lib.TOKMIX_ERR_UNSUPPORTED, _lib.TOKMIX_OK


# ------------------------------------------------------------------------------------ attention
@pytest.mark.parametrize("changes,code", [
    (dict(batch=-1), INVALID), (dict(hq=0), INVALID), (dict(hkv=0), INVALID), (dict(hq=6, hkv=4), INVALID),
    (dict(sq=-1), INVALID), (dict(skv=-1), INVALID), (dict(d=96), UNSUPPORTED), (dict(layout=2), INVALID),
    (dict(scale=0.0), INVALID), (dict(scale=math.nan), INVALID), (dict(scale=math.inf), INVALID), (dict(do=None), INVALID),
    (dict(q=ODD), INVALID), (dict(k=None), INVALID), (dict(v=ODD), INVALID), (dict(o=None), INVALID), (dict(lse=None), INVALID),
    (dict(dq=None), INVALID), (dict(dk=ODD), INVALID), (dict(dv=None), INVALID), (dict(skv=0), INVALID),
    (dict(batch=0), OK), (dict(sq=0, skv=0), OK),
])
def test_attention_gradient_rejects_bad_arguments(changes, code):
    args = dict(do=P, q=P, k=P, v=P, o=P, lse=P, dq=P, dk=P, dv=P, batch=2, hq=4, hkv=2, sq=130, skv=130, d=128, layout=0,
                causal=1, scale=0.1, ws=P, ws_bytes=1 << 40, status=None, stream=None)
    args.update(changes)
    assert _lib.load().tokmix_fa2_bwd(*args.values()) == code
    if code != OK:
        assert _lib.last_error()


def test_attention_gradient_workspace():
    need = _lib.load().tokmix_fa2_bwd_workspace_bytes
    for d in (64, 128, 256):
        assert need(8, 32, 32, 1000, 1000, d, 1) >= 8 * 32 * 1000 * d * 4     # a sum in fp32 per element of dq
        assert need(8, 32, 32, 1000, 128, d, 1) < 8 * 32 * 1000 * d * 4       # one key tile: none
        assert need(1, 8, 1, 2048, 2048, d, 1) > 8 * 2048 * d * 4             # few key tiles: parts of dk and dv beside them
    assert need(0, 4, 2, 10, 10, 64, 1) >= 0 and need(1, 1, 1, 0, 10, 64, 0) >= 0
    assert need(-1, 4, 2, 10, 10, 64, 1) == -1 and need(1, 0, 1, 10, 10, 64, 1) == -1 and need(1, 1, 1, 10, 10, 96, 1) == -1
    assert need(1, 3, 2, 10, 10, 64, 1) == -1
    # a long batch: sizes beyond 32 bits
    assert need(64, 64, 64, 65536, 65536, 256, 1) >= 64 * 64 * 65536 * 256 * 4


def test_attention_forward_with_lse_rejects_bad_arguments():
    lib = _lib.load()
    assert lib.tokmix_fa2_fwd_lse(None, P, P, P, P, 1, 8, 8, 128, 128, 128, 0, 1, 0.1, None, None) == INVALID
    assert lib.tokmix_fa2_fwd_lse(P, P, P, P, P, 1, 6, 4, 128, 128, 128, 0, 1, 0.1, None, None) == INVALID
    assert lib.tokmix_fa2_fwd_lse(P, P, P, P, None, 0, 8, 8, 128, 128, 128, 0, 1, 0.1, None, None) == OK


def _attn(**changes):
    q = torch.zeros(1, 4, 8, 64, dtype=torch.bfloat16)
    k = torch.zeros(1, 2, 8, 64, dtype=torch.bfloat16)
    args = dict(do=q, q=q, k=k, v=k, o=q, lse=torch.zeros(1, 4, 8))
    args.update(changes)
    return args


@pytest.mark.parametrize("changes", [{}, dict(v=torch.zeros(1, 2, 9, 64, dtype=torch.bfloat16)), dict(layout="sbhd"),
                                     dict(q=torch.zeros(4, 8, 64, dtype=torch.bfloat16)),
                                     dict(k=torch.zeros(1, 3, 8, 64, dtype=torch.bfloat16),
                                          v=torch.zeros(1, 3, 8, 64, dtype=torch.bfloat16))])
def test_attention_gradient_raises_on_cpu(changes):
    with pytest.raises(ValueError):
        flash_attention_2_bwd.kernel_fn(**_attn(**changes))


# ------------------------------------------------------------------------------------ norm and rotation
AXIS = (ctypes.c_uint8 * 16)(*([0, 1, 2] * 5 + [0]))
BAD_AXIS = (ctypes.c_uint8 * 16)(*([0] * 15 + [3]))


def _rope(**changes):
    a = dict(q=16, k=16, q_weight=16, k_weight=16, cos=16, sin=16, positions=None, pair_axis=None, dq=16, dk=16, q_out=16, k_out=16)
    a.update({f"{t}_{x}_stride": 64 for t in ("q", "k", "dq", "dk") for x in ("batch", "token", "head")})
    a.update(batch=2, seqlen=5, heads_q=4, heads_k=2, head_dim=64, half=16, nope=32, axes=1, table_rows=5, dtype=0, weight_dtype=0,
             eps=1e-6)
    a.update(changes)
    return _lib.QkNormRope(**a)


BAD_ROPES = [
    (dict(batch=-1), INVALID), (dict(seqlen=-1), INVALID), (dict(heads_q=0), INVALID), (dict(heads_k=0), INVALID),
    (dict(head_dim=96), UNSUPPORTED), (dict(dtype=1), UNSUPPORTED), (dict(weight_dtype=2), UNSUPPORTED), (dict(half=0), INVALID),
    (dict(half=12), INVALID), (dict(nope=4), INVALID), (dict(nope=40), INVALID), (dict(nope=-8), INVALID), (dict(axes=0), INVALID),
    (dict(axes=5, positions=16, pair_axis=ctypes.addressof(AXIS)), INVALID), (dict(axes=3, positions=16), INVALID),
    (dict(axes=3, pair_axis=ctypes.addressof(AXIS)), INVALID),
    (dict(axes=3, positions=16, pair_axis=ctypes.addressof(BAD_AXIS)), INVALID), (dict(eps=-1.0), INVALID),
    (dict(eps=math.nan), INVALID), (dict(table_rows=4), INVALID), (dict(table_rows=0, positions=16), INVALID),
    (dict(q_token_stride=4), INVALID), (dict(q=None), INVALID), (dict(k=24), INVALID), (dict(q_out=None), INVALID),
    (dict(k_out=24), INVALID), (dict(cos=None), INVALID), (dict(sin=8), INVALID), (dict(q_weight=None), INVALID),
]


@pytest.mark.parametrize("changes,code", BAD_ROPES + [(dict(batch=0), OK), (dict(seqlen=0), OK)])
def test_rope_rejects_bad_arguments(changes, code):
    assert _lib.load().tokmix_qk_norm_rope_fwd(ctypes.byref(_rope(**changes)), None, None) == code


@pytest.mark.parametrize("changes,code", BAD_ROPES + [(dict(dq=None), INVALID), (dict(dk=24), INVALID),
                                                      (dict(dk_head_stride=12), INVALID)])
def test_rope_gradient_rejects_bad_arguments(changes, code):
    assert _lib.load().tokmix_qk_norm_rope_bwd(ctypes.byref(_rope(**changes)), P, P, P, 1 << 40, None, None) == code


def test_rope_null_arguments():
    lib = _lib.load()
    assert lib.tokmix_qk_norm_rope_fwd(None, None, None) == INVALID
    assert lib.tokmix_qk_norm_rope_bwd(None, P, P, P, 1 << 40, None, None) == INVALID
    assert lib.tokmix_qk_norm_rope_bwd(ctypes.byref(_rope()), None, P, P, 1 << 40, None, None) == INVALID
    assert lib.tokmix_qk_norm_rope_bwd_workspace_bytes(-1, 1, 1, 64) == -1
    assert lib.tokmix_qk_norm_rope_bwd_workspace_bytes(10, 1, 1, 96) == -1


@pytest.mark.parametrize("half,sections,interleaved,ok", [
    (64, (16, 24, 24), False, True), (64, (24, 20, 20), True, True), (64, (16, 24, 24), True, False), (8, (8,), False, True),
    (8, (8,), True, True), (16, (4, 4, 4, 4), True, True), (16, (16, 0), False, True), (16, (16, 0), True, True),
    (16, (8, 9), False, False), (16, (17, -1), False, False), (16, (4, 4, 4, 2, 2), False, False), (16, (), False, False),
    (24, (20, 4), True, True), (24, (4, 20), True, False),
])
def test_pair_axes(half, sections, interleaved, ok):
    if not ok:
        with pytest.raises(ValueError):
            qk_norm_rope._pair_axis(half, sections, interleaved)
        return
    axis = list(qk_norm_rope._pair_axis(half, sections, interleaved))
    assert [axis.count(a) for a in range(len(sections))] == list(sections)
    if interleaved and len(sections) > 1:
        assert axis[:2] == ([0, 1] if sections[1] else [0, 0])
    else:
        assert axis == sorted(axis)


def _rope_args(**changes):
    q, k = torch.zeros(2, 5, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 5, 2, 64, dtype=torch.bfloat16)
    w, t = torch.zeros(64, dtype=torch.bfloat16), torch.zeros(8, 16)
    args = dict(q=q, k=k, q_weight=w, k_weight=w, cos=t, sin=t)
    args.update(changes)
    return args


@pytest.mark.parametrize("changes", [
    {}, dict(q=torch.zeros(2, 5, 4, 96, dtype=torch.bfloat16)), dict(k=torch.zeros(2, 6, 2, 64, dtype=torch.bfloat16)),
    dict(k=torch.zeros(2, 5, 2, 64)), dict(q=torch.zeros(5, 4, 64, dtype=torch.bfloat16)),
])
def test_rope_modules_raise_on_cpu(changes):
    args = _rope_args(**changes)
    with pytest.raises(ValueError):
        qk_norm_rope.kernel_fn(**args)
    with pytest.raises(ValueError):
        qk_norm_rope_bwd.kernel_fn(args["q"], args["k"], **args)


def test_rope_description_as_bytes():
    """The module packs the C description's fields; the structure of the same fields has the same bytes."""
    values = list(range(1, len(_lib.QkNormRope._fields_))) + [0.5]
    assert bytes(_lib.QkNormRope(*values)) == _lib.QK_NORM_ROPE.pack(*values)
