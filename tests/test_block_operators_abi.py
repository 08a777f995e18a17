"""Host checks of a linear attention block's operators (no GPU): the C entry points
refuse bad sizes, types, pointers and workspaces before any launch, and the Python
operators raise before any call."""
import ctypes
import math

import pytest
import torch

import sparc_amd
from sparc_amd import _lib

FAKE = ctypes.c_void_p(256)  # never dereferenced: a check fails first
F32, BF16 = torch.float32, torch.bfloat16


def _error():
    return _lib.load().sparc_last_error()


def _rotary(**kw):
    d = dict(batch=2, length=3, q_heads=4, k_heads=2, head_dim=16, rotary_dim=8, table_rows=10, io_dtype=0,
             param_dtype=0, interleaved=0, eps=1e-6)
    return ctypes.byref(_lib.RotaryDesc(**{**d, **kw}))


@pytest.mark.parametrize("kw,msg", [
    (dict(batch=-1), b"negative"), (dict(q_heads=0), b"positive"), (dict(head_dim=0), b"1 to 512"),
    (dict(head_dim=513), b"1 to 512"), (dict(rotary_dim=7), b"even"), (dict(rotary_dim=18), b"at most"),
    (dict(table_rows=-1), b"table_rows"), (dict(io_dtype=2), b"io_dtype"), (dict(param_dtype=1), b"parameters"),
    (dict(eps=-1.0), b"eps"), (dict(eps=math.nan), b"eps"), (dict(batch=1 << 20, length=1 << 20), b"too large"),
    (dict(batch=1 << 20, length=1 << 10, k_heads=2), b"too large"),
])
def test_rotary_entry_points_validate(kw, msg):
    lib = _lib.load()
    assert lib.sparc_qk_norm_rotary_forward(_rotary(**kw), *([FAKE] * 8), None) == 1 and msg in _error()
    assert lib.sparc_qk_norm_rotary_backward(_rotary(**kw), *([FAKE] * 13), 1 << 30, None) == 1 and msg in _error()
    assert lib.sparc_qk_norm_rotary_workspace_bytes(_rotary(**kw)) == 0


def test_rotary_entry_points_check_pointers():
    lib = _lib.load()
    fwd, bwd = lib.sparc_qk_norm_rotary_forward, lib.sparc_qk_norm_rotary_backward
    assert fwd(None, *([FAKE] * 8), None) == 1
    assert fwd(_rotary(), None, *([FAKE] * 7), None) == 1 and b"NULL" in _error()
    assert fwd(_rotary(), FAKE, FAKE, None, None, None, None, FAKE, FAKE, None) == 1 and b"NULL" in _error()
    assert fwd(_rotary(batch=0), *([None] * 8), None) == 0
    need = lib.sparc_qk_norm_rotary_workspace_bytes(_rotary())
    assert bwd(_rotary(), *([FAKE] * 13), need - 1, None) == 4 and b"workspace" in _error()
    assert bwd(_rotary(), *([FAKE] * 12), None, need, None) == 4
    assert bwd(_rotary(), FAKE, FAKE, None, None, FAKE, None, None, *([FAKE] * 6), need, None) == 1


def _linear(**kw):
    d = dict(batch=2, length=3, heads=4, kv_heads=2, key_dim=16, value_dim=8, io_dtype=0, scale=1.0)
    far = (ctypes.c_int64 * 3)(1 << 20, 1 << 12, 256)
    return ctypes.byref(_lib.LinearDesc(**{**d, "q_stride": far, "k_stride": far, "v_stride": far, **kw}))


@pytest.mark.parametrize("kw,msg", [
    (dict(batch=-1), b"negative"), (dict(length=-1), b"negative"), (dict(heads=0), b"multiple"),
    (dict(kv_heads=3), b"multiple"), (dict(kv_heads=0), b"multiple"), (dict(key_dim=0), b"1 to 256"),
    (dict(value_dim=257), b"1 to 256"), (dict(io_dtype=4), b"io_dtype"), (dict(batch=1 << 23), b"too large"),
    (dict(length=1 << 33), b"too large"), (dict(q_stride=(ctypes.c_int64 * 3)(0, 15, 1)), b"time strides"),
    (dict(v_stride=(ctypes.c_int64 * 3)(0, 1 << 22, 1)), b"time strides"),
])
def test_linear_attention_entry_points_validate(kw, msg):
    lib = _lib.load()
    calls = (lambda d: lib.sparc_linear_attention_forward(d, *([FAKE] * 9), 1 << 40, None),
             lambda d: lib.sparc_linear_attention_backward(d, *([FAKE] * 13), 1 << 40, None),
             lambda d: lib.sparc_linear_attention_step(d, *([FAKE] * 7), None))
    for call in calls:
        assert call(_linear(**kw)) == 1 and msg in _error()
    for backward in (0, 1):
        assert lib.sparc_linear_attention_workspace_bytes(_linear(**kw), backward) == 0


def test_linear_attention_entry_points_check_pointers():
    lib = _lib.load()
    fwd, bwd, step = (getattr(lib, f"sparc_linear_attention_{n}") for n in ("forward", "backward", "step"))
    assert fwd(None, *([FAKE] * 9), 0, None) == 1
    assert fwd(_linear(), None, *([FAKE] * 8), 0, None) == 1 and b"NULL" in _error()
    assert fwd(_linear(batch=0), *([None] * 9), 0, None) == 0
    long = dict(batch=1, length=100000, heads=2)
    need = lib.sparc_linear_attention_workspace_bytes(_linear(**long), 0)
    assert need > 0 and fwd(_linear(**long), *([FAKE] * 9), need - 1, None) == 4 and b"workspace" in _error()
    need = lib.sparc_linear_attention_workspace_bytes(_linear(**long), 1)
    assert need > 0 and bwd(_linear(**long), *([FAKE] * 13), need - 1, None) == 4
    assert bwd(_linear(**long), *([FAKE] * 12), None, need, None) == 4
    # sums over shared heads pass through the workspace
    assert lib.sparc_linear_attention_workspace_bytes(_linear(), 1) >= 4 * 2 * 3 * 4 * (16 + 8)
    assert lib.sparc_linear_attention_workspace_bytes(_linear(kv_heads=4), 1) == 0
    assert step(_linear(), *([FAKE] * 7), None) == 1 and b"length 1" in _error()
    assert step(_linear(length=1), *([FAKE] * 4), None, FAKE, FAKE, None) == 1 and b"NULL" in _error()


def test_gated_entry_points_validate():
    lib = _lib.load()

    def fwd(rows=4, dim=8, hidden=16, io=0, act=0, x=FAKE, y=FAKE):
        return lib.sparc_gated_forward(rows, dim, hidden, io, act, x, FAKE, FAKE, y, None)

    assert fwd(rows=-1) == 1 and fwd(dim=0) == 1 and fwd(hidden=0) == 1
    assert fwd(io=2) == 1 and b"io_dtype" in _error()
    assert fwd(act=4) == 1 and fwd(act=-1) == 1 and b"activation" in _error()
    assert fwd(rows=1 << 31) == 1 and b"too large" in _error()
    assert fwd(x=None) == 1 and b"NULL" in _error()
    assert fwd(rows=0, x=None, y=None) == 0
    assert lib.sparc_gated_workspace_bytes(4, 0, 16, 0) == 0
    need = lib.sparc_gated_workspace_bytes(4, 8, 16, 1)
    assert need >= 2 * 4 * 16 * 2
    bwd = lib.sparc_gated_backward
    assert bwd(4, 8, 16, 1, 0, *([FAKE] * 8), need - 1, None) == 4 and b"workspace" in _error()
    assert bwd(4, 8, 16, 1, 0, *([FAKE] * 5), FAKE, None, FAKE, need, None) == 1 and b"NULL" in _error()


def _raises(error, match, call, *a, **kw):
    with pytest.raises(error, match=match):
        call(*a, **kw)


def test_rotary_refuses():
    q, k, w, table = torch.zeros(2, 3, 4, 16), torch.zeros(2, 3, 2, 16), torch.ones(16), torch.zeros(5, 8)
    call = sparc_amd.qk_norm_rotary
    _raises(ValueError, "must be .B, T, H, D.", call, q[0], k, w, w, table)
    _raises(ValueError, "must be .B, T, H, D.", call, q, k[:, :2], w, w, table)
    _raises(ValueError, "up to 512", call, torch.zeros(1, 1, 1, 514), torch.zeros(1, 1, 1, 514), None, None, table)
    _raises(ValueError, "eps", call, q, k, w, w, table, eps=-1.0)
    _raises(TypeError, "float32 or bfloat16", call, q.double(), k.double(), w, w, table)
    _raises(ValueError, "alike", call, q, k.bfloat16(), w, w, table)
    _raises(ValueError, "q_weight must be", call, q, k, w[:8], w, table)
    _raises(ValueError, "k_weight must be", call, q, k, w, w.double(), table)
    _raises(ValueError, "alike", call, q.bfloat16(), k.bfloat16(), w, w.bfloat16(), table)
    _raises(ValueError, "table must be", call, q, k, w, w, torch.zeros(5, 18))
    _raises(ValueError, "table must be", call, q, k, w, w, torch.zeros(5, 7))
    _raises(ValueError, "positions must be int", call, q, k, w, w, table, torch.zeros(2, 3))
    _raises(ValueError, "positions must be", call, q, k, w, w, table, torch.zeros(3, 3, dtype=torch.int64))
    _raises(RuntimeError, "GPU tensors", call, q, k, w, w, table)


def test_linear_attention_refuses():
    q, k, v, decay = torch.zeros(2, 5, 4, 8), torch.zeros(2, 5, 2, 8), torch.zeros(2, 5, 2, 6), torch.zeros(4)
    call = sparc_amd.linear_attention
    _raises(ValueError, "must be .B, T, H, K.", call, q[0], k, v, decay)
    _raises(ValueError, "must be .B, T, H, K.", call, q, k[:, :4], v, decay)
    _raises(ValueError, "must be .B, T, H, K.", call, q, k[..., :7], v, decay)
    _raises(ValueError, "multiple", call, q[:, :, :3], k, v, decay[:3])
    _raises(ValueError, "1 to 256", call, q, k, torch.zeros(2, 5, 2, 257), decay)
    _raises(TypeError, "float32 or bfloat16", call, q.half(), k.half(), v.half(), decay)
    _raises(ValueError, "alike", call, q, k.bfloat16(), v, decay)
    _raises(ValueError, "log_decay", call, q, k, v, decay[:2])
    _raises(ValueError, "log_decay", call, q, k, v, decay.bfloat16())
    _raises(ValueError, "state", call, q, k, v, decay, state=torch.zeros(2, 4, 6, 8))
    _raises(ValueError, "lengths", call, q, k, v, decay, lengths=torch.zeros(3, dtype=torch.int64))
    _raises(ValueError, "lengths", call, q, k, v, decay, lengths=torch.zeros(2))
    _raises(RuntimeError, "GPU tensors", call, q, k, v, decay)
    step, state = sparc_amd.linear_attention_step, torch.zeros(2, 4, 8, 6)
    _raises(ValueError, "must be .B, H, K.", step, q, k, v, decay, state)
    one = (q[:, 0], k[:, 0], v[:, 0], decay)
    _raises(ValueError, "state", step, *one, state[:1])
    _raises(ValueError, "out_state", step, *one, state, out_state=state.bfloat16())
    _raises(ValueError, "contiguous", step, *one, state, out_state=torch.zeros(2, 4, 6, 8).transpose(2, 3))
    _raises(RuntimeError, "GPU tensors", step, *one, state)


def test_gated_linear_unit_refuses():
    x, w = torch.zeros(3, 8), torch.zeros(16, 8)
    call = sparc_amd.gated_linear_unit
    _raises(ValueError, "unknown activation", call, x, w, w, activation="tanh")
    _raises(ValueError, "D > 0", call, torch.zeros(3, 0), w, w)
    _raises(ValueError, "weights must both", call, x, w[:, :7], w)
    _raises(ValueError, "weights must both", call, x, w, w[:4])
    _raises(TypeError, "float32 or bfloat16", call, x.half(), w.half(), w.half())
    _raises(ValueError, "alike", call, x, w.bfloat16(), w)
    _raises(RuntimeError, "GPU tensors", call, x, w, w)


def test_stack_refuses():
    from sparc_amd.stack import LinearAttentionBlock, SPARCStack
    _raises(ValueError, "unknown mixer", SPARCStack, 1, 32, 2, mixer="other")
    _raises(ValueError, "needs heads", SPARCStack, 1, 32, 2, mixer="linear")
    _raises(ValueError, "multiple", LinearAttentionBlock, 30, heads=4)
    _raises(ValueError, "multiple", LinearAttentionBlock, 32, heads=4, kv_heads=3)
    _raises(ValueError, "even multiple", LinearAttentionBlock, 12, heads=4)
    assert len(SPARCStack(2, 32, 2, mixer="linear", heads=2, feed_forward=16, max_length=4).blocks) == 2
