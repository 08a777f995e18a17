"""Host checks of the operators around the block stack (no GPU): the C entry
points refuse bad sizes, types, pointers and workspaces before any launch, and
the Python operators raise before any call."""
import ctypes
import math

import pytest
import torch

import sparc_amd
from oracle import lm_oracle as L
from sparc_amd import _lib
from sparc_amd import clip as clip_module

FAKE = ctypes.c_void_p(256)  # never dereferenced: a check fails first


def _error():
    return _lib.load().sparc_last_error()


def test_layer_norm_entry_points_validate():
    lib = _lib.load()
    eps = ctypes.c_float(1e-5)

    def fwd(rows, cols, io=0, pt=0, x=FAKE, e=eps, y=FAKE, mean=FAKE, rstd=FAKE):
        return lib.sparc_layer_norm_forward(rows, cols, io, pt, x, None, None, e, y, mean, rstd, None)

    assert fwd(-1, 8) == 1 and fwd(4, 0) == 1 and fwd(1 << 31, 8) == 1
    assert fwd(4, 8, io=3) == 1 and b"io_dtype" in _error()
    assert fwd(4, 8, io=0, pt=1) == 1 and b"parameters" in _error()
    assert fwd(4, 8, x=None) == 1 and b"NULL" in _error()
    assert fwd(4, 8, mean=None) == 1 and b"together" in _error()
    assert fwd(4, 8, e=ctypes.c_float(-1.0)) == 1 and b"eps" in _error()
    assert fwd(4, 8, e=ctypes.c_float(math.nan)) == 1
    assert fwd(0, 8, x=None, y=None) == 0
    assert lib.sparc_layer_norm_workspace_bytes(4, 0) == 0
    assert lib.sparc_layer_norm_workspace_bytes(10, 24) >= 2 * 10 * 24 * 4
    bwd = lib.sparc_layer_norm_backward
    assert bwd(4, 8, 0, 0, *([FAKE] * 9), 0, None) == 4 and b"workspace" in _error()
    assert bwd(4, 8, 0, 0, None, *([FAKE] * 8), 1 << 20, None) == 1 and b"NULL" in _error()
    assert bwd(4, 8, 0, 0, *([FAKE] * 8), ctypes.c_void_p(258), 1 << 20, None) == 1 and b"aligned" in _error()


def test_embedding_entry_points_validate():
    lib = _lib.load()
    one = ctypes.c_float(1.0)

    def fwd(n, vocab, dim, io=0, ids=8, t=FAKE, w=FAKE, y=FAKE):
        return lib.sparc_embedding_forward(n, vocab, dim, io, ids, t, w, one, y, None)

    assert fwd(-1, 8, 8) == 1 and fwd(4, 0, 8) == 1 and fwd(4, 8, 0) == 1
    assert fwd(4, 8, 8, io=2) == 1 and b"io_dtype" in _error()
    assert fwd(4, 8, 8, ids=2) == 1 and b"32- or 64-bit" in _error()
    assert fwd(4, 8, 8, t=None) == 1 and b"NULL" in _error()
    assert fwd(4, 1 << 31, 8) == 1 and b"too large" in _error()
    assert fwd(0, 8, 8, t=None, w=None, y=None) == 0
    assert lib.sparc_embedding_workspace_bytes(4, 8, 0) == 0
    need = lib.sparc_embedding_workspace_bytes(1000, 50, 24)
    assert need >= 4 * 1000 * 4 + 50
    bwd = lib.sparc_embedding_backward
    assert bwd(1000, 50, 24, 0, 8, FAKE, -1, FAKE, one, FAKE, FAKE, need - 1, None) == 4
    assert bwd(1000, 50, 24, 0, 8, FAKE, -1, FAKE, one, None, FAKE, need, None) == 1
    assert bwd(1000, 50, 24, 0, 8, FAKE, -1, FAKE, one, FAKE, ctypes.c_void_p(264), need, None) == 1
    assert b"aligned" in _error()


def test_grad_norm_entry_points_validate():
    lib = _lib.load()
    data, sizes, codes = (ctypes.c_void_p * 2)(256, 512), (ctypes.c_int64 * 2)(4, 4), (ctypes.c_int32 * 2)(0, 1)
    assert lib.sparc_grad_norm_workspace_bytes(-1) == 0
    need = lib.sparc_grad_norm_workspace_bytes(2)
    assert 0 < need <= lib.sparc_grad_norm_workspace_bytes(1000)
    norm = lib.sparc_grad_norm
    assert norm(-1, data, sizes, codes, FAKE, FAKE, need, None) == 1
    assert norm(2, None, sizes, codes, FAKE, FAKE, need, None) == 1
    assert norm(2, data, sizes, codes, None, FAKE, need, None) == 1
    assert norm(2, data, sizes, codes, FAKE, FAKE, need - 1, None) == 4
    assert norm(2, data, (ctypes.c_int64 * 2)(4, -1), codes, FAKE, FAKE, need, None) == 1
    assert norm(2, data, sizes, (ctypes.c_int32 * 2)(0, 7), FAKE, FAKE, need, None) == 1 and b"dtype" in _error()
    assert norm(2, (ctypes.c_void_p * 2)(258, 512), sizes, codes, FAKE, FAKE, need, None) == 1 and b"aligned" in _error()
    assert norm(2, (ctypes.c_void_p * 2)(None, 512), sizes, codes, FAKE, FAKE, need, None) == 1 and b"NULL" in _error()
    clip = lib.sparc_clip_grad_norm
    for bad in (-1.0, math.nan):
        assert clip(2, data, sizes, codes, ctypes.c_float(bad), FAKE, FAKE, need, None) == 1 and b"max_norm" in _error()


def test_beam_entry_points_validate():
    lib = _lib.load()
    need = lib.sparc_beam_workspace_bytes(2, 4, 100)
    assert need > 0
    for bad in ((2, 0, 100), (2, 33, 100), (2, 4, 0), (-1, 4, 100), (1 << 22, 4, 100), (2, 32, 1 << 27)):
        assert lib.sparc_beam_workspace_bytes(*bad) == 0

    def step(batch=2, beams=4, vocab=100, stride=100, io=0, logits=FAKE, finished=None, eos=-1, size=need):
        return lib.sparc_beam_step(batch, beams, vocab, stride, io, logits, FAKE, finished, eos, *([FAKE] * 3), None,
                                   FAKE, size, None)

    assert step(io=4) == 1 and b"io_dtype" in _error()
    assert step(stride=99) == 1 and b"row_stride" in _error()
    assert step(eos=100) == 1 and step(eos=-2) == 1 and b"eos_id" in _error()
    assert step(finished=FAKE) == 1 and b"eos_id" in _error()
    assert step(logits=None) == 1 and b"NULL" in _error()
    assert step(size=need - 1) == 4 and b"workspace" in _error()
    assert step(batch=0) == 0
    ptrs, rb = (ctypes.c_void_p * 1)(256), (ctypes.c_int64 * 1)(64)
    order = lib.sparc_reorder_states
    assert order(2, 33, 1, ptrs, ptrs, rb, FAKE, None) == 1
    assert order(2, 4, 1, ptrs, ptrs, rb, None, None) == 1 and b"NULL" in _error()
    assert order(2, 4, 1, ptrs, ptrs, (ctypes.c_int64 * 1)(7), FAKE, None) == 1 and b"even" in _error()
    assert order(2, 4, 1, (ctypes.c_void_p * 1)(257), ptrs, rb, FAKE, None) == 1 and b"aligned" in _error()
    assert order(2, 4, 0, None, None, None, None, None) == 0


def test_python_operators_refuse():
    f, b = torch.zeros(3, 8), torch.zeros(3, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="D > 0"):
        sparc_amd.layer_norm(torch.zeros(3, 0))
    with pytest.raises(ValueError, match="eps"):
        sparc_amd.layer_norm(f, eps=-1.0)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        sparc_amd.layer_norm(f.double())
    with pytest.raises(ValueError, match="weight must be"):
        sparc_amd.layer_norm(f, torch.zeros(7))
    with pytest.raises(ValueError, match="dtype"):
        sparc_amd.layer_norm(f, torch.zeros(8, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="alike"):
        sparc_amd.layer_norm(b, torch.zeros(8), torch.zeros(8, dtype=torch.bfloat16))
    ids = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="table"):
        sparc_amd.embedding(ids, torch.zeros(8))
    with pytest.raises(TypeError, match="int64 or int32"):
        sparc_amd.embedding(ids.float(), f)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        sparc_amd.embedding(ids, f.half())
    with pytest.raises(ValueError, match="padding_idx"):
        sparc_amd.embedding(ids, f, padding_idx=3)
    for call in (lambda: sparc_amd.layer_norm(f), lambda: sparc_amd.embedding(ids, f),
                 lambda: sparc_amd.grad_norm([f]),
                 lambda: sparc_amd.beam_search_step(torch.zeros(1, 2, 8), torch.zeros(1, 2)),
                 lambda: sparc_amd.reorder_states([f], torch.zeros(1, 3, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="need GPU tensors"):
            call()


def test_clip_refuses():
    p = torch.nn.Parameter(torch.zeros(3, 8))
    assert float(sparc_amd.clip_grad_norm_([p], 1.0)) == 0.0  # no gradient
    p.grad = torch.zeros(3, 8)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            sparc_amd.clip_grad_norm_([p], bad)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        sparc_amd.grad_norm([torch.zeros(3, dtype=torch.float16)])
    with pytest.raises(ValueError, match="dense"):
        sparc_amd.grad_norm([torch.zeros(3, 8).to_sparse()])
    p.grad = torch.zeros(1, 8).expand(3, 8)
    with pytest.raises(ValueError, match="more than once"):
        sparc_amd.clip_grad_norm_([p], 1.0)


@pytest.mark.parametrize("make,dense,repeats", [
    (lambda t: t, True, False),
    (lambda t: t.permute(2, 0, 1), True, False),
    (lambda t: t[:, 1:2].transpose(0, 2), False, False),
    (lambda t: t[..., ::2], False, False),
    (lambda t: t[:1, :1].expand(4, 6, 5), False, True),
    (lambda t: t.reshape(-1).as_strided((5, 3), (1, 1)), False, True),
    (lambda t: t[:0], True, False),
])
def test_memory_layout_of_gradients(make, dense, repeats):
    t = make(torch.zeros(4, 6, 5))
    assert clip_module._dense(t) is dense and clip_module._repeats(t) is repeats


def test_beam_step_refuses():
    x, s = torch.zeros(2, 4, 10), torch.zeros(2, 4)
    for bad in (torch.zeros(4, 10), torch.zeros(2, 33, 10), torch.zeros(2, 0, 10), torch.zeros(2, 4, 0)):
        with pytest.raises(ValueError, match=r"\[B, K, V\]"):
            sparc_amd.beam_search_step(bad, s)
    with pytest.raises(ValueError, match="scores"):
        sparc_amd.beam_search_step(x, s.double())
    with pytest.raises(ValueError, match="eos_id"):
        sparc_amd.beam_search_step(x, s, finished=torch.zeros(2, 4, dtype=torch.bool))
    with pytest.raises(ValueError, match="finished"):
        sparc_amd.beam_search_step(x, s, finished=torch.zeros(2, 4), eos_id=1)
    with pytest.raises(ValueError, match="vocabulary"):
        sparc_amd.beam_search_step(x, s, eos_id=10)
    parents = torch.zeros(2, 4, dtype=torch.int64)
    with pytest.raises(ValueError, match="rows"):
        sparc_amd.reorder_states([torch.zeros(7, 3)], parents)
    with pytest.raises(ValueError, match="parents"):
        sparc_amd.reorder_states([torch.zeros(8, 3)], parents.int())


def test_oracle_gradients_against_differences():
    """The oracle's gradient formulas against central differences of its forward."""
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    x, w, b, dy, h = r(5, 7), r(7), r(7), r(5, 7), 1e-5
    grads = L.layer_norm_grads(x, w, 1e-5, dy)
    for at, (v, got) in enumerate(zip((x, w, b), grads)):
        u = r(*v.shape)
        args = lambda s: [t + s * h * u if i == at else t for i, t in enumerate((x, w, b))]  # noqa: E731
        diff = sum(s * (L.layer_norm(*args(s), 1e-5) * dy).sum() for s in (1, -1)) / (2 * h)
        assert abs(float(diff - (got * u).sum())) < 1e-7
    tokens, table, dy = torch.tensor([[1, 4, 1], [0, 2, 9]]), r(5, 3), r(2, 3, 3)
    dw, u = L.embedding_grad(tokens, 5, dy, 3.0), r(5, 3)
    diff = sum(s * (L.embedding(tokens, table + s * u, 3.0) * dy).nansum() for s in (1, -1)) / 2
    assert abs(float(diff - (dw * u).sum())) < 1e-12


def test_layer_norm_workspace_holds_the_partial_rows():
    """Two partial rows for each workgroup that the widths' forms launch, not more:
    512 for rows of a wave, 1024 for 4 waves, 256 for 16, 64 for rows that no
    workgroup holds."""
    need = _lib.load().sparc_layer_norm_workspace_bytes
    for rows, cols, partials in ((1 << 20, 768, 512), (1 << 20, 1536, 1024), (8192, 24576, 256), (70000, 32768, 256),
                                 (9000, 131072, 64), (40, 131072, 40), (10, 24576, 10)):
        assert need(rows, cols) <= 2 * partials * cols * 4 + 256, (rows, cols)
        assert need(rows, cols) >= 2 * min(partials, rows // 2) * cols * 4, (rows, cols)


def test_language_model_refuses_padding_outside_the_vocabulary():
    from sparc_amd import lm
    for bad in (7, -8):
        with pytest.raises(ValueError, match="padding_idx"):
            lm.SPARCLanguageModel(7, 1, 16, 4, padding_idx=bad)
    assert lm.SPARCLanguageModel(7, 1, 16, 4, padding_idx=-7).padding_idx == 0
