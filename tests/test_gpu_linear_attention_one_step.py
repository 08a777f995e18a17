"""linear_attention over one step whose inputs have any stride of time: torch leaves it
free where there is one step, and so does the C header.  Tolerances as in
test_gpu_linear_attention.py."""
import ctypes

import pytest
import torch

from oracle import block_oracle as O
from sparc_amd import _lib
from test_gpu_linear_attention import BF16, F32, IDS, _case, _check, _run

pytestmark = pytest.mark.gpu
B, H, G = 2, 4, 2


def _with_time_stride(x, stride):
    """The same values [B, 1, n, d] with another stride of the one step."""
    s = list(x.stride())
    s[1] = stride
    return x.as_strided(x.shape, s)


@pytest.mark.parametrize("dtype", [F32, BF16], **IDS)
@pytest.mark.parametrize("K,V", [(64, 64), (128, 128), (16, 24), (20, 44), (256, 256)])
@pytest.mark.parametrize("stride", [0, 1, 7, 1 << 22, (1 << 30) + 1, 1 << 31])
def test_any_time_stride(stride, K, V, dtype):
    """1 << 30 and more: multiples of its bytes wrap to small ones in 32 bits."""
    print(f"[case] one step, time stride {stride}, {K} x {V} {dtype}", flush=True)
    s, do, ds = _case(B, 1, H, G, K, V, dtype, seed=K + V, state=True)
    for n in ("q", "k", "v"):
        s[n] = _with_time_stride(s[n], stride)
    _run(s, do, ds, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16], **IDS)
@pytest.mark.parametrize("form", ["expanded", "permuted"])
def test_views_of_one_step(form, dtype):
    """Views that a program makes: torch takes the permuted one for contiguous."""
    K, V = 32, 64
    s, do, ds = _case(B, 1, H, G, K, V, dtype, seed=5, state=True)
    for n in ("q", "k", "v"):
        heads, d = s[n].shape[2:]
        if form == "expanded":
            s[n] = s[n][:, 0].unsqueeze(1).expand(B, 3, heads, d)[:, :1]
            s[n] = _with_time_stride(s[n], 0)
        else:
            s[n] = s[n][:, 0].contiguous()[..., None].permute(0, 3, 1, 2)
            assert s[n].stride(1) == 1 and s[n].is_contiguous()
    _run(s, do, ds, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16], **IDS)
@pytest.mark.parametrize("stride", [0, 1 << 31])
def test_the_c_entry_points(stride, dtype):
    """Through the C header, whose time strides are free at length 1."""
    K, V = 64, 64
    s, do, ds = _case(B, 1, H, G, K, V, dtype, seed=9, state=True)
    lib, g = _lib.load(), {n: x.cuda() for n, x in s.items()}
    d = _lib.LinearDesc(batch=B, length=1, heads=H, kv_heads=G, key_dim=K, value_dim=V,
                        io_dtype=_lib.io_code(dtype), scale=K ** -0.5)
    for name, heads, width in (("q", H, K), ("k", G, K), ("v", G, V)):
        getattr(d, name + "_stride")[:] = [heads * width, stride, width]
    o, after = torch.empty(B, 1, H, V, dtype=dtype, device="cuda"), torch.empty(B, H, K, V, device="cuda")
    grads = {n: torch.empty(g[n].shape, dtype=g[n].dtype, device="cuda") for n in ("q", "k", "v", "state")}
    do, ds = do.cuda(), ds.cuda()
    need = [lib.sparc_linear_attention_workspace_bytes(ctypes.byref(d), back) for back in (0, 1)]
    ws = torch.empty(max(*need, 1), dtype=torch.uint8, device="cuda")
    P, stream = _lib.ptr, _lib.stream_of(o.device)
    _lib.check(lib.sparc_linear_attention_forward(
        ctypes.byref(d), P(g["q"]), P(g["k"]), P(g["v"]), P(g["log_decay"]), None, P(g["state"]), P(o), P(after),
        P(ws), need[0], stream), "forward")
    _lib.check(lib.sparc_linear_attention_backward(
        ctypes.byref(d), P(g["q"]), P(g["k"]), P(g["v"]), P(g["log_decay"]), None, P(g["state"]), P(do), P(ds),
        P(grads["q"]), P(grads["k"]), P(grads["v"]), P(grads["state"]), P(ws), need[1], stream), "backward")

    def oracle(x, *back):
        x = {n: t.double().requires_grad_(n != "log_decay") for n, t in x.items()}
        y = O.linear_attention(**x)
        got = torch.autograd.grad(y, [x[n] for n in grads], back)
        return {"o": y[0].detach(), "after": y[1].detach(), **dict(zip(grads, got))}
    back = [t.cpu().double() for t in (do, ds)]
    size = oracle({n: x if n == "log_decay" else x.abs() for n, x in s.items()}, *(t.abs() for t in back))
    _check({"o": o, "after": after, **grads}, oracle(s, *back), size, 1 + max(K, V) * (H // G) + 64, dtype == BF16)
