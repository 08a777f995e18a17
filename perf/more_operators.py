"""The operators of a block of linear attention and a gated feed-forward block, and
what a pass through each has to do.

Four kinds of call, each over the sizes, data types and options it is used with:

* ``rotary`` -- ``qk_norm_rotary``: RMS norms of queries and keys for each head and
                the rotation by their positions; for training with all gradients
* ``linear`` -- ``linear_attention``: a decay for each head, over a prompt or a
                training batch, with the state before and after; for training with
                all gradients
* ``step``   -- ``linear_attention_step``: the same for one token, the state in place
* ``gated``  -- ``gated_linear_unit``: act(x Wg^T) * (x Wu^T); for training with all
                gradients

``own`` chooses between the framework's calls and their plain form in elementary
torch operations.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # the next token of 256 streams at d_model 2048 (the decode configuration), 16
        # heads of 128: nothing but latency
        dict(name="rotary_decode", kind="rotary", train=False, B=256, T=1, H=16, G=16, D=128, R=128, dtype="bf16",
             pdtype="bf16", interleaved=False, far=40000),
        # the 12-layer stack's batch (16 x 2048 tokens, d_model 768), 12 heads of 64
        dict(name="rotary_train", kind="rotary", train=True, B=16, T=2048, H=12, G=12, D=64, R=64, dtype="bf16",
             pdtype="bf16", interleaved=False, far=0),
        # six query heads to a key head, a part of an uneven head rotated by
        # neighbouring pairs, full precision
        dict(name="rotary_odd", kind="rotary", train=True, B=3, T=1237, H=6, G=1, D=90, R=42, dtype="fp32",
             pdtype="fp32", interleaved=True, far=0),
        # one long prompt at d_model 2048: 16 chains, each as long as the scan's stress case
        dict(name="linear_prompt", kind="linear", train=False, B=1, T=65536, H=16, G=16, K=128, V=128, dtype="bf16",
             padded=False, state=False),
        # the 12-layer stack's training batch
        dict(name="linear_train", kind="linear", train=True, B=16, T=2048, H=12, G=12, K=64, V=64, dtype="bf16",
             padded=False, state=False),
        # the headline's batch (8 x 4096 tokens, d_model 1024), 8 heads of 128
        dict(name="linear_train_wide", kind="linear", train=True, B=8, T=4096, H=8, G=8, K=128, V=128, dtype="bf16",
             padded=False, state=False),
        # padded documents that continue others, full precision, three heads of an
        # uneven width to one head of keys and values
        dict(name="linear_odd", kind="linear", train=True, B=3, T=1237, H=6, G=2, K=40, V=72, dtype="fp32",
             padded=True, state=True),
        # the next token of one stream, and of 256 (the decode configuration)
        dict(name="step_one", kind="step", B=1, H=16, G=16, K=128, V=128, dtype="bf16"),
        dict(name="step_large", kind="step", B=256, H=16, G=16, K=128, V=128, dtype="bf16"),
        # a feed-forward block behind that step, four times as wide as the stream
        dict(name="gated_decode", kind="gated", train=False, N=256, D=2048, F=8192, dtype="bf16", act="silu"),
        # the 12-layer stack's training batch, the three products of a block together
        # as large as one of eight times the square of d_model
        dict(name="gated_train", kind="gated", train=True, N=32768, D=768, F=2048, dtype="bf16", act="silu"),
        # widths that no vector divides, full precision
        dict(name="gated_odd", kind="gated", train=True, N=1237, D=1001, F=2731, dtype="fp32", act="gelu"),
    ]


ACTS = ("silu", "gelu", "relu", "sigmoid")


def _log(rng, lo, hi):
    """A whole number between lo and hi, evenly spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    """Query heads, and the key heads that divide them."""
    g = rng.choice((1, 2, 3, 4, 8, 12, 16))
    return g * rng.choice([m for m in (1, 1, 2, 3, 4, 6) if g * m <= 16]), g


def draw(rng):
    kind = rng.choice(("rotary", "rotary", "linear", "linear", "linear", "step", "gated", "gated"))
    dtype = rng.choice(("fp32", "bf16", "bf16"))
    h, g = _heads(rng)
    train = rng.random() < 0.6
    if kind == "rotary":
        d = rng.choice((64, 128, _log(rng, 2, 256)))
        r = min(d, rng.choice((d, d, _log(rng, 2, d)))) // 2 * 2
        n = min(_log(rng, 1, 32768), (1 << 24) // ((h + g) * d))
        b = _log(rng, 1, min(n, 256))
        return dict(kind=kind, train=train, B=b, T=n // b, H=h, G=g, D=d, R=r, dtype=dtype,
                    pdtype=rng.choice((dtype, "fp32")), interleaved=rng.random() < 0.4,
                    far=_log(rng, 1, 40000) if rng.random() < 0.4 else 0)
    if kind in ("linear", "step"):
        k, v = rng.choice(((64, 64), (128, 128), (_log(rng, 8, 128), _log(rng, 8, 256))))
        if kind == "step":
            b = max(1, min(_log(rng, 1, 256), (1 << 26) // (h * k * v)))
            return dict(kind=kind, B=b, H=h, G=g, K=k, V=v, dtype=dtype)
        n = max(1, min(_log(rng, 1, 16384 if train else 65536), (1 << (24 if train else 26)) // (h * max(k, v))))
        b = _log(rng, 1, min(n, 64))
        return dict(kind=kind, train=train, B=b, T=n // b, H=h, G=g, K=k, V=v, dtype=dtype, padded=rng.random() < 0.4,
                    state=rng.random() < 0.4)
    n, d, f = _log(rng, 1, 32768), _log(rng, 32, 4096), _log(rng, 32, 8192)
    if rng.random() < 0.6:
        d, f = max(32, d // 32 * 32), max(32, f // 32 * 32)
    while d * f > 1 << 24:
        d, f = d // 2, f * 3 // 4
    n = max(1, min(n, (1 << (35 if dtype == "bf16" else 33)) // (d * f)))
    return dict(kind=kind, train=train, N=n, D=d, F=f, dtype=dtype, act=rng.choice(ACTS))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
class _Inputs:
    """Random tensors on the GPU, from the seed alone."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(int(seed))

    def randn(self, *shape, dtype=torch.float32, scale=1.0, mean=0.0):
        return torch.randn(*shape, device="cuda", generator=self.g).mul_(scale).add_(mean).to(dtype)

    def rand(self, *shape):
        return torch.rand(*shape, device="cuda", generator=self.g)

    def unit(self, *shape, dtype):
        """Rows of a mean square of one, as a norm leaves them."""
        x = torch.randn(*shape, device="cuda", generator=self.g)
        return x.mul_(torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)).to(dtype)


def prepare(case, seed):
    r, dt, kind = _Inputs(seed), DTYPES[case["dtype"]], case["kind"]
    s = {"case": case}
    if kind == "rotary":
        b, t, h, g, d, rot, pdt = (case[x] for x in ("B", "T", "H", "G", "D", "R", "pdtype"))
        # queries and keys are parts of one projection's output, values behind them
        both = r.randn(b, t, (h + 2 * g) * d, dtype=dt, scale=1.3)
        s["q"] = both[..., :h * d].unflatten(-1, (h, d)).detach()
        s["k"] = both[..., h * d:(h + g) * d].unflatten(-1, (g, d)).detach()
        s["wq"], s["wk"] = (r.randn(d, dtype=DTYPES[pdt], scale=0.2, mean=1.0) for _ in range(2))
        # cosines and sines of every position, from angles in 64 bits
        s["positions"] = (r.rand(b, 1) * case["far"]).long() + torch.arange(t, device="cuda") if case["far"] else None
        angle = torch.arange(case["far"] + t, device="cuda", dtype=torch.float64)[:, None] * \
            10000.0 ** (torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / -rot)
        s["table"] = torch.cat((angle.cos(), angle.sin()), dim=-1).float()
        if case["train"]:
            s["inputs"] = [x.requires_grad_() for x in (s["q"], s["k"], s["wq"], s["wk"])]
            s["dq"], s["dk"] = r.randn(b, t, h, d, dtype=dt), r.randn(b, t, g, d, dtype=dt)
    elif kind in ("linear", "step"):
        b, h, g, k, v = (case[x] for x in ("B", "H", "G", "K", "V"))
        steps = (b, case["T"]) if kind == "linear" else (b,)
        s["q"], s["k"] = r.unit(*steps, h, k, dtype=dt), r.unit(*steps, g, k, dtype=dt)
        # values straight from the projection that made queries and keys too
        s["v"] = r.randn(*steps, h * k + g * (k + v), dtype=dt)[..., h * k + g * k:].unflatten(-1, (g, v)).detach()
        # from 32 steps of memory to 4096
        s["decay"] = torch.log1p(-torch.exp2(-5.0 - 7.0 * torch.arange(h, device="cuda") / max(1, h - 1)))
        if kind == "step":
            s["state"] = r.randn(b, h, k, v, scale=0.5)
            return s
        s["state"] = r.randn(b, h, k, v, scale=0.5) if case["state"] else None
        s["lengths"] = (r.rand(b) * (case["T"] + 1)).long().clamp_(max=case["T"]) if case["padded"] else None
        if case["train"]:
            s["inputs"] = [x.requires_grad_() for x in (s["q"], s["k"], s["v"], s["state"]) if x is not None]
            s["do"] = r.randn(*steps, h, v, dtype=dt)
            s["dstate"] = r.randn(b, h, k, v, scale=0.1) if case["state"] else None
    else:
        n, d, f = case["N"], case["D"], case["F"]
        s["x"] = r.unit(n, d, dtype=dt)
        s["wg"], s["wu"] = (r.randn(f, d, dtype=dt, scale=d ** -0.5) for _ in range(2))
        if case["train"]:
            s["inputs"] = [x.requires_grad_() for x in (s["x"], s["wg"], s["wu"])]
            s["dy"] = r.randn(n, f, dtype=dt)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return (_own if own else _plain)(state, state["case"])


def _own(s, case):
    import sparc_amd
    kind = case["kind"]
    if kind == "rotary":
        q, k = sparc_amd.qk_norm_rotary(s["q"], s["k"], s["wq"], s["wk"], s["table"], positions=s["positions"],
                                        interleaved=case["interleaved"], eps=1e-6)
        if not case["train"]:
            return [q, k]
        return [q.detach(), k.detach(), *torch.autograd.grad((q, k), s["inputs"], (s["dq"], s["dk"]))]
    if kind == "linear":
        o, state = sparc_amd.linear_attention(s["q"], s["k"], s["v"], s["decay"], state=s["state"],
                                              lengths=s["lengths"])
        if not case["train"]:
            return [o, state]
        outs, grads = ((o, state), (s["do"], s["dstate"])) if case["state"] else ((o,), (s["do"],))
        return [o.detach(), state.detach(), *torch.autograd.grad(outs, s["inputs"], grads)]
    if kind == "step":
        return list(sparc_amd.linear_attention_step(s["q"], s["k"], s["v"], s["decay"], s["state"],
                                                    out_state=s["state"]))
    y = sparc_amd.gated_linear_unit(s["x"], s["wg"], s["wu"], activation=case["act"])
    if not case["train"]:
        return y
    return [y.detach(), *torch.autograd.grad(y, s["inputs"], s["dy"])]


def _plain(s, case):
    kind, dt = case["kind"], DTYPES[case["dtype"]]
    if kind == "rotary":
        table, inter = s["table"][:case["T"]] if s["positions"] is None else s["table"][s["positions"]], case["interleaved"]
        both, sums = [], []
        for x, w, dy in ((s["q"], s["wq"], s.get("dq")), (s["k"], s["wk"], s.get("dk"))):
            x, w = x.detach().float(), w.detach().float()
            rstd = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
            both.append(_turn(x * rstd * w, table, inter, 1.0).to(dt))
            if case["train"]:
                g = _turn(dy.float(), table, inter, -1.0)
                xhat, gw = x * rstd, g * w
                both.append((rstd * (gw - xhat * (gw * xhat).mean(-1, keepdim=True))).to(dt))
                sums.append((g * xhat).sum((0, 1, 2)).to(s["wq"].dtype))
        return [*both[::2], *both[1::2], *sums] if case["train"] else both
    if kind == "linear":
        h, g = case["H"], case["G"]
        q, do = s["q"].detach().float() * case["K"] ** -0.5, s.get("do")
        k, v = (x.detach().float().repeat_interleave(h // g, dim=2) for x in (s["k"], s["v"]))
        length = s["lengths"] if case["padded"] else torch.full((case["B"],), case["T"], device="cuda")
        there = (torch.arange(case["T"], device="cuda") < length[:, None])[..., None, None]
        q, k, v = (torch.where(there, x, 0.0) for x in (q, k, v))
        before = s["state"].detach() if case["state"] else q.new_zeros(case["B"], h, case["K"], case["V"])
        o, after = _chunks(q, k, v, s["decay"], before, length, True)
        if not case["train"]:
            return [o.to(dt), after]
        do = torch.where(there, do.float(), 0.0)
        dlast = s["dstate"] if case["state"] else torch.zeros_like(before)
        dq, _ = _chunks(do, v, k, s["decay"], before.transpose(-1, -2), length, True)
        back = lambda x: _reversed(x, length)
        dk, _ = _chunks(back(v), back(do), back(q), s["decay"], dlast.transpose(-1, -2), length, False)
        dv, dfirst = _chunks(back(k), back(q), back(do), s["decay"], dlast, length, False)
        dk, dv = (back(x).unflatten(2, (g, h // g)).sum(3) for x in (dk, dv))
        grads = [(dq * case["K"] ** -0.5).to(dt), dk.to(dt), dv.to(dt), dfirst]
        return [o.to(dt), after, *(grads if case["state"] else grads[:3])]
    if kind == "step":
        m = case["H"] // case["G"]
        q, k, v = s["q"].float() * case["K"] ** -0.5, s["k"].float(), s["v"].float()
        k, v = k.repeat_interleave(m, dim=1), v.repeat_interleave(m, dim=1)
        s["state"].mul_(torch.exp(s["decay"])[:, None, None]).add_(k[..., None] * v[..., None, :])
        return [(q[..., None] * s["state"]).sum(-2).to(dt), s["state"]]
    x, wg, wu = (s[n].detach().float() for n in ("x", "wg", "wu"))
    g, u = x @ wg.T, x @ wu.T
    a, da = _act(g, case["act"])
    y = (a * u).to(dt)
    if not case["train"]:
        return y
    dy = s["dy"].float()
    dg, du = dy * u * da, dy * a
    return [y, (dg @ wg + du @ wu).to(dt), (dg.T @ x).to(dt), (du.T @ x).to(dt)]


def _turn(x, table, interleaved, sign):
    """The first values of each head, in pairs, turned by the angles of ``table`` [.., T, R]."""
    r = table.shape[-1]
    cos, sin = table[..., None, :r // 2], table[..., None, r // 2:] * sign
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    c, d = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((c, d), dim=-1).flatten(-2) if interleaved else torch.cat((c, d), dim=-1)
    return torch.cat((turned, x[..., r:]), dim=-1)


def _chunks(q, k, v, decay, before, length, inclusive, C=64):
    """o_t = q_t S_t and the last S, S_t = a S_(t-1) + k_t v_t^T, over chunks of C steps.
    Not inclusive: the state given is S behind the last step, undecayed, and the one
    returned is decayed once more."""
    B, T, H, _ = q.shape
    N = -(-T // C)
    q, k, v = (torch.nn.functional.pad(x, (0, 0, 0, 0, 0, N * C - T)).view(B, N, C, H, -1).permute(0, 3, 1, 2, 4)
               for x in (q, k, v))
    i, extra = torch.arange(C, device=q.device), int(inclusive)
    power = lambda n: torch.exp(decay[:, None, None, None] * n)
    lower = torch.where(i[:, None] >= i, power((i[:, None] - i).clamp(min=0)), 0.0)
    scores = (q @ k.transpose(-1, -2)) * lower
    # steps of each chunk that a row has
    have = (length[:, None] - torch.arange(N, device=q.device) * C).clamp(0, C)[:, None, :, None, None]
    local = (k * power((have - extra - i[:, None]).clamp(min=0))).transpose(-1, -2).contiguous() @ v
    states, s = [], before
    for n in range(N):
        states.append(s)
        s = s * power(have[:, :, n:n + 1])[:, :, 0] + local[:, :, n]
    o = scores @ v + (q * power(i[:, None] + extra)) @ torch.stack(states, dim=2)
    return o.permute(0, 2, 3, 1, 4).reshape(B, N * C, H, -1)[:, :T], s


def _reversed(x, length):
    """The steps of each row in reverse order, those behind its end where they are."""
    t = torch.arange(x.shape[1], device=x.device)
    at = torch.where(t < length[:, None], length[:, None] - 1 - t, t)
    return x.gather(1, at[..., None, None].expand(-1, -1, *x.shape[2:]))


def _act(g, name):
    """An activation and its derivative."""
    if name == "relu":
        return g.clamp(min=0.0), (g > 0).to(g.dtype)
    if name == "gelu":
        phi = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * phi, phi + g * torch.exp(-0.5 * g * g) * (0.5 / math.pi) ** 0.5
    sig = 1.0 / (1.0 + torch.exp(-g))
    if name == "sigmoid":
        return sig, sig * (1.0 - sig)
    return g * sig, sig * (1.0 + g * (1.0 - sig))


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    """Inputs read once, outputs and gradients written once; the operations of the
    recurrent form for linear attention."""
    kind, es = case["kind"], 2 if case["dtype"] == "bf16" else 4
    if kind == "rotary":
        n, ps = case["B"] * case["T"], 2 if case["pdtype"] == "bf16" else 4
        el = n * (case["H"] + case["G"]) * case["D"]
        fixed = 2 * case["D"] * ps + min(n, case["far"] + case["T"]) * case["R"] * 4 + (8 * n if case["far"] else 0)
        if case["train"]:  # x in, y out; x and dy in, dx out
            return {"bytes": 5 * el * es + 3 * fixed, "flops": 24 * el}
        return {"bytes": 2 * el * es + fixed, "flops": 8 * el}
    if kind in ("linear", "step"):
        h, g, k, v = (case[x] for x in ("H", "G", "K", "V"))
        n, states = case["B"] * case.get("T", 1), case["B"] * h * k * v
        ins, out = n * (h * k + g * (k + v)) * es, n * h * v * es
        if kind == "step":
            return {"bytes": ins + out + 8 * states, "flops": 5 * states}
        first = 4 * states * (2 if case["state"] else 1)
        if case["train"]:  # the inputs and do once more, their gradients
            return {"bytes": 3 * ins + 2 * out + 2 * first, "flops": 16 * n * h * k * v}
        return {"bytes": ins + out + first, "flops": 4 * n * h * k * v}
    n, d, f = case["N"], case["D"], case["F"]
    if case["train"]:  # x, both weights, y; these and dy once more, three gradients
        return {"bytes": (3 * (n * d + 2 * f * d) + 2 * n * f) * es, "flops": 12 * n * d * f}
    return {"bytes": (n * d + 2 * f * d + n * f) * es, "flops": 4 * n * d * f}


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "rotary":
        with torch.enable_grad():
            leaves = [s[n].detach().double().requires_grad_() for n in ("q", "k", "wq", "wk")]
            at = torch.arange(case["T"], device="cuda").expand(case["B"], -1) if s["positions"] is None else s["positions"]
            half = case["R"] // 2
            # pairs as complex numbers, multiplied by those of the angles
            turn = torch.complex(s["table"].double()[:, :half], s["table"].double()[:, half:])[at][:, :, None]
            first, second = (torch.arange(half, device="cuda") * m + o for m, o in
                             (((2, 0), (2, 1)) if case["interleaved"] else ((1, 0), (1, half))))
            ys = []
            for x, w in zip(leaves[:2], leaves[2:]):
                y = x * w / torch.sqrt(torch.linalg.vecdot(x, x)[..., None] / case["D"] + 1e-6)
                z = torch.complex(y[..., first], y[..., second]) * turn
                ys.append(y.index_copy(-1, first, z.real).index_copy(-1, second, z.imag))
            if not case["train"]:
                return ys
            return [*[y.detach() for y in ys],
                    *torch.autograd.grad(ys, leaves, (s["dq"].double(), s["dk"].double()))]
    if kind == "gated":
        with torch.enable_grad():
            x, wg, wu = leaves = [s[n].detach().double().requires_grad_() for n in ("x", "wg", "wu")]
            g = torch.nn.functional.linear(x, wg)
            y = getattr(torch.nn.functional if case["act"] != "sigmoid" else torch, case["act"])(g) * \
                torch.nn.functional.linear(x, wu)
            if not case["train"]:
                return y.detach()
            return [y.detach(), *torch.autograd.grad(y, leaves, s["dy"].double())]
    # one step after another
    with torch.enable_grad():
        names = [n for n in ("q", "k", "v", "state") if s[n] is not None]
        leaves = {n: s[n].detach().double().requires_grad_(case.get("train", False)) for n in names}
        B, h, m = case["B"], case["H"], case["H"] // case["G"]
        state = leaves.get("state", torch.zeros(B, h, case["K"], case["V"], device="cuda", dtype=torch.float64))
        q, k, v = (leaves[n] if kind == "linear" else leaves[n][:, None] for n in ("q", "k", "v"))
        q, k, v = (x.unbind(1) for x in (q / math.sqrt(case["K"]), k.repeat_interleave(m, 2), v.repeat_interleave(m, 2)))
        a = s["decay"].double().exp()[:, None, None]
        outs = []
        for t, (qt, kt, vt) in enumerate(zip(q, k, v)):
            new = torch.addcmul(a * state, kt[..., None], vt[..., None, :])
            ot = torch.matmul(qt[..., None, :], new)[..., 0, :]
            if case.get("padded"):
                there = (t < s["lengths"])[:, None, None]
                new, ot = torch.where(there[..., None], new, state), torch.where(there, ot, 0.0)
            state = new
            outs.append(ot)
        if kind == "step":
            return [outs[0], state]
        o = torch.stack(outs, dim=1)
        if not case["train"]:
            return [o, state]
        ys, dys = ((o, state), (s["do"].double(), s["dstate"].double())) if case["state"] else ((o,), (s["do"].double(),))
        return [o.detach(), state.detach(), *torch.autograd.grad(ys, list(leaves.values()), dys)]
