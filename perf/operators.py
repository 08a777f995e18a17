"""The operators of a language model around the block stack, and what a pass through each has to do.

Four kinds of call, each over the sizes, data types and options it is used with:

* ``embed`` -- ``embedding``: rows of a table for token ids, scaled; for training
               with the table's dense gradient
* ``norm``  -- ``layer_norm`` over the last dimension; for training with the
               gradients of the input, the weight and the bias
* ``clip``  -- ``clip_grad_norm_``: the norm over all gradients of a model, and
               the gradients scaled in place
* ``beam``  -- ``beam_search_step``: the best continuations over beams and
               vocabulary, and the recurrent states in the new beams' order

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
        # the next token of 256 streams at d_model 2048 (the decode configuration):
        # nothing but latency
        dict(name="embed_decode", kind="embed", train=False, B=256, T=1, D=2048, V=32768, dtype="bf16", pad=False),
        # the 12-layer stack's batch (16 x 2048 tokens, d_model 768) from its table
        dict(name="embed_train", kind="embed", train=True, B=16, T=2048, D=768, V=32768, dtype="bf16", pad=False),
        # padded documents in full precision, nothing a power of two
        dict(name="embed_odd", kind="embed", train=True, B=3, T=1237, D=1001, V=50001, dtype="fp32", pad=True),
        # a norm between two decode steps: 256 rows, no gradient
        dict(name="norm_decode", kind="norm", train=False, R=256, D=2048, dtype="bf16", pdtype="bf16", bias=True),
        # a block's pre-norm in the 12-layer stack, forward and backward
        dict(name="norm_train", kind="norm", train=True, R=32768, D=768, dtype="bf16", pdtype="bf16", bias=True),
        # rows that no vector width divides, full precision, a weight alone
        dict(name="norm_odd", kind="norm", train=True, R=3711, D=1001, dtype="fp32", pdtype="fp32", bias=False),
        # a norm over the mixer's width in the stack (2 * 768 * 16 channels), with
        # the parameters kept in full precision
        dict(name="norm_wide", kind="norm", train=True, R=8192, D=24576, dtype="bf16", pdtype="fp32", bias=True),
        # one layer's mixer parameters and its small projections, in full
        # precision: launches and host work
        dict(name="clip_small", kind="clip", layers=1, D=64, N=16, dtype="fp32", clips=True),
        # all gradients of the 12-layer stack (d_model 768, 16 states a channel)
        dict(name="clip_stack", kind="clip", layers=12, D=768, N=16, dtype="bf16", clips=True),
        # one prompt, four beams, the states of the 12-layer stack
        dict(name="beam_one", kind="beam", B=1, K=4, V=32768, layers=12, M=12288, dtype="bf16", first=False,
             in_place=False),
        # 32 prompts at an odd vocabulary, logits in full precision, states in place
        dict(name="beam_odd", kind="beam", B=32, K=5, V=50001, layers=3, M=3000, dtype="fp32", first=False,
             in_place=True),
        # a serving batch: 1024 beams over a large vocabulary, d_model 2048 with 16 states
        dict(name="beam_large", kind="beam", B=128, K=8, V=131072, layers=2, M=32768, dtype="bf16", first=False,
             in_place=False),
    ]


def _off(n):
    """n, or its neighbour where n is 3 * 2^10 or a multiple of it."""
    return n if n % 3072 else n - 1


def _log(rng, lo, hi):
    """A whole number between lo and hi, evenly spread over its logarithm."""
    return _off(max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))))


def draw(rng):
    kind = rng.choice(("embed", "embed", "norm", "norm", "clip", "beam", "beam"))
    dtype = rng.choice(("fp32", "bf16"))
    if kind == "embed":
        d, v = _log(rng, 32, 4096), _log(rng, 250, 131072)
        if rng.random() < 0.7:
            d = d // 40 * 40 if d >= 40 else 32
        while v * d > 1 << 26:
            v = _off(v // 2)
        n = min(_log(rng, 1, 65536), (1 << 26) // d)
        b = _log(rng, 1, min(n, 64))
        return dict(kind=kind, train=rng.random() < 0.7, B=b, T=_off(n // b), D=d, V=v, dtype=dtype, pad=rng.random() < 0.3)
    if kind == "norm":
        d = _log(rng, 32, 32768)
        if rng.random() < 0.7:
            d = d // 40 * 40 if d >= 40 else 32
        r = _off(min(_log(rng, 1, 65536), 100_000_000 // d))
        return dict(kind=kind, train=rng.random() < 0.7, R=r, D=d, dtype=dtype, pdtype=rng.choice((dtype, "fp32")),
                    bias=rng.random() < 0.7)
    if kind == "clip":
        n, d = rng.choice((4, 8, 16)), _log(rng, 33, 1024) | 1
        layers = _log(rng, 1, 24)
        while layers * 4 * d * d * n > 1 << 27:
            layers, d = max(1, layers // 2), d * 3 // 4 | 1
        return dict(kind=kind, layers=layers, D=d, N=n, dtype=dtype, clips=rng.random() < 0.7)
    k, v, b = _log(rng, 1, 32), _log(rng, 250, 131072), _log(rng, 1, 256)
    while b * k * v > 1 << 26:
        b = max(1, b // 2)
    layers, m = _log(rng, 1, 24), _log(rng, 64, 32768)
    if rng.random() < 0.7:
        m = m // 80 * 80 if m >= 80 else 64
    while b * k * layers * m > 1 << 25:
        layers, m = max(1, layers // 2), _off(max(64, m // 2))
    return dict(kind=kind, B=b, K=k, V=v, layers=layers, M=m, dtype=dtype, first=rng.random() < 0.2,
                in_place=rng.random() < 0.5)


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


def _shapes(layers, d, n):
    """The parameters of the block stack: per block the norm, the two projections
    and the mixer's; the last norm."""
    w = 2 * d * n
    block = [(d,), (w, d), (d, w), *[(w // 2,)] * 2, *[(w + 1,)] * 2, *[(w // 2,)] * 4]
    return block * layers + [(d,)]


def _grad_sizes(case):
    """Shapes, starts in one buffer (each at a multiple of 128 values, as separate
    allocations would start) and the buffer's length."""
    shapes, starts, at = _shapes(case["layers"], case["D"], case["N"]), [], 0
    for s in shapes:
        starts.append(at)
        at += -(-math.prod(s) // 128) * 128
    return shapes, starts, at


def _embed_scale(case):
    return math.sqrt(case["D"])


def prepare(case, seed):
    r, dt, kind = _Inputs(seed), DTYPES[case["dtype"]], case["kind"]
    s = {"case": case}
    if kind == "embed":
        b, t, d, v = case["B"], case["T"], case["D"], case["V"]
        # words by their rank: the share of the k-th most frequent falls as 1 / k
        rank = torch.exp(r.rand(b, t) * math.log(v + 1)).long().sub_(1).clamp_(0, v - 1)
        s["tokens"] = (rank * 7919 + 11) % v
        if case["pad"]:  # documents of different lengths, filled up with id 0
            length = (r.rand(b, 1) * t).long()
            s["tokens"] = torch.where(torch.arange(t, device="cuda") <= length, s["tokens"], 0)
        s["weight"] = r.randn(v, d, dtype=dt, scale=d ** -0.5)
        if case["train"]:
            s["weight"].requires_grad_()
            s["dy"] = r.randn(b, t, d, dtype=dt)
    elif kind == "norm":
        rows, d, pdt = case["R"], case["D"], DTYPES[case["pdtype"]]
        s["x"] = r.randn(rows, d, dtype=dt, scale=1.7, mean=0.4)
        s["weight"] = r.randn(d, dtype=pdt, scale=0.2, mean=1.0)
        s["bias"] = r.randn(d, dtype=pdt, scale=0.1) if case["bias"] else None
        if case["train"]:
            s["inputs"] = [t.requires_grad_() for t in (s["x"], s["weight"], s["bias"]) if t is not None]
            s["dy"] = r.randn(rows, d, dtype=dt)
    elif kind == "clip":
        shapes, starts, total = _grad_sizes(case)
        s["flat"] = torch.zeros(total, device="cuda", dtype=dt)
        s["params"] = []
        for shape, at in zip(shapes, starts):
            p = torch.nn.Parameter(torch.zeros(shape, device="cuda", dtype=dt))
            p.grad = s["flat"][at:at + p.numel()].view(shape)
            p.grad.copy_(r.randn(*shape, dtype=dt, scale=0.02))
            s["params"].append(p)
        norm = 0.02 * math.sqrt(sum(math.prod(x) for x in shapes))
        s["limit"] = (0.5 if case["clips"] else 1e4) * norm
    else:
        b, k, v = case["B"], case["K"], case["V"]
        s["logits"] = r.randn(b, k, v, scale=3.0).to(dt)
        scores = -torch.cumsum(r.rand(b, k) * 2.0, dim=1) - 20.0 * r.rand(b, 1)
        s["finished"] = r.rand(b, k) < 0.1
        if case["first"]:  # before the first token every beam but one is empty
            scores[:, 0], scores[:, 1:] = 0.0, -math.inf
            s["finished"] = torch.zeros_like(s["finished"])
        s["scores"], s["eos"] = scores, v // 3
        s["states"] = [tuple(r.randn(b * k, case["M"], scale=0.1) for _ in range(2)) for _ in range(case["layers"])]
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return (_own if own else _plain)(state, state["case"])


def _limit(state):
    """The norm that this pass clips to: a little less from pass to pass, so that
    each of them scales the gradients that the one before it has clipped."""
    if state["case"]["clips"]:
        state["limit"] *= 0.9999
    return state["limit"]


def _own(s, case):
    import sparc_amd
    kind = case["kind"]
    if kind == "embed":
        pad = 0 if case["pad"] else None
        y = sparc_amd.embedding(s["tokens"], s["weight"], scale=_embed_scale(case), padding_idx=pad)
        if not case["train"]:
            return y
        return [y.detach(), *torch.autograd.grad(y, [s["weight"]], s["dy"])]
    if kind == "norm":
        y = sparc_amd.layer_norm(s["x"], s["weight"], s["bias"], eps=1e-5)
        if not case["train"]:
            return y
        return [y.detach(), *torch.autograd.grad(y, s["inputs"], s["dy"])]
    if kind == "clip":
        norm = sparc_amd.clip_grad_norm_(s["params"], _limit(s))
        return {"norm": norm, "grads": s["flat"]}
    step = sparc_amd.beam_search_step(s["logits"], s["scores"], finished=s["finished"], eos_id=s["eos"],
                                      states=s["states"], out_states=s["states"] if case["in_place"] else None)
    return {"tokens": step.tokens, "parents": step.parents, "scores": step.scores, "finished": step.finished,
            "states": step.states}


def _plain(s, case):
    kind = case["kind"]
    if kind == "embed":
        tok, w, scale = s["tokens"].reshape(-1), s["weight"].detach(), _embed_scale(case)
        y = (w[tok].float() * scale).to(w.dtype).view(*s["tokens"].shape, -1)
        if not case["train"]:
            return y
        dy = s["dy"].reshape(len(tok), -1).float() * scale
        if case["pad"]:
            dy = dy * (tok != 0)[:, None]
        return [y, torch.zeros(w.shape, device="cuda").index_add_(0, tok, dy).to(w.dtype)]
    if kind == "norm":
        x = s["x"].detach().float()
        w = s["weight"].detach().float()
        c = x - x.mean(-1, keepdim=True)
        rstd = 1.0 / torch.sqrt((c * c).mean(-1, keepdim=True) + 1e-5)
        xhat = c * rstd
        y = xhat * w
        if case["bias"]:
            y = y + s["bias"].detach().float()
        y = y.to(s["x"].dtype)
        if not case["train"]:
            return y
        dy = s["dy"].float()
        g = dy * w
        dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
        out = [y, dx.to(s["x"].dtype), (dy * xhat).sum(0).to(s["weight"].dtype)]
        return [*out, dy.sum(0).to(s["bias"].dtype)] if case["bias"] else out
    if kind == "clip":
        limit = _limit(s)
        norm = torch.stack([p.grad.float().square().sum() for p in s["params"]]).sum().sqrt()
        factor = (limit / (norm + 1e-6)).clamp(max=1.0)
        [p.grad.copy_(p.grad.float() * factor) for p in s["params"]]
        return {"norm": norm, "grads": s["flat"]}
    b, k, v = case["B"], case["K"], case["V"]
    x, done = s["logits"].float(), s["finished"]
    top = x.amax(-1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    cand = s["scores"][..., None] + (x - lse)
    cand = torch.where(done[..., None], -math.inf, cand)
    cand[..., s["eos"]] = torch.where(done, s["scores"], cand[..., s["eos"]])
    scores, at = torch.sort(cand.view(b, k * v), dim=-1, descending=True, stable=True)
    scores, at = scores[:, :k].clone(), at[:, :k]
    parents, tokens = at // v, at % v
    rows = (parents + k * torch.arange(b, device="cuda")[:, None]).reshape(-1)
    states = [tuple(p[rows] for p in layer) for layer in s["states"]]
    if case["in_place"]:
        states = [tuple(p.copy_(q) for p, q in zip(*both)) for both in zip(s["states"], states)]
    return {"tokens": tokens, "parents": parents, "scores": scores,
            "finished": done.gather(1, parents) | (tokens == s["eos"]), "states": states}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    """Inputs read once, outputs and gradients written once."""
    kind, es = case["kind"], 2 if case["dtype"] == "bf16" else 4
    if kind == "embed":
        n, d, v = case["B"] * case["T"], case["D"], case["V"]
        fwd = 8 * n + (min(n, v) + n) * d * es
        return {"bytes": fwd + ((n + v) * d * es if case["train"] else 0), "flops": n * d * (3 if case["train"] else 1)}
    if kind == "norm":
        el, ps = case["R"] * case["D"], 2 if case["pdtype"] == "bf16" else 4
        params = case["D"] * ps * (2 if case["bias"] else 1)
        if case["train"]:  # x in, y out; x, dy in, dx out; the parameters and their gradients
            return {"bytes": 5 * el * es + 3 * params, "flops": 20 * el}
        return {"bytes": 2 * el * es + params, "flops": 8 * el}
    if kind == "clip":
        n = sum(math.prod(x) for x in _shapes(case["layers"], case["D"], case["N"]))
        return {"bytes": n * es * (2 if case["clips"] else 1), "flops": n * (3 if case["clips"] else 2)}
    rows = case["B"] * case["K"]
    return {"bytes": rows * (case["V"] * es + 16 * case["layers"] * case["M"] + 31), "flops": 5 * rows * case["V"]}


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "embed":
        tok, w = s["tokens"], s["weight"].detach().double() * _embed_scale(case)
        y = torch.nn.functional.one_hot(tok, case["V"]).double() @ w if tok.numel() * case["V"] < 1 << 22 else \
            torch.gather(w, 0, tok.reshape(-1, 1).expand(-1, case["D"])).view(*tok.shape, -1)
        if not case["train"]:
            return y
        keep = tok.reshape(-1) != (0 if case["pad"] else -1)
        rows = (s["dy"].double() * _embed_scale(case)).reshape(-1, case["D"])[keep]
        at = tok.reshape(-1)[keep][:, None].expand(-1, case["D"])
        return [y, torch.zeros_like(w).scatter_add_(0, at, rows)]
    if kind == "norm":
        x, w = s["x"].detach().double(), s["weight"].detach().double()
        var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
        sd = torch.sqrt(var + 1e-5)
        xhat = (x - mean) / sd
        y = torch.addcmul(s["bias"].detach().double(), xhat, w) if case["bias"] else xhat * w
        if not case["train"]:
            return y
        dy = s["dy"].double()
        g = dy * w
        along = torch.linalg.vecdot(g, xhat)[:, None] * xhat + g.sum(-1, keepdim=True)
        grads = [(g - along / case["D"]) / sd, torch.einsum("rd,rd->d", dy, xhat)]
        return [y, *grads, dy.sum(0)] if case["bias"] else [y, *grads]
    if kind == "clip":
        flat = s["flat"].double()
        norm = torch.dot(flat, flat).sqrt()
        return {"norm": norm, "grads": flat * min(1.0, _limit(s) / (float(norm) + 1e-6))}
    logp = torch.log_softmax(s["logits"].double(), dim=-1)
    done = s["finished"][..., None]
    ends = torch.arange(case["V"], device="cuda") == s["eos"]
    logp = torch.where(done, torch.where(ends, 0.0, -math.inf), logp)
    best = (s["scores"].double()[..., None] + logp).flatten(1).topk(case["K"], dim=-1).values
    return {"tokens": None, "parents": None, "scores": best, "finished": None,
            "states": [(None, None) for _ in range(case["layers"])]}
