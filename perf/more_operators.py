"""The rest of a training step around the experts' products and the output head, as a program that uses them would call them:
the gated feed-forward block (dense, over the experts' rows, and for single tokens), the embedding in front of it, and the
clipping of all gradients by their global norm.

A case is a dict of plain values. `op` names the path:

  gated          h = act(x Wg^T, x Wu^T), and the gate and up values for the backward pass where `keep` says so
  gated_dgrad    dh = dy W2, from it and the kept gate and up values their gradients, and h again (for W2's gradient)
  embed          rows of a table by token, times a scale
  embed_grad     the table's gradient: every row's tokens summed, zeros for rows without tokens, another gradient added or not
  clip           the norm over a list of gradients of both types, and every gradient times min(1, max_norm / norm)

E = 0: a dense block; otherwise rows grouped by expert, `unused` rows behind the last. act "silu": silu(g) u; "swiglu_oai": the clamped
form with its constants 1.702 and 7. `interleaved`: gate and up rows of the weights alternate instead of standing one below the other.
`masked`: share of tokens that are padding (id -1). Token ids are distributed as 1 / rank.
Where `own` is false, `run` computes the plain form in elementary torch operations.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_OPS = ("gated", "gated", "gated_dgrad", "gated_dgrad", "embed", "embed_grad", "embed_grad", "clip")
_ALPHA, _LIMIT = 1.702, 7.0
_GATED_FLOPS = 4.0 * 8192 * 4096 * 14336
_GATED_WEIGHTS = 128 * 2880 * 2880
_ROW_ELEMENTS = 65536 * 7168
_TABLE_ELEMENTS = 201088 * 2880 * 2
_CLIP_ELEMENTS = 1 << 30


def listed():
    return [
        # decode: one token through the gate and up projection of a dense block of the FP8 layer's sizes; the weights are all there is
        {"name": "gated_one", "op": "gated", "R": 1, "E": 0, "I": 2048, "K": 7168, "act": "silu", "interleaved": False, "keep": False},
        # decode of a batch: 48 tokens, a wide block
        {"name": "gated_few", "op": "gated", "R": 48, "E": 0, "I": 14336, "K": 4096, "act": "silu", "interleaved": False, "keep": False},
        # training step of a dense block, 8192 tokens: the largest product
        {"name": "gated_batch", "op": "gated", "R": 8192, "E": 0, "I": 14336, "K": 4096, "act": "silu", "interleaved": False,
         "keep": True},
        # gate and up projection of the GPT-OSS-like layer's experts in training: 4096 tokens of 4 choices, rows alternating, clamped
        {"name": "gated_experts", "op": "gated", "R": 16500, "E": 128, "I": 2880, "K": 2880, "act": "swiglu_oai", "interleaved": True,
         "keep": True, "unused": 116},
        # backward of a small dense block: odd number of tokens, one round of tiles
        {"name": "gated_dgrad_odd", "op": "gated_dgrad", "R": 1111, "E": 0, "I": 2816, "N": 1024, "act": "silu", "interleaved": False},
        # backward through the down projection on one of eight GPUs that share the DeepSeek-V3-like layer's 256 experts
        {"name": "gated_dgrad_experts", "op": "gated_dgrad", "R": 65536, "E": 32, "I": 2048, "N": 7168, "act": "silu",
         "interleaved": False, "unused": 0},
        # embedding of a short prompt: one launch of a few microseconds
        {"name": "embed_few", "op": "embed", "T": 17, "V": 129280, "H": 7168, "masked": 0.0, "scale": 1.0},
        # embedding of a long batch, scaled by the root of the width
        {"name": "embed_long", "op": "embed", "T": 32768, "V": 201088, "H": 2880, "masked": 0.1, "scale": 2880.0 ** 0.5},
        # gradient of a small model's table: most rows have no token
        {"name": "embed_grad_odd", "op": "embed_grad", "T": 1111, "V": 50257, "H": 1024, "masked": 0.1, "scale": 1.0, "out": "bf16",
         "add": False},
        # a tied table: the head's gradient in fp32 and the embedding's, a long batch with a few very frequent tokens
        {"name": "embed_grad_tied", "op": "embed_grad", "T": 32768, "V": 201088, "H": 2880, "masked": 0.1, "scale": 2880.0 ** 0.5,
         "out": "fp32", "add": True},
        # gradients of a small model: many tensors, a few hundred thousand elements in all
        {"name": "clip_small", "op": "clip", "tensors": 60, "elements": 300_000, "fp32": 0.5, "max_norm": 1.0},
        # gradients of a billion parameters in bf16, a few in fp32
        {"name": "clip_large", "op": "clip", "tensors": 310, "elements": 1 << 30, "fp32": 0.1, "max_norm": 1.0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(_OPS)
    while True:
        if op in ("gated", "gated_dgrad"):
            E = rng.choice([0, 0, _log_int(rng, 2, 128)])
            R = _log_int(rng, 1, 65536 if E else 8192)
            wide = 8 * _log_int(rng, 64, 896)
            case = {"op": op, "R": R, "E": E, "I": 8 * _log_int(rng, 32, 1792), "act": rng.choice(["silu", "swiglu_oai"]),
                    "interleaved": rng.random() < 0.5}
            if op == "gated":
                case |= {"K": wide, "keep": rng.random() < 0.5}
            else:
                case |= {"N": wide}
            if E:
                case["unused"] = rng.choice([0, R // 10])
            flops = (4.0 if op == "gated" else 2.0) * R * case["I"] * wide
            if flops <= _GATED_FLOPS and max(1, E) * case["I"] * wide <= _GATED_WEIGHTS and R * case["I"] <= 8192 * 14336:
                return case
        elif op == "clip":
            return {"op": op, "tensors": _log_int(rng, 1, 400), "elements": _log_int(rng, 1000, _CLIP_ELEMENTS),
                    "fp32": rng.choice([0.0, 0.1, 0.5, 1.0]), "max_norm": rng.choice([0.1, 1.0, 1e6])}
        else:
            case = {"op": op, "T": _log_int(rng, 1, 65536), "V": _log_int(rng, 1000, 201088), "H": 8 * _log_int(rng, 64, 896),
                    "masked": rng.choice([0.0, 0.1, 0.5])}
            case["scale"] = rng.choice([1.0, case["H"] ** 0.5])
            cells = case["V"] * case["H"]
            if op == "embed_grad":
                case |= {"out": rng.choice(["bf16", "fp32"]), "add": rng.random() < 0.5}
                cells *= (2 if case["out"] == "fp32" else 1) * (2 if case["add"] else 1)
            if case["T"] * case["H"] <= _ROW_ELEMENTS and cells <= _TABLE_ELEMENTS:
                return case


# ------------------------------------------------------------------------------------------------ inputs

def _randn(g, *shape, std=1.0, dtype=torch.bfloat16):
    t = torch.empty(shape, dtype=dtype, device="cuda")
    t.normal_(0.0, std, generator=g)
    return t


def _zeros(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype, device="cuda")


def _offsets(g, R, E, unused):
    """Offsets of E experts of uneven popularity over the first R - unused rows; a few experts have none."""
    share = torch.randn(E, device="cuda", generator=g).mul_(0.5).exp_()
    share[torch.rand(E, device="cuda", generator=g) < 0.05] = 0
    if float(share.sum()) == 0:
        share[:] = 1
    rows = torch.sort(torch.multinomial(share, R - unused, replacement=True, generator=g)).values
    return torch.searchsorted(rows, torch.arange(E + 1, device="cuda")).to(torch.int32)


def _ids(g, T, V, masked):
    """Token ids, the r-th most frequent one with a share of about 1 / (r log V), in an order of frequency of its own; -1: padding."""
    u = torch.rand(T, device="cuda", generator=g, dtype=torch.float64)
    rank = torch.exp(u * math.log(V + 1)).long().sub_(1).clamp_(0, V - 1)
    ids = torch.randperm(V, device="cuda", generator=g)[rank]
    ids[torch.rand(T, device="cuda", generator=g) < masked] = -1
    return ids


def _sizes(case):
    """Lengths of the list's tensors: matrices of a few sizes and, one in three, vectors; odd ones among them."""
    n, total = case["tensors"], case["elements"]
    shares = [1e-4 if i % 3 == 2 else 1.0 + (i * 7 % 5) for i in range(n)]
    scale = total / sum(shares)
    return [max(1, int(s * scale)) for s in shares]


def _is_fp32(case, i):
    return (i * 0.618034) % 1.0 < case["fp32"]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    s = {"case": case}
    if op in ("gated", "gated_dgrad"):
        R, E, I = case["R"], case["E"], case["I"]
        s["offsets"] = _offsets(g, R, E, case["unused"]) if E else None
        stack = (E,) if E else ()
        if op == "gated":
            K = case["K"]
            s["x"] = _randn(g, R, K)
            s["w13"] = _randn(g, *stack, 2 * I, K, std=1.5 * K ** -0.5)
            s["h"] = _zeros(R, I)
            s["gate_up"] = _zeros(R, 2 * I) if case["keep"] else None
        else:
            N = case["N"]
            s["dy"] = _randn(g, R, N, std=0.01)
            s["w2"] = _randn(g, *stack, N, I, std=I ** -0.5)
            s["gate_up"] = _randn(g, R, 2 * I, std=1.5)
            s["dgate_up"] = _zeros(R, 2 * I)
            s["h"] = _zeros(R, I)
    elif op == "clip":
        # the tensors are pieces of one flat buffer of each type, as programs that exchange gradients hold them; each begins at a
        # multiple of 64 elements
        sizes = _sizes(case)
        types = [torch.float32 if _is_fp32(case, i) else torch.bfloat16 for i in range(len(sizes))]
        flat, out, at = {}, {}, {torch.float32: 0, torch.bfloat16: 0}
        starts = []
        for n, t in zip(sizes, types):
            starts.append(at[t])
            at[t] += (n + 63) // 64 * 64
        for t, n in at.items():
            flat[t], out[t] = _zeros(n, dtype=t), _zeros(n, dtype=t)
        s["grads"] = [flat[t][a:a + n] for n, t, a in zip(sizes, types, starts)]
        outs = [out[t][a:a + n] for n, t, a in zip(sizes, types, starts)]
        for i, grad in enumerate(s["grads"]):
            grad.normal_(0.0, 10.0 ** (-3 + i % 3), generator=g)
        s["flat"] = [flat[t] for t in flat if at[t]]
        s["out"] = [out[t] for t in out if at[t]]
        s["norm"] = _zeros(1, dtype=torch.float32)
        if own:
            from hipkittens_amd import tk_kernel as tk
            s["plan"] = tk.GradTensors(s["grads"], outs)
            s["workspace"] = torch.empty(tk.grad_norm_workspace_bytes(), dtype=torch.uint8, device="cuda")
    else:
        T, V, H = case["T"], case["V"], case["H"]
        s["ids"] = _ids(g, T, V, case["masked"])
        if op == "embed":
            s["table"] = _randn(g, V, H, std=0.02)
            s["out"] = _zeros(T, H)
        else:
            dtype = torch.float32 if case["out"] == "fp32" else torch.bfloat16
            s["dout"] = _randn(g, T, H, std=0.01)
            s["add"] = _randn(g, V, H, std=0.01, dtype=dtype) if case["add"] else None
            s["dtable"] = _zeros(V, H, dtype=dtype)
            if own:
                from hipkittens_amd import tk_kernel as tk
                s["workspace"] = torch.empty(tk.embedding_backward_workspace_bytes(T, V, H), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    return s


# --------------------------------------------------------------------------------------------------- run

def _run_own(s):
    from hipkittens_amd import tk_kernel as tk
    case = s["case"]
    op = case["op"]
    if op == "gated":
        tk.dispatch_gated_gemm(s["x"], s["w13"], s["h"], s["gate_up"], expert_offsets=s["offsets"], interleaved=case["interleaved"],
                               activation=case["act"], alpha=_ALPHA, limit=_LIMIT)
        return (s["h"], s["gate_up"]) if case["keep"] else s["h"]
    if op == "gated_dgrad":
        tk.dispatch_gated_gemm_dgrad(s["dy"], s["w2"], s["gate_up"], s["dgate_up"], s["h"], expert_offsets=s["offsets"],
                                     interleaved=case["interleaved"], activation=case["act"], alpha=_ALPHA, limit=_LIMIT)
        return s["dgate_up"], s["h"]
    if op == "embed":
        tk.dispatch_embedding(s["ids"], s["table"], s["out"], scale=case["scale"])
        return s["out"]
    if op == "embed_grad":
        tk.dispatch_embedding_backward(s["ids"], s["dout"], s["dtable"], s["workspace"], scale=case["scale"], add=s["add"])
        return s["dtable"]
    tk.dispatch_grad_norm(s["plan"], s["norm"], s["workspace"])
    tk.dispatch_grad_clip(s["plan"], s["norm"], case["max_norm"])
    return s["norm"], s["out"]


def _experts(s):
    """(rows, expert) of the groups; a dense block is one group without an expert."""
    if s["offsets"] is None:
        return [(slice(0, s["case"]["R"]), None)]
    off = s["offsets"].tolist()
    return [(slice(a, b), e) for e, (a, b) in enumerate(zip(off, off[1:])) if b > a]


def _of(w, e):
    return (w if e is None else w[e]).float()


def run(s):
    if own:
        return _run_own(s)
    case = s["case"]
    op = case["op"]
    if op == "gated":
        R, I = case["R"], case["I"]
        h = _zeros(R, I)
        gate_up = _zeros(R, 2 * I) if case["keep"] else None
        for rows, e in _experts(s):
            gu = s["x"][rows].float() @ _of(s["w13"], e).t()
            if case["keep"]:
                gate_up[rows] = gu.bfloat16()
            g, u = (gu[:, 0::2], gu[:, 1::2]) if case["interleaved"] else (gu[:, :I], gu[:, I:])
            if case["act"] == "silu":
                h[rows] = (g / (1 + torch.exp(-g)) * u).bfloat16()
            else:
                g, u = g.clamp(max=_LIMIT), u.clamp(-_LIMIT, _LIMIT)
                h[rows] = ((u + 1) * (g / (1 + torch.exp(-_ALPHA * g)))).bfloat16()
        return (h, gate_up) if case["keep"] else h
    if op == "gated_dgrad":
        R, I = case["R"], case["I"]
        h, dgate_up = _zeros(R, I), _zeros(R, 2 * I)
        for rows, e in _experts(s):
            dh = s["dy"][rows].float() @ _of(s["w2"], e)
            gu = s["gate_up"][rows].float()
            g, u = (gu[:, 0::2], gu[:, 1::2]) if case["interleaved"] else (gu[:, :I], gu[:, I:])
            if case["act"] == "silu":
                sig = 1 / (1 + torch.exp(-g))
                h[rows] = (g * sig * u).bfloat16()
                dg, du = dh * u * sig * (1 + g * (1 - sig)), dh * g * sig
            else:
                gc, uc = g.clamp(max=_LIMIT), u.clamp(-_LIMIT, _LIMIT)
                sig = 1 / (1 + torch.exp(-_ALPHA * gc))
                h[rows] = ((uc + 1) * gc * sig).bfloat16()
                dg = torch.where(g <= _LIMIT, dh * (uc + 1) * sig * (1 + _ALPHA * gc * (1 - sig)), 0.0)
                du = torch.where(u.abs() <= _LIMIT, dh * gc * sig, 0.0)
            if case["interleaved"]:
                dgate_up[rows] = torch.stack((dg, du), dim=2).reshape(-1, 2 * I).bfloat16()
            else:
                dgate_up[rows] = torch.cat((dg, du), dim=1).bfloat16()
        return dgate_up, h
    if op == "embed":
        rows = s["table"][s["ids"].clamp(min=0)].float() * case["scale"]
        return torch.where(s["ids"][:, None] >= 0, rows, 0.0).bfloat16()
    if op == "embed_grad":
        V, H = case["V"], case["H"]
        live = torch.nonzero(s["ids"] >= 0).squeeze(1)
        sums = torch.zeros(V, H, dtype=torch.float32, device="cuda")
        sums.index_add_(0, s["ids"][live], s["dout"][live].float())
        sums *= case["scale"]
        if case["add"]:
            sums += s["add"].float()
        return sums.to(s["dtable"].dtype)
    squares = [(t.double() * t.double()).sum() for t in s["grads"]]
    norm = torch.stack(squares).sum().sqrt().float().reshape(1)
    factor = (case["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    return norm, [(t.float() * factor).to(t.dtype) for t in s["flat"]]


# ------------------------------------------------------------------------------------------- work, exact

def _distinct(T, V):
    """Rows of the table that T tokens are expected to name."""
    k = np.arange(1, V + 1, dtype=np.float64)
    p = np.log1p(1.0 / k) / math.log(V + 1)
    return float(-np.expm1(T * np.log1p(-np.minimum(p, 1 - 1e-12))).sum())


def work(case):
    op = case["op"]
    if op in ("gated", "gated_dgrad"):
        E, I, R = case["E"], case["I"], case["R"] - case.get("unused", 0)
        used = min(E, R) if E else 1   # experts without rows need not be read
        if op == "gated":
            K = case["K"]
            return {"bytes": 2.0 * R * K + 4.0 * used * I * K + (6.0 if case["keep"] else 2.0) * R * I, "flops": 4.0 * R * I * K}
        N = case["N"]
        return {"bytes": 2.0 * R * N + 2.0 * used * I * N + 10.0 * R * I, "flops": 2.0 * R * I * N}
    if op == "clip":
        size = sum(n * (4.0 if _is_fp32(case, i) else 2.0) for i, n in enumerate(_sizes(case)))
        return {"bytes": 2.0 * size, "flops": 3.0 * sum(_sizes(case))}
    T, V, H = case["T"] * (1.0 - case["masked"]), case["V"], case["H"]
    if op == "embed":
        return {"bytes": 8.0 * case["T"] + 2.0 * H * (_distinct(T, V) + case["T"]), "flops": T * H}
    cell = 4.0 if case["out"] == "fp32" else 2.0
    return {"bytes": 8.0 * case["T"] + 2.0 * T * H + cell * V * H * (2 if case["add"] else 1), "flops": T * H}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    f64 = torch.float64
    if op in ("gated", "gated_dgrad"):
        R, I, silu = case["R"], case["I"], case["act"] == "silu"
        bounds = [0, R] if s["offsets"] is None else s["offsets"].tolist()
        at_gate = slice(0, None, 2) if case["interleaved"] else slice(0, I)
        at_up = slice(1, None, 2) if case["interleaved"] else slice(I, 2 * I)
        h = torch.zeros(R, I, dtype=f64, device="cuda")
        wide = torch.zeros(R, 2 * I, dtype=f64, device="cuda") if op == "gated_dgrad" or case["keep"] else None
        for e in range(len(bounds) - 1):
            for a in range(bounds[e], bounds[e + 1], 4096):   # some thousand rows at a time
                rows = slice(a, min(a + 4096, bounds[e + 1]))
                if op == "gated":
                    w = (s["w13"] if s["offsets"] is None else s["w13"][e]).to(f64)
                    both = torch.mm(s["x"][rows].to(f64), w.t())
                    if case["keep"]:
                        wide[rows] = both
                else:
                    both = s["gate_up"][rows].to(f64)
                g, u = both[:, at_gate], both[:, at_up]
                top = g if silu else torch.minimum(g, torch.full_like(g, _LIMIT))
                lin = u if silu else torch.minimum(torch.maximum(u, torch.full_like(u, -_LIMIT)), torch.full_like(u, _LIMIT)) + 1
                sig = torch.sigmoid(top if silu else _ALPHA * top)
                h[rows] = lin * top * sig
                if op == "gated_dgrad":
                    w = (s["w2"] if s["offsets"] is None else s["w2"][e]).to(f64)
                    dh = torch.mm(s["dy"][rows].to(f64), w)
                    slope = sig + top * sig * (1 - sig) * (1.0 if silu else _ALPHA)
                    wide[rows, at_gate] = dh * lin * slope * (1.0 if silu else (g <= _LIMIT).to(f64))
                    wide[rows, at_up] = dh * top * sig * (1.0 if silu else (u.abs() <= _LIMIT).to(f64))
        if op == "gated":
            return (h, wide) if case["keep"] else h
        return wide, h
    if op == "embed":
        out = torch.zeros(case["T"], case["H"], dtype=f64, device="cuda")
        ok = s["ids"] >= 0
        out[ok] = s["table"][s["ids"][ok]].to(f64) * case["scale"]
        return out
    if op == "embed_grad":
        # tokens in the order of their ids, a row's as the difference of the running sums at its ends, some columns at a time
        V, H = case["V"], case["H"]
        ids, order = torch.sort(s["ids"], stable=True)
        ends = torch.searchsorted(ids, torch.arange(-1, V, device="cuda"), right=True)
        out = s["add"].to(f64) if case["add"] else torch.zeros(V, H, dtype=f64, device="cuda")
        for c in range(0, H, 512):
            running = torch.zeros(case["T"] + 1, min(512, H - c), dtype=f64, device="cuda")
            torch.cumsum(s["dout"][order, c:c + 512].to(f64), dim=0, out=running[1:])
            out[:, c:c + 512] += (running[ends[1:]] - running[ends[:-1]]) * case["scale"]
        return out
    total = sum((t.to(f64) ** 2).sum() for t in s["grads"])
    norm = torch.sqrt(total).reshape(1)
    factor = torch.minimum(case["max_norm"] / (norm + 1e-6), torch.ones_like(norm))
    return norm, [t.to(f64) * factor for t in s["flat"]]
