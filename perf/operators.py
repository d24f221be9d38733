"""Training next to the MoE layers and the bf16 GEMM: tokens to their experts and back, the experts' products and the output
head with its loss, each with its gradient, as a program that uses them would call them.

A case is a dict of plain values. `op` names the path:

  permute             rows of x copied to their places in the order of the experts
  permute_backward    the gradient of that: every token's rows of the experts' order summed, with a residual or without
  unpermute_backward  the gradient of the weighted sum over a token's experts: of the experts' rows and of the weights
  experts             y = x W[e]^T for the rows of each expert
  experts_dgrad       dx = dy W[e]
  experts_wgrad       dW[e] = dy^T x over the rows of each expert, in bf16 or fp32
  head_loss           log-sum-exp and cross entropy of the logits x W^T, one loss per row
  head_grad           the same and, from the losses' gradients, those of x and W

Rows of T tokens with k choices each are routed over E experts; `masked` is the share of tokens (or labels) that are padding.
Where `own` is false, `run` computes the plain form in elementary torch operations.
"""
from __future__ import annotations

import math

import torch

own = False

_ROUTED = ("permute", "permute_backward", "unpermute_backward")
_EXPERTS = ("experts", "experts_dgrad", "experts_wgrad")
_HEAD = ("head_loss", "head_grad")
_ROW_ELEMENTS = 8192 * 8 * 7168          # the largest permuted buffer that is drawn: the listed one
_EXPERT_FLOPS = 2.0 * 65536 * 4096 * 7168
_EXPERT_WEIGHTS = 128 * 5760 * 2880
_HEAD_FLOPS = 2.0 * 8192 * 129280 * 7168
_HEAD_GRAD_FLOPS = 6.0 * 4096 * 201088 * 2880


def listed():
    return [
        # decode step or a very short sequence: one launch of a few microseconds
        {"name": "permute_few", "op": "permute", "T": 4, "k": 4, "E": 128, "H": 2880, "masked": 0.0},
        # a batch of 8192 tokens of the DeepSeek-V3-like layer: 0.9 GB written
        {"name": "permute_long", "op": "permute", "T": 8192, "k": 8, "E": 256, "H": 7168, "masked": 0.0},
        # backward of the GPT-OSS-like layer's permute, a tenth of the tokens padding, the router's gradient added
        {"name": "permute_backward", "op": "permute_backward", "T": 4096, "k": 4, "E": 128, "H": 2880, "masked": 0.1,
         "add": True},
        # backward of the DeepSeek-V3-like layer's weighted sum, a ragged number of tokens
        {"name": "unpermute_backward", "op": "unpermute_backward", "T": 8001, "k": 8, "E": 256, "H": 7168, "masked": 0.0},
        # gate and up projection for 64 tokens on a quarter of the GPT-OSS-like layer's experts: the weights dominate
        {"name": "experts_few", "op": "experts", "R": 256, "E": 32, "N": 5760, "K": 2880, "unused": 0},
        # gate and up projection of the GPT-OSS-like layer, 4096 tokens: 128 rows an expert on average
        {"name": "experts_batch", "op": "experts", "R": 16384, "E": 128, "N": 5760, "K": 2880, "unused": 0},
        # one of eight GPUs that share the DeepSeek-V3-like layer's 256 experts, 8192 tokens on each: backward of gate and up
        {"name": "experts_dgrad_long", "op": "experts_dgrad", "R": 65536, "E": 32, "N": 4096, "K": 7168, "unused": 0},
        # weight gradient of the down projection of the GPT-OSS-like layer, fp32 as an optimiser takes it, unused rows behind
        {"name": "experts_wgrad", "op": "experts_wgrad", "R": 16500, "E": 128, "N": 2880, "K": 2880, "unused": 116,
         "out": "fp32"},
        # the loss of one short document
        {"name": "head_loss_short", "op": "head_loss", "M": 100, "V": 32000, "K": 2880, "masked": 0.0},
        # evaluation of 8192 tokens with a vocabulary of 129280
        {"name": "head_loss_long", "op": "head_loss", "M": 8192, "V": 129280, "K": 7168, "masked": 0.0},
        # a small model's training step: odd vocabulary, ragged number of rows
        {"name": "head_grad_odd", "op": "head_grad", "M": 1111, "V": 50257, "K": 1024, "masked": 0.1},
        # a training step of 4096 tokens with a vocabulary of 201088, prompt tokens without a loss
        {"name": "head_grad_long", "op": "head_grad", "M": 4096, "V": 201088, "K": 2880, "masked": 0.25},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(_ROUTED + _EXPERTS + _HEAD)
    while True:
        if op in _ROUTED:
            k = rng.randint(1, 8)
            case = {"op": op, "T": _log_int(rng, 1, 8192), "k": k, "E": _log_int(rng, max(2, k), 256),
                    "H": 8 * _log_int(rng, 64, 896), "masked": rng.choice([0.0, 0.1, 0.3])}
            if op == "permute_backward":
                case["add"] = rng.random() < 0.5
            if case["T"] * k * case["H"] <= _ROW_ELEMENTS:
                return case
        elif op in _EXPERTS:
            R = _log_int(rng, 1, 65536)
            case = {"op": op, "R": R, "E": _log_int(rng, 1, 128), "N": 8 * _log_int(rng, 64, 896),
                    "K": 8 * _log_int(rng, 64, 896), "unused": rng.choice([0, R // 10])}
            if op == "experts_wgrad":
                case["out"] = rng.choice(["bf16", "fp32"])
            if (2.0 * R * case["N"] * case["K"] <= _EXPERT_FLOPS and
                    case["E"] * case["N"] * case["K"] <= _EXPERT_WEIGHTS):
                return case
        else:
            case = {"op": op, "M": _log_int(rng, 1, 8192), "V": _log_int(rng, 1000, 201088), "K": 8 * _log_int(rng, 64, 896),
                    "masked": rng.choice([0.0, 0.1, 0.5])}
            flops = 2.0 * case["M"] * case["V"] * case["K"]
            if flops <= _HEAD_FLOPS if op == "head_loss" else 3 * flops <= _HEAD_GRAD_FLOPS:
                return case


# ------------------------------------------------------------------------------------------------ inputs

def _randn(g, *shape, std=1.0):
    t = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
    t.normal_(0.0, std, generator=g)
    return t


def _route(g, T, k, E, masked):
    """Top-k of noise around a popularity of the experts, padded tokens without experts, slots sorted by expert."""
    scores = torch.randn(T, E, device="cuda", generator=g) + 0.5 * torch.randn(E, device="cuda", generator=g)
    top, ids = scores.topk(k, dim=1)
    if masked:
        ids[torch.rand(T, device="cuda", generator=g) < masked] = -1
    ids = ids.to(torch.int32).reshape(-1)
    order = torch.sort(torch.where(ids < 0, E, ids), stable=True).indices
    slots = order[: int((ids >= 0).sum())]
    slot_to_pos = torch.full((T * k,), -1, dtype=torch.int32, device="cuda")
    slot_to_pos[slots] = torch.arange(slots.numel(), dtype=torch.int32, device="cuda")
    return slot_to_pos, torch.softmax(top, dim=1).contiguous()


def _offsets(g, R, E, unused):
    """Offsets of E experts of uneven popularity over the first R - unused rows; a few experts have none."""
    share = torch.randn(E, device="cuda", generator=g).mul_(0.5).exp_()
    share[torch.rand(E, device="cuda", generator=g) < 0.05] = 0
    if float(share.sum()) == 0:
        share[:] = 1
    rows = torch.sort(torch.multinomial(share, R - unused, replacement=True, generator=g)).values if R > unused else \
        torch.empty(0, dtype=torch.int64, device="cuda")
    return torch.searchsorted(rows, torch.arange(E + 1, device="cuda")).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    s = {"case": case}
    if op in _ROUTED:
        T, k, H = case["T"], case["k"], case["H"]
        s["slot_to_pos"], s["weights"] = _route(g, T, k, case["E"], case["masked"])
        if op == "permute":
            s["x"] = _randn(g, T, H)
            s["xp"] = torch.zeros(T * k, H, dtype=torch.bfloat16, device="cuda")
        elif op == "permute_backward":
            s["dxp"] = _randn(g, T * k, H)
            s["add"] = _randn(g, T, H) if case["add"] else None
            s["dx"] = torch.zeros(T, H, dtype=torch.bfloat16, device="cuda")
        else:
            s["dy"] = _randn(g, T, H)
            s["o"] = _randn(g, T * k, H)
            s["do"] = torch.zeros(T * k, H, dtype=torch.bfloat16, device="cuda")
            s["dweights"] = torch.zeros(T, k, dtype=torch.float32, device="cuda")
    elif op in _EXPERTS:
        R, E, N, K = case["R"], case["E"], case["N"], case["K"]
        s["offsets"] = _offsets(g, R, E, case["unused"])
        if op != "experts_wgrad":
            s["w"] = _randn(g, E, N, K, std=K ** -0.5 if op == "experts" else N ** -0.5)
        if op != "experts_dgrad":
            s["x"] = _randn(g, R, K)
        if op != "experts":
            s["dy"] = _randn(g, R, N)
        if op == "experts":
            s["y"] = torch.zeros(R, N, dtype=torch.bfloat16, device="cuda")
        elif op == "experts_dgrad":
            s["dx"] = torch.zeros(R, K, dtype=torch.bfloat16, device="cuda")
        else:
            s["dw"] = torch.zeros(E, N, K, dtype=torch.float32 if case["out"] == "fp32" else torch.bfloat16, device="cuda")
    else:
        M, V, K = case["M"], case["V"], case["K"]
        s["x"] = _randn(g, M, K)
        s["w"] = _randn(g, V, K, std=2.0 * K ** -0.5)
        labels = torch.randint(0, V, (M,), device="cuda", generator=g)
        labels[torch.rand(M, device="cuda", generator=g) < case["masked"]] = -100
        s["labels"] = labels
        s["loss"] = torch.zeros(M, dtype=torch.float32, device="cuda")
        s["lse"] = torch.zeros(M, dtype=torch.float32, device="cuda")
        if op == "head_grad":
            # a mean over the rows that count, rows weighted unevenly
            s["dloss"] = (0.5 + torch.rand(M, device="cuda", generator=g)) / max(1, int((labels >= 0).sum()))
            s["dx"] = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
            s["dw"] = torch.zeros(V, K, dtype=torch.bfloat16, device="cuda")
        if own:
            from hipkittens_amd import tk_kernel as tk
            n = tk.linear_cross_entropy_workspace_bytes(M, V, K, backward=op == "head_grad")
            s["workspace"] = torch.empty(n, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    return s


# --------------------------------------------------------------------------------------------------- run

def _run_own(s):
    from hipkittens_amd import tk_kernel as tk
    op = s["case"]["op"]
    if op == "permute":
        tk.dispatch_moe_permute(s["x"], s["slot_to_pos"], s["xp"])
        return s["xp"]
    if op == "permute_backward":
        tk.dispatch_moe_permute_backward(s["dxp"], s["slot_to_pos"], s["dx"], add=s["add"])
        return s["dx"]
    if op == "unpermute_backward":
        tk.dispatch_moe_unpermute_backward(s["dy"], s["o"], s["weights"], s["slot_to_pos"], s["do"], s["dweights"])
        return s["do"], s["dweights"]
    if op == "experts":
        tk.dispatch_moe_grouped_gemm(s["x"], s["w"], s["offsets"], s["y"])
        return s["y"]
    if op == "experts_dgrad":
        tk.dispatch_moe_grouped_gemm_dgrad(s["dy"], s["w"], s["offsets"], s["dx"])
        return s["dx"]
    if op == "experts_wgrad":
        tk.dispatch_moe_grouped_gemm_wgrad(s["dy"], s["x"], s["offsets"], s["dw"])
        return s["dw"]
    tk.dispatch_linear_cross_entropy(s["x"], s["w"], s["labels"], s["loss"], s["lse"], s["workspace"])
    if op == "head_loss":
        return s["loss"], s["lse"]
    tk.dispatch_linear_cross_entropy_backward(s["x"], s["w"], s["labels"], s["lse"], s["dloss"], s["dx"], s["dw"],
                                              s["workspace"])
    return s["loss"], s["lse"], s["dx"], s["dw"]


def run(s):
    if own:
        return _run_own(s)
    case = s["case"]
    op = case["op"]
    if op in _ROUTED:
        T, k, H = case["T"], case["k"], case["H"]
        pos = s["slot_to_pos"].long()
        live = torch.nonzero(pos >= 0).squeeze(1)
        at, token = pos[live], live // k
        if op == "permute":
            xp = torch.zeros(T * k, H, dtype=torch.bfloat16, device="cuda")
            xp[at] = s["x"][token]
            return xp
        if op == "permute_backward":
            dx = s["add"].float() if case["add"] else torch.zeros(T, H, device="cuda")
            p = pos.reshape(T, k)
            for j in range(k):   # one choice of every token at a time, in order
                dx += torch.where(p[:, j:j + 1] >= 0, s["dxp"][p[:, j].clamp(min=0)].float(), 0.0)
            return dx.bfloat16()
        dy = s["dy"].float()
        do = torch.zeros(T * k, H, dtype=torch.bfloat16, device="cuda")
        do[at] = (s["weights"].reshape(-1)[live, None] * dy[token]).bfloat16()
        dw = torch.zeros(T * k, device="cuda")
        dw[live] = (s["o"][at].float() * dy[token]).sum(dim=1)
        return do, dw.reshape(T, k)
    if op in _EXPERTS:
        off = s["offsets"].tolist()
        if op == "experts_wgrad":
            dw = torch.zeros(case["E"], case["N"], case["K"], device="cuda",
                             dtype=torch.float32 if case["out"] == "fp32" else torch.bfloat16)
            for e, (a, b) in enumerate(zip(off, off[1:])):
                if b > a:
                    dw[e] = s["dy"][a:b].float().t() @ s["x"][a:b].float()
            return dw
        src, width = (s["x"], case["N"]) if op == "experts" else (s["dy"], case["K"])
        out = torch.zeros(case["R"], width, dtype=torch.bfloat16, device="cuda")
        for e, (a, b) in enumerate(zip(off, off[1:])):
            if b > a:
                w = s["w"][e].float()
                out[a:b] = src[a:b].float() @ (w.t() if op == "experts" else w)
        return out
    x, w, labels = s["x"].float(), s["w"].float(), s["labels"]
    logits = x @ w.t()
    top = logits.max(dim=1, keepdim=True).values
    p = torch.exp(logits - top)
    z = p.sum(dim=1, keepdim=True)
    lse = top + torch.log(z)
    counts = labels >= 0
    at = labels.clamp(min=0)[:, None]
    loss = torch.where(counts, (lse - logits.gather(1, at)).squeeze(1), 0.0)
    if op == "head_loss":
        return loss, lse.squeeze(1)
    del logits
    scale = torch.where(counts, s["dloss"], 0.0)[:, None]
    dl = p.mul_(scale / z)
    dl.scatter_add_(1, at, -scale)
    return loss, lse.squeeze(1), (dl @ w).bfloat16(), (dl.t() @ x).bfloat16()


# ------------------------------------------------------------------------------------------- work, exact

def work(case):
    op = case["op"]
    if op in _ROUTED:
        T, S, H = case["T"], case["T"] * case["k"], case["H"]
        live = S * (1.0 - case["masked"])
        if op == "permute":
            return {"bytes": 2.0 * H * (T * (1.0 - case["masked"]) + live) + 4.0 * S, "flops": 0.0}
        if op == "permute_backward":
            return {"bytes": 2.0 * H * (T * (2 if case["add"] else 1) + live) + 4.0 * S, "flops": live * H}
        return {"bytes": 2.0 * H * (T * (1.0 - case["masked"]) + 2 * live) + 12.0 * S, "flops": 3.0 * live * H}
    if op in _EXPERTS:
        R, E, N, K = case["R"] - case["unused"], case["E"], case["N"], case["K"]
        rows = 2.0 * R * (N + K)
        weights = E * N * K * (4.0 if case.get("out") == "fp32" else 2.0)
        if op != "experts_wgrad":
            weights *= min(1.0, R / E)   # experts without rows need not be read
        return {"bytes": rows + weights, "flops": 2.0 * R * N * K}
    M, V, K = case["M"], case["V"], case["K"]
    product = 2.0 * M * V * K
    if op == "head_loss":
        return {"bytes": 2.0 * K * (M + V) + 16.0 * M, "flops": product}
    return {"bytes": 4.0 * K * (M + V) + 20.0 * M, "flops": 3 * product}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    f64 = torch.float64
    if op in _ROUTED:
        T, k, H = case["T"], case["k"], case["H"]
        pos = s["slot_to_pos"].long().reshape(T, k)
        if op == "permute":
            out = torch.zeros(T * k, H, dtype=f64, device="cuda")
            for j in range(k):
                ok = pos[:, j] >= 0
                out[pos[ok, j]] = s["x"][ok].to(f64)
            return out
        if op == "permute_backward":
            out = s["add"].to(f64) if case["add"] else torch.zeros(T, H, dtype=f64, device="cuda")
            for j in range(k):
                ok = pos[:, j] >= 0
                out[ok] += s["dxp"][pos[ok, j]].to(f64)
            return out
        do = torch.zeros(T * k, H, dtype=f64, device="cuda")
        dw = torch.zeros(T, k, dtype=f64, device="cuda")
        for j in range(k):
            ok = pos[:, j] >= 0
            dy = s["dy"][ok].to(f64)
            do[pos[ok, j]] = dy * s["weights"][ok, j:j + 1].to(f64)
            dw[ok, j] = (dy * s["o"][pos[ok, j]].to(f64)).sum(dim=1)
        return do, dw
    if op in _EXPERTS:
        off = s["offsets"].tolist()
        E, N, K = case["E"], case["N"], case["K"]
        if op == "experts_wgrad":
            out = torch.zeros(E, N, K, dtype=f64, device="cuda")
            for e in range(E):
                rows = slice(off[e], off[e + 1])
                if off[e + 1] > off[e]:
                    out[e] = torch.mm(s["dy"][rows].to(f64).t().contiguous(), s["x"][rows].to(f64))
            return out
        out = torch.zeros(case["R"], N if op == "experts" else K, dtype=f64, device="cuda")
        for e in range(E):
            rows = slice(off[e], off[e + 1])
            if off[e + 1] > off[e]:
                w = s["w"][e].to(f64)
                out[rows] = torch.mm(s["x"][rows].to(f64), w.t().contiguous()) if op == "experts" else \
                    torch.mm(s["dy"][rows].to(f64), w)
        return out
    M, V, K = case["M"], case["V"], case["K"]
    w = s["w"].to(f64)
    loss = torch.zeros(M, dtype=f64, device="cuda")
    lse = torch.zeros(M, dtype=f64, device="cuda")
    grad = op == "head_grad"
    dx = torch.zeros(M, K, dtype=f64, device="cuda") if grad else None
    dw = torch.zeros(V, K, dtype=f64, device="cuda") if grad else None
    for a in range(0, M, 1024):   # a thousand rows of logits at a time
        rows = slice(a, min(a + 1024, M))
        x, labels = s["x"][rows].to(f64), s["labels"][rows]
        logits = torch.mm(x, w.t())
        lse[rows] = torch.logsumexp(logits, dim=1)
        n = torch.nonzero(labels >= 0).squeeze(1)
        loss[a + n] = lse[a + n] - logits[n, labels[n]]
        if grad:
            dl = torch.exp(logits - lse[rows, None])
            dl[n, labels[n]] -= 1.0
            dl *= torch.where(labels >= 0, s["dloss"][rows].to(f64), 0.0)[:, None]
            dx[rows] = torch.mm(dl, w)
            dw += torch.mm(dl.t(), x)
    return (loss, lse, dx, dw) if grad else (loss, lse)
