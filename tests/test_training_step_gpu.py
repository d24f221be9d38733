"""The training entry points together, as a step of a small model with a tied table uses them: embedding, a dense gated block and a gated block
of experts with residuals, head and loss, everything back, the table's two gradients in one, the norm of all gradients and their
clipping; against the same step by autograd in 64 bits, on another stream, in a graph, and without the native dispatchers."""
import pathlib

import pytest
import torch

from hipkittens_amd import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ALPHA, LIMIT = 1.702, 7.0


class Step:
    """One step; everything is written into buffers made once."""

    def __init__(self, hk, T, V, H, I, E, k, Ie, seed, masked, max_norm):
        self.tk = tk = hk.tk_kernel
        g = torch.Generator(device=DEV).manual_seed(seed)
        bf = lambda *s, std=1.0: (torch.randn(*s, device=DEV, generator=g) * std).to(torch.bfloat16)
        self.T, self.V, self.H, self.I, self.E, self.k, self.Ie, self.max_norm = T, V, H, I, E, k, Ie, max_norm
        self.scale = H**0.5
        self.table = bf(V, H, std=H**-0.5)
        self.w13, self.w2 = bf(2 * I, H, std=1.5 * H**-0.5), bf(H, I, std=I**-0.5)
        self.w13e, self.w2e = bf(E, 2 * Ie, H, std=1.5 * H**-0.5), bf(E, H, Ie, std=Ie**-0.5)
        self.logits = torch.randn(T, E, device=DEV, generator=g)
        u = torch.rand(T, device=DEV, generator=g)
        self.ids = ((V + 1.0) ** u).long().sub(1).clamp(0, V - 1)
        self.mask = torch.rand(T, device=DEV, generator=g) < masked
        self.ids[self.mask] = -1
        self.labels = torch.randint(0, V, (T,), device=DEV, generator=g)
        self.labels[self.mask] = -100
        self.dloss = torch.full((T,), 1.0 / max(1, int((~self.mask).sum())), device=DEV)
        e = lambda *s, dtype=torch.bfloat16: torch.full(s, 77, dtype=dtype, device=DEV)
        f, i, b = torch.float32, torch.int32, torch.uint8
        S = T * k
        self.x0, self.h, self.gu, self.y1 = e(T, H), e(T, I), e(T, 2 * I), e(T, H)
        self.choice, self.weights, self.sorted, self.offsets, self.pos = e(T, k, dtype=i), e(T, k, dtype=f), e(S, dtype=i), e(E + 1, dtype=i), e(S, dtype=i)
        self.sort_ws = e(tk.moe_sort_workspace_bytes(T, k, E), dtype=b)
        self.xp, self.he, self.gue, self.o, self.y2 = e(S, H), e(S, Ie), e(S, 2 * Ie), e(S, H), e(T, H)
        self.loss, self.lse = e(T, dtype=f), e(T, dtype=f)
        self.head_ws = e(tk.linear_cross_entropy_workspace_bytes(T, V, H), dtype=b)
        self.dy2, self.do, self.dweights, self.dgue, self.dxp = e(T, H), e(S, H), e(T, k, dtype=f), e(S, 2 * Ie), e(S, H)
        self.dy1, self.dgu, self.dx, self.h2, self.he2 = e(T, H), e(T, 2 * I), e(T, H), e(T, I), e(S, Ie)
        self.dtable = e(V, H, dtype=f)
        self.dw13, self.dw2 = e(2 * I, H), e(H, I, dtype=f)
        self.dw13e, self.dw2e = e(E, 2 * Ie, H, dtype=f), e(E, H, Ie)
        self.embed_ws = e(tk.embedding_backward_workspace_bytes(T, V, H), dtype=b)
        self.grads = tk.GradTensors([self.dtable, self.dw13, self.dw2, self.dw13e, self.dw2e])
        self.norm, self.norm_ws = e(1, dtype=f), e(tk.grad_norm_workspace_bytes(), dtype=b)
        self.outs = [self.loss, self.norm, self.dweights, self.dtable, self.dw13, self.dw2, self.dw13e, self.dw2e]

    def run(self):
        tk = self.tk
        experts = dict(expert_offsets=self.offsets, interleaved=True, activation="swiglu_oai", alpha=ALPHA, limit=LIMIT)
        tk.dispatch_embedding(self.ids, self.table, self.x0, scale=self.scale)
        tk.dispatch_gated_gemm(self.x0, self.w13, self.h, self.gu)
        tk.dispatch_bf16_gemm(self.h, self.w2, self.y1)
        self.y1.add_(self.x0)
        tk.dispatch_moe_topk_softmax(self.logits, self.choice, self.weights)
        self.choice.masked_fill_(self.mask[:, None], -1)
        self.pos.fill_(-1)
        tk.dispatch_moe_sort(self.choice, self.sorted, self.offsets, self.pos, self.sort_ws)
        tk.dispatch_moe_permute(self.y1, self.pos, self.xp)
        tk.dispatch_gated_gemm(self.xp, self.w13e, self.he, self.gue, **experts)
        tk.dispatch_moe_grouped_gemm(self.he, self.w2e, self.offsets, self.o)
        tk.dispatch_moe_unpermute(self.o, self.weights, self.pos, self.y2)
        self.y2.add_(self.y1)
        tk.dispatch_linear_cross_entropy(self.y2, self.table, self.labels, self.loss, self.lse, self.head_ws)

        tk.dispatch_linear_cross_entropy_backward(self.y2, self.table, self.labels, self.lse, self.dloss, self.dy2, self.dtable, self.head_ws)
        tk.dispatch_moe_unpermute_backward(self.dy2, self.o, self.weights, self.pos, self.do, self.dweights)
        tk.dispatch_gated_gemm_dgrad(self.do, self.w2e, self.gue, self.dgue, self.he2, **experts)
        tk.dispatch_moe_grouped_gemm_wgrad(self.do, self.he2, self.offsets, self.dw2e)
        tk.dispatch_moe_grouped_gemm_wgrad(self.dgue, self.xp, self.offsets, self.dw13e)
        tk.dispatch_moe_grouped_gemm_dgrad(self.dgue, self.w13e, self.offsets, self.dxp)
        tk.dispatch_moe_permute_backward(self.dxp, self.pos, self.dy1, add=self.dy2)
        tk.dispatch_gated_gemm_dgrad(self.dy1, self.w2, self.gu, self.dgu, self.h2)
        tk.dispatch_bf16_gemm_wgrad(self.dy1, self.h2, self.dw2)
        tk.dispatch_bf16_gemm_wgrad(self.dgu, self.x0, self.dw13)
        tk.dispatch_bf16_gemm_dgrad(self.dgu, self.w13, self.dx)
        self.dx.add_(self.dy1)
        tk.dispatch_embedding_backward(self.ids, self.dx, self.dtable, self.embed_ws, scale=self.scale, add=self.dtable)
        tk.dispatch_grad_norm(self.grads, self.norm, self.norm_ws)
        tk.dispatch_grad_clip(self.grads, self.norm, self.max_norm)

    def reference(self):
        """The same step in 64 bits with autograd, on the CPU."""
        c = lambda t: t.detach().double().cpu().requires_grad_(True)
        table, w13, w2, w13e, w2e = c(self.table), c(self.w13), c(self.w2), c(self.w13e), c(self.w2e)
        ids, live = self.ids.cpu(), ~self.mask.cpu()
        x0 = torch.where(live[:, None], table[ids.clamp(min=0)] * self.scale, 0.0)
        gate, up = (x0 @ w13.t()).chunk(2, dim=1)
        y1 = (torch.nn.functional.silu(gate) * up) @ w2.t() + x0
        top, choice = self.logits.double().cpu().topk(self.k, dim=1)
        weights = torch.softmax(top, dim=1).requires_grad_(True)
        rows = []
        for t in range(self.T):
            y = y1[t]
            if live[t]:
                for j in range(self.k):
                    e = int(choice[t, j])
                    both = w13e[e] @ y1[t]
                    gate, up = both[0::2].clamp(max=LIMIT), both[1::2].clamp(-LIMIT, LIMIT)
                    y = y + weights[t, j] * (w2e[e] @ ((up + 1) * gate * torch.sigmoid(ALPHA * gate)))
            rows.append(y)
        logits = torch.stack(rows) @ table.t()
        loss = torch.nn.functional.cross_entropy(logits, self.labels.cpu(), reduction="none", ignore_index=-100)
        (loss * self.dloss.double().cpu()).sum().backward()
        grads = [t.grad for t in (table, w13, w2, w13e, w2e)]
        norm = torch.sqrt(sum((t**2).sum() for t in grads))
        factor = min(1.0, self.max_norm / (norm.item() + 1e-6))
        return [loss.detach(), norm.reshape(1), weights.grad] + [t * factor for t in grads]


@pytest.mark.parametrize("T,V,H,I,E,k,Ie,masked,max_norm", [(37, 333, 72, 104, 5, 2, 40, 0.2, 0.05), (160, 1000, 136, 256, 8, 4, 64, 0.0, 1e6),
                                                            (1, 50, 64, 32, 3, 1, 32, 0.0, 0.1)])
def test_against_autograd(hk, T, V, H, I, E, k, Ie, masked, max_norm):
    """Relative in the Frobenius norm. On the longest way lie x0, the kept gate and up values, h, y1 and its sum with x0, the experts' same three, o,
    y2 and its sum, dl, dy2, do, the experts' gradients and dxp, dy1, the block's gradients, dx and its sum, a weight gradient and its clipping:
    22 roundings to bf16, each off by at most 2^-8 of its value and independent of one another; sqrt(22) 2^-8 = 0.018 for
    uncorrelated errors, twice that is asked for."""
    print(f"whole step T={T} V={V} H={H} I={I} E={E} k={k}", flush=True)
    step = Step(hk, T, V, H, I, E, k, Ie, T, masked, max_norm)
    step.run()
    torch.cuda.synchronize()
    names = ("loss", "norm", "dweights", "dtable", "dw13", "dw2", "dw13e", "dw2e")
    for name, got, want in zip(names, step.outs, step.reference()):
        got = got.double().cpu()
        assert torch.isfinite(got).all(), name
        err = float((got - want).norm() / want.norm())
        assert err <= 0.036, (name, err)


def _bytes(t):
    return t.reshape(-1).view(torch.uint8)


def test_on_another_stream(hk):
    """Everything goes to the current stream: the inputs are only there once that stream has made them."""
    print("whole step on a side stream", flush=True)
    step = Step(hk, 300, 2000, 136, 264, 8, 2, 64, 5, 0.1, 0.05)
    step.run()
    torch.cuda.synchronize()
    want = [o.clone() for o in step.outs]
    inputs = [step.table, step.w13, step.ids, step.w2e]
    kept = [t.clone() for t in inputs]
    for t in inputs:
        t.zero_()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        big = torch.empty(1 << 26, device=DEV)
        for _ in range(20):
            big.add_(1.0)            # holds the stream back
        for t, v in zip(inputs, kept):
            t.copy_(v)
        step.run()
    side.synchronize()
    for got, w in zip(step.outs, want):
        assert torch.equal(_bytes(got), _bytes(w))


def test_in_a_graph(hk):
    print("whole step in a graph", flush=True)
    step = Step(hk, 5000, 3000, 264, 520, 8, 4, 128, 6, 0.1, 0.05)
    step.run()
    torch.cuda.synchronize()
    want = [o.clone() for o in step.outs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.run()
    for rep in range(3):
        for o in step.outs + [step.xp, step.o, step.do, step.dgu, step.dgue]:
            o.fill_(5)
        for ws in (step.head_ws, step.sort_ws, step.embed_ws, step.norm_ws):
            ws.fill_(0xFF)     # nothing in the workspaces is kept from one call to the next
        graph.replay()
        torch.cuda.synchronize()
        for got, w in zip(step.outs, want):
            assert torch.equal(_bytes(got), _bytes(w)), rep


def test_without_the_native_dispatchers(hk, monkeypatch):
    """The Python dispatchers give the same bits."""
    print("whole step without the native dispatchers", flush=True)
    step = Step(hk, 130, 500, 72, 104, 4, 2, 40, 7, 0.1, 0.05)
    step.run()
    torch.cuda.synchronize()
    want = [o.clone() for o in step.outs]
    assert hk.tk_kernel._native is not None and hk.tk_kernel._native is not hk.tk_kernel._NoNative
    monkeypatch.setattr(_lib, "_DISPATCH_PATH", pathlib.Path("/nonexistent/_dispatch.so"))
    monkeypatch.setattr(_lib, "_dispatch", None)
    monkeypatch.setattr(hk.tk_kernel, "_native", None)
    for o in step.outs:
        o.fill_(5)
    with pytest.warns(RuntimeWarning, match="check their arguments in Python"):
        step.run()
    torch.cuda.synchronize()
    for got, w in zip(step.outs, want):
        assert torch.equal(_bytes(got), _bytes(w))


def test_native_dispatchers_take_ordinary_calls(hk):
    """Each takes its ordinary call, and leaves what it does not know to Python."""
    print("native dispatchers of the training step", flush=True)
    nat = _lib.load_dispatch()
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(s, dtype=dtype, device=DEV)
    x, w13, h, gu, w2 = z(4, 64), z(128, 64), z(4, 64), z(4, 128), z(64, 64)
    off, ids = z(2, dtype=torch.int32), z(4, dtype=torch.int64)
    assert nat.gated_gemm(x, w13, h, None, None, False, 0, 1.0, 7.0) == 0
    assert nat.gated_gemm(x, w13[None], h, gu, off, True, 1, 1.0, 7.0) == 0
    assert nat.gated_gemm(x, w13, h, None, None, False, None, 1.0, 7.0) is None
    assert nat.gated_gemm(x, w13, h, None, off, False, 0, 1.0, 7.0) is None
    assert nat.gated_gemm(x, w13, h, h, None, False, 0, 1.0, 7.0) is None
    assert nat.gated_gemm(x, w13, None, gu, None, False, 0, 1.0, 7.0) is None
    assert nat.gated_gemm_dgrad(x, w2, gu, gu, None, None, False, 0, 1.0, 7.0) == 0
    assert nat.gated_gemm_dgrad(x, w2[None], gu, z(4, 128), h, off, False, 0, 1.0, 7.0) == 0
    assert nat.gated_gemm_dgrad(x, w2, gu, h, None, None, False, 0, 1.0, 7.0) is None
    assert nat.gated_gemm_dgrad(x, w2, None, gu, None, None, False, 0, 1.0, 7.0) is None
    assert nat.bf16_gemm_dgrad(x, w2, h) == 0 and nat.bf16_gemm_dgrad(x, w13, h) is None
    assert nat.bf16_gemm_wgrad(x, h, w2) == 0 and nat.bf16_gemm_wgrad(x, h, z(64, 64, dtype=torch.float32)) == 0
    assert nat.bf16_gemm_wgrad(x, h, w13) is None
    ws = z(hk.tk_kernel.embedding_backward_workspace_bytes(4, 10, 64), dtype=torch.uint8)
    assert nat.embedding(ids, z(10, 64), x, 2.0) == 0 and nat.embedding(ids, z(10, 64), x, 2) is None
    assert nat.embedding(ids[:3], z(10, 64), x, 2.0) is None
    assert nat.embedding_backward(ids, x, z(10, 64), ws, 1.0, None) == 0
    assert nat.embedding_backward(ids, x, z(10, 64), ws, 1.0, z(10, 64, dtype=torch.float32)) is None
    assert nat.embedding_backward(ids, x, z(10, 64, dtype=torch.float32), ws, 1.0, z(10, 64, dtype=torch.float32)) == 0
    plan = hk.tk_kernel.GradTensors([x, h])
    norm, nws = z(1, dtype=torch.float32), z(hk.tk_kernel.grad_norm_workspace_bytes(), dtype=torch.uint8)
    assert nat.grad_norm(plan.list, plan.n, plan.chunks, norm, nws) == 0 and nat.grad_clip(plan.list, plan.n, plan.chunks, norm, 1.0) == 0
    assert nat.grad_clip(plan.list, plan.n, plan.chunks, norm, 1) is None and nat.grad_norm(plan.list, plan.n, plan.chunks, x, nws) is None
    torch.cuda.synchronize()
