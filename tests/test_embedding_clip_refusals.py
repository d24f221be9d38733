"""Refusals of the embedding's and the gradients' entry points, without a GPU, and the workspace's size."""
import ctypes

import pytest
import torch

import hipkittens_amd as hk

NULL, SHAPE, ALIGN, WORKSPACE, UNSUPPORTED = -1, -2, -3, -4, -6


@pytest.fixture(scope="module")
def p():
    buf = ctypes.create_string_buffer(4096)
    yield (ctypes.addressof(buf) + 63) & ~63   # an aligned host pointer that is never followed


def test_embedding(p):
    lib = hk.load_library()
    big = 1 << 50
    for at in (0, 2, 4):
        args = [p, 0, p, 0, p, 4, 100, 64, 1.0, None]
        args[at] = None
        assert lib.hk_embedding(*args) == NULL
    for at in (0, 2, 4):
        args = [p, 0, p, p, p, 0, 4, 100, 64, 1.0, p, big, None]
        args[at] = None
        assert lib.hk_embedding_backward(*args) == NULL
    for T, V, H in ((0, 100, 64), (4, 0, 64), (4, 100, 0), (4, 100, 60), (1 << 24, 100, 64), (4, 1 << 30, 64), (4, 100, (1 << 21) + 8), (-1, 100, 64),
                    (4, 1 << 29, 8192), (1 << 23, 100, 1 << 15)):   # (the last two: more than 2^38 elements)
        assert lib.hk_embedding(p, 0, p, 0, p, T, V, H, 1.0, None) == SHAPE
        assert lib.hk_embedding_backward(p, 0, p, p, p, 0, T, V, H, 1.0, p, big, None) == SHAPE
        assert lib.hk_embedding_backward_workspace_bytes(T, V, H) == 0
    for a, b in ((2, 0), (-1, 0), (0, 2), (0, -1)):
        assert lib.hk_embedding(p, a, p, b, p, 4, 100, 64, 1.0, None) == UNSUPPORTED
        assert lib.hk_embedding_backward(p, a, p, p, p, b, 4, 100, 64, 1.0, p, big, None) == UNSUPPORTED
    assert lib.hk_embedding(p, 0, p + 8, 0, p, 4, 100, 64, 1.0, None) == ALIGN
    assert lib.hk_embedding(p, 0, p, 0, p + 2, 4, 100, 64, 1.0, None) == ALIGN
    for at in (2, 3, 4, 10):
        args = [p, 0, p, p, p, 0, 4, 100, 64, 1.0, p, big, None]
        args[at] = p + 8
        assert lib.hk_embedding_backward(*args) == ALIGN
    assert lib.hk_embedding(p + 2, 0, p, 0, p, 4, 100, 64, 1.0, None) == ALIGN and lib.hk_embedding(p + 4, 1, p, 0, p, 4, 100, 64, 1.0, None) == ALIGN
    assert lib.hk_embedding_backward(p + 4, 1, p, p, p, 0, 4, 100, 64, 1.0, p, big, None) == ALIGN
    need = lib.hk_embedding_backward_workspace_bytes(4, 100, 64)
    assert lib.hk_embedding_backward(p, 0, p, p, p, 0, 4, 100, 64, 1.0, p, need - 1, None) == WORKSPACE
    assert lib.hk_embedding_backward(p, 0, p, p, p, 0, 4, 100, 64, 1.0, None, need, None) == WORKSPACE


def test_workspace_never_falls_with_more_tokens():
    lib = hk.load_library()
    for V, H in ((1, 8), (100, 520), (50257, 1024), (201088, 2880), (1 << 29, 256)):
        sizes = [lib.hk_embedding_backward_workspace_bytes(T, V, H) for T in sorted(
            {1, 2, 7} | {a << s for s in range(0, 24) for a in (1,)} | {(a << s) + d for s in range(4, 23) for a in (1, 3) for d in (-1, 1)})
            if T < 1 << 24]
        assert all(a <= b for a, b in zip(sizes, sizes[1:])) and sizes[0] > 0
    steps = [lib.hk_embedding_backward_workspace_bytes(T, 50257, 1024) for T in range(30000, 140000, 7)]   # across the block lengths' edges
    assert all(a <= b for a, b in zip(steps, steps[1:]))


def _fill(lib, p, n=2, counts=(4, 4), types=(0, 1), out_types=(0, 1), grads=None, outs="same", bytes_=None):
    host = ctypes.create_string_buffer(4096)
    ptrs = lambda v: (ctypes.c_void_p * n)(*v)
    g = grads if grads is not None else [p + 64 * i for i in range(n)]
    o = None if outs is None else ptrs(g if outs == "same" else outs)
    chunks = ctypes.c_int64(-1)
    st = lib.hk_grad_list_fill(ptrs(g), o, (ctypes.c_int64 * n)(*counts), (ctypes.c_int32 * n)(*types), (ctypes.c_int32 * n)(*out_types), n,
                               ctypes.addressof(host), 4096 if bytes_ is None else bytes_, ctypes.byref(chunks))
    return st, chunks.value


def test_gradient_lists(p):
    lib = hk.load_library()
    assert lib.hk_grad_list_bytes(0) == lib.hk_grad_list_bytes(-1) == lib.hk_grad_list_bytes((1 << 20) + 1) == 0
    assert lib.hk_grad_list_bytes(2) == 2 * lib.hk_grad_list_bytes(1) > 0
    assert _fill(lib, p) == (0, 2) and _fill(lib, p, outs=None) == (0, 2)
    assert _fill(lib, p, counts=(0, 1 << 20))[0] == 0
    assert _fill(lib, p, counts=(0, 0), grads=[None, None]) == (0, 0)
    assert _fill(lib, p, counts=(-1, 4))[0] == SHAPE and _fill(lib, p, counts=(1 << 40, 4))[0] == SHAPE
    assert _fill(lib, p, types=(0, 2))[0] == UNSUPPORTED and _fill(lib, p, out_types=(3, 1))[0] == UNSUPPORTED
    assert _fill(lib, p, out_types=(1, 1))[0] == UNSUPPORTED   # in place, but another type
    assert _fill(lib, p, grads=[None, p])[0] == NULL and _fill(lib, p, outs=[p, None])[0] == NULL
    assert _fill(lib, p, grads=[p + 1, p + 64])[0] == ALIGN and _fill(lib, p, grads=[p, p + 66])[0] == ALIGN
    assert _fill(lib, p, bytes_=lib.hk_grad_list_bytes(2) - 1)[0] == WORKSPACE
    need = lib.hk_grad_norm_workspace_bytes()
    for at in (0, 3):
        args = [p, 2, 2, p, p, need, None]
        args[at] = None
        assert lib.hk_grad_norm(*args) == NULL
    for n, chunks in ((0, 1), (2, -1), (2, 1 << 40), ((1 << 20) + 1, 1)):
        assert lib.hk_grad_norm(p, n, chunks, p, p, need, None) == SHAPE
        assert lib.hk_grad_clip(p, n, chunks, p, 1.0, None) == SHAPE
    assert lib.hk_grad_norm(p, 2, 2, p, p, need - 1, None) == WORKSPACE and lib.hk_grad_norm(p, 2, 2, p, None, need, None) == WORKSPACE
    assert lib.hk_grad_norm(p + 4, 2, 2, p, p, need, None) == ALIGN and lib.hk_grad_norm(p, 2, 2, p + 2, p, need, None) == ALIGN
    assert lib.hk_grad_clip(p, 2, 2, p + 1, 1.0, None) == ALIGN
    assert lib.hk_grad_clip(None, 2, 2, p, 1.0, None) == NULL and lib.hk_grad_clip(p, 2, 2, None, 1.0, None) == NULL
    assert lib.hk_grad_clip(p, 2, 2, p, -1.0, None) == UNSUPPORTED and lib.hk_grad_clip(p, 2, 2, p, float("nan"), None) == UNSUPPORTED
    assert lib.hk_grad_clip(p, 2, 0, p, 1.0, None) == 0   # nothing to do, nothing launched


def test_python_boundary():
    tk = hk.tk_kernel
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)
    ids, ws = torch.zeros(4, dtype=torch.int64), torch.zeros(64, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="GPU"):
        tk.dispatch_embedding(ids, bf(10, 64), bf(4, 64))
    with pytest.raises(RuntimeError, match="Tensor"):
        tk.dispatch_embedding_backward(None, bf(4, 64), bf(10, 64), ws)
    for bad in ([], [bf(4)], [None], [bf(8, 4).t()]):
        with pytest.raises(RuntimeError):
            tk.GradTensors(bad)
    with pytest.raises(RuntimeError, match="GradTensors"):
        tk.dispatch_grad_norm([bf(4)], torch.zeros(1), ws)
    with pytest.raises(RuntimeError, match="GradTensors"):
        tk.dispatch_grad_clip(None, torch.zeros(1), 1.0)


@pytest.mark.gpu
def test_python_boundary_shapes_and_types():
    tk = hk.tk_kernel
    d = "cuda:0"
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device=d)
    f32 = lambda *s: torch.zeros(s, device=d)
    ids = torch.zeros(4, dtype=torch.int64, device=d)
    ws = torch.zeros(tk.embedding_backward_workspace_bytes(4, 10, 64), dtype=torch.uint8, device=d)
    flat = bf(100)
    plan = tk.GradTensors([flat])
    nws = torch.zeros(tk.grad_norm_workspace_bytes(), dtype=torch.uint8, device=d)
    for call in (lambda: tk.dispatch_embedding(ids, bf(10, 64), bf(5, 64)),
                 lambda: tk.dispatch_embedding(ids, bf(10, 64), bf(4, 72)),
                 lambda: tk.dispatch_embedding(ids, bf(10, 64), f32(4, 64)),
                 lambda: tk.dispatch_embedding(ids, bf(10, 60), bf(4, 60)),
                 lambda: tk.dispatch_embedding(ids.reshape(2, 2), bf(10, 64), bf(4, 64)),
                 lambda: tk.dispatch_embedding(f32(4), bf(10, 64), bf(4, 64)),
                 lambda: tk.dispatch_embedding(ids[:0], bf(10, 64), bf(0, 64)),
                 lambda: tk.dispatch_embedding_backward(ids, bf(4, 64), bf(10, 64), ws[:-1]),
                 lambda: tk.dispatch_embedding_backward(ids, bf(4, 64), bf(10, 64), ws, add=f32(10, 64)),
                 lambda: tk.dispatch_embedding_backward(ids, bf(4, 64), bf(10, 64), ws, add=bf(11, 64)),
                 lambda: tk.dispatch_embedding_backward(ids, f32(4, 64), bf(10, 64), ws),
                 lambda: tk.GradTensors([flat, flat]),
                 lambda: tk.GradTensors([flat[:60], flat[59:]]),
                 lambda: tk.GradTensors([flat[:50]], [flat[1:51]]),
                 lambda: tk.GradTensors([flat[:50], flat[50:]], [flat[50:], flat[:50]]),
                 lambda: tk.GradTensors([flat], [f32(99)]),
                 lambda: tk.GradTensors([flat], []),
                 lambda: tk.GradTensors([torch.zeros(4, dtype=torch.float16, device=d)]),
                 lambda: tk.GradTensors([flat, torch.zeros(4)]),
                 lambda: tk.dispatch_grad_norm(plan, f32(2), nws),
                 lambda: tk.dispatch_grad_norm(plan, bf(1), nws),
                 lambda: tk.dispatch_grad_norm(plan, f32(1), nws[:-1]),
                 lambda: tk.dispatch_grad_clip(plan, f32(1), -1.0),
                 lambda: tk.dispatch_grad_clip(plan, f32(1), float("nan"))):
        with pytest.raises(RuntimeError):
            call()
    tk.GradTensors([flat[:50], flat[50:]], [flat[:50], bf(50)])   # in place and elsewhere
    torch.cuda.synchronize()
