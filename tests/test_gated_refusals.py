"""Refusals of the gated blocks' entry points, without a GPU: status codes before anything is launched, and the Python boundary's errors."""
import ctypes

import pytest
import torch

import hipkittens_amd as hk

NULL, SHAPE, ALIGN, UNSUPPORTED = -1, -2, -3, -6
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def p():
    buf = ctypes.create_string_buffer(4096)
    yield (ctypes.addressof(buf) + 63) & ~63   # an aligned host pointer that is never followed


def _forward(lib, p, R=4, E=1, I=64, K=64, offsets=None, act=0, alpha=1.0, limit=7.0, **ptrs):
    q = {"x": p, "w": p, "h": p, "gu": p} | ptrs
    return lib.hk_gated_gemm(q["x"], q["w"], offsets, q["h"], q["gu"], R, E, I, K, 0, act, alpha, limit, None)


def _backward(lib, p, R=4, E=1, N=64, I=64, offsets=None, act=0, alpha=1.0, limit=7.0, **ptrs):
    q = {"dy": p, "w": p, "gu": p, "dgu": p, "h": p} | ptrs
    return lib.hk_gated_gemm_dgrad(q["dy"], q["w"], offsets, q["gu"], q["dgu"], q["h"], R, E, N, I, 0, act, alpha, limit, None)


def test_status_codes(p):
    lib = hk.load_library()
    for name in ("x", "w", "h"):
        assert _forward(lib, p, **{name: None}) == NULL
    for name in ("dy", "w", "gu", "dgu"):
        assert _backward(lib, p, **{name: None}) == NULL
    for name in ("x", "w", "h", "gu"):
        assert _forward(lib, p, **{name: p + 8}) == ALIGN
    for name in ("dy", "w", "gu", "dgu", "h"):
        assert _backward(lib, p, **{name: p + 2}) == ALIGN
    for bad in (dict(R=0), dict(R=-1), dict(R=1 << 30), dict(I=0), dict(I=60), dict(I=(1 << 20) + 8), dict(E=0), dict(E=513, offsets=p),
                dict(E=2)):   # (several experts need offsets)
        assert _forward(lib, p, **bad) == SHAPE, bad
        assert _backward(lib, p, **bad) == SHAPE, bad
    for wide in (0, 4, -8, (1 << 21) + 8):
        assert _forward(lib, p, K=wide) == SHAPE and _backward(lib, p, N=wide) == SHAPE
    # more tiles than a launch has workgroups
    assert _forward(lib, p, R=1 << 29, I=1 << 18) == SHAPE
    assert _backward(lib, p, R=1 << 29, I=1 << 19) == SHAPE
    for act, alpha, limit in ((2, 1.0, 7.0), (-1, 1.0, 7.0), (1, NAN, 7.0), (1, INF, 7.0), (1, 1.7, NAN), (1, 1.7, 0.0), (1, 1.7, -7.0)):
        assert _forward(lib, p, act=act, alpha=alpha, limit=limit) == UNSUPPORTED
        assert _backward(lib, p, act=act, alpha=alpha, limit=limit) == UNSUPPORTED


def test_dense_gradients(p):
    lib = hk.load_library()
    for at in (0, 1, 2):
        args = [p, p, p, 4, 64, 64, None]
        args[at] = None
        assert lib.hk_bf16_gemm_dgrad(*args) == NULL
        assert lib.hk_bf16_gemm_wgrad(*args[:3], 0, *args[3:]) == NULL
        args[at] = p + 4
        assert lib.hk_bf16_gemm_dgrad(*args) == ALIGN
        assert lib.hk_bf16_gemm_wgrad(*args[:3], 1, *args[3:]) == ALIGN
    for M, N, K in ((0, 64, 64), (4, 60, 64), (4, 64, 4), (1 << 30, 64, 64), (4, (1 << 21) + 8, 64)):
        assert lib.hk_bf16_gemm_dgrad(p, p, p, M, N, K, None) == SHAPE
        assert lib.hk_bf16_gemm_wgrad(p, p, p, 0, M, N, K, None) == SHAPE
    assert lib.hk_bf16_gemm_wgrad(p, p, p, 2, 4, 64, 64, None) == UNSUPPORTED


def test_experts_products_still_need_offsets(p):
    lib = hk.load_library()
    assert lib.hk_moe_grouped_gemm(p, p, None, p, 4, 1, 64, 64, None) == NULL
    assert lib.hk_moe_grouped_gemm_dgrad(p, p, None, p, 4, 1, 64, 64, None) == NULL
    assert lib.hk_moe_grouped_gemm_wgrad(p, p, None, p, 0, 4, 1, 64, 64, None) == NULL


def test_python_boundary():
    tk = hk.tk_kernel
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU"):
        tk.dispatch_gated_gemm(bf(4, 64), bf(128, 64), bf(4, 64))
    with pytest.raises(RuntimeError, match="Tensor"):
        tk.dispatch_gated_gemm([1], bf(128, 64), bf(4, 64))
    with pytest.raises(RuntimeError, match="Tensor"):
        tk.dispatch_gated_gemm(None, bf(128, 64), bf(4, 64))
    with pytest.raises(RuntimeError, match="activation"):
        tk.dispatch_gated_gemm(bf(4, 64), bf(128, 64), bf(4, 64), activation="relu")
    with pytest.raises(RuntimeError, match="Tensor"):
        tk.dispatch_gated_gemm_dgrad(bf(4, 64), bf(64, 64), None, bf(4, 128))
    with pytest.raises(RuntimeError, match="GPU"):
        tk.dispatch_gated_gemm_dgrad(bf(4, 64), bf(64, 64), bf(4, 128), bf(4, 128))
    with pytest.raises(RuntimeError, match="GPU"):
        tk.dispatch_bf16_gemm_dgrad(bf(4, 64), bf(64, 64), bf(4, 64))
    with pytest.raises(RuntimeError, match="contiguous"):
        tk.dispatch_bf16_gemm_wgrad(bf(64, 4).t(), bf(4, 64), bf(64, 64))


@pytest.mark.gpu
def test_python_boundary_shapes_and_types():
    tk = hk.tk_kernel
    d = "cuda:0"
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device=d)
    f32 = lambda *s: torch.zeros(s, device=d)
    i32 = lambda n: torch.zeros(n, dtype=torch.int32, device=d)
    for call in (lambda: tk.dispatch_gated_gemm(bf(4, 64), bf(128, 72), bf(4, 64)),
                 lambda: tk.dispatch_gated_gemm(bf(4, 64), bf(136, 64), bf(4, 64)),
                 lambda: tk.dispatch_gated_gemm(bf(4, 64), bf(128, 64), bf(5, 64)),
                 lambda: tk.dispatch_gated_gemm(bf(4, 64), bf(128, 64), bf(4, 64), bf(4, 64)),
                 lambda: tk.dispatch_gated_gemm(bf(4, 64), bf(128, 64), f32(4, 64)),
                 lambda: tk.dispatch_gated_gemm(f32(4, 64), bf(128, 64), bf(4, 64)),
                 lambda: tk.dispatch_gated_gemm(bf(4, 64), bf(2, 128, 64), bf(4, 64)),
                 lambda: tk.dispatch_gated_gemm(bf(4, 64), bf(128, 64), bf(4, 64), expert_offsets=i32(2)),
                 lambda: tk.dispatch_gated_gemm(bf(4, 64), bf(2, 128, 64), bf(4, 64), expert_offsets=i32(2)),
                 lambda: tk.dispatch_gated_gemm(bf(4, 64), bf(2, 128, 64), bf(4, 64), expert_offsets=f32(3)),
                 lambda: tk.dispatch_gated_gemm(bf(4, 60), bf(128, 60), bf(4, 64)),
                 lambda: tk.dispatch_gated_gemm(bf(4, 64), bf(128, 64), bf(4, 64), activation="swiglu_oai", limit=-1.0),
                 lambda: tk.dispatch_gated_gemm(bf(4, 64), bf(128, 64), None),
                 lambda: tk.dispatch_gated_gemm(bf(4, 64), bf(128, 64), None, bf(4, 128)),
                 lambda: tk.dispatch_gated_gemm(bf(0, 64), bf(128, 64), bf(0, 64)),
                 lambda: tk.dispatch_gated_gemm_dgrad(bf(4, 64), bf(64, 72), bf(4, 128), bf(4, 128)),
                 lambda: tk.dispatch_gated_gemm_dgrad(bf(4, 64), bf(64, 64), bf(4, 128), bf(4, 64)),
                 lambda: tk.dispatch_gated_gemm_dgrad(bf(4, 64), bf(64, 64), bf(4, 127), bf(4, 128)),
                 lambda: tk.dispatch_gated_gemm_dgrad(bf(4, 64), bf(64, 64), bf(4, 128), bf(4, 128), bf(4, 72)),
                 lambda: tk.dispatch_gated_gemm_dgrad(bf(4, 64), bf(64, 64), bf(4, 128), f32(4, 128)),
                 lambda: tk.dispatch_bf16_gemm_dgrad(bf(4, 64), bf(64, 64), bf(4, 72)),
                 lambda: tk.dispatch_bf16_gemm_wgrad(bf(4, 64), bf(5, 64), bf(64, 64)),
                 lambda: tk.dispatch_bf16_gemm_wgrad(bf(4, 64), bf(4, 64), torch.zeros(64, 64, dtype=torch.float64, device=d))):
        with pytest.raises(RuntimeError):
            call()
    torch.cuda.synchronize()
