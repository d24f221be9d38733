"""Refusals of the training entry points, without a GPU: status codes before anything is launched, and the Python boundary's
errors."""
import ctypes

import pytest
import torch

import hipkittens_amd as hk

NULL, SHAPE, ALIGN, WORKSPACE, UNSUPPORTED = -1, -2, -3, -4, -6
IMAX = 2**31 - 1


@pytest.fixture(scope="module")
def p():
    buf = ctypes.create_string_buffer(4096)
    yield (ctypes.addressof(buf) + 63) & ~63   # an aligned host pointer that is never followed


def test_permute_family(p):
    lib = hk.load_library()
    for at in (0, 1, 5):
        args = [p, p, 4, 2, 64, p, None]
        args[at] = None
        assert lib.hk_moe_permute(*args) == NULL
    for T, k, H in ((1 << 24, 1, 64), (0, 2, 64), (4, 0, 64), (4, 2, 0), (4, 2, 60), (-1, 2, 64), (1 << 29, 3, 64), (IMAX, IMAX, 8)):
        assert lib.hk_moe_permute(p, p, T, k, H, p, None) == SHAPE
        assert lib.hk_moe_permute_backward(p, p, T, k, H, None, p, None) == SHAPE
        assert lib.hk_moe_unpermute_backward(p, p, p, p, T, k, H, p, p, None) == SHAPE
    assert lib.hk_moe_permute(p + 2, p, 4, 2, 64, p, None) == ALIGN
    assert lib.hk_moe_permute_backward(p, p, 4, 2, 64, p + 8, p, None) == ALIGN
    assert lib.hk_moe_permute_backward(p, p, 4, 2, 64, None, None, None) == NULL
    assert lib.hk_moe_unpermute_backward(p, p, p, p, 4, 2, 64, p + 8, p, None) == ALIGN
    assert lib.hk_moe_unpermute_backward(p, p, p, p, 4, 2, 64, p, None, None) == NULL
    assert lib.hk_moe_unpermute_backward(p, p, p, p, 1, 65536, 64, p, p, None) == SHAPE


def test_grouped_products(p):
    lib = hk.load_library()
    for at in (0, 1, 2, 3):
        args = [p, p, p, p, 4, 2, 64, 64, None]
        args[at] = None
        assert lib.hk_moe_grouped_gemm(*args) == NULL
        assert lib.hk_moe_grouped_gemm_dgrad(*args) == NULL
        assert lib.hk_moe_grouped_gemm_wgrad(*args[:4], 0, *args[4:]) == NULL
    for R, E, N, K in ((0, 2, 64, 64), (4, 0, 64, 64), (4, 513, 64, 64), (4, 2, 60, 64), (4, 2, 64, 4), (4, 2, 0, 64),
                       (1 << 30, 2, 64, 64), (4, 2, (1 << 21) + 8, 64), (4, 2, 64, IMAX - 7)):
        assert lib.hk_moe_grouped_gemm(p, p, p, p, R, E, N, K, None) == SHAPE
        assert lib.hk_moe_grouped_gemm_dgrad(p, p, p, p, R, E, N, K, None) == SHAPE
        assert lib.hk_moe_grouped_gemm_wgrad(p, p, p, p, 0, R, E, N, K, None) == SHAPE
    # more tiles than a launch has workgroups
    assert lib.hk_moe_grouped_gemm(p, p, p, p, 1 << 29, 1, 1 << 20, 64, None) == SHAPE
    assert lib.hk_moe_grouped_gemm_wgrad(p, p, p, p, 0, 64, 512, 1 << 16, 1 << 16, None) == SHAPE
    assert lib.hk_moe_grouped_gemm(p + 8, p, p, p, 4, 2, 64, 64, None) == ALIGN
    assert lib.hk_moe_grouped_gemm_dgrad(p, p + 2, p, p, 4, 2, 64, 64, None) == ALIGN
    assert lib.hk_moe_grouped_gemm_wgrad(p, p, p, p + 4, 1, 4, 2, 64, 64, None) == ALIGN
    assert lib.hk_moe_grouped_gemm_wgrad(p, p, p, p, 2, 4, 2, 64, 64, None) == UNSUPPORTED


def test_linear_cross_entropy(p):
    lib = hk.load_library()
    big = 1 << 50
    for at in (0, 1, 2, 4, 5):
        args = [p, p, p, 1, p, p, 4, 100, 64, p, big, None]
        args[at] = None
        assert lib.hk_linear_cross_entropy(*args) == NULL
    for at in (0, 1, 2, 4, 5):
        args = [p, p, p, 1, p, p, p, p, 0, 4, 100, 64, p, big, None]
        args[at] = None
        assert lib.hk_linear_cross_entropy_backward(*args) == NULL
    assert lib.hk_linear_cross_entropy_backward(p, p, p, 1, p, p, None, None, 0, 4, 100, 64, p, big, None) == NULL
    for M, V, K in ((0, 100, 64), (4, 0, 64), (4, 100, 0), (4, 100, 60), (1 << 30, 100, 64), (4, 1 << 30, 64),
                    (1 << 25, 1 << 25, 64), (1 << 20, 1 << 20, 64), (4, 100, (1 << 21) + 8)):
        assert lib.hk_linear_cross_entropy(p, p, p, 1, p, p, M, V, K, p, big, None) == SHAPE
        assert lib.hk_linear_cross_entropy_backward(p, p, p, 1, p, p, p, p, 0, M, V, K, p, big, None) == SHAPE
        assert lib.hk_linear_cross_entropy_workspace_bytes(M, V, K, 0) == 0
        assert lib.hk_linear_cross_entropy_workspace_bytes(M, V, K, 1) == 0
    assert lib.hk_linear_cross_entropy(p, p, p, 2, p, p, 4, 100, 64, p, big, None) == UNSUPPORTED
    assert lib.hk_linear_cross_entropy_backward(p, p, p, 1, p, p, p, p, 3, 4, 100, 64, p, big, None) == UNSUPPORTED
    for at in (0, 1, 9):
        args = [p, p, p, 1, p, p, 4, 100, 64, p, big, None]
        args[at] += 8
        assert lib.hk_linear_cross_entropy(*args) == ALIGN
    need = lib.hk_linear_cross_entropy_workspace_bytes(4, 100, 64, 0)
    both = lib.hk_linear_cross_entropy_workspace_bytes(4, 100, 64, 1)
    assert 0 < need <= both
    assert lib.hk_linear_cross_entropy(p, p, p, 1, p, p, 4, 100, 64, p, need - 1, None) == WORKSPACE
    assert lib.hk_linear_cross_entropy(p, p, p, 1, p, p, 4, 100, 64, None, need, None) == WORKSPACE
    assert lib.hk_linear_cross_entropy_backward(p, p, p, 1, p, p, p, p, 0, 4, 100, 64, None, both, None) == WORKSPACE
    # the logits are not kept: far less than M x V bytes for many rows and classes, and no overflow in the sizes
    assert 0 < lib.hk_linear_cross_entropy_workspace_bytes(16384, 201088, 2880, 1) < 16384 * 201088 // 4
    assert lib.hk_linear_cross_entropy_workspace_bytes(1 << 19, 201088, 64, 0) >= (1 << 19) * 201088 // 128 * 8


def test_python_boundary():
    tk = hk.tk_kernel
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)
    i32 = lambda n: torch.zeros(n, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        tk.dispatch_moe_permute(bf(4, 64), i32(8), bf(8, 64))
    with pytest.raises(RuntimeError, match="contiguous"):
        tk.dispatch_moe_permute(bf(64, 4).t(), i32(8), bf(8, 64))
    with pytest.raises(RuntimeError, match="Tensor"):
        tk.dispatch_moe_permute_backward(bf(8, 64), i32(8), None)
    with pytest.raises(RuntimeError, match="GPU"):
        tk.dispatch_moe_unpermute_backward(bf(4, 64), bf(8, 64), torch.zeros(4, 2), i32(8), bf(8, 64), torch.zeros(4, 2))
    with pytest.raises(RuntimeError, match="GPU"):
        tk.dispatch_moe_grouped_gemm(bf(4, 64), bf(2, 64, 64), i32(3), bf(4, 64))
    with pytest.raises(RuntimeError, match="GPU"):
        tk.dispatch_linear_cross_entropy(bf(4, 64), bf(100, 64), i32(4), torch.zeros(4), torch.zeros(4),
                                         torch.zeros(64, dtype=torch.uint8))


@pytest.mark.gpu
def test_python_boundary_shapes_and_types():
    tk = hk.tk_kernel
    d = "cuda:0"
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device=d)
    f32 = lambda *s: torch.zeros(s, device=d)
    i32 = lambda n: torch.zeros(n, dtype=torch.int32, device=d)
    ws = torch.zeros(tk.linear_cross_entropy_workspace_bytes(4, 100, 64), dtype=torch.uint8, device=d)
    for call in (lambda: tk.dispatch_moe_permute(bf(4, 64), i32(8), bf(9, 64)),
                 lambda: tk.dispatch_moe_permute(bf(4, 64), i32(7), bf(8, 64)),
                 lambda: tk.dispatch_moe_permute(bf(4, 64), i32(8), bf(8, 72)),
                 lambda: tk.dispatch_moe_permute(bf(4, 64), i32(8), f32(8, 64)),
                 lambda: tk.dispatch_moe_permute_backward(bf(8, 64), i32(8), bf(4, 64), add=bf(5, 64)),
                 lambda: tk.dispatch_moe_unpermute_backward(bf(4, 64), bf(8, 64), f32(4, 3), i32(8), bf(8, 64), f32(4, 2)),
                 lambda: tk.dispatch_moe_unpermute_backward(bf(4, 64), bf(8, 64), f32(4, 2), i32(8), bf(8, 64), bf(4, 2)),
                 lambda: tk.dispatch_moe_grouped_gemm(bf(4, 64), bf(2, 72, 64), i32(4), bf(4, 72)),
                 lambda: tk.dispatch_moe_grouped_gemm(bf(4, 64), bf(2, 72, 64), i32(3), bf(5, 72)),
                 lambda: tk.dispatch_moe_grouped_gemm_dgrad(bf(4, 72), bf(2, 72, 64), i32(3), bf(4, 72)),
                 lambda: tk.dispatch_moe_grouped_gemm_wgrad(bf(4, 72), bf(4, 64), i32(3), i32(8).reshape(2, 2, 2)),
                 lambda: tk.dispatch_moe_grouped_gemm(bf(4, 60), bf(2, 72, 60), i32(3), bf(4, 72)),
                 lambda: tk.dispatch_linear_cross_entropy(bf(4, 64), bf(100, 64), f32(4), f32(4), f32(4), ws),
                 lambda: tk.dispatch_linear_cross_entropy(bf(4, 64), bf(100, 64), i32(5), f32(4), f32(4), ws),
                 lambda: tk.dispatch_linear_cross_entropy(bf(4, 64), bf(100, 64), i32(4), f32(4), f32(5), ws),
                 lambda: tk.dispatch_linear_cross_entropy(bf(4, 64), bf(100, 64), i32(4), f32(4), f32(4), ws[:16]),
                 lambda: tk.dispatch_linear_cross_entropy_backward(bf(4, 64), bf(100, 64), i32(4), f32(4), f32(4), None, None, ws),
                 lambda: tk.dispatch_linear_cross_entropy_backward(bf(4, 64), bf(100, 64), i32(4), f32(4), f32(4), f32(4, 64), None, ws),
                 lambda: tk.dispatch_linear_cross_entropy_backward(bf(4, 64), bf(100, 64), i32(4), f32(4), f32(4), None, bf(99, 64), ws)):
        with pytest.raises(RuntimeError):
            call()
    torch.cuda.synchronize()


def test_linear_cross_entropy_rows_of_one_launch(p):
    """Launches of 64 threads a row, and of a workgroup per eight rows and per 256 classes beside the tiles', hold fewer than
    2^32 threads: more rows are refused, not left to the launch."""
    lib = hk.load_library()
    for M, V in ((1 << 25, 100), (1 << 26, 1), (1 << 27, 100), ((1 << 30) - 1, 8)):
        assert lib.hk_linear_cross_entropy(p, p, p, 1, p, p, M, V, 8, p, 1 << 60, None) == SHAPE
        assert lib.hk_linear_cross_entropy_backward(p, p, p, 1, p, p, p, p, 0, M, V, 8, p, 1 << 60, None) == SHAPE
        assert lib.hk_linear_cross_entropy_workspace_bytes(M, V, 8, 1) == 0
    assert lib.hk_linear_cross_entropy_workspace_bytes((1 << 25) - 1, 100, 8, 1) > 0
