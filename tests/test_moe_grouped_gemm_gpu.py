"""The experts' products in bf16 and both gradients against the definitions in 64 bits: experts without rows, one row, rows
on both sides of a tile, unused rows, NaNs in what must not be read, widths that end inside a tile and a 16-byte chunk."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

# rows of each expert, unused rows behind
ROWS = [([1], 0), ([0, 3, 0], 2), ([127, 128, 129], 0), ([1, 255, 0, 256, 257, 2], 5), ([700], 1), ([0, 0, 0], 4),
        ([5] * 40 + [0] * 5 + [130, 64, 63, 65], 0)]
WIDTHS = [(8, 8), (64, 72), (136, 520), (256, 256), (392, 1000), (1032, 264)]


def _bf(t):
    return t.to(torch.bfloat16)


def _case(rows, unused, N, K, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    off = [0]
    for r in rows:
        off.append(off[-1] + r)
    R, E = off[-1] + unused, len(rows)
    mk = lambda *s: _bf(torch.randn(*s, device=DEV, generator=g))
    x, dy, w = mk(R, K), mk(R, N), mk(E, N, K)
    x[off[-1]:] = float("nan")    # rows behind the last expert's are not read
    dy[off[-1]:] = float("nan")
    return off, torch.tensor(off, dtype=torch.int32, device=DEV), x, dy, w


def _close(got, want, size, terms, half_step):
    """|got - want| at most: `terms` products summed in fp32 (a step of fp32 of the sum so far each, doubled for the order
    and rounding inside a matrix instruction, which are not specified), then the result's half step."""
    bound = want.abs() * half_step + size * 2 * (terms + 8) * 2**-24
    bad = (got.double() - want).abs() > bound
    assert not bad.any(), (int(bad.sum()), torch.nonzero(bad)[:4].tolist(), float((got.double() - want).abs().max()))
    assert torch.isfinite(got).all()


# enough tiles for the 256x256 kernels in every product: rows on both sides of a tile, K-steps on both sides of one and two
LARGE = [([2049, 0, 255, 257, 1, 3000, 63, 65, 129], 3, 2312, 2056), ([4000, 1000, 4500], 0, 1544, 1800), ([9000], 9, 1800, 72),
         ([100, 0, 64, 65, 127, 128, 129, 191, 257, 1] * 4, 0, 776, 840)]   # (tiles enough for the single-stage kernel, several K-steps)


@pytest.mark.parametrize("case", range(len(LARGE)))
def test_large_products_and_gradients(hk, case):
    rows, unused, N, K = LARGE[case]
    _products_and_gradients(hk, rows, unused, N, K, 1000 + case)


@pytest.mark.parametrize("N,K", WIDTHS)
@pytest.mark.parametrize("case", range(len(ROWS)))
def test_products_and_gradients(hk, case, N, K):
    _products_and_gradients(hk, *ROWS[case], N, K, 17 * case + N + K)


def _products_and_gradients(hk, rows, unused, N, K, seed):
    off, offsets, x, dy, w = _case(rows, unused, N, K, seed)
    R, E = x.shape[0], len(rows)
    print(f"grouped rows={rows[:8]} unused={unused} N={N} K={K}", flush=True)
    y = torch.full((R + 1, N), 777.0, dtype=torch.bfloat16, device=DEV)
    dx = torch.full((R + 1, K), 777.0, dtype=torch.bfloat16, device=DEV)
    dw = torch.full((E + 1, N, K), 777.0, dtype=torch.bfloat16, device=DEV)
    dw32 = torch.full((E + 1, N, K), 777.0, dtype=torch.float32, device=DEV)
    tk = hk.tk_kernel
    tk.dispatch_moe_grouped_gemm(x, w, offsets, y[:R])
    tk.dispatch_moe_grouped_gemm_dgrad(dy, w, offsets, dx[:R])
    tk.dispatch_moe_grouped_gemm_wgrad(dy, x, offsets, dw[:E])
    tk.dispatch_moe_grouped_gemm_wgrad(dy, x, offsets, dw32[:E])
    for e in range(E):
        a, b = off[e], off[e + 1]
        xe, ge, we = x[a:b].double(), dy[a:b].double(), w[e].double()
        if b > a:
            wt = we.t().contiguous()
            _close(y[a:b], xe @ wt, xe.abs() @ wt.abs(), K, 2**-8)
            _close(dx[a:b], ge @ we, ge.abs() @ we.abs(), N, 2**-8)
        gt = ge.t().contiguous()
        want, size = gt @ xe, gt.abs() @ xe.abs()
        _close(dw[e], want, size, b - a, 2**-8)
        _close(dw32[e], want, size, b - a, 2**-24)
    for t in (y[off[-1]:], dx[off[-1]:], dw[E], dw32[E]):
        assert torch.all(t == t.new_tensor(777.0))


@pytest.mark.parametrize("N,K", [(136, 264), (520, 520)])
def test_an_experts_nans_stay_with_it(hk, N, K):
    rows = [70, 33, 0, 130]
    off, offsets, x, dy, w = _case(rows, 0, N, K, 3)
    print(f"grouped NaN isolation N={N} K={K}", flush=True)
    x[off[1]:off[2]] = float("nan")
    dy[off[1]:off[2]] = float("inf")
    w[1] = float("nan")
    y, dx, dw = torch.empty_like(dy), torch.empty_like(x), torch.empty_like(w)
    tk = hk.tk_kernel
    tk.dispatch_moe_grouped_gemm(x, w, offsets, y)
    tk.dispatch_moe_grouped_gemm_dgrad(dy, w, offsets, dx)
    tk.dispatch_moe_grouped_gemm_wgrad(dy, x, offsets, dw)
    assert torch.isnan(y[off[1]:off[2]]).all() and torch.isnan(dx[off[1]:off[2]]).all() and torch.isnan(dw[1]).all()
    for e in (0, 2, 3):
        a, b = off[e], off[e + 1]
        assert torch.isfinite(y[a:b]).all() and torch.isfinite(dx[a:b]).all() and torch.isfinite(dw[e]).all()
    # one row's NaN stays in that row
    x = torch.zeros_like(x)
    x[7] = float("nan")
    tk.dispatch_moe_grouped_gemm(x, w, offsets, y)
    assert torch.isnan(y[7]).all() and torch.isfinite(y[:7]).all() and torch.isfinite(y[8:off[1]]).all()


def test_results_do_not_depend_on_the_other_experts(hk):
    """The same bits for an expert alone and among others, and on every call."""
    rows = [300, 1, 517, 0, 64]
    N, K = 776, 520
    off, offsets, x, dy, w = _case(rows, 0, N, K, 5)
    tk = hk.tk_kernel
    print("grouped independence", flush=True)

    def run(x, dy, w, offsets):
        y, dx, dw = torch.empty_like(dy), torch.empty_like(x), torch.empty(w.shape, device=DEV)
        tk.dispatch_moe_grouped_gemm(x, w, offsets, y)
        tk.dispatch_moe_grouped_gemm_dgrad(dy, w, offsets, dx)
        tk.dispatch_moe_grouped_gemm_wgrad(dy, x, offsets, dw)
        return y, dx, dw

    y, dx, dw = run(x, dy, w, offsets)
    for again in run(x, dy, w, offsets):
        assert any(torch.equal(again, t) for t in (y, dx, dw) if t.shape == again.shape and t.dtype == again.dtype)
    for e in (0, 2):
        a, b = off[e], off[e + 1]
        alone = run(x[a:b].clone(), dy[a:b].clone(), w[e:e + 1].clone(),
                    torch.tensor([0, b - a], dtype=torch.int32, device=DEV))
        assert torch.equal(alone[0], y[a:b]) and torch.equal(alone[1], dx[a:b]) and torch.equal(alone[2][0], dw[e])


def test_offsets_out_of_order_or_range_stay_inside_the_buffers(hk):
    """Offsets are held inside [0, R] and in order: nothing outside the R rows is written, an expert in order is right."""
    N, K, R = 136, 72, 50
    print("grouped broken offsets", flush=True)
    g = torch.Generator(device=DEV).manual_seed(11)
    x, dy = _bf(torch.randn(R, K, device=DEV, generator=g)), _bf(torch.randn(R, N, device=DEV, generator=g))
    w = _bf(torch.randn(3, N, K, device=DEV, generator=g))
    offsets = torch.tensor([-5, 20, 10, 2**31 - 1], dtype=torch.int32, device=DEV)
    y = torch.full((R + 1, N), 777.0, dtype=torch.bfloat16, device=DEV)
    dw = torch.full((4, N, K), 777.0, device=DEV)
    hk.tk_kernel.dispatch_moe_grouped_gemm(x, w, offsets, y[:R])
    hk.tk_kernel.dispatch_moe_grouped_gemm_wgrad(dy, x, offsets, dw[:3])
    assert torch.all(y[R] == 777.0) and torch.all(dw[3] == 777.0)
    want = dy[:20].double().t().contiguous() @ x[:20].double()
    _close(dw[0], want, dy[:20].double().abs().t().contiguous() @ x[:20].double().abs(), 20, 2**-24)
    assert torch.all(dw[1] == 0)   # [20, 20)


@pytest.mark.parametrize("E", [1, 511, 512])
def test_many_experts(hk, E):
    g = torch.Generator(device=DEV).manual_seed(E)
    N, K, R = 72, 136, 2 * E + 3
    print(f"grouped E={E}", flush=True)
    ids = torch.sort(torch.randint(0, E, (R,), device=DEV, generator=g)).values
    offsets = torch.searchsorted(ids, torch.arange(E + 1, device=DEV)).to(torch.int32)
    x, w = _bf(torch.randn(R, K, device=DEV, generator=g)), _bf(torch.randn(E, N, K, device=DEV, generator=g))
    y = torch.empty(R, N, dtype=torch.bfloat16, device=DEV)
    hk.tk_kernel.dispatch_moe_grouped_gemm(x, w, offsets, y)
    we = w[ids].double()
    want = (we * x[:, None].double()).sum(dim=2)
    _close(y, want, (we * x[:, None].double()).abs().sum(dim=2), K, 2**-8)


def test_weight_gradient_of_a_long_expert(hk):
    """More than 2^32 bytes of one expert's rows: the sum over 300001 rows is a count where all elements are 1."""
    R, N, K = 300001, 8192, 64
    print(f"grouped wgrad R={R} N={N} K={K}", flush=True)
    dy = torch.ones(R, N, dtype=torch.bfloat16, device=DEV)
    x = torch.ones(R, K, dtype=torch.bfloat16, device=DEV)
    dy[-1], x[-1] = 64.0, 2.0
    dw = torch.empty(1, N, K, device=DEV)
    hk.tk_kernel.dispatch_moe_grouped_gemm_wgrad(dy, x, torch.tensor([0, R], dtype=torch.int32, device=DEV), dw)
    assert torch.all(dw == R - 1 + 128)   # below 2^24: exact in fp32
    dx = torch.zeros(R, K, dtype=torch.bfloat16, device=DEV)
    w = torch.zeros(1, N, K, dtype=torch.bfloat16, device=DEV)
    w[0, -1] = 1.0
    hk.tk_kernel.dispatch_moe_grouped_gemm_dgrad(dy, w, torch.tensor([0, R], dtype=torch.int32, device=DEV), dx)
    assert torch.all(dx[:-1] == 1) and torch.all(dx[-1] == 64)


@pytest.mark.parametrize("N,K", [(2056, 1544), (776, 3080), (2056, 8)])
@pytest.mark.parametrize("rows,unused", [([300, 200, 500], 0), ([700], 3), ([3, 0, 9, 1], 0), ([1500], 0)])
def test_products_between_the_tile_sizes(hk, rows, unused, N, K):
    """More tiles of 64x64 than CUs and fewer of 128x128, or just as many of the former, and contractions of one K-step to dozens."""
    _products_and_gradients(hk, rows, unused, N, K, 5000 + N + K + rows[0])
