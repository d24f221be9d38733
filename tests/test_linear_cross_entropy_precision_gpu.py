"""Digits of the head's results where single precision or bf16 could lose them: logits that fp32 holds exactly (operands are
small multiples of 1/8), so that every difference from the definitions in 64 bits is the epilogues' and the gradients' own."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _exact_case(M, V, K, seed, size=8, ignored=0.1):
    """x and w: multiples of 1/8 up to size / 8; logits: multiples of 1/64 below 2^18 / 64. Every other row's label is its largest logit."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    eighths = lambda *s: (torch.randint(-size, size + 1, s, device=DEV, generator=g) / 8).to(torch.bfloat16)
    x, w = eighths(M, K), eighths(V, K)
    l = x.double() @ w.double().t().contiguous()
    assert float(l.abs().max()) < 2**12
    labels = torch.randint(0, V, (M,), device=DEV, generator=g)
    labels = torch.where(torch.arange(M, device=DEV) % 2 == 0, l.argmax(dim=1), labels)
    labels[torch.rand(M, device=DEV, generator=g) < ignored] = -100
    return x, w, l, labels, torch.randn(M, device=DEV, generator=g)


def _gradients(hk, x, w, labels, lse, dloss, dw_dtype):
    tk = hk.tk_kernel
    (M, K), V = x.shape, w.shape[0]
    ws = torch.full((tk.linear_cross_entropy_workspace_bytes(M, V, K),), 0xFF, dtype=torch.uint8, device=DEV)
    dx, dw = torch.empty_like(x), torch.full((V + 1, K), 777.0, dtype=dw_dtype, device=DEV)
    tk.dispatch_linear_cross_entropy_backward(x, w, labels, lse, dloss, dx, dw[:V], ws)
    assert torch.all(dw[V] == 777.0)
    return dx, dw[:V]


def _dl(l, labels, lse, dloss):
    """dl for the lse that the call is given, |dl| and the error of |dl| before it is rounded to fewer bits: the exponential's argument
    in fp32 (half a step of lse log2 e and of the difference), the instruction by a step, the products and the difference by half of one."""
    counts = labels >= 0
    hot = torch.zeros_like(l)
    hot[counts, labels[counts]] = 1.0
    scale = torch.where(counts, dloss.double(), 0.0)[:, None]
    lse = lse.double()[:, None]
    p = torch.exp(l - lse)
    arg = (lse.abs() + (l - lse).abs()) * 2**-23
    return scale * (p - hot), scale.abs() * (p * (arg + 2**-21) + (p + hot) * 2**-22) + (scale.abs() + 1) * 2.0**-126


@pytest.mark.parametrize("M,V,K", [(45, 333, 8), (130, 1000, 64), (700, 3000, 64), (973, 1187, 792), (2000, 9001, 264), (40000, 7777, 64)])
def test_weight_gradient_in_fp32_has_more_digits_than_bf16(hk, M, V, K):
    print(f"linear cross entropy, fp32 dw M={M} V={V} K={K}", flush=True)
    x, w, l, labels, dloss = _exact_case(M, V, K, M + K)
    lse = torch.logsumexp(l, dim=1).float()
    _, dw = _gradients(hk, x, w, labels, lse, dloss, torch.float32)
    want, err, size = (torch.zeros(V, K, dtype=torch.float64, device=DEV) for _ in range(3))
    for a in range(0, M, 8000):
        s = slice(a, a + 8000)
        dl, d = _dl(l[s], labels[s], lse[s], dloss[s])
        xd = x[s].double()
        want += dl.t().contiguous() @ xd
        # what is left of dl behind two numbers of bf16: half a step of half a step
        err += (d + (dl.abs() + d) * 2**-16).t().contiguous() @ xd.abs()
        size += dl.abs().t().contiguous() @ xd.abs()
    # 2 M products added in fp32, a step each, doubled for what a matrix instruction does inside; the smallest number of bf16 and fp32
    err += size * 2 * (2 * M + 8) * 2**-24 + 2 * (M + 1) * 2.0**-126
    bad = (dw.double() - want).abs() > err + want.abs() * 2**-24
    assert not bad.any(), (int(bad.sum()), float((dw.double() - want).norm() / want.norm()))


def test_loss_of_confident_rows_and_large_logits(hk):
    """Logits of hundreds: the loss is the sum's logarithm over the label's term and does not carry the rounding of lse, which is
    a hundred times larger than the loss of a confident row; no loss is negative. lse is rounded once."""
    M, V, K = 500, 777, 64
    print("linear cross entropy, loss of large logits", flush=True)
    x, w, l, labels, _ = _exact_case(M, V, K, 3, size=64)
    l0 = l.max(dim=1).values
    tk = hk.tk_kernel
    ws = torch.full((tk.linear_cross_entropy_workspace_bytes(M, V, K, backward=False),), 0xFF, dtype=torch.uint8, device=DEV)
    loss, lse = torch.empty(M, device=DEV), torch.empty(M, device=DEV)
    tk.dispatch_linear_cross_entropy(x, w, labels, loss, lse, ws)
    counts = labels >= 0
    want = torch.logsumexp(l, dim=1)
    mine = l.gather(1, labels.clamp(min=0)[:, None]).squeeze(1)
    # the sum relative to the largest term: at most 100 additions in a row, each half a step, the exponentials' arguments and
    # the instruction a few steps more
    total = 2**-17
    assert ((lse.double() - want).abs() <= want.abs() * 2**-24 + total).all()
    want_loss = torch.where(counts, torch.log(torch.exp(l - mine[:, None]).sum(dim=1)), 0.0)
    want_loss = torch.where(counts & (l0 - mine > 300), want - mine, want_loss)
    # the label's distance from the largest logit times log2 e and ln 2: three roundings of what is at most the loss
    assert ((loss.double() - want_loss).abs() <= total + want_loss * 2**-22).all(), float((loss.double() - want_loss).abs().max())
    assert (loss >= 0).all() and torch.all(loss[~counts] == 0)


def test_gradients_of_confident_rows_and_large_logits(hk):
    """p - 1 of a confident row is far smaller than a rounding of lse log2 e where lse is several hundred: that rounding is not added."""
    M, V, K = 64, 777, 64
    print("linear cross entropy, gradients of confident rows", flush=True)
    g = torch.Generator(device=DEV).manual_seed(4)
    x, w, _, _, dloss = _exact_case(M, V, K, 4, size=64, ignored=0.0)
    # rows of three classes within a few units of one another at the top of some hundred logits
    at = torch.randint(0, V - 3, (M,), device=DEV, generator=g)
    w[1::3], w[2::3] = w[0::3][: w[1::3].shape[0]], w[0::3][: w[2::3].shape[0]]
    top = at // 3 * 3
    x = w[top].clone()
    x[:, 0] = 8.0
    w[:, 0] = ((torch.arange(V, device=DEV) % 3 == 0).float() * 0.875).to(torch.bfloat16)   # 7 ahead of its copies: p - 1 about -2e-3
    l = x.double() @ w.double().t().contiguous()
    lse = torch.logsumexp(l, dim=1).float()
    labels = top.clone()
    dx, dw = _gradients(hk, x, w, labels, lse, dloss, torch.float32)
    hot = torch.zeros_like(l)
    hot[torch.arange(M, device=DEV), labels] = 1.0
    p = torch.exp(l - lse.double()[:, None])
    assert float((1 - p.gather(1, labels[:, None])).max()) < 0.01 and float(lse.abs().min()) > 300
    scale = dloss.double()[:, None]
    dl = scale * (p - hot)
    # as in _dl, without a rounding of lse: the argument's own, which counts where the exponential does (|a| e^a < 1)
    d = scale.abs() * (2**-22 + p * 2**-21 + (p + hot) * 2**-22) + (scale.abs() + 1) * 2.0**-126
    d = torch.where((l - lse.double()[:, None]) < -60, scale.abs() * 2**-60, d)
    half = (dl.abs() + d) * 2**-8 * (1 - hot)
    dx_err = (d + half) @ w.double().abs() + (dl.abs() @ w.double().abs()) * 2 * (V + 8) * 2**-24
    bad = (dx.double() - dl @ w.double()).abs() > dx_err * (1 + 2**-8) + (dl @ w.double()).abs() * 2**-8
    assert not bad.any(), int(bad.sum())
    want = dl.t().contiguous() @ x.double()
    dw_err = ((d + (dl.abs() + d) * 2**-16).t().contiguous() + dl.abs().t().contiguous() * 2 * (2 * M + 8) * 2**-24) @ x.double().abs()
    bad = (dw.double() - want).abs() > dw_err + want.abs() * 2**-24
    assert not bad.any(), (int(bad.sum()), float((dw.double() - want).norm() / want.norm()))


@pytest.mark.parametrize("M,V,K", [(5000, 2, 72), (3001, 17, 264), (4000, 130, 1032), (2500, 40, 8), (6000, 1000, 520)])
@pytest.mark.parametrize("kind", ["spread", "sorted", "one"])
@pytest.mark.parametrize("dw_dtype", [torch.bfloat16, torch.float32])
def test_many_rows_of_each_class(hk, M, V, K, kind, dw_dtype):
    """Hundreds to thousands of rows with a label among the classes of one wave, in the order of the classes or mixed, or all of one
    class: the label's remainder is added for each of them."""
    print(f"linear cross entropy, many rows a class M={M} V={V} K={K} {kind} {dw_dtype}", flush=True)
    x, w, l, labels, dloss = _exact_case(M, V, K, M + V)
    if kind == "sorted":
        labels = labels.sort().values
    elif kind == "one":
        labels = torch.where(labels >= 0, V - 1, labels)
    lse = torch.logsumexp(l, dim=1).float()
    dx, dw = _gradients(hk, x, w, labels, lse, dloss, dw_dtype)
    dl, d = _dl(l, labels, lse, dloss)
    hot = torch.zeros_like(l)
    hot[labels >= 0, labels[labels >= 0]] = 1.0
    xd, wd = x.double(), w.double()
    half = (dl.abs() + d) * 2**-8 * (1 - hot)   # one number of bf16, but for the label's term
    dlt = dl.t().contiguous()
    want = dlt @ xd
    err = (d + (half if dw_dtype == torch.bfloat16 else (dl.abs() + d) * 2**-16)).t().contiguous() @ xd.abs()
    err += (dlt.abs() @ xd.abs()) * 2 * (2 * M + 8) * 2**-24 + 2 * (M + 1) * 2.0**-126
    step = 2**-8 if dw_dtype == torch.bfloat16 else 2**-24
    bad = (dw.double() - want).abs() > err * (1 + step) + want.abs() * step
    assert not bad.any(), (int(bad.sum()), float((dw.double() - want).norm() / want.norm()))
    want = dl @ wd
    err = (d + half) @ wd.abs() + (dl.abs() @ wd.abs()) * 2 * (V + 8) * 2**-24 + 2 * (V + 1) * 2.0**-126
    bad = (dx.double() - want).abs() > err * (1 + 2**-8) + want.abs() * 2**-8
    assert not bad.any(), int(bad.sum())


@pytest.mark.parametrize("M,V,K", [(600, 5, 200), (1500, 40, 504), (2000, 2, 1000)])
@pytest.mark.parametrize("kind", ["spread", "one"])
def test_each_rows_label_term_of_many(hk, M, V, K, kind):
    """Rows of x with one element other than 0: an element of dw is the sum of three rows' products, in which one row's missing or
    misplaced remainder shows."""
    print(f"linear cross entropy, rows of one element M={M} V={V} K={K} {kind}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(M + K)
    _, w, _, labels, dloss = _exact_case(M, V, K, M + V)
    x = torch.zeros(M, K, dtype=torch.bfloat16, device=DEV)
    x[torch.arange(M, device=DEV), torch.arange(M, device=DEV) % K] = (torch.randint(1, 9, (M,), device=DEV, generator=g) / 8).to(torch.bfloat16)
    if kind == "one":
        labels = torch.where(labels >= 0, V // 2, labels)
    l = x.double() @ w.double().t().contiguous()
    lse = torch.logsumexp(l, dim=1).float()
    _, dw = _gradients(hk, x, w, labels, lse, dloss, torch.float32)
    dl, d = _dl(l, labels, lse, dloss)
    hot = torch.zeros_like(l)
    hot[labels >= 0, labels[labels >= 0]] = 1.0
    xd, dlt = x.double(), dl.t().contiguous()
    # two numbers of bf16 and the remainder's two: at most 12 products other than 0, half a step of fp32 each, doubled
    err = (d + (dl.abs() + d) * 2**-16 * (1 - hot)).t().contiguous() @ xd + (dlt.abs() @ xd) * 24 * 2**-24 + 24 * 2.0**-126
    want = dlt @ xd
    bad = (dw.double() - want).abs() > err + want.abs() * 2**-24
    assert not bad.any(), (int(bad.sum()), float((dw.double() - want).norm() / want.norm()))
