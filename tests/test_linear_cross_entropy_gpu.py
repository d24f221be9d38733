"""Softmax cross entropy from the hidden states and its gradients against the definitions in 64 bits, with bounds that follow
the kernels' arithmetic: fp32 sums, the hardware's exponential, dl and the gradients rounded to bf16."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SHAPES = [(1, 1, 8), (1, 1000, 64), (7, 129, 72), (64, 128, 64), (100, 777, 264), (129, 257, 136), (256, 512, 512),
          (300, 2049, 72), (1025, 1300, 200)]
# rows, classes and widths at which 256x256 tiles take over in one product or another, dx cut into several pieces of its sum
LARGE = [(2, 20011, 264), (513, 33000, 520), (2000, 9001, 1032), (3000, 17000, 776)]


def _case(M, V, K, seed, label_dtype=torch.int64, spread=2.0, ignored=0.2):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(M, K, device=DEV, generator=g).to(torch.bfloat16)
    w = (torch.randn(V, K, device=DEV, generator=g) * spread * K**-0.5).to(torch.bfloat16)
    labels = torch.randint(0, V, (M,), device=DEV, generator=g)
    out = torch.tensor([-100, V, -1, 2**31 - 1], device=DEV)
    labels = torch.where(torch.rand(M, device=DEV, generator=g) < ignored, out[torch.arange(M, device=DEV) % 4], labels)
    dloss = torch.randn(M, device=DEV, generator=g)
    return x, w, labels.to(label_dtype), dloss


def _reference(x, w, labels, dloss):
    """Values and error bounds, all in 64 bits."""
    M, K = x.shape
    V = w.shape[0]
    xd, wd = x.double(), w.double()
    wt = wd.t().contiguous()
    l = xd @ wt
    # K products in fp32, a step each, doubled for what a matrix instruction does inside
    dl_err = (xd.abs() @ wt.abs()) * 2 * (K + 8) * 2**-24
    lse = torch.logsumexp(l, dim=1)
    counts = (labels >= 0) & (labels < V)
    at = torch.where(counts, labels.long(), 0)
    mine = l.gather(1, at[:, None]).squeeze(1)
    loss = torch.where(counts, lse - mine, 0.0)
    # lse moves no more than the logit that moves most; the exponentials' and the sums' relative error: an argument a is
    # off by |a| 2^-23 where e^a counts (|a| e^a < 1), the instruction and the additions (at most 256 deep) by 2^-16
    lse_err = dl_err.max(dim=1).values + 2**-16 + lse.abs() * 2**-23
    loss_err = torch.where(counts, lse_err + dl_err.gather(1, at[:, None]).squeeze(1) + (lse.abs() + mine.abs()) * 2**-23, 0.0)
    p = torch.exp(l - lse[:, None])
    hot = torch.zeros_like(p)
    hot[counts, at[counts]] = 1.0
    scale = torch.where(counts, dloss.double(), 0.0)[:, None]
    dl = scale * (p - hot)
    # p is off by its exponent's error, the difference by a step of fp32 of its larger side, dl by half a step of bf16 but for the label's
    d = scale.abs() * (p * (dl_err + lse_err[:, None] + 2**-19) + (p + hot) * 2**-22)
    # fp32 and bf16 hold no normal number below 2^-126: an exponential, a dl, a product or a sum below it may come out as 0
    # (a logit 88 below lse: p < 2^-126), once each
    tiny = 2.0**-126
    d = d + (dl.abs() + d) * 2**-8 * (1 - hot) + (scale.abs() + 1) * tiny   # the label's remainder is kept: no half step there
    dx, dw = dl @ wd, dl.t().contiguous() @ xd
    dx_err = d @ wd.abs() + (dl.abs() @ wd.abs()) * 2 * (V + 8) * 2**-24 + 2 * (V + 1) * tiny
    dw_err = d.t().contiguous() @ xd.abs() + (dl.abs().t().contiguous() @ xd.abs()) * 2 * (M + 8) * 2**-24 + 2 * (M + 1) * tiny
    return (lse, lse_err), (loss, loss_err), (dx, dx_err), (dw, dw_err), counts


def _within(got, want, err, half_step=0.0):
    bad = ~((got.double() - want).abs() <= err * (1 + half_step) + want.abs() * half_step)
    assert not bad.any(), (int(bad.sum()), torch.nonzero(bad)[:4].tolist(), float((got.double() - want).abs().max()))


def _run(hk, x, w, labels, dloss, dw_dtype=torch.bfloat16, workspace=None, want_dx=True, want_dw=True):
    tk = hk.tk_kernel
    (M, K), V = x.shape, w.shape[0]
    if workspace is None:
        workspace = torch.full((tk.linear_cross_entropy_workspace_bytes(M, V, K),), 0xFF, dtype=torch.uint8, device=DEV)
    full = lambda *s, dtype=torch.float32: torch.full(s, 777.0, dtype=dtype, device=DEV)
    loss, lse = full(M + 1), full(M + 1)
    dx = full(M + 1, K, dtype=torch.bfloat16) if want_dx else None
    dw = full(V + 1, K, dtype=dw_dtype) if want_dw else None
    tk.dispatch_linear_cross_entropy(x, w, labels, loss[:M], lse[:M], workspace)
    tk.dispatch_linear_cross_entropy_backward(x, w, labels, lse[:M], dloss, dx[:M] if want_dx else None,
                                              dw[:V] if want_dw else None, workspace)
    for t in (loss[M], lse[M], *((dx[M],) if want_dx else ()), *((dw[V],) if want_dw else ())):
        assert torch.all(t == t.new_tensor(777.0))
    return loss[:M], lse[:M], dx[:M] if want_dx else None, dw[:V] if want_dw else None


@pytest.mark.parametrize("M,V,K", SHAPES + LARGE)
@pytest.mark.parametrize("label_dtype", [torch.int32, torch.int64])
def test_loss_and_gradients(hk, M, V, K, label_dtype):
    print(f"linear cross entropy M={M} V={V} K={K} {label_dtype}", flush=True)
    x, w, labels, dloss = _case(M, V, K, M + V + K, label_dtype)
    if M == 1:
        labels[0] = V // 2
    lse_r, loss_r, dx_r, dw_r, counts = _reference(x, w, labels, dloss)
    dw_dtype = torch.float32 if label_dtype == torch.int32 else torch.bfloat16
    loss, lse, dx, dw = _run(hk, x, w, labels, dloss, dw_dtype)
    _within(lse, *lse_r)
    _within(loss, *loss_r)
    _within(dx, *dx_r, 2**-8)
    _within(dw, *dw_r, 2**-8 if dw_dtype == torch.bfloat16 else 2**-24)
    assert torch.all(loss[~counts] == 0) and torch.all(dx[~counts] == 0)


def test_large_and_far_logits(hk):
    """Logits of several hundred, equal logits and a maximum in the last, ragged tile."""
    M, V, K = 70, 1031, 64
    print("linear cross entropy, large logits", flush=True)
    x, w, labels, dloss = _case(M, V, K, 1, spread=120.0)
    x[3] = 0                      # all logits equal
    w[V - 1] = w[V - 1].sign() * 3
    x[5] = w[V - 1].sign() * 8     # its maximum is the last logit
    labels[5], labels[3] = V - 1, 0
    lse_r, loss_r, dx_r, dw_r, _ = _reference(x, w, labels, dloss)
    loss, lse, dx, dw = _run(hk, x, w, labels, dloss)
    _within(lse, *lse_r)
    _within(loss, *loss_r)
    _within(dx, *dx_r, 2**-8)
    _within(dw, *dw_r, 2**-8)


def test_every_row_ignored_and_rows_that_do_not_count(hk):
    M, V, K = 130, 300, 72
    print("linear cross entropy, ignored rows", flush=True)
    x, w, labels, dloss = _case(M, V, K, 2, ignored=0.0)
    none = torch.full_like(labels, -100)
    loss, lse, dx, dw = _run(hk, x, w, none, torch.full_like(dloss, float("nan")))
    assert torch.all(loss == 0) and torch.all(dx == 0) and torch.all(dw == 0)
    # rows without a label take no part, whatever they hold
    pad = torch.arange(M, device=DEV) % 7 == 3
    some = torch.where(pad, -100, labels)
    clean = _run(hk, x, w, some, dloss)
    x2 = x.clone()
    x2[pad] = float("nan")
    x2[3] = float("inf")
    got = _run(hk, x2, w, some, torch.where(pad, float("nan"), dloss))
    assert torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2]) and torch.equal(got[3], clean[3])
    # a row's NaN or infinity stays in its row of loss, lse and dx
    labels[10] = -100
    x2 = x.clone()
    x2[20] = float("nan")
    x2[21, 0] = float("inf")
    clean = _run(hk, x, w, labels, dloss)
    loss, lse, dx, _ = _run(hk, x2, w, labels, dloss, want_dw=False)
    rest = torch.ones(M, dtype=torch.bool, device=DEV)
    rest[20:22] = False
    assert torch.isnan(loss[20]) and torch.isnan(lse[20]) and torch.isnan(dx[20]).all() and not torch.isfinite(loss[21])
    assert torch.equal(loss[rest], clean[0][rest]) and torch.equal(dx[rest], clean[2][rest])


@pytest.mark.parametrize("M,V,K", [(700, 300, 72), (2100, 17000, 776)])
def test_labels_that_crowd_a_few_classes(hk, M, V, K):
    """Hundreds of rows with one label, and more than 64 among the classes of one wave: none in the blocks around them."""
    print(f"linear cross entropy, crowded labels M={M} V={V} K={K}", flush=True)
    x, w, labels, dloss = _case(M, V, K, 12)
    kind = torch.arange(M, device=DEV) % 3
    labels = torch.where(kind == 0, 37, torch.where(kind == 1, V - 1 - torch.arange(M, device=DEV) % 130, labels))
    lse_r, loss_r, dx_r, dw_r, _ = _reference(x, w, labels, dloss)
    loss, lse, dx, dw = _run(hk, x, w, labels, dloss, torch.float32)
    _within(loss, *loss_r)
    _within(dx, *dx_r, 2**-8)
    _within(dw, *dw_r, 2**-24)
    # every label the same
    same = torch.full_like(labels, V // 2)
    _, _, dx_r, dw_r, _ = _reference(x, w, same, dloss)
    _, _, dx, dw = _run(hk, x, w, same, dloss, torch.float32)
    _within(dx, *dx_r, 2**-8)
    _within(dw, *dw_r, 2**-24)


def test_one_gradient_alone_has_the_same_bits(hk):
    x, w, labels, dloss = _case(200, 700, 136, 4)
    print("linear cross entropy, one gradient", flush=True)
    both = _run(hk, x, w, labels, dloss)
    assert torch.equal(_run(hk, x, w, labels, dloss, want_dw=False)[2], both[2])
    assert torch.equal(_run(hk, x, w, labels, dloss, want_dx=False)[3], both[3])
    assert torch.equal(_run(hk, x, w, labels, dloss)[3], both[3])


def test_gradients_against_differences(hk):
    """(loss(x + h d) - loss(x - h d)) / 2h along directions d that bf16 holds exactly, against <dx, d> and <dw, d>."""
    M, V, K = 40, 333, 64
    print("linear cross entropy, differences", flush=True)
    g = torch.Generator(device=DEV).manual_seed(9)
    quarter = lambda *s: (torch.randint(-8, 9, s, device=DEV, generator=g) / 8).to(torch.bfloat16)
    x, w = quarter(M, K), quarter(V, K)
    _, _, labels, dloss = _case(M, V, K, 9)
    _, _, dx, dw = _run(hk, x, w, labels, dloss, torch.float32)
    h = 2.0**-6
    for name in ("x", "w"):
        d = torch.randint(-1, 2, (x if name == "x" else w).shape, device=DEV, generator=g).to(torch.bfloat16)
        total = []
        for sign in (1, -1):
            moved = ((x if name == "x" else w).float() + sign * h * d.float()).to(torch.bfloat16)   # exact: eighths and 64ths below 2
            xs, ws = (moved, w) if name == "x" else (x, moved)
            total.append((_run(hk, xs, ws, labels, dloss)[0].double() * dloss.double()).sum())
        slope = (total[0] - total[1]) / (2 * h)
        want = ((dx if name == "x" else dw).double() * d.double()).sum()
        # third derivative of a row's loss along d: at most 2 (spread of the logits' motion)^3, the motion <= sum |.| <= K
        lse_r, loss_r, dx_r, dw_r, counts = _reference(x, w, labels, dloss)
        move = (d.double() @ w.double().t().contiguous() if name == "x" else x.double() @ d.double().t().contiguous()).abs().max(dim=1).values
        cut = (dloss.double().abs() * counts * 2 * (2 * move) ** 3).sum() * h * h / 6
        noise = (loss_r[1] * dloss.double().abs()).sum() * 1.5 / h
        grad_err = ((dx_r if name == "x" else dw_r)[1] + (dx_r if name == "x" else dw_r)[0].abs() * 2**-8) * d.double().abs()
        assert (slope - want).abs() <= cut + noise + grad_err.sum()


def test_pieces_of_the_vocabulary(hk):
    """Rows enough that the vocabulary takes several pieces, the last one ragged; against rows taken a few at a time."""
    M, V, K = 40000, 7777, 64
    print("linear cross entropy, pieces", flush=True)
    x, w, labels, dloss = _case(M, V, K, 6)
    tk = hk.tk_kernel
    assert tk.linear_cross_entropy_workspace_bytes(M, V, K) < 2 * M * V     # not the whole of dl
    loss, lse, dx, dw = _run(hk, x, w, labels, dloss, torch.float32)
    total = torch.zeros(V, K, dtype=torch.float64, device=DEV)
    bound = torch.zeros_like(total)
    for a in range(0, M, 8000):
        s = slice(a, a + 8000)
        lse_r, loss_r, dx_r, dw_r, _ = _reference(x[s], w, labels[s], dloss[s])
        _within(lse[s], *lse_r)
        _within(loss[s], *loss_r)
        _within(dx[s], *dx_r, 2**-8)
        total += dw_r[0]
        bound += dw_r[1] * 5      # 40000 rows' additions instead of 8000
    _within(dw, total, bound, 2**-24)


@pytest.mark.parametrize("M,V", [(40000, 30011), (3000, 100003)])
def test_pieces_by_the_tiles_of_either_gradient(hk, M, V):
    """Many rows of few columns: pieces larger than for few rows, dw's tiles the longer items of a launch; few rows and many classes:
    dx's. Both in more than one piece."""
    K = 64
    print(f"linear cross entropy, pieces M={M} V={V}", flush=True)
    x, w, labels, dloss = _case(M, V, K, 7)
    assert hk.tk_kernel.linear_cross_entropy_workspace_bytes(M, V, K) < 2 * M * V     # not the whole of dl
    loss, lse, dx, dw = _run(hk, x, w, labels, dloss, torch.float32)
    total = torch.zeros(V, K, dtype=torch.float64, device=DEV)
    bound = torch.zeros_like(total)
    parts = -(-M // 8000)
    for a in range(0, M, 8000):
        s = slice(a, a + 8000)
        lse_r, loss_r, dx_r, dw_r, _ = _reference(x[s], w, labels[s], dloss[s])
        _within(lse[s], *lse_r)
        _within(loss[s], *loss_r)
        _within(dx[s], *dx_r, 2**-8)
        total += dw_r[0]
        bound += dw_r[1] * parts   # M rows' additions instead of one part's
    _within(dw, total, bound, 2**-24)


@pytest.mark.parametrize("M,V,K", [(973, 1187, 792), (311, 2478, 1480), (64, 64, 2056), (130, 6000, 136)])
@pytest.mark.parametrize("crowded", [False, True])
def test_few_tiles(hk, M, V, K, crowded):
    """No more tiles than CUs in the logits, the gradients or both, with labels all over and on a few classes."""
    print(f"linear cross entropy, few tiles M={M} V={V} K={K} crowded={crowded}", flush=True)
    x, w, labels, dloss = _case(M, V, K, M + K)
    if crowded:
        labels = torch.where(torch.arange(M, device=DEV) % 2 == 0, V // 2 + torch.arange(M, device=DEV) % 17, labels)
    lse_r, loss_r, dx_r, dw_r, _ = _reference(x, w, labels, dloss)
    for dw_dtype, half in ((torch.bfloat16, 2**-8), (torch.float32, 2**-24)):
        loss, lse, dx, dw = _run(hk, x, w, labels, dloss, dw_dtype)
        _within(lse, *lse_r)
        _within(loss, *loss_r)
        _within(dx, *dx_r, 2**-8)
        _within(dw, *dw_r, half)
