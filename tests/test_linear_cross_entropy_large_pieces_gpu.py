"""A piece of dl larger than 2 GB, as the head's gradients make them for many rows: rows and classes on both sides of every 2 GB."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dw_dtype", [torch.bfloat16, torch.float32])
def test_piece_beyond_two_gigabytes(hk, dw_dtype):
    M, V, K = 131072, 32011, 64
    print(f"linear cross entropy, large piece M={M} V={V} K={K} {dw_dtype}", flush=True)
    tk = hk.tk_kernel
    g = torch.Generator(device=DEV).manual_seed(21)
    x = torch.randn(M, K, device=DEV, generator=g).to(torch.bfloat16)
    w = (torch.randn(V, K, device=DEV, generator=g) * 2 * K**-0.5).to(torch.bfloat16)
    labels = torch.randint(0, V, (M,), device=DEV, generator=g)
    labels[::9] = -100
    dloss = torch.randn(M, device=DEV, generator=g)
    size = tk.linear_cross_entropy_workspace_bytes(M, V, K)
    assert size > 3 << 30
    ws = torch.empty(size, dtype=torch.uint8, device=DEV)
    ws.fill_(0xFF)
    loss, lse, dx, dw = torch.empty(M, device=DEV), torch.empty(M, device=DEV), torch.empty_like(x), torch.empty(V, K, dtype=dw_dtype, device=DEV)
    tk.dispatch_linear_cross_entropy(x, w, labels, loss, lse, ws)
    tk.dispatch_linear_cross_entropy_backward(x, w, labels, lse, dloss, dx, dw, ws)
    counts = labels >= 0

    def dl_of(rows, classes):
        """dl [rows, classes] in 64 bits for the call's own lse, and its error: logits' (K products in fp32, doubled), lse's and the
        exponential's argument's roundings, the instruction, and half a step of bf16."""
        xr, wc = x[rows].double(), w[classes].double().t().contiguous()
        l, l_err = xr @ wc, (xr.abs() @ wc.abs()) * 2 * (K + 8) * 2**-24
        hot = (labels[rows][:, None] == classes[None]).double()
        scale = torch.where(counts[rows], dloss[rows].double(), 0.0)[:, None]
        own = lse[rows].double()[:, None]
        p = torch.exp(l - own)
        d = scale.abs() * (p * (l_err + (own.abs() + (l - own).abs()) * 2**-23 + 2**-21) + (p + hot) * 2**-22)
        dl = scale * (p - hot)
        return dl, d + (dl.abs() + d) * 2**-8 * (1 - hot) + (scale.abs() + 1) * 2.0**-126

    every_row, every_class = torch.arange(M, device=DEV), torch.arange(V, device=DEV)
    # rows at both ends, in the middle and around the multiples of 2 GB of a piece's rows of 8 to 32 KB
    rows = torch.cat([torch.arange(a - 20, a + 20, device=DEV) for a in (20, 32768, 65536, 98304, M - 20)] + [torch.randint(0, M, (200,), device=DEV, generator=g)])
    dl, d = dl_of(rows, every_class)
    wd = w.double()
    want = dl @ wd
    bad = (dx[rows].double() - want).abs() > (d @ wd.abs() + (dl.abs() @ wd.abs()) * 2 * (V + 8) * 2**-24) * (1 + 2**-8) + want.abs() * 2**-8
    assert not bad.any(), int(bad.sum())
    classes = torch.cat([torch.arange(a - 16, a + 16, device=DEV) for a in (16, 8192, 16384, 24576, V - 16)])
    dl, d = dl_of(every_row, classes)
    dlt, xd = dl.t().contiguous(), x.double()
    want = dlt @ xd
    err = d.t().contiguous() @ xd.abs() + (dlt.abs() @ xd.abs()) * 2 * (2 * M + 8) * 2**-24
    bad = (dw[classes].double() - want).abs() > err * (1 + 2**-8) + want.abs() * (2**-8 if dw_dtype == torch.bfloat16 else 2**-24)
    assert not bad.any(), int(bad.sum())
