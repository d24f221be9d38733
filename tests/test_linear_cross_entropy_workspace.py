"""The head's workspace never shrinks when there are more rows: a program that allocates it once for its largest batch runs every
smaller one in it."""
import pytest
import torch

import hipkittens_amd as hk

tk = hk.tk_kernel


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("V,K", [(129280, 7168), (32000, 1024), (50257, 1024), (14000, 1024), (201088, 2880), (1000, 64), (2, 8), (300, 8),
                                 (100003, 64), (1046, 5128), (7777, 64), (200, 1 << 15)])
def test_size_never_shrinks_with_more_rows(V, K, backward):
    most = min((1 << 25) - 1, 128 * (((1 << 23) - 1) // max(-(-V // 128), -(-K // 128))))
    Ms = set(range(1, 3000)) | {m + d for m in range(2900, 40000, 251) for d in (-1, 0, 1)} | set(range(40000, 300000, 7919))
    Ms |= {1 << i for i in range(25)} | {most}
    Ms = sorted(m for m in Ms if m <= most)
    sizes = [tk.linear_cross_entropy_workspace_bytes(M, V, K, backward=backward) for M in Ms]
    assert all(s > 0 for s in sizes)
    shrinks = [(a, b, s, t) for a, b, s, t in zip(Ms, Ms[1:], sizes, sizes[1:]) if t < s]
    assert not shrinks, (len(shrinks), shrinks[:3])


@pytest.mark.gpu
@pytest.mark.parametrize("V,K,largest,batches", [(14000, 1024, 65, (64, 33, 1)), (32000, 1024, 300, (256, 129, 128, 7)),
                                                 (2083, 4272, 700, (600, 300, 38)), (7777, 64, 40000, (39000, 5000))])
@pytest.mark.parametrize("dw_dtype", [torch.bfloat16, torch.float32])
def test_small_batches_in_the_largest_ones_workspace(V, K, largest, batches, dw_dtype):
    dev = "cuda:0"
    print(f"linear cross entropy, one workspace V={V} K={K} {largest} {dw_dtype}", flush=True)
    g = torch.Generator(device=dev).manual_seed(V)
    w = (torch.randn(V, K, device=dev, generator=g) * 2 * K**-0.5).to(torch.bfloat16)
    for backward in (False, True):
        size = tk.linear_cross_entropy_workspace_bytes(largest, V, K, backward=backward)
        ws = torch.empty(size + 4096, dtype=torch.uint8, device=dev)
        for M in (largest, *batches):
            x = torch.randn(M, K, device=dev, generator=g).to(torch.bfloat16)
            labels, dloss = torch.randint(0, V, (M,), device=dev, generator=g), torch.randn(M, device=dev, generator=g)
            own = torch.empty(tk.linear_cross_entropy_workspace_bytes(M, V, K), dtype=torch.uint8, device=dev)
            out = []
            for buf in (ws[:size], own):
                ws.fill_(0xFF)
                own.fill_(0xFF)
                loss, lse = torch.empty(M, device=dev), torch.empty(M, device=dev)
                dx, dw = torch.empty_like(x), torch.empty(V, K, dtype=dw_dtype, device=dev)
                tk.dispatch_linear_cross_entropy(x, w, labels, loss, lse, buf)
                if backward:
                    tk.dispatch_linear_cross_entropy_backward(x, w, labels, lse, dloss, dx, dw, buf)
                out.append((loss, lse) + ((dx, dw) if backward else ()))
            for a, b in zip(*out):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
            assert torch.all(ws[size:] == 0xFF)   # nothing is written behind the workspace
