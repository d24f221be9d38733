"""Offsets that are out of range or out of order: the experts' rows are those of the offsets held inside [0, R] with a running maximum,
so that no row belongs to two experts, in the products and in both gradients."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("R,E,N,K,broken", [(50, 3, 136, 72, {0: -5, 1: 20, 2: 10, 3: 2**31 - 1}),
                                            (700, 6, 264, 520, {0: 30, 1: 400, 2: 100, 3: 90, 4: 650, 5: -2**31, 6: 690}),
                                            (3000, 130, 72, 136, {0: 0, 3: 2500, 40: 2600, 100: 7, 128: 5000, 129: 1, 130: 2}),
                                            (5000, 512, 72, 64, {0: 100, 1: 9, 8: 50, 9: 3000, 511: 4999, 512: 0})])
def test_out_of_order_offsets_are_a_running_maximum(hk, R, E, N, K, broken):
    print(f"grouped offsets out of order R={R} E={E}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(R + E)
    bf = lambda *s: torch.randn(*s, device=DEV, generator=g).to(torch.bfloat16)
    x, dy, w = bf(R, K), bf(R, N), bf(E, N, K)
    host = [broken.get(e, R * e // E) for e in range(E + 1)]
    offsets = torch.tensor(host, dtype=torch.int32, device=DEV)
    held, top = [], 0
    for o in host:
        top = max(top, min(max(o, 0), R))
        held.append(top)
    tk = hk.tk_kernel

    def run(table):
        y, dx, dw = torch.full((R, N), 777.0, dtype=torch.bfloat16, device=DEV), torch.full_like(x, 777.0), torch.full_like(w, 777.0)
        tk.dispatch_moe_grouped_gemm(x, w, table, y)
        tk.dispatch_moe_grouped_gemm_dgrad(dy, w, table, dx)
        tk.dispatch_moe_grouped_gemm_wgrad(dy, x, table, dw)
        return y, dx, dw

    got = run(offsets)
    for a, b in zip(got, run(torch.tensor(held, dtype=torch.int32, device=DEV))):
        assert torch.equal(a, b)
    # and those rows are right: K (N) products in fp32, a step each, doubled, then half a step of bf16
    for e in range(E):
        a, b = held[e], held[e + 1]
        if b == a:
            assert torch.all(got[2][e] == 0)
            continue
        we, xe, ge = w[e].double(), x[a:b].double(), dy[a:b].double()
        wt, gt = we.t().contiguous(), ge.t().contiguous()
        for t, want, size, terms in ((got[0][a:b], xe @ wt, xe.abs() @ wt.abs(), K), (got[1][a:b], ge @ we, ge.abs() @ we.abs(), N),
                                     (got[2][e], gt @ xe, gt.abs() @ xe.abs(), b - a)):
            assert ((t.double() - want).abs() <= want.abs() * 2**-8 + size * 2 * (terms + 8) * 2**-24).all()
    for t in (got[0], got[1]):
        assert torch.all(t[:held[0]] == 777.0) and torch.all(t[held[-1]:] == 777.0)
