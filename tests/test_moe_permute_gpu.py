"""Rows to the order of their experts and the gradients around the weighted un-permute, against the definitions in 64 bits:
every form of the choice count, widths around a workgroup's column chunks, slots without a row, rows that no slot names."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SHAPES = [(1, 1, 8), (1, 4, 504), (3, 4, 512), (4, 5, 520), (16, 8, 7168), (2, 10, 1032), (255, 2, 576), (256, 2, 576),
          (257, 3, 2056), (300, 9, 2880), (33, 64, 64)]


def _rand(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g).to(torch.bfloat16)


def _positions(g, T, k, drop):
    """A permutation of the slots, the slots of some tokens and some single ones without a row: (slot_to_pos, live slots)"""
    S = T * k
    pos = torch.randperm(S, device=DEV, generator=g).to(torch.int32)
    if drop:
        dead = torch.rand(S, device=DEV, generator=g) < 0.2
        dead |= (torch.rand(T, device=DEV, generator=g) < 0.2).repeat_interleave(k)
        bad = torch.tensor([-1, S, S + 7, -2**31, 2**31 - 1], dtype=torch.int32, device=DEV)
        pos = torch.where(dead, bad[torch.arange(S, device=DEV) % 5], pos)
    live = torch.nonzero((pos >= 0) & (pos < S)).squeeze(1)
    return pos, live


@pytest.mark.parametrize("T,k,H", SHAPES)
@pytest.mark.parametrize("drop", [False, True])
def test_permute_copies_every_row_and_no_other(hk, T, k, H, drop):
    print(f"permute T={T} k={k} H={H} drop={drop}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(T * 131 + H)
    x = _rand(g, T, H)
    pos, live = _positions(g, T, k, drop)
    xp = torch.full((T * k + 1, H), 777.0, dtype=torch.bfloat16, device=DEV)
    want = xp.clone()
    want[pos[live].long()] = x[live // k]
    hk.tk_kernel.dispatch_moe_permute(x, pos, xp[:-1])
    assert torch.equal(xp.view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("T,k,H", SHAPES)
@pytest.mark.parametrize("drop", [False, True])
@pytest.mark.parametrize("add", [None, "other", "itself"])
def test_permute_backward_sums_a_tokens_rows(hk, T, k, H, drop, add):
    print(f"permute backward T={T} k={k} H={H} drop={drop} add={add}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(T * 137 + H)
    dxp = _rand(g, T * k, H)
    pos, live = _positions(g, T, k, drop)
    if drop:   # what no slot names is not read
        named = torch.zeros(T * k, dtype=torch.bool, device=DEV)
        named[pos[live].long()] = True
        dxp[~named] = float("nan")
    dx = torch.full((T + 1, H), 777.0, dtype=torch.bfloat16, device=DEV)
    res = None
    want, size = torch.zeros(T, H, dtype=torch.float64, device=DEV), torch.zeros(T, H, dtype=torch.float64, device=DEV)
    if add is not None:
        res = _rand(g, T, H)
        want += res.double()
        size += res.double().abs()
        if add == "itself":
            dx[:T] = res
            res = dx[:T]
    want.index_add_(0, live // k, dxp[pos[live].long()].double())
    size.index_add_(0, live // k, dxp[pos[live].long()].double().abs())
    hk.tk_kernel.dispatch_moe_permute_backward(dxp, pos, dx[:T], add=res)
    # k additions in fp32 of what is at most `size`, then half a step of bf16
    bound = want.abs() * 2**-8 + size * (k + 1) * 2**-23
    assert ((dx[:T].double() - want).abs() <= bound).all()
    assert torch.all(dx[T] == dx.new_tensor(777.0))


@pytest.mark.parametrize("T,k,H", SHAPES)
@pytest.mark.parametrize("drop", [False, True])
def test_unpermute_backward(hk, T, k, H, drop):
    print(f"unpermute backward T={T} k={k} H={H} drop={drop}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(T * 139 + H)
    dy, o = _rand(g, T, H), _rand(g, T * k, H)
    pos, live = _positions(g, T, k, drop)
    w = torch.rand(T, k, device=DEV, generator=g)
    w[0, 0] = 0.0
    at, token = pos[live].long(), live // k
    if drop:
        named = torch.zeros(T * k, dtype=torch.bool, device=DEV)
        named[at] = True
        o[~named] = float("nan")
    do = torch.full((T * k + 1, H), 777.0, dtype=torch.bfloat16, device=DEV)
    want = do.double()
    want[at] = w.reshape(-1)[live, None].double() * dy[token].double()
    dw = torch.full((T + 1, k), 777.0, device=DEV)
    hk.tk_kernel.dispatch_moe_unpermute_backward(dy, o, w, pos, do[:-1], dw[:T])
    # a product in fp32, half a step of bf16
    assert ((do.double() - want).abs() <= want.abs() * (2**-8 + 2**-22)).all()
    terms = o[at].double() * dy[token].double()
    dwant = torch.zeros(T * k, dtype=torch.float64, device=DEV)
    dsize = torch.zeros_like(dwant)
    dwant[live], dsize[live] = terms.sum(dim=1), terms.abs().sum(dim=1)
    # H products, each added once with at most half a step of fp32 of the sum so far
    assert ((dw[:T].reshape(-1).double() - dwant).abs() <= dsize * (H + 8) * 2**-24).all()
    assert torch.all(dw[T] == 777.0)
    dead = torch.ones(T * k, dtype=torch.bool, device=DEV)
    dead[live] = False
    assert torch.all(dw[:T].reshape(-1)[dead] == 0)


def test_offsets_beyond_32_bits(hk):
    """Permuted rows whose byte offsets pass 2^32: the last token's rows at both ends of a 4.3 GB buffer."""
    T, k, H = 150001, 1, 14336
    print(f"permute T={T} k={k} H={H}", flush=True)
    x = torch.empty(T, H, dtype=torch.bfloat16, device=DEV)
    x.normal_()
    pos = torch.arange(T - 1, -1, -1, dtype=torch.int32, device=DEV)
    xp = torch.zeros(T, H, dtype=torch.bfloat16, device=DEV)
    hk.tk_kernel.dispatch_moe_permute(x, pos, xp)
    for a in range(0, T, 10000):
        b = min(T, a + 10000)
        assert torch.equal(xp[T - b:T - a].flip(0).view(torch.int16), x[a:b].view(torch.int16))
    back = torch.zeros_like(x)
    hk.tk_kernel.dispatch_moe_permute_backward(xp, pos, back)
    assert torch.equal(back[-100:], x[-100:]) and torch.equal(back[:100], x[:100])
    w, dw = torch.full((T, 1), 2.0, device=DEV), torch.zeros(T, 1, device=DEV)
    hk.tk_kernel.dispatch_moe_unpermute_backward(x, xp, w, pos, back, dw)
    assert torch.equal(back[:100].double(), x[-100:].flip(0).double() * 2)
    sq = x[-100:].double().square().sum(dim=1)
    assert ((dw[-100:, 0].double() - sq).abs() <= sq * (H + 8) * 2**-24).all()
