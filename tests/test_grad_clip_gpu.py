"""The global norm of gradients and clipping against the definitions in 64 bits: lists of both types, lengths from nothing to several chunks,
views at any alignment, in place and into other types, values whose squares leave fp32.

Tolerances. The sum of squares is made in 64 bits (2^-50 of it at these lengths), its root rounded to fp32: 2^-24. The factor: the norm's rounding,
the sum with 1e-6 and a division, within 4 x 2^-24 (fp32 division is within 2.5 steps). A product: 2^-24, then half a step of its type."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = {torch.bfloat16: 2**-8, torch.float32: 0.0}
BF, F32 = torch.bfloat16, torch.float32


def _norm(tk, plan):
    norm = torch.full((2,), -1.0, device=DEV)
    ws = torch.full((tk.grad_norm_workspace_bytes() + 64,), 0xA5, dtype=torch.uint8, device=DEV)
    tk.dispatch_grad_norm(plan, norm[:1], ws[:-64])
    assert norm[1] == -1.0 and torch.all(ws[-64:] == 0xA5)
    return norm[:1]


def _make(sizes, types, seed, shift=0, std=1.0):
    """Tensors of these lengths, each a view `shift` elements behind an aligned address with elements of 777 around it."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    bufs = [torch.full((n + 40,), 777.0, dtype=t, device=DEV) for n, t in zip(sizes, types)]
    views = [b[shift:shift + n] for b, n in zip(bufs, sizes)]
    for i, v in enumerate(views):
        v.copy_((torch.randn(v.shape, device=DEV, generator=g) * std * (1 + i % 3)).to(v.dtype))
    return bufs, views


def _check(tk, grads, outs, max_norm):
    before = [t.clone() for t in grads]
    plan = tk.GradTensors(grads, outs)
    norm = _norm(tk, plan)
    want = torch.sqrt(sum((t.double() ** 2).sum() for t in before)).item()
    assert abs(norm.item() - want) <= want * 2**-23
    tk.dispatch_grad_clip(plan, norm, max_norm)
    factor = min(1.0, max_norm / (want + 1e-6))
    for a, b in zip(before, plan.outs):
        exact = a.double() * factor
        tol = exact.abs() * (6 * 2**-24 + HALF[b.dtype]) + 1e-37
        assert ((b.double() - exact).abs() <= tol).all(), (b.shape, b.dtype)
    if outs is not None:
        for a, t in zip(before, grads):
            assert torch.equal(a, t)
    return norm


SIZES = [0, 1, 2, 3, 7, 8, 9, 63, 64, 65, 1000, 16383, 16384, 16385, 0, 40000, 5, 100001, 0]


@pytest.mark.parametrize("shift", [0, 1, 3, 8])
@pytest.mark.parametrize("max_norm", [0.5, 1e9])
def test_in_place(hk, shift, max_norm):
    print(f"clip in place shift={shift} max={max_norm}", flush=True)
    types = [(BF, F32)[(i * 7 // 3) % 2] for i in range(len(SIZES))]
    bufs, grads = _make(SIZES, types, shift, shift)
    before = [g.clone() for g in grads]
    _check(hk.tk_kernel, grads, None, max_norm)
    for b, n in zip(bufs, SIZES):
        assert torch.all(b[:shift] == 777.0) and torch.all(b[shift + n:] == 777.0)
    if max_norm > 1e6:   # a factor of one: the same bits
        assert all(torch.equal(a, b) for a, b in zip(before, grads))


@pytest.mark.parametrize("src_shift,dst_shift", [(0, 0), (0, 1), (2, 2), (3, 0), (8, 4)])
@pytest.mark.parametrize("src,dst", [(BF, BF), (F32, F32), (BF, F32), (F32, BF)])
@pytest.mark.parametrize("max_norm", [0.5, 1e9])
def test_into_others(hk, src, dst, src_shift, dst_shift, max_norm):
    print(f"clip {src} {dst} {src_shift} {dst_shift} {max_norm}", flush=True)
    _, grads = _make(SIZES, [src] * len(SIZES), 1, src_shift)
    bufs, outs = _make(SIZES, [dst] * len(SIZES), 2, dst_shift)
    _check(hk.tk_kernel, grads, outs, max_norm)
    for b, n in zip(bufs, SIZES):
        assert torch.all(b[:dst_shift] == 777.0) and torch.all(b[dst_shift + n:] == 777.0)


@pytest.mark.parametrize("sizes", [[1], [0], [0, 0, 1], [3] * 3000, [50_000_001], [17] * 50 + [9_000_000] + [0] * 9 + [33] * 2100, [16384] * 2049])
def test_lists(hk, sizes):
    print(f"clip of {len(sizes)} tensors, {sum(sizes)} elements", flush=True)
    types = [(BF, F32)[i % 2] for i in range(len(sizes))]
    flat = {t: torch.empty(sum(n for n, u in zip(sizes, types) if u is t), dtype=t, device=DEV).normal_() for t in (BF, F32)}
    at, grads = {BF: 0, F32: 0}, []
    for n, t in zip(sizes, types):
        grads.append(flat[t][at[t]:at[t] + n])
        at[t] += n
    tk = hk.tk_kernel
    want = torch.sqrt(sum((t.double() ** 2).sum() for t in flat.values())).item()
    plan = tk.GradTensors(grads)
    norm = _norm(tk, plan)
    assert abs(norm.item() - want) <= want * 2**-23
    before = {t: f.clone() for t, f in flat.items()}
    tk.dispatch_grad_clip(plan, norm, 0.5)
    factor = min(1.0, 0.5 / (want + 1e-6))
    for t, f in flat.items():
        exact = before[t].double() * factor
        assert ((f.double() - exact).abs() <= exact.abs() * (6 * 2**-24 + HALF[t]) + 1e-37).all()


def test_shapes_and_parameters(hk):
    tk = hk.tk_kernel
    a = torch.nn.Parameter(torch.ones(3, 4, 5, device=DEV))
    b = torch.full((2, 2, 2, 2, 2), 2.0, dtype=BF, device=DEV)
    c = torch.full((), 3.0, device=DEV)
    plan = tk.GradTensors([a.detach(), b, c])
    norm = _norm(tk, plan)
    assert abs(norm.item() - (60 + 128 + 9) ** 0.5) < 1e-5
    tk.dispatch_grad_clip(plan, norm, 1.0)
    assert abs(c.item() - 3 / 197**0.5) < 1e-6


def test_values_whose_squares_leave_fp32(hk):
    tk = hk.tk_kernel
    for value, n in ((1e30, 1000), (3e38, 1), (1e-30, 1000), (0.0, 10)):
        g = torch.full((n,), value, device=DEV)
        norm = _norm(tk, tk.GradTensors([g]))
        want = (g.double() ** 2).sum().sqrt().item()
        assert abs(norm.item() - want) <= want * 2**-23
    big = torch.full((100,), 3e38, device=DEV)   # a norm beyond fp32
    plan = tk.GradTensors([big])
    norm = _norm(tk, plan)
    assert torch.isinf(norm).all()
    tk.dispatch_grad_clip(plan, norm, 1.0)
    assert torch.all(big == 0)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_not_a_number_and_infinity(hk, dtype):
    tk = hk.tk_kernel
    for at in (0, 77, 20000):
        g = torch.ones(20001, dtype=dtype, device=DEV)
        g[at] = float("nan")
        other = torch.ones(5, device=DEV)
        plan = tk.GradTensors([g, other])
        norm = _norm(tk, plan)
        assert torch.isnan(norm).all()
        tk.dispatch_grad_clip(plan, norm, 1.0)
        assert torch.isnan(g).all() and torch.isnan(other).all()
    g = torch.ones(20001, dtype=dtype, device=DEV)
    g[5] = float("-inf")
    plan = tk.GradTensors([g])
    norm = _norm(tk, plan)
    assert torch.isinf(norm).all()
    tk.dispatch_grad_clip(plan, norm, 1.0)
    assert torch.isnan(g[5]) and torch.all(g[:5] == 0) and torch.all(g[6:] == 0)


def test_max_norm_of_zero_and_infinity(hk):
    tk = hk.tk_kernel
    g = torch.ones(100, device=DEV)
    plan = tk.GradTensors([g])
    norm = _norm(tk, plan)
    tk.dispatch_grad_clip(plan, norm, float("inf"))
    assert torch.all(g == 1)
    tk.dispatch_grad_clip(plan, norm, 0.0)
    assert torch.all(g == 0)


def test_captured_and_the_same_on_every_call(hk):
    print("clip capture", flush=True)
    tk = hk.tk_kernel
    g = torch.Generator(device=DEV).manual_seed(9)
    _, grads = _make([70_000, 3, 0, 250_001, 64], [BF, F32, BF, F32, F32], 4)
    outs = [torch.zeros_like(t, dtype=F32) for t in grads]
    plan = tk.GradTensors(grads, outs)
    norm, ws = torch.zeros(1, device=DEV), torch.empty(tk.grad_norm_workspace_bytes(), dtype=torch.uint8, device=DEV)

    def step(plan, norm, ws):
        tk.dispatch_grad_norm(plan, norm, ws)
        tk.dispatch_grad_clip(plan, norm, 0.3)
    step(plan, norm, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(plan, norm, ws)
    for i in range(4):
        for t in grads:
            t.copy_(torch.randn(t.shape, device=DEV, generator=g).to(t.dtype) * 10.0 ** (i - 2))
        outs2 = [torch.zeros_like(t) for t in outs]
        plan2, norm2, ws2 = tk.GradTensors(grads, outs2), torch.zeros(1, device=DEV), torch.full_like(ws, i)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(plan2, norm2, ws2)
        torch.cuda.current_stream().wait_stream(side)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, norm2) and all(torch.equal(a, b) for a, b in zip(outs, outs2)), i


# (elements of gradient and result, types): lists whose chunks are more than 8192, which the kernels read and write past the caches
LONG = {"one tensor beyond 2^32 bytes": [(2**31 + 12_345, BF, BF), (100_003, F32, F32), (1, BF, BF), (0, F32, F32), (16_385, BF, BF)],
        "fp32 beyond 2^32 bytes": [(77, BF, BF), (2**30 + 4_097, F32, F32), (16_384, BF, BF), (3, F32, F32)],
        "many": [(n, (BF, F32)[i % 3 % 2], (BF, F32)[i % 3 % 2]) for i, n in enumerate([999_999, 1, 2_000_001, 16_384, 0] * 46)],
        "into others": [(90_000_001, BF, F32), (50_000_007, F32, BF), (20_000_003, BF, BF), (33, F32, F32), (8_000_000, F32, F32)]}


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("name,elsewhere", [(n, e) for n in LONG for e in (False, True) if e or n != "into others"])
def test_lists_beyond_the_caches(hk, name, elsewhere, shift):
    """Every gradient `shift` elements behind an aligned address and every result there or one element further, with elements of 777 around
    them; compared some million elements at a time."""
    print(f"clip of a long list: {name}, elsewhere={elsewhere}, shift={shift}", flush=True)
    tk, parts = hk.tk_kernel, LONG[name]
    assert sum((n + 16383) // 16384 for n, _, _ in parts) > 8192
    g = torch.Generator(device=DEV).manual_seed(shift + len(parts))
    room = lambda n, t: torch.full((n + 24,), 777.0, dtype=t, device=DEV)
    bufs = [room(n, t) for n, t, _ in parts]
    grads = [b[8 + shift:8 + shift + n] for b, (n, _, _) in zip(bufs, parts)]
    for i, t in enumerate(grads):
        t.normal_(0.0, 1.0 + i % 3, generator=g)
    before = [t.clone() for t in grads]
    out_bufs = [room(n, t) for n, _, t in parts] if elsewhere else bufs
    skip = [8 + shift + (i % 2 if elsewhere else 0) for i in range(len(parts))]
    outs = [b[s:s + n] for b, s, (n, _, _) in zip(out_bufs, skip, parts)]
    plan = tk.GradTensors(grads, outs if elsewhere else None)
    norm = _norm(tk, plan)
    pieces = lambda t: t.split(1 << 26) if t.numel() else ()
    want = sum((p.double() ** 2).sum().item() for t in before for p in pieces(t)) ** 0.5
    assert abs(norm.item() - want) <= want * 2**-23
    assert want > 2000.0
    tk.dispatch_grad_clip(plan, norm, 1000.0)
    factor = 1000.0 / (want + 1e-6)
    for i, (a, b) in enumerate(zip(before, outs)):
        for p, q in zip(pieces(a), pieces(b)):
            exact = p.double() * factor
            assert ((q.double() - exact).abs() <= exact.abs() * (6 * 2**-24 + HALF[b.dtype]) + 1e-37).all(), i
        assert torch.all(out_bufs[i][:skip[i]] == 777.0) and torch.all(out_bufs[i][skip[i] + b.numel():] == 777.0), i
    if elsewhere:
        assert all(torch.equal(a.view(torch.int16 if a.dtype is BF else torch.int32), b.view(torch.int16 if a.dtype is BF else torch.int32))
                   for a, b in zip(before, grads))
