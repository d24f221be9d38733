"""The gated feed-forward block's kernels against the definitions in 64 bits: dense and over experts' rows, one row and more, widths
that end inside a tile and a 16-byte chunk, saturated and clamped values, NaNs in what must not be read, rows that are left alone.

Tolerances. A projection is K products summed in fp32: at most 2 (K + 8) 2^-24 times the sum of their sizes off (a step of fp32 of the sum so
far each, doubled for the order and rounding inside a matrix instruction, which are not specified). The logistic function of z comes from
an exponential whose argument carries up to two roundings, |z| 2^-23, and three functions and operations of at most 2^-22 in all: relative
error (|z| + 4) 2^-22; where it lies below 2^-126, the smallest normal number of fp32 (1 / (1 + e) with e from 2^126 on), the reciprocal
is flushed to zero, which is off by less than 2^-126 itself: FLUSH times whatever the function is multiplied by. The slope of t s(a t) is below 1.1. Results are rounded to bf16 once: half a step, 2^-8 of the value."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ALPHA, LIMIT = 1.702, 7.0
HALF = 2**-8
TINY = 1e-36   # results below this may be denormal or flushed
FLUSH = 2**-126


def _rand(g, *shape, std=1.0):
    return (torch.randn(*shape, device=DEV, generator=g) * std).to(torch.bfloat16)


def _sum_error(a, b, terms):
    """Bound of a product's fp32 sums: a [m,k], b [k,n] in 64 bits."""
    return (a.abs() @ b.abs()) * 2 * (terms + 8) * 2**-24


def _split(gu, interleaved):
    I = gu.shape[-1] // 2
    return (gu[..., 0::2], gu[..., 1::2]) if interleaved else (gu[..., :I], gu[..., I:])


def _join(g, u, interleaved):
    return torch.stack((g, u), dim=-1).flatten(-2) if interleaved else torch.cat((g, u), dim=-1)


def _gate(act, g, u):
    """t, v, s, z, alpha of the formulas in 64 bits"""
    a, lim, b = (1.0, math.inf, 0.0) if act == "silu" else (ALPHA, LIMIT, 1.0)
    t, v = g.clamp(max=lim), u.clamp(-lim, lim) + b
    return t, v, torch.sigmoid(a * t), a * t, a


def _check(got, want, bound, what):
    d = (got.double() - want).abs()
    bad = d > bound + TINY
    assert not bad.any(), (what, int(bad.sum()), torch.nonzero(bad)[:4].tolist(), float((d / (bound + TINY)).max()))
    assert torch.isfinite(got).all(), what


def _check_forward(h, gate_up, x, w, act, interleaved):
    """One group's rows: x [r,K], w [2I,K]."""
    x, wt, K = x.double(), w.double().t().contiguous(), x.shape[1]
    gu, err = x @ wt, _sum_error(x, wt, K)
    if gate_up is not None:
        _check(gate_up, gu, err + gu.abs() * HALF, "gate_up")
    g, u = _split(gu, interleaved)
    eg, eu = _split(err, interleaved)
    t, v, s, z, _ = _gate(act, g, u)
    want = v * t * s
    bound = 1.1 * v.abs() * eg + (t * s).abs() * eu + eg * (eu + eg * v.abs()) + want.abs() * ((z.abs() + 4) * 2**-22 + 4 * 2**-24)
    bound = bound + FLUSH * (v * t).abs()
    _check(h, want, bound * (1 + HALF) + want.abs() * HALF, "h")


def _check_backward(dgate_up, h, dy, w2, gate_up, act, interleaved):
    dy, w2, N = dy.double(), w2.double(), dy.shape[1]
    dh, err = dy @ w2, _sum_error(dy, w2, N)
    g, u = _split(gate_up.double(), interleaved)
    t, v, s, z, a = _gate(act, g, u)
    es = (z.abs() + 4) * 2**-22
    if h is not None:
        want = v * t * s
        _check(h, want, (want.abs() * (es + 4 * 2**-24) + FLUSH * (v * t).abs()) * (1 + HALF) + want.abs() * HALF, "h")
    k = s * (1 + z * (1 - s))
    dg, du = dh * v * k, dh * t * s
    ek = s * (1 + z.abs()) * (es + 2**-22) + FLUSH * (1 + z.abs())
    eg = err * (v * k).abs() + (dh.abs() + err) * v.abs() * ek + dg.abs() * 4 * 2**-24
    eu = err * (t * s).abs() + (dh.abs() + err) * t.abs() * (s * (es + 2**-22) + FLUSH)
    if act != "silu":
        held_g, held_u = g > LIMIT, u.abs() > LIMIT
        dg, eg = dg.masked_fill(held_g, 0), eg.masked_fill(held_g, 0)
        du, eu = du.masked_fill(held_u, 0), eu.masked_fill(held_u, 0)
    got_g, got_u = _split(dgate_up, interleaved)
    _check(got_g, dg, eg * (1 + HALF) + dg.abs() * HALF, "dgate")
    _check(got_u, du, eu * (1 + HALF) + du.abs() * HALF, "dup")


def _run(hk, rows, unused, I, wide, act, interleaved, seed, dense, scale=1.5, keep=True):
    """Forward and backward of one case; `rows` of each expert, or of a dense block."""
    tk = hk.tk_kernel
    g = torch.Generator(device=DEV).manual_seed(seed)
    off = [0]
    for r in rows:
        off.append(off[-1] + r)
    R, E = off[-1] + unused, len(rows)
    print(f"gated rows={rows[:8]} unused={unused} I={I} wide={wide} {act} interleaved={interleaved} dense={dense}", flush=True)
    x, w13 = _rand(g, R, wide), _rand(g, E, 2 * I, wide, std=scale * wide**-0.5)
    dy, w2 = _rand(g, R, wide), _rand(g, E, wide, I, std=I**-0.5)
    x[off[-1]:] = float("nan")
    dy[off[-1]:] = float("nan")
    offsets = None if dense else torch.tensor(off, dtype=torch.int32, device=DEV)
    strip = (lambda w: w[0]) if dense else (lambda w: w)
    mk = lambda n: torch.full((R + 1, n), 777.0, dtype=torch.bfloat16, device=DEV)
    h, gu, dgu, h2 = mk(I), mk(2 * I), mk(2 * I), mk(I)
    opts = dict(expert_offsets=offsets, interleaved=interleaved, activation=act, alpha=ALPHA, limit=LIMIT)
    tk.dispatch_gated_gemm(x, strip(w13), h[:R], gu[:R] if keep else None, **opts)
    for e in range(E):
        a, b = off[e], off[e + 1]
        if b > a:
            _check_forward(h[a:b], gu[a:b] if keep else None, x[a:b], w13[e], act, interleaved)
    if not keep:
        gu[:off[-1]] = _rand(g, off[-1], 2 * I, std=4.0)
    kept = gu.clone()
    tk.dispatch_gated_gemm_dgrad(dy, strip(w2), gu[:R], dgu[:R], h2[:R] if keep else None, **opts)
    for e in range(E):
        a, b = off[e], off[e + 1]
        if b > a:
            _check_backward(dgu[a:b], h2[a:b] if keep else None, dy[a:b], w2[e], gu[a:b], act, interleaved)
    assert torch.equal(gu.view(torch.int16), kept.view(torch.int16))
    for t in (h, gu, dgu) + ((h2,) if keep else ()):
        assert torch.all(t[off[-1]:] == 777.0)
    # in place of gate_up: the same bits
    tk.dispatch_gated_gemm_dgrad(dy, strip(w2), gu[:R], gu[:R], None, **opts)
    assert torch.equal(gu.view(torch.int16), dgu.view(torch.int16))


WIDTHS = [(8, 8), (16, 72), (64, 64), (136, 520), (256, 256), (392, 1000), (1032, 264)]


@pytest.mark.parametrize("I,wide", WIDTHS)
@pytest.mark.parametrize("R", [1, 2, 15, 16, 17, 33, 63, 64, 65, 130, 257])
def test_dense(hk, R, I, wide):
    n = R + I + wide
    _run(hk, [R], 0, I, wide, ("silu", "swiglu_oai")[n % 2], n % 3 == 0, n, True, keep=n % 5 != 0)


EXPERTS = [([1], 0), ([0, 3, 0], 2), ([127, 128, 129], 0), ([1, 255, 0, 256, 257, 2], 5), ([0, 0, 0], 4),
           ([5] * 40 + [0] * 5 + [130, 64, 63, 65], 0)]


@pytest.mark.parametrize("I,wide", WIDTHS)
@pytest.mark.parametrize("case", range(len(EXPERTS)))
def test_experts(hk, case, I, wide):
    n = case + I // 8 + wide // 8
    _run(hk, *EXPERTS[case], I, wide, ("swiglu_oai", "silu")[n % 2], n % 3 != 0, 7 * n, False)


# sizes at which each of the tile kernels is taken, in both directions: more tiles than CUs of every size, and few large ones
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,unused,I,wide,dense", [
    ([4100], 0, 2312, 1032, True), ([1111], 0, 2816, 1024, True), ([515], 0, 1288, 520, True), ([9000], 9, 904, 72, False),
    ([2049, 0, 255, 257, 1, 3000, 63, 65, 129], 3, 2312, 520, False), ([100, 0, 64, 65, 127, 128, 129, 191, 257, 1] * 4, 0, 776, 840, False)])
def test_large(hk, rows, unused, I, wide, dense, interleaved):
    _run(hk, rows, unused, I, wide, "swiglu_oai" if interleaved else "silu", interleaved, I + wide, dense)


@pytest.mark.parametrize("act", ["silu", "swiglu_oai"])
@pytest.mark.parametrize("R", [5, 300])
def test_saturated_values(hk, R, act):
    """Gates and ups far outside the clamp, and where the exponential leaves fp32."""
    _run(hk, [R], 0, 264, 72, act, False, 11, True, scale=100.0)


def test_values_at_the_clamp(hk):
    """Exactly the limit: the value is the limit's and the gradient passes; the next number behind it: no gradient. (One term per
    projection, so that both are exact.)"""
    print("gated at the clamp", flush=True)
    tk, I, K = hk.tk_kernel, 16, 8
    over = 7.03125   # the next bf16 above 7
    gates = torch.tensor([7.0, over, -7.0, 1.0, 0.0, -over, 100.0, -100.0], device=DEV)
    ups = torch.tensor([7.0, over, -7.0, -over, 0.0, 1.0, -100.0, 100.0], device=DEV)
    w13 = torch.zeros(2 * I, K, dtype=torch.bfloat16, device=DEV)
    w13[:8, 0], w13[I:I + 8, 0] = gates, ups
    x = torch.zeros(1, K, dtype=torch.bfloat16, device=DEV)
    x[0, 0] = 1
    h, gu = torch.zeros(1, I, dtype=torch.bfloat16, device=DEV), torch.zeros(1, 2 * I, dtype=torch.bfloat16, device=DEV)
    tk.dispatch_gated_gemm(x, w13, h, gu, activation="swiglu_oai", alpha=ALPHA, limit=LIMIT)
    assert torch.equal(gu[0].float(), w13[:, 0].float())
    _check_forward(h, gu, x, w13, "swiglu_oai", False)
    dy, w2 = torch.ones(1, 8, dtype=torch.bfloat16, device=DEV), torch.ones(8, I, dtype=torch.bfloat16, device=DEV)
    dgu = torch.zeros_like(gu)
    tk.dispatch_gated_gemm_dgrad(dy, w2, gu, dgu, activation="swiglu_oai", alpha=ALPHA, limit=LIMIT)
    _check_backward(dgu, None, dy, w2, gu, "swiglu_oai", False)
    dg, du = dgu[0, :8].float(), dgu[0, I:I + 8].float()
    assert dg[0] != 0 and dg[1] == 0 and dg[6] == 0 and du[0] != 0 and du[1] == 0 and du[2] != 0 and du[3] == 0 and du[7] == 0


def test_gradients_against_differences(hk):
    """dgate_up from the kernel against central differences of the activation in 64 bits at the kept values."""
    print("gated differences", flush=True)
    tk, R, I, N = hk.tk_kernel, 33, 72, 16
    g = torch.Generator(device=DEV).manual_seed(2)
    gu, dy, w2 = _rand(g, R, 2 * I, std=3.0), _rand(g, R, N), _rand(g, N, I)
    for act in ("silu", "swiglu_oai"):
        dgu = torch.empty_like(gu)
        tk.dispatch_gated_gemm_dgrad(dy, w2, gu, dgu, activation=act, alpha=ALPHA, limit=LIMIT)
        dh = dy.double() @ w2.double()

        def f(v):
            t, lin, s, _, _ = _gate(act, v[:, :I], v[:, I:])
            return lin * t * s
        step = 1e-5
        for half in (0, 1):
            d = torch.zeros(R, 2 * I, dtype=torch.float64, device=DEV)
            d[:, half * I:(half + 1) * I] = step
            want = dh * (f(gu.double() + d) - f(gu.double() - d)) / (2 * step)
            got = dgu[:, half * I:(half + 1) * I].double()
            near = (gu[:, half * I:(half + 1) * I].double().abs() - LIMIT).abs() < 2 * step   # (a difference across the clamp's corner)
            # second-order error of the differences below 1e-8; sums and functions in fp32 below 1e-4 of sum |dy| |w2| (1 + |v|)
            size = (dy.double().abs() @ w2.double().abs()) * (2 + gu.double().abs().max())
            assert (((got - want).abs() <= HALF * want.abs() + 1e-4 * size) | near).all()


def test_nans_and_infinities(hk):
    """They reach the rows and columns that they belong to and no others."""
    print("gated NaN and inf", flush=True)
    tk, R, I, K = hk.tk_kernel, 140, 72, 136
    g = torch.Generator(device=DEV).manual_seed(4)
    for act in ("silu", "swiglu_oai"):
        x, w13 = _rand(g, R, K), _rand(g, 2 * I, K)
        x[7] = float("nan")
        w13[3] = float("nan")        # gate of column 3
        w13[I + 5] = float("nan")    # up of column 5
        h, gu = _rand(g, R, I), _rand(g, R, 2 * I)
        tk.dispatch_gated_gemm(x, w13, h, gu, activation=act)
        bad = torch.zeros(R, I, dtype=torch.bool, device=DEV)
        bad[7] = bad[:, 3] = bad[:, 5] = True
        assert torch.equal(torch.isnan(h), bad)
        dy, w2 = _rand(g, R, K), _rand(g, K, I)
        gu = _rand(g, R, 2 * I)
        gu[9, 4], gu[9, I + 6] = float("nan"), float("nan")
        dy[11] = float("inf")
        dgu, h = torch.zeros_like(gu), torch.zeros_like(h)
        tk.dispatch_gated_gemm_dgrad(dy, w2, gu, dgu, h, activation=act)
        fine = torch.ones(R, 2 * I, dtype=torch.bool, device=DEV)
        fine[11] = False
        fine[9, 4] = fine[9, I + 4] = fine[9, 6] = fine[9, I + 6] = False
        assert torch.isfinite(dgu[fine]).all() and torch.isnan(dgu[9, 4]) and torch.isnan(dgu[9, I + 4]) and torch.isnan(dgu[9, 6])
        assert not torch.isfinite(dgu[11]).any()
        assert torch.isnan(h[9, 4]) and torch.isnan(h[9, 6]) and int(torch.isnan(h).sum()) == 2


def test_an_expert_alone_and_among_others(hk):
    """The same bits, whatever the others hold; offsets out of order give no row to two experts."""
    print("gated expert isolation", flush=True)
    tk, I, K = hk.tk_kernel, 136, 200
    rows = [70, 0, 130, 33]
    g = torch.Generator(device=DEV).manual_seed(6)
    off = [0, 70, 70, 200, 233]
    offsets = torch.tensor(off, dtype=torch.int32, device=DEV)
    x, w13, w2, dy = _rand(g, 233, K), _rand(g, 4, 2 * I, K), _rand(g, 4, K, I), _rand(g, 233, K)
    mk = lambda n: torch.zeros(233, n, dtype=torch.bfloat16, device=DEV)
    h, gu, dgu = mk(I), mk(2 * I), mk(2 * I)
    tk.dispatch_gated_gemm(x, w13, h, gu, expert_offsets=offsets)
    tk.dispatch_gated_gemm_dgrad(dy, w2, gu, dgu, expert_offsets=offsets)
    x2, w2b, w13b, dy2 = x.clone(), w2.clone(), w13.clone(), dy.clone()
    for t, at in ((x2, slice(0, 70)), (dy2, slice(0, 70)), (x2, slice(200, 233)), (dy2, slice(200, 233))):
        t[at] = float("nan")
    for t in (w13b, w2b):
        t[0], t[1], t[3] = float("nan"), float("nan"), float("inf")
    h2, gu2, dgu2 = mk(I), mk(2 * I), mk(2 * I)
    tk.dispatch_gated_gemm(x2, w13b, h2, gu2, expert_offsets=offsets)
    tk.dispatch_gated_gemm_dgrad(dy2, w2b, gu2, dgu2, expert_offsets=offsets)
    for a, b in ((h, h2), (gu, gu2), (dgu, dgu2)):
        assert torch.equal(a[70:200].view(torch.int16), b[70:200].view(torch.int16))
    broken = torch.tensor([0, 100, 40, 10_000_000, -5], dtype=torch.int32, device=DEV)
    h3 = mk(I)
    tk.dispatch_gated_gemm(x, w13, h3, None, expert_offsets=broken)
    _check_forward(h3[:100], None, x[:100], w13[0], "silu", False)
    _check_forward(h3[100:], None, x[100:], w13[2], "silu", False)


@pytest.mark.parametrize("M,N,K", [(1, 8, 8), (64, 72, 136), (257, 264, 520), (1111, 1024, 2816), (5000, 2056, 1032)])
def test_dense_product_gradients(hk, M, N, K):
    print(f"dense gradients {M} {N} {K}", flush=True)
    tk = hk.tk_kernel
    g = torch.Generator(device=DEV).manual_seed(M)
    dy, x, w = _rand(g, M, N), _rand(g, M, K), _rand(g, N, K)
    dx = torch.full((M + 1, K), 777.0, dtype=torch.bfloat16, device=DEV)
    tk.dispatch_bf16_gemm_dgrad(dy, w, dx[:M])
    d, xd, wd = dy.double(), x.double(), w.double()
    want = d @ wd
    _check(dx[:M], want, _sum_error(d, wd, N) + want.abs() * HALF, "dx")
    dt = d.t().contiguous()
    want, err = dt @ xd, _sum_error(dt, xd, M)
    for dtype, half in ((torch.bfloat16, HALF), (torch.float32, 2**-24)):
        dw = torch.full((N + 1, K), 777.0, dtype=dtype, device=DEV)
        tk.dispatch_bf16_gemm_wgrad(dy, x, dw[:N])
        _check(dw[:N], want, err + want.abs() * half, "dw")
        assert torch.all(dw[N] == 777.0)
    assert torch.all(dx[M] == 777.0)


def test_captured_and_on_another_stream(hk):
    """Captured on a side stream and replayed with other inputs, next to eager work: the eager results each time."""
    print("gated capture", flush=True)
    tk, R, I, K = hk.tk_kernel, 200, 264, 136
    g = torch.Generator(device=DEV).manual_seed(8)
    x, w13, dy, w2 = _rand(g, R, K), _rand(g, 2 * I, K), _rand(g, R, K), _rand(g, K, I)
    mk = lambda n: torch.zeros(R, n, dtype=torch.bfloat16, device=DEV)
    out = [mk(I), mk(2 * I), mk(2 * I), mk(I)]

    def step(o):
        tk.dispatch_gated_gemm(x, w13, o[0], o[1])
        tk.dispatch_gated_gemm_dgrad(dy, w2, o[1], o[2], o[3])
    step(out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(out)
    for i in range(4):
        x.copy_(_rand(g, R, K))
        dy.copy_(_rand(g, R, K))
        want = [mk(I), mk(2 * I), mk(2 * I), mk(I)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(want)
        torch.cuda.current_stream().wait_stream(side)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16)), i


@pytest.mark.parametrize("act,interleaved", [("silu", False), ("silu", True), ("swiglu_oai", False), ("swiglu_oai", True)])
def test_about_half_a_large_tile_of_rows_per_expert(hk, act, interleaved):
    """The forward kernel of 128 rows and 256 columns: rows on both sides of its tile, columns that end in its halves, K-steps on both sides of its
    three stages."""
    rows = [100, 0, 64, 65, 127, 128, 129, 191, 1, 257] * 3 + [90, 110]
    for I, K in ((1032, 1800), (1160, 1672), (2056, 840)):
        _run(hk, rows, 5, I, K, act, interleaved, I + K, False)


@pytest.mark.parametrize("act,interleaved", [("silu", True), ("swiglu_oai", False)])
@pytest.mark.parametrize("R", [1, 16, 17, 32, 33, 48, 49, 64])
def test_few_rows_of_wide_blocks(hk, R, act, interleaved):
    """Decode: every number of row fragments, with 16, 32 and 64 rows of weights a workgroup, K that ends inside a K-step, kept values or not."""
    for I, K, keep in ((8, 2056, True), (1032, 136, True), (4104, 1096, False), (9000, 2120, R % 2 == 0)):
        _run(hk, [R], 0, I, K, act, interleaved, R + I, True, keep=keep)


@pytest.mark.parametrize("act,interleaved", [("silu", True), ("swiglu_oai", False), ("silu", False), ("swiglu_oai", True)])
@pytest.mark.parametrize("rows,unused,I,K", [
    ([0, 1, 3, 0, 1], 0, 136, 2120), ([0, 0, 0, 17, 0, 0, 33], 6, 264, 584), ([5, 2, 0, 1, 0, 0, 20] * 6, 3, 520, 1096), ([1, 0, 7] * 21, 0, 392, 1032),
    ([16, 17, 7, 12], 1, 264, 1096), ([12, 31, 0, 33, 8, 15, 20] * 9, 40, 520, 1032), ([9, 20, 40, 3] * 14, 0, 1032, 1160), ([1] * 200, 0, 72, 1992)])
def test_few_rows_of_experts(hk, rows, unused, I, K, act, interleaved):
    """Decode with experts: one and two row fragments and every number of columns a workgroup in both directions, experts with more rows than a
    workgroup takes, without any, and with rows behind the last."""
    _run(hk, rows, unused, I, K, act, interleaved, I + K + len(rows), False, keep=len(rows) % 2 == 0)


@pytest.mark.parametrize("act,interleaved", [("silu", True), ("swiglu_oai", False), ("silu", False), ("swiglu_oai", True)])
@pytest.mark.parametrize("rows,unused,I,wide,dense", [
    ([200], 0, 2632, 128, True), ([500], 0, 2312, 64, True), ([449], 0, 2504, 576, True), ([100, 0, 30, 65] * 5, 4, 328, 320, False),
    ([100, 0, 30, 65] * 5, 0, 712, 256, False)])
def test_two_small_tiles_a_cu(hk, rows, unused, I, wide, dense, act, interleaved):
    """64x64 tiles, more of them than CUs and no more than two a CU, forward or backward; fewer K-steps than stages, as many, and more."""
    _run(hk, rows, unused, I, wide, act, interleaved, I + wide, dense)


@pytest.mark.parametrize("act,interleaved", [("silu", True), ("swiglu_oai", False), ("silu", False), ("swiglu_oai", True)])
@pytest.mark.parametrize("rows,unused,I,wide,dense", [
    ([2100], 0, 2056, 840, True), ([1150], 0, 2056, 1800, True), ([1150], 0, 4616, 520, True), ([700, 0, 1200, 513] * 2, 7, 2056, 520, False)])
def test_large_tiles(hk, rows, unused, I, wide, dense, act, interleaved):
    """Each of the kernels of 128 and 256 rows dense and over experts, with every activation and order of the weights' rows."""
    _run(hk, rows, unused, I, wide, act, interleaved, I + wide + 1, dense)


@pytest.mark.parametrize("act,interleaved", [("silu", True), ("swiglu_oai", False)])
@pytest.mark.parametrize("rows,I,wide,dense", [
    ([1], 4160, 1088, True), ([8], 2048, 2112, True), ([17], 4160, 1088, True), ([40], 8256, 2176, True), ([64], 2112, 2112, True),
    ([0, 1, 3, 0, 1], 192, 2112, False), ([0, 0, 0, 17, 0, 0, 33], 256, 640, False), ([5, 2, 0, 1, 0, 0, 20] * 6, 576, 1088, False),
    ([1, 0, 7] * 21, 384, 1024, False), ([12, 31, 0, 33, 8, 15, 20] * 9, 576, 1024, False), ([1, 0, 2] * 8, 576, 2112, False),
    ([16, 17, 7, 12], 256, 1088, False)])
def test_few_rows_with_weights_past_the_caches(hk, rows, I, wide, dense, act, interleaved):
    """Rows of weights that are whole cache lines, as most checkpoints', of every kernel for few rows in both directions."""
    _run(hk, rows, 0, I, wide, act, interleaved, I + wide + len(rows), dense)


def test_few_rows_with_weights_inside_a_cache_line(hk):
    """The same weights at an address that is no multiple of a cache line's: the same values."""
    print("gated weights inside a line", flush=True)
    tk, R, I, K = hk.tk_kernel, 3, 2112, 2112
    g = torch.Generator(device=DEV).manual_seed(31)
    x, dy, gu = _rand(g, R, K), _rand(g, R, K), _rand(g, R, 2 * I)
    pools = [torch.empty(2 * I * K + 64, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    w = _rand(g, 2 * I * K, std=K**-0.5)
    got = []
    for pool, skip in zip(pools, (0, 8)):
        at = pool[skip:skip + 2 * I * K]
        at.copy_(w)
        h, d = torch.empty(R, I, dtype=torch.bfloat16, device=DEV), torch.empty(R, 2 * I, dtype=torch.bfloat16, device=DEV)
        tk.dispatch_gated_gemm(x, at.view(2 * I, K), h)
        tk.dispatch_gated_gemm_dgrad(dy, at[:I * K].view(K, I), gu, d)
        got.append((h, d))
    for a, b in zip(*got):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,other,kept,I,wide", [
    ([1, 1, 1, 5, 1, 1], [3, 0, 0, 5, 1, 1], 3, 392, 2056), ([1, 1, 1, 5, 1, 1], [0, 0, 4, 5, 0, 1], 3, 1096, 2056),
    ([12, 14, 10, 12], [20, 0, 10, 18], 2, 776, 2056),
    ([1, 2, 0, 3] * 10, [3, 0] * 12 + [0, 0, 0, 3, 6, 0, 3, 0] + [3, 0] * 4, 27, 1096, 1032),
    ([12, 9] * 16, [21, 0] * 3 + [12, 9] + [21, 0] * 12, 7, 1160, 1096), ([12, 9] * 16, [21, 0] * 3 + [12, 9] + [21, 0] * 12, 7, 1152, 1088)])
def test_an_expert_of_few_rows_among_others(hk, rows, other, kept, I, wide, interleaved):
    """As many rows in all, spread over the other experts in another way, and `kept`'s elsewhere: the bits of its rows stay. (Each of the forward
    kernels for few rows of experts and the backward ones, one row fragment and two, weights through the caches and past them.)"""
    print(f"gated expert of few rows {rows[:6]} {other[:6]} I={I} wide={wide} interleaved={interleaved}", flush=True)
    tk, E = hk.tk_kernel, len(rows)
    g = torch.Generator(device=DEV).manual_seed(I + E)
    assert sum(rows) == sum(other)
    n = min(rows[kept], other[kept])
    w13, w2 = _rand(g, E, 2 * I, wide, std=1.5 * wide**-0.5), _rand(g, E, wide, I, std=I**-0.5)
    mine, mine_dy, mine_gu = _rand(g, n, wide), _rand(g, n, wide), _rand(g, n, 2 * I)
    got = []
    for each in (rows, other):
        R, at = sum(each), sum(each[:kept])
        x, dy, kept_gu = _rand(g, R, wide), _rand(g, R, wide), _rand(g, R, 2 * I)
        x[at:at + n], dy[at:at + n], kept_gu[at:at + n] = mine, mine_dy, mine_gu
        offsets = torch.tensor([sum(each[:e]) for e in range(E + 1)], dtype=torch.int32, device=DEV)
        mk = lambda c: torch.zeros(R, c, dtype=torch.bfloat16, device=DEV)
        h, gu, dgu, h2 = mk(I), mk(2 * I), mk(2 * I), mk(I)
        tk.dispatch_gated_gemm(x, w13, h, gu, expert_offsets=offsets, interleaved=interleaved)
        tk.dispatch_gated_gemm_dgrad(dy, w2, kept_gu, dgu, h2, expert_offsets=offsets, interleaved=interleaved)
        got.append([t[at:at + n].clone() for t in (h, gu, dgu, h2)])
    for name, a, b in zip(("h", "gate_up", "dgate_up", "h again"), *got):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16)), (name, int((a != b).sum()))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("experts,R,I,N", [(0, 3, 136, 264), (0, 40, 136, 264), (0, 300, 264, 136), (0, 2100, 2056, 200), (3, 9, 136, 1032), (3, 700, 264, 136)])
def test_gradients_of_the_lowest_gate_values(hk, experts, R, I, N, interleaved):
    """Gate values whose product with alpha leaves fp32, the type's lowest as a mask among them: the logistic function is 0 there, and so are h and
    both gradients, exactly; without a limit, far above, it is 1, and the slope too."""
    print(f"gated lowest values experts={experts} R={R} I={I} N={N} interleaved={interleaved}", flush=True)
    tk = hk.tk_kernel
    g = torch.Generator(device=DEV).manual_seed(R + I)
    dy, w2 = _rand(g, R, N), _rand(g, max(experts, 1), N, I, std=N**-0.5)
    gu = _rand(g, R, 2 * I)
    gate, up = _split(gu, interleaved)
    low, far = -torch.finfo(torch.bfloat16).max, torch.finfo(torch.bfloat16).max
    gate[0, 1], gate[1, :], gate[R - 1, I - 1], gate[2, 5] = low, low, -2.5e38, far
    up[2, 5] = 0.5
    offsets = torch.tensor([0] + [R * (e + 1) // experts for e in range(experts)], dtype=torch.int32, device=DEV) if experts else None
    mk = lambda n: torch.full((R, n), 777.0, dtype=torch.bfloat16, device=DEV)
    for limit in (LIMIT, math.inf):
        dgu, h = mk(2 * I), mk(I)
        tk.dispatch_gated_gemm_dgrad(dy, w2 if experts else w2[0], gu, dgu, h, expert_offsets=offsets, interleaved=interleaved,
                                     activation="swiglu_oai", alpha=ALPHA, limit=limit)
        dg, du = _split(dgu, interleaved)
        assert torch.isfinite(dgu).all() or limit == math.inf
        for at in ((0, 1), (1, slice(None)), (R - 1, I - 1)):
            assert torch.all(dg[at] == 0) and torch.all(du[at] == 0) and torch.all(h[at] == 0), (limit, at)
        if limit == math.inf:   # dg = dh (u + 1)
            dh = float(dy[2].double() @ w2[0][:, 5].double())
            size = float(dy[2].double().abs() @ w2[0][:, 5].double().abs())
            assert abs(float(dg[2, 5]) - 1.5 * dh) <= abs(1.5 * dh) * (HALF + 2**-20) + 1.5 * size * 2 * (N + 8) * 2**-24
