"""The embedding and its gradient against the definitions in 64 bits: one token and many, ids all alike, all different and outside the table,
NaNs in what must not be read, sums over several blocks and workgroups, another gradient added, in place too.

Tolerances. Forward: a product in fp32 (2^-24 of it) and the rounding to bf16 (2^-8). Gradient: n terms summed in fp32 in some order, each sum
off by at most 2^-24 of the sum of the terms' sizes; the scale and `add` one rounding more; then half a step of the result's type."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = {torch.bfloat16: 2**-8, torch.float32: 2**-24}


def _ids(kind, T, V, g):
    if kind == "one":
        ids = torch.full((T,), V // 2, device=DEV)
    elif kind == "different":
        ids = torch.randperm(max(T, V), device=DEV, generator=g)[:T] % V
    elif kind == "falling":
        ids = (V - 1 - torch.arange(T, device=DEV) * V // max(T, V)).clamp(min=0)
    elif kind == "frequent":   # a few ids have most tokens
        u = torch.rand(T, device=DEV, generator=g)
        ids = ((V + 1.0) ** u).long().sub(1).clamp(0, V - 1)
    elif kind == "outside":
        ids = torch.randint(0, V, (T,), device=DEV, generator=g)
        far = torch.tensor([-1, V, -100, 2**31 - 1, -2**31], device=DEV)
        where = torch.rand(T, device=DEV, generator=g) < 0.4
        ids = torch.where(where, far[torch.randint(0, 5, (T,), device=DEV, generator=g)], ids)
    else:
        assert kind == "none"
        ids = torch.full((T,), -1, device=DEV)
    return ids.long()


def _backward(hk, T, V, H, kind, dtype, id_type, add, scale, seed, ids=None):
    tk = hk.tk_kernel
    g = torch.Generator(device=DEV).manual_seed(seed)
    print(f"embedding backward T={T} V={V} H={H} {kind} {dtype} {id_type} add={add}", flush=True)
    ids = _ids(kind, T, V, g) if ids is None else ids
    dout = torch.randn(T, H, device=DEV, generator=g).bfloat16()
    live = (ids >= 0) & (ids < V)
    dout[~live] = float("nan")
    base = torch.randn(V, H, device=DEV, generator=g).to(dtype)
    buf = torch.full((V + 1, H), 777.0, dtype=dtype, device=DEV)
    dtable = buf[:V]
    if add == "in place":
        dtable.copy_(base)
    ws = torch.full((tk.embedding_backward_workspace_bytes(T, V, H) + 64,), 0xA5, dtype=torch.uint8, device=DEV)
    given = {"no": None, "yes": base, "in place": dtable}[add]
    tk.dispatch_embedding_backward(ids.to(id_type), dout, dtable, ws[:-64], scale=scale, add=given)
    assert torch.all(ws[-64:] == 0xA5) and torch.all(buf[V] == 777.0)
    want = torch.zeros(V, H, dtype=torch.float64, device=DEV)
    size = torch.zeros_like(want)
    want.index_add_(0, ids[live], dout[live].double())
    size.index_add_(0, ids[live], dout[live].double().abs())
    n = torch.bincount(ids[live], minlength=V).double()[:, None]
    want, size = want * scale, size * abs(scale)
    bound = size * (n + 2) * 2**-24
    if add != "no":
        want = want + base.double()
        bound = bound + want.abs() * 2**-24
    bad = (dtable.double() - want).abs() > bound * (1 + HALF[dtype]) + want.abs() * HALF[dtype] + 1e-37
    assert not bad.any(), (int(bad.sum()), torch.nonzero(bad)[:4].tolist())
    assert torch.isfinite(dtable).all()
    untouched = n[:, 0] == 0
    assert torch.equal(dtable[untouched], base[untouched] if add != "no" else torch.zeros_like(base[untouched]))
    return dout, dtable


@pytest.mark.parametrize("T", [1, 2, 7, 8, 9, 64, 65, 1000, 4095, 4096])
@pytest.mark.parametrize("V,H", [(1, 8), (2, 64), (513, 520), (3001, 72)])
def test_gradient(hk, T, V, H):
    n = T + V + H
    kinds = ["one", "different", "falling", "frequent", "outside"]
    for i in range(2):
        _backward(hk, T, V, H, kinds[(n + 2 * i) % 5], (torch.bfloat16, torch.float32)[(n + i) % 2], (torch.int32, torch.int64)[n // 2 % 2],
                  ("no", "yes", "in place")[(n + i) % 3], (1.0, -0.37)[i], n)


@pytest.mark.parametrize("kind", ["one", "different", "falling", "frequent", "outside", "none"])
@pytest.mark.parametrize("T,V,H", [(4097, 100, 64), (9001, 50257, 136), (20000, 70000, 24), (12288, 1 << 19, 8), (9000, 300, 8200), (8500, 700, 16400), (8192, 777, 72), (8193, 777, 72)])
def test_gradient_over_several_workgroups(hk, T, V, H, kind):
    n = T + V + len(kind)
    _backward(hk, T, V, H, kind, (torch.bfloat16, torch.float32)[n % 2], (torch.int64, torch.int32)[n // 2 % 2], ("no", "yes", "in place")[n % 3],
              1.5, n)


@pytest.mark.parametrize("T,V,H", [(150000, 1000, 8), (300000, 1 << 20, 8)])
def test_many_tokens(hk, T, V, H):
    _backward(hk, T, V, H, "frequent", torch.float32, torch.int64, "no", 1.0, 5)


def test_a_rows_tokens_are_added_in_their_order(hk):
    """A row's terms that cancel only in one order: large, then its negative, then small ones. Inside a block the sum is exact."""
    print("embedding order", flush=True)
    tk, V, H = hk.tk_kernel, 5, 8
    ids = torch.tensor([3, 1, 3, 1, 3], device=DEV)
    dout = torch.zeros(5, H, dtype=torch.bfloat16, device=DEV)
    dout[0], dout[2], dout[4] = 2.0**100, -2.0**100, 1.0
    dtable = torch.zeros(V, H, device=DEV)
    ws = torch.empty(tk.embedding_backward_workspace_bytes(5, V, H), dtype=torch.uint8, device=DEV)
    tk.dispatch_embedding_backward(ids, dout, dtable, ws)
    assert torch.all(dtable[3] == 1.0) and torch.all(dtable[[0, 1, 2, 4]] == 0)


def test_the_same_on_every_call_and_in_a_graph(hk):
    print("embedding capture", flush=True)
    tk, T, V, H = hk.tk_kernel, 9001, 3000, 264
    g = torch.Generator(device=DEV).manual_seed(3)
    ids, dout = _ids("frequent", T, V, g), torch.randn(T, H, device=DEV, generator=g).bfloat16()
    table, out = torch.randn(V, H, device=DEV, generator=g).bfloat16(), torch.zeros(T, H, dtype=torch.bfloat16, device=DEV)
    dtable = torch.zeros(V, H, device=DEV)
    ws = torch.empty(tk.embedding_backward_workspace_bytes(T, V, H), dtype=torch.uint8, device=DEV)

    def step(out, dtable, ws):
        tk.dispatch_embedding(ids, table, out, scale=3.0)
        tk.dispatch_embedding_backward(ids, dout, dtable, ws, scale=3.0)
    step(out, dtable, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(out, dtable, ws)
    for i in range(4):
        ids.copy_(_ids("frequent" if i % 2 else "outside", T, V, g))
        out2, dtable2, ws2 = torch.zeros_like(out), torch.zeros_like(dtable), torch.full_like(ws, i)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(out2, dtable2, ws2)
        torch.cuda.current_stream().wait_stream(side)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, out2) and torch.equal(dtable.view(torch.int32), dtable2.view(torch.int32)), i


def test_workspace_of_the_largest_batch_serves_smaller_ones(hk):
    tk, V, H = hk.tk_kernel, 40, 264
    ws = tk.embedding_backward_workspace_bytes(70000, V, H)
    for T in (1, 100, 4096, 4097, 65535, 65536, 69999):
        assert tk.embedding_backward_workspace_bytes(T, V, H) <= ws


@pytest.mark.parametrize("T,V,H", [(1, 1, 8), (3, 10, 64), (17, 1000, 520), (64, 300, 2048), (65, 300, 2056), (1000, 77, 4104)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("id_type", [torch.int32, torch.int64])
def test_lookup(hk, T, V, H, dtype, id_type):
    tk = hk.tk_kernel
    g = torch.Generator(device=DEV).manual_seed(T + H)
    print(f"embedding T={T} V={V} H={H} {dtype} {id_type}", flush=True)
    table = torch.randn(V, H, device=DEV, generator=g).to(dtype)
    for kind, scale in (("different", 1.0), ("outside", H**0.5)):
        ids = _ids(kind, T, V, g)
        live = ((ids >= 0) & (ids < V))[:, None]
        out = torch.full((T + 1, H), 777.0, dtype=torch.bfloat16, device=DEV)
        tk.dispatch_embedding(ids.to(id_type), table, out[:T], scale=scale)
        want = torch.where(live, table[ids.clamp(0, V - 1)].double() * scale, 0.0)
        assert ((out[:T].double() - want).abs() <= want.abs() * (2**-8 + 2**-23)).all()
        if scale == 1.0 and dtype == torch.bfloat16:
            assert torch.equal(out[:T], table[ids])
        assert torch.all(out[T] == 777.0)
    table[0] = float("inf")
    table[V - 1] = float("nan")
    ids = torch.full((T,), -1, device=DEV)
    tk.dispatch_embedding(ids, table, out[:T], scale=2.0)
    assert torch.all(out[:T] == 0)
    ids[:] = V - 1
    tk.dispatch_embedding(ids, table, out[:T], scale=2.0)
    assert torch.isnan(out[:T]).all()


def test_outputs_beyond_the_caches(hk):
    """A lookup of more than 96 MB and gradients of a table of more than 256 MB, whose stores go past the caches."""
    print("embedding beyond the caches", flush=True)
    tk, T, V, H = hk.tk_kernel, 20011, 3000, 2600
    g = torch.Generator(device=DEV).manual_seed(1)
    ids, table = _ids("outside", T, V, g), torch.randn(V, H, device=DEV, generator=g).bfloat16()
    out = torch.full((T + 1, H), 777.0, dtype=torch.bfloat16, device=DEV)
    tk.dispatch_embedding(ids, table, out[:T], scale=3.0)
    live = ((ids >= 0) & (ids < V))[:, None]
    want = torch.where(live, table[ids.clamp(0, V - 1)].double() * 3.0, 0.0)
    assert ((out[:T].double() - want).abs() <= want.abs() * (2**-8 + 2**-23)).all() and torch.all(out[T] == 777.0)
    for add in ("no", "yes", "in place"):
        _backward(hk, 5000, 40000, 2056, "frequent", torch.float32, torch.int64, add, 0.5, 9)


def test_a_table_that_passes_32_bits(hk):
    """Rows behind 2^32 bytes of the table, in both directions (fp32: 4.4 GB)."""
    print("embedding of a large table", flush=True)
    tk, V, H = hk.tk_kernel, 270_000, 4096
    table = torch.zeros(V, H, device=DEV)
    ids = torch.tensor([V - 1, 0, V - 1, 262_144, 262_143, -1], device=DEV)
    table[ids[:5]] = torch.arange(5, dtype=torch.float32, device=DEV)[:, None] + 1
    out = torch.empty(6, H, dtype=torch.bfloat16, device=DEV)
    tk.dispatch_embedding(ids, table, out)
    assert torch.equal(out[:5].float(), table[ids[:5]]) and torch.all(out[5] == 0)
    dout = torch.ones(6, H, dtype=torch.bfloat16, device=DEV)
    table.fill_(5.0)
    ws = torch.empty(tk.embedding_backward_workspace_bytes(6, V, H), dtype=torch.uint8, device=DEV)
    tk.dispatch_embedding_backward(ids, dout, table, ws)
    counts = torch.zeros(V, device=DEV)
    counts[[V - 1, 0, 262_144, 262_143]] = torch.tensor([2.0, 1.0, 1.0, 1.0], device=DEV)
    assert torch.equal(table[:, 0], counts) and torch.equal(table[:, -1], counts)
    assert float(table.sum(dtype=torch.float64)) == 5.0 * H


@pytest.mark.parametrize("T", [1023, 1024, 1025])
def test_gradient_at_one_token_a_thread(hk, T):
    for kind in ("outside", "frequent"):
        _backward(hk, T, 5000, 136, kind, torch.float32, torch.int64, "yes", 1.0, T)


@pytest.mark.parametrize("first", [0, 3, 8, 27])
def test_rows_of_about_as_many_blocks_as_a_wave_joins(hk, first):
    """Rows of 120 to 160 tokens behind `first` single ones (blocks of eight: 15 to 21 of them), two long ones and a run that ends the list."""
    lengths = [1] * first + list(range(120, 161, 3)) + [700, 1500, 2, 129]
    ids = torch.repeat_interleave(torch.arange(len(lengths), device=DEV), torch.tensor(lengths, device=DEV))
    g = torch.Generator(device=DEV).manual_seed(first)
    ids = ids[torch.randperm(ids.numel(), device=DEV, generator=g)]
    for dtype, add in ((torch.float32, "yes"), (torch.bfloat16, "no"), (torch.float32, "in place")):
        _backward(hk, ids.numel(), len(lengths) + 3, 584, "given", dtype, torch.int32, add, 0.5, first, ids=ids)
