"""The table of a GradTensors is memory that the list itself takes from torch's allocator, on the stream it is made on. Calls on another stream
have to tell the allocator of that stream: it otherwise gives the table's memory away when the list is dropped, while kernels that read it are
still to run."""
import pytest
import torch

import hipkittens_amd as hk

tk = hk.tk_kernel
DEV = "cuda:0"


class _Table:
    device = torch.device("cuda", 0)

    def __init__(self):
        self.streams = []

    def record_stream(self, stream):
        self.streams.append(stream)


@pytest.mark.parametrize("call", ["norm", "clip"])
def test_a_call_on_another_stream_is_recorded(monkeypatch, call):
    """On the CPU: the dispatchers with a stream and a launch in the places of the GPU's."""
    current = [7]
    launched = []

    class Native:
        grad_norm = staticmethod(lambda *a: launched.append(current[0]) or 0)
        grad_clip = grad_norm

    monkeypatch.setattr(tk, "_native", Native)
    monkeypatch.setattr(tk, "_raw_stream", lambda index: current[0])
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: ("stream", current[0]))
    monkeypatch.setattr(tk.GradTensors, "__init__", lambda self: None)
    grads = tk.GradTensors()
    grads.list, grads.n, grads.chunks, grads.device, grads.stream = _Table(), 1, 1, _Table.device, 7
    run = lambda: tk.dispatch_grad_norm(grads, None, None) if call == "norm" else tk.dispatch_grad_clip(grads, None, 1.0)
    run()
    assert launched == [7] and grads.list.streams == []   # the table's own stream: the allocator knows it
    current[0] = 9
    run()
    assert launched == [7, 9] and grads.list.streams == [("stream", 9)]


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_the_table_of_a_dropped_list_waits_for_the_other_stream(monkeypatch, native):
    """A list is used on a side stream behind work that takes a while, and dropped at once: its table's memory is not given to new tensors before
    the calls have run."""
    print(f"table of a dropped list, native={native}", flush=True)
    if not native:
        monkeypatch.setattr(tk, "_native", tk._NoNative)
    grad = torch.full((100_001,), 2.0, device=DEV)
    norm, ws = torch.zeros(1, device=DEV), torch.empty(tk.grad_norm_workspace_bytes(), dtype=torch.uint8, device=DEV)
    plan = tk.GradTensors([grad])
    size, table = plan.list.numel(), plan.list.data_ptr()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    busy, done = torch.ones(4096, 4096, device=DEV), torch.cuda.Event()
    with torch.cuda.stream(side):
        for _ in range(200):   # some ms at least
            busy @ busy
        tk.dispatch_grad_norm(plan, norm, ws)
        tk.dispatch_grad_clip(plan, norm, 1.0)
        done.record(side)
    del plan
    taken = [torch.empty(size, dtype=torch.uint8, device=DEV) for _ in range(8)]   # (nothing is written to them)
    waited = not done.query()
    places = [t.data_ptr() for t in taken]
    torch.cuda.synchronize()
    assert waited and table not in places
    assert abs(norm.item() - 2 * 100_001**0.5) < 1e-3 and abs(grad[77].item() * 100_001**0.5 - 1) < 1e-5
