"""The binding's own workspaces belong to the stream that the call runs on.

Memory from another stream's pool may have belonged to a tensor that work still
pending there reads or writes, and nothing makes the call's stream wait for that
work. Taken from the call's own stream, a workspace is ordered with it in both
directions. The CPU tests watch where the memory is asked for, on a library that
only counts; the GPU tests run the operators behind and before pending work."""
from __future__ import annotations

import contextlib
import types

import pytest


class Recorder:
    """The library's calls and torch's stream contexts and allocations, on a
    host without a device: every query asks for `need` bytes."""

    def __init__(self, cb, torch, need):
        self.cb, self.need, self.stack, self.asked, self.ran = cb, need, ["current"], [], []
        self.real_empty = torch.empty

    def query(self, desc, out):
        out._obj.workspace_bytes = out._obj.workspace_min_bytes = self.need
        return 0

    def run(self, desc, workspace, size, stream):
        if workspace is None or size < self.need:
            return self.cb.ERR_WORKSPACE
        self.ran.append(stream)
        return 0

    def empty(self, *size, **kw):
        if kw.get("dtype") is not None and str(kw["dtype"]) == "torch.uint8":
            self.asked.append(self.stack[-1])
        return self.real_empty(*size, **kw)

    @contextlib.contextmanager
    def on(self, stream):
        self.stack.append(stream)
        yield
        self.stack.pop()


class FakeStream:
    def __init__(self, cuda_stream):
        self.cuda_stream = cuda_stream


@pytest.fixture
def recorder(cb, monkeypatch):
    import torch
    r = Recorder(cb, torch, 512)
    lib = types.SimpleNamespace(
        choreo_gemm_query=r.query, choreo_gemm=r.run, choreo_gated_ffn_query=r.query, choreo_gated_ffn=r.run,
        choreo_gated_ffn_backward_query=r.query, choreo_gated_ffn_backward=r.run)
    lib.choreo_last_error = lambda: b""
    monkeypatch.setattr(cb, "lib", lib)
    monkeypatch.setattr(torch, "empty", r.empty)
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda self, s: None)
    monkeypatch.setattr(torch.cuda, "stream", r.on)
    monkeypatch.setattr(torch.cuda, "Stream", FakeStream)
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda ptr, device=None: ("external", ptr))
    monkeypatch.setattr(torch.cuda, "default_stream", lambda device=None: "default")
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 0x77, raising=False)
    return r


def calls(cb):
    """Each operator that may need a workspace, as a function of the stream."""
    import torch
    x, w, h = torch.zeros(4, 8).bfloat16(), torch.zeros(8, 6).bfloat16(), torch.zeros(4, 6).bfloat16()
    dx = torch.zeros(4, 8).bfloat16()
    return {
        "gemm": lambda s: cb.gemm(x, w, h, stream=s),
        "gated_ffn": lambda s: cb.gated_ffn(x, w, w, h, stream=s),
        "gated_ffn_backward": lambda s: cb.gated_ffn_backward(h, x, w, w, dx=dx, stream=s),
    }


@pytest.mark.parametrize("op", ["gemm", "gated_ffn", "gated_ffn_backward"])
def test_workspace_is_asked_for_on_the_calls_stream(cb, recorder, op):
    stream = FakeStream(0x1230)
    calls(cb)[op](stream)
    assert recorder.asked == [stream] and recorder.ran == [0x1230]


@pytest.mark.parametrize("op", ["gemm", "gated_ffn", "gated_ffn_backward"])
@pytest.mark.parametrize("ptr,where", [(0x4560, ("external", 0x4560)), (0, "default"), (1, "default")])
def test_workspace_follows_a_raw_stream_handle(cb, recorder, op, ptr, where):
    """0 and 1 both name the legacy default stream."""
    calls(cb)[op](ptr)
    assert recorder.asked == [where] and recorder.ran == [ptr]


@pytest.mark.parametrize("op", ["gemm", "gated_ffn", "gated_ffn_backward"])
def test_workspace_without_a_stream_is_the_current_streams(cb, recorder, op):
    calls(cb)[op](None)
    assert recorder.asked == ["current"] and recorder.ran == [0x77]


@pytest.mark.parametrize("op", ["gemm", "gated_ffn", "gated_ffn_backward"])
def test_workspace_of_the_current_stream_by_handle(cb, recorder, op):
    calls(cb)[op](0x77)
    assert recorder.asked == ["current"] and recorder.ran == [0x77]


def _problem(op):
    """(run(cb, out, stream), out shape and type, workspace bytes) of a call that needs a workspace."""
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(3)

    def rand(rows, cols, std, pad=0):
        return (torch.randn(rows, cols + pad, generator=g, device="cuda") * std).bfloat16()[:, :cols]

    m, n, k = 500, 1003, 331   # odd rows: the operands are repacked
    x, dh = rand(m, k, 1.0), rand(m, n, 0.5)
    wg, wu = rand(k, n, k ** -0.5), rand(k, n, k ** -0.5)
    if op == "gemm":
        return lambda cb, out, s: cb.gemm(x, wg, out, stream=s), (m, n)
    if op == "gated_ffn":
        return lambda cb, out, s: cb.gated_ffn(x, wg, wu, out, stream=s), (m, n)
    return lambda cb, out, s: cb.gated_ffn_backward(dh, x, wg, wu, dx=out, stream=s), (m, k)


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["gemm", "gated_ffn", "gated_ffn_backward"])
@pytest.mark.parametrize("raw", [False, True])
def test_pending_work_on_freed_memory_is_left_alone(cb, cuda, op, raw):
    """The current stream still has to read tensors that were freed on the host
    when the call on another stream takes its workspace, and allocates and fills
    new ones after it."""
    import torch
    run, shape = _problem(op)
    ref = torch.empty(*shape, device="cuda", dtype=torch.bfloat16)
    run(cb, ref, None)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    stream = side.cuda_stream if raw else side
    sizes = [1 << 20, 2 << 20, 3 << 20, 4 << 20, 5 << 20, 6 << 20, 8 << 20]   # around what the calls ask for
    outs = [torch.empty_like(ref) for _ in range(4)]
    kept = [[torch.zeros(s, dtype=torch.uint8, device="cuda") for s in sizes] for _ in outs]
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        owners = [torch.full((s,), 17 + i, dtype=torch.uint8, device="cuda") for s in sizes]
        torch.cuda._sleep(4_000_000)                  # some milliseconds of the current stream
        for dst, src in zip(kept[i], owners):
            dst.copy_(src)
        del owners, src                               # free on the host, still to be read on the device
        run(cb, out, stream)
        later = [torch.full((s,), 0x7F, dtype=torch.uint8, device="cuda") for s in sizes]
        del later
    torch.cuda.synchronize()
    cb.sync_status()
    for i, out in enumerate(outs):
        assert torch.equal(out, ref), i
        for dst in kept[i]:
            assert (dst == 17 + i).all(), i


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["gemm", "gated_ffn", "gated_ffn_backward"])
@pytest.mark.parametrize("raw", [False, True])
def test_captured_on_a_joined_stream(cb, cuda, op, raw):
    """A graph whose calls run on a second stream that joined the capture: the
    workspaces are the graph's, and two graphs replayed in turn with new
    allocations between them keep their results."""
    import torch
    run, shape = _problem(op)
    ref = torch.empty(*shape, device="cuda", dtype=torch.bfloat16)
    run(cb, ref, None)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graphs = []
    for _ in range(2):
        out, graph = torch.zeros_like(ref), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            side.wait_stream(torch.cuda.current_stream())
            for _ in range(2):
                run(cb, out, side.cuda_stream if raw else side)
            torch.cuda.current_stream().wait_stream(side)
        graphs.append((graph, out))
    for _ in range(3):
        for graph, out in graphs:
            out.zero_()
            graph.replay()
            torch.full((8 << 20,), 0x7F, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    cb.sync_status()
    for _, out in graphs:
        assert torch.equal(out, ref)
