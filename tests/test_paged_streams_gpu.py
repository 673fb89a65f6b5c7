"""The workspace of the paged attention between streams and graph branches
(marked gpu)."""
import ctypes
import subprocess
import sys
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")
from test_paged_gpu import BF16, make, ops  # noqa: E402, F401

pytestmark = pytest.mark.gpu

KERNEL_NODE = 0


def captured_edges(graph):
    """(kernel nodes, edges) of a captured graph."""
    rt = ctypes.CDLL("libcudart.so.12")
    raw = ctypes.c_void_p(graph.raw_cuda_graph())
    count = ctypes.c_size_t()
    assert rt.cudaGraphGetNodes(raw, None, ctypes.byref(count)) == 0
    nodes = (ctypes.c_void_p * count.value)()
    assert rt.cudaGraphGetNodes(raw, nodes, ctypes.byref(count)) == 0
    kernels = []
    for node in nodes:
        kind = ctypes.c_int()
        assert rt.cudaGraphNodeGetType(ctypes.c_void_p(node), ctypes.byref(kind)) == 0
        if kind.value == KERNEL_NODE:
            kernels.append(node)
    assert rt.cudaGraphGetEdges_v2(raw, None, None, None, ctypes.byref(count)) == 0
    if count.value == 0:
        return kernels, set()
    first, second = (ctypes.c_void_p * count.value)(), (ctypes.c_void_p * count.value)()
    data = (ctypes.c_uint64 * count.value)()  # eight bytes an edge
    assert rt.cudaGraphGetEdges_v2(raw, first, second, data, ctypes.byref(count)) == 0
    return kernels, set(zip(first, second))


def fork(ops, calls, stream=None, also_on_main=False):  # noqa: F811
    """A graph with each call on a branch of its own (captured from `stream`; the first once more at the end)."""
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    sides = [torch.cuda.Stream() for _ in calls[1:]]
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        main = torch.cuda.current_stream()
        for side in sides:
            side.wait_stream(main)
        for stream, (made, max_q, out) in zip([main] + sides, calls):
            with torch.cuda.stream(stream):
                ops.attention(*made, max_q=max_q, out=out)
        if also_on_main:
            made, max_q, out = calls[0]
            ops.attention(*made, max_q=max_q, out=out)
        for side in sides:
            main.wait_stream(side)
    return graph


def some_calls():
    calls = []
    for seed, requests in enumerate(([(1, 9000), (1, 500)], [(2, 5000), (1, 7000), (1, 12)], [(1, 3000)] * 5)):
        made = make(requests, 8, 2, 128, 64, BF16, seed=seed)
        calls.append((made, max(n for n, _ in requests), torch.empty_like(made[0])))
    return calls


@pytest.mark.parametrize("used_before", [False, True])
@pytest.mark.parametrize("also_on_main", [False, True])
def test_branches_of_a_graph_are_ordered(ops, used_before, also_on_main):  # noqa: F811
    for _ in range(2):  # also in a second capture
        calls, stream = some_calls(), torch.cuda.Stream()
        if used_before:  # the stream of the last call outside is the one that is captured then
            with torch.cuda.stream(stream):
                ops.attention(*calls[0][0], max_q=calls[0][1])
        graph = fork(ops, calls, stream, also_on_main)
        kernels, edges = captured_edges(graph)
        assert len(kernels) == 3 + also_on_main
        reach = {k: {b for a, b in edges if a == k} for k in kernels}
        for _ in kernels:
            reach = {k: r.union(*(reach[x] for x in r)) for k, r in reach.items()}
        assert sorted(len(r) for r in reach.values()) == list(range(len(kernels)))
        del graph


def test_replayed_branches_agree(ops):  # noqa: F811
    calls = some_calls()
    want = [ops.attention(*made, max_q=max_q) for made, max_q, _ in calls]
    graph = fork(ops, calls)
    for _ in range(20):
        for _, _, out in calls:
            out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for (_, _, out), w in zip(calls, want):
            assert torch.equal(out, w)
    again = [ops.attention(*made, max_q=max_q) for made, max_q, _ in calls]
    assert all(torch.equal(a, b) for a, b in zip(again, want))
    ops.sync()
    del graph


def test_a_stream_under_capture_is_not_waited_for(ops):  # noqa: F811
    """A call outside a capture, with the previous one's stream inside: refused, and neither is drawn into the other."""
    from bnn_b200 import accel
    made, max_q, out = some_calls()[0]
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        want = ops.attention(*made, max_q=max_q)
    torch.cuda.synchronize()
    other, another = torch.cuda.Stream(), torch.empty_like(out)
    with torch.cuda.graph(graph, stream=side):
        ops.attention(*made, max_q=max_q, out=out)
        with torch.cuda.stream(other), pytest.raises(accel.BnnError) as e:
            ops.attention(*made, max_q=max_q, out=another)
        assert e.value.status == accel.EBUSY
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    assert torch.equal(ops.attention(*made, max_q=max_q), want)
    del graph


@pytest.mark.parametrize("rounds", [30])
def test_calls_on_many_streams(ops, rounds):  # noqa: F811
    calls = some_calls()
    want = [ops.attention(*made, max_q=max_q) for made, max_q, _ in calls]
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    got = []
    for i in range(rounds):
        with torch.cuda.stream(streams[i * 7 % 4]):
            made, max_q, _ = calls[i % 3]
            got.append(ops.attention(*made, max_q=max_q))
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        assert torch.equal(x, want[i % 3])


def test_threads_share_a_workspace(ops):  # noqa: F811
    """Four threads, each on a stream of its own, call at once; every result is the lone call's."""
    import threading
    calls = some_calls()
    want = [ops.attention(*made, max_q=max_q) for made, max_q, _ in calls]
    torch.cuda.synchronize()
    wrong, begin = [], threading.Barrier(4)

    def work(nth):
        with torch.cuda.stream(torch.cuda.Stream()):
            begin.wait()
            for i in range(100):
                made, max_q, _ = calls[(i + nth) % 3]
                if not torch.equal(ops.attention(*made, max_q=max_q), want[(i + nth) % 3]):
                    wrong.append((nth, i))

    interval = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    try:
        threads = [threading.Thread(target=work, args=(n,)) for n in range(4)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    finally:
        sys.setswitchinterval(interval)
    assert not wrong
    ops.sync()


def test_a_dropped_workspace_is_not_handed_out(ops):  # noqa: F811
    """An operators' object that goes while another stream works on its workspace: only the next such object
    gets the memory, and only when that work is done."""
    from bnn_b200 import paged
    made, max_q, _ = some_calls()[0]
    want = ops.attention(*made, max_q=max_q)
    for _ in range(3):
        torch.cuda.synchronize()
        own = paged.Paged(ops.device)
        size, at = own._workspace.numel(), own._workspace.data_ptr()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            own.attention(*made, max_q=max_q)
            torch.cuda._sleep(200_000_000)  # a tenth of a second
            got = own.attention(*made, max_q=max_q)
        del own
        fresh = torch.empty(size, dtype=torch.uint8, device="cuda")
        assert fresh.data_ptr() != at and not side.query()
        heir = paged.Paged(ops.device)
        assert heir._workspace.data_ptr() == at and side.query()
        assert torch.equal(heir.attention(*made, max_q=max_q), want) and torch.equal(got, want)
        del heir
        ops.sync()


def test_a_workspace_of_one_stream_goes_back(ops):  # noqa: F811
    from bnn_b200 import paged
    made, max_q, _ = some_calls()[0]
    torch.cuda.synchronize()
    waiting = [paged.Paged(ops.device) for _ in range(8)]  # those that other tests left
    own = paged.Paged(ops.device)
    size, at = own._workspace.numel(), own._workspace.data_ptr()
    own.attention(*made, max_q=max_q)
    del own
    assert torch.empty(size, dtype=torch.uint8, device="cuda").data_ptr() == at
    del waiting


def test_the_handles_stream_may_go_first():
    """Calls on the device handle's own stream, the handle closed, then the operators' object dropped (in a
    process of its own: an exception there would end it)."""
    code = """if True:
        import ctypes, gc, sys
        sys.path[:0] = sys.argv[1:]
        import torch
        from bnn_b200 import accel, paged
        from test_paged_gpu import BF16, make
        for _ in range(5):
            dev = accel.Device(0)
            ops = paged.Paged(dev)
            fn = dev.api.dll.bnn_b200_device_stream
            fn.restype, fn.argtypes = ctypes.c_void_p, [ctypes.c_void_p]
            made = make([(1, 900), (2, 50)], 4, 2, 128, 16, BF16)
            want = ops.attention(*made, max_q=2)
            torch.cuda.synchronize()
            with torch.cuda.stream(torch.cuda.ExternalStream(fn(dev.handle))):
                got = ops.attention(*made, max_q=2)
                ops.sync()
            assert torch.equal(got, want)
            dev.close()
            del ops
            gc.collect()
            torch.zeros(1 << 25, device="cuda")
            torch.cuda.synchronize()
        print("through")
    """
    here = Path(__file__).resolve()
    got = subprocess.run([sys.executable, "-c", code, str(here.parent), str(here.parents[1] / "bnn-train-infer_b200")], capture_output=True,
                         text=True, timeout=300)
    assert got.returncode == 0 and "through" in got.stdout, got.stderr[-2000:]
