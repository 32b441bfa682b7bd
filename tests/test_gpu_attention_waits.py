"""The joins' waits: their limit, and that what one launch leaves behind does not
reach the next replay of a captured one."""
import ctypes
import os
import shutil
import subprocess
import sys
import threading

import pytest

torch = pytest.importorskip("torch")
from attention_cases import SENTINEL, Batch  # noqa: E402

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(autouse=True)
def healthy(cuda, qmv):
    qmv.device_status(clear=True)
    yield
    assert qmv.device_status(clear=True) == 0


@pytest.fixture(scope="module")
def check(qmv, tmp_path_factory):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    so = str(tmp_path_factory.mktemp("wait") / "wait_check.so")
    csrc = os.path.join(os.path.dirname(HERE), "my-inference-engine_b200", "csrc")
    subprocess.run([nvcc, "-O2", "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-Xcompiler", "-fPIC", "-I", csrc,
                    "-o", so, os.path.join(HERE, "attention_wait_check.cu")], check=True, capture_output=True)
    lib = ctypes.CDLL(so)
    lib.check_wait.argtypes = [ctypes.c_void_p, ctypes.c_uint64, ctypes.c_uint64, ctypes.c_void_p]
    lib.check_set.argtypes = [ctypes.c_void_p, ctypes.c_uint64]
    lib.check_number.argtypes = [ctypes.c_void_p, ctypes.c_uint64, ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p]
    return lib


def test_a_wait_for_a_flag_that_nobody_sets_ends(qmv, check):
    """It gives up after its limit and reports bit 6; what runs afterwards is right."""
    flag, status = torch.zeros(1, dtype=torch.int64, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    assert check.check_wait(flag.data_ptr(), 12345, 50_000_000, status.data_ptr()) == 0
    assert int(status) == 64
    status.zero_()
    torch.cuda.synchronize()
    assert check.check_set(flag.data_ptr(), 12345) == 0
    assert check.check_wait(flag.data_ptr(), 12345, 50_000_000, status.data_ptr()) == 0
    assert int(status) == 0
    b = Batch(qmv, "bf16", 14, 2, 64, [50, 1], [3000, 700])
    b.run_paged()
    b.check(False)


def _nodes(rt, graph):
    def ok(result):
        assert result[0] == rt.cudaError_t.cudaSuccess, result
        return result[1:]

    raw = rt.cudaGraph_t(graph.raw_cuda_graph())
    nodes = ok(rt.cudaGraphGetNodes(raw, ok(rt.cudaGraphGetNodes(raw))[1]))[0]
    return ok, raw, [(ok(rt.cudaGraphNodeGetType(n))[0].name.replace("cudaGraphNodeType", ""), n) for n in nodes]


def test_every_replay_of_a_captured_launch_has_a_number(check):
    """All CTAs of a replay, and no other replay's: a flag that was set too late to
    be waited for cannot be taken for a later replay's."""
    ctas = 500
    count = torch.zeros(1, dtype=torch.int64, device="cuda")
    out = torch.zeros(ctas, dtype=torch.int64, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        assert check.check_number(out.data_ptr(), 7000, count.data_ptr(), ctas, torch.cuda.current_stream().cuda_stream) == 0
    for k in range(20):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.all(out == 7000 + k)
    assert check.check_number(out.data_ptr(), 9, None, ctas, None) == 0
    torch.cuda.synchronize()
    assert torch.all(out == 9)


@pytest.mark.parametrize("t,new,packed", [("bf16", 1, False), ("bf16", 50, False), ("f32", 1, False), ("f32", 50, False), ("bf16", 50, True), ("f32", 50, True)])
def test_a_captured_launch_counts_its_replays(qmv, t, new, packed):
    rt, drv = pytest.importorskip("cuda.bindings.runtime"), pytest.importorskip("cuda.bindings.driver")
    b = Batch(qmv, t, 14, 2, 64, [new, new + 600 * packed], [2900, 700 + 600 * packed])
    run = b.run_packed if packed else b.run_paged
    run()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        for _ in range(2):
            run(stream=torch.cuda.current_stream().cuda_stream)
    _, _, nodes = _nodes(rt, graph)
    assert not any(k == "Memset" for k, _ in nodes)
    counts, ctas = [], []
    for k, node in nodes:
        if k != "Kernel":
            continue
        error, params = drv.cuGraphKernelNodeGetParams(drv.CUgraphNode(int(node)))
        assert error == drv.CUresult.CUDA_SUCCESS
        if packed and t == "f32" and params.blockDimX == 256:
            continue  # the split of keys and values
        # the tag is the last parameter: a number and the count's address
        at = ctypes.cast(int(params.kernelParams), ctypes.POINTER(ctypes.c_void_p))[4 if new == 1 else 5]
        counts.append(ctypes.cast(at, ctypes.POINTER(ctypes.c_uint64))[1])
        ctas.append(params.gridDimX)
    assert len(counts) == 2 and len(set(counts)) == 2 and all(counts)
    graph.instantiate()
    for k in range(3):
        b.out.fill_(SENTINEL)
        graph.replay()
        b.check(packed)
        for at, n in zip(counts, ctas):
            have = (ctypes.c_uint64 * 1)()
            assert rt.cudaMemcpy(ctypes.addressof(have), at, 8, rt.cudaMemcpyKind.cudaMemcpyDeviceToHost)[0] == rt.cudaError_t.cudaSuccess
            assert have[0] == (k + 1) * n


def test_captured_launches_beyond_the_counts(qmv):
    """More captured launches than have counts of their own: those clear their
    flags on the stream, and are right all the same.  In a process of its own,
    since counts are not given back."""
    code = """
import sys
import threading
sys.path.insert(0, %r)
import torch, conftest
from cuda.bindings import runtime as rt
qmv = conftest.load_package(); qmv.load_library()
from attention_cases import SENTINEL, Batch
from test_gpu_attention_waits import _nodes
b = Batch(qmv, "bf16", 14, 2, 64, [1, 1], [2900, 700])
b.run_paged()
graph = torch.cuda.CUDAGraph(keep_graph=True)
with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
    for _ in range(4100):
        b.run_paged(stream=torch.cuda.current_stream().cuda_stream)
kinds = [k for k, _ in _nodes(rt, graph)[2]]
assert kinds.count("Kernel") == 4100 and kinds.count("Memset") == 4, (kinds.count("Kernel"), kinds.count("Memset"))
graph.instantiate()
for _ in range(3):
    b.out.fill_(SENTINEL)
    graph.replay()
    b.check(False)
assert qmv.device_status() == 0
print("all right")
""" % HERE
    pytest.importorskip("cuda.bindings.runtime")
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "all right" in done.stdout, done.stderr[-2000:]


# ------------------------------------------------- calls that run side by side

def _side_by_side(qmv):
    return [Batch(qmv, "bf16", 14, 2, 64, [1, 1], [5000, 4000], page=64), Batch(qmv, "f16", 8, 2, 128, [200], [1500], page=32, seed=1),
            Batch(qmv, "f32", 14, 2, 64, [90, 3], [900, 2000], seed=2)]


def test_every_call_of_two_streams(qmv):
    """Each of the calls in flight together against its result alone, bit for bit."""
    work = [(b, run) for b in _side_by_side(qmv) for run in (b.run_paged, b.run_packed)]
    alone = []
    for b, run in work:
        out = torch.full_like(b.out, SENTINEL)
        run(out=out)
        alone.append(out)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = [[torch.full_like(b.out, SENTINEL) for _ in range(10 * len(streams))] for b, _ in work]
    torch.cuda.synchronize()
    for i in range(10 * len(streams)):
        for j, (b, run) in enumerate(work):
            run(stream=streams[(i + j) % 3].cuda_stream, out=outs[j][i])
    torch.cuda.synchronize()
    for want, got in zip(alone, outs):
        assert all(torch.equal(want, x) for x in got)


def test_every_call_of_two_threads(qmv):
    bs = _side_by_side(qmv)
    alone = []
    for b in bs:
        out = torch.full_like(b.out, SENTINEL)
        b.run_paged(out=out)
        alone.append(out)
    outs = [[torch.full_like(b.out, SENTINEL) for _ in range(50)] for b in bs]
    streams = [torch.cuda.Stream() for _ in bs]
    torch.cuda.synchronize()
    failures = []

    def work(b, stream, mine):
        try:
            for out in mine:
                b.run_paged(stream=stream.cuda_stream, out=out)
        except Exception as e:  # noqa: BLE001 - handed to the test's thread
            failures.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(bs, streams, outs)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failures
    for want, got in zip(alone, outs):
        assert all(torch.equal(want, x) for x in got)


def test_two_captured_graphs_at_once(qmv):
    """Replays of two graphs on two streams, each with scratch of its own."""
    bs = _side_by_side(qmv)
    graphs = []
    for b in bs:
        b.run_paged()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=torch.cuda.Stream()):
            b.run_paged(stream=torch.cuda.current_stream().cuda_stream)
        graphs.append((b, g, b.out.clone(), torch.zeros((), dtype=torch.int64, device="cuda"), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(30):
        for b, g, want, wrong, stream in graphs:
            with torch.cuda.stream(stream):
                b.out.fill_(SENTINEL)
                g.replay()
                wrong += (b.out != want).sum()
    torch.cuda.synchronize()
    assert [int(x[3]) for x in graphs] == [0, 0, 0]
