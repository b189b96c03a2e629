"""Calls that are captured into graphs: forward and gradients, by the thread that captures and by autograd's, and what graphs leave behind."""
import ctypes

import pytest
import torch

import mops_b200
import mops_b200.torch as mt
from mops_b200 import _lib
from test_block_ops import norm_arguments, normal, offsets_of

pytestmark = pytest.mark.gpu


def array(t):
    return _lib.make_array(t.data_ptr(), str(t.dtype).split(".")[1], tuple(t.shape), t.stride())


class Lookup:
    """embedding_lookup through the C ABI, without waiting, on a stream."""

    def __init__(self):
        self.W, self.indices = torch.arange(40.0, device="cuda").reshape(10, 4), torch.arange(5, dtype=torch.int32, device="cuda")
        self.out = torch.empty(5, 4, device="cuda")
        self.arguments = [array(t) for t in (self.out, self.W, self.indices)] + [ctypes.c_double(1.0)]
        self.lib = _lib.library()
        torch.cuda.synchronize()

    def __call__(self, stream):
        self.lib.mops_b200_set_stream(ctypes.c_void_p(stream))
        self.lib.mops_b200_set_wait(0)
        try:
            _lib.call("mops_b200_cuda_embedding_lookup", self.arguments)
        finally:
            self.lib.mops_b200_set_stream(None)
            self.lib.mops_b200_set_wait(1)


def new_stream(rt):
    handle = ctypes.c_void_p()
    assert rt.cudaStreamCreateWithFlags(ctypes.byref(handle), 1) == 0
    return handle.value


def capture(rt, stream, call):
    graph = ctypes.c_void_p()
    assert rt.cudaStreamBeginCapture(ctypes.c_void_p(stream), 1) == 0  # (this thread's calls only)
    call(stream)
    assert rt.cudaStreamEndCapture(ctypes.c_void_p(stream), ctypes.byref(graph)) == 0
    return graph


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,columns", [(500, 64), (17000, 40), (300, 33)])
def test_gradients_in_a_graph(dtype, tokens, columns):
    """A recorded pass and its gradients, replayed on new values: tokens sorted by one block and by kernels of their own, rows that are copied first."""
    table = normal((900, columns), dtype, 1).requires_grad_(True)
    indices = (torch.arange(tokens, device="cuda", dtype=torch.int32) * 7) % 900
    W, offsets = normal((3, columns, columns), dtype, 2, columns ** -0.5).requires_grad_(True), offsets_of([tokens // 2, 0, tokens - tokens // 2])
    (x, _, gate, *weights), grads = norm_arguments(tokens, columns, 2, dtype)
    leaves = [table, W] + [t.requires_grad_(True) for t in [x, gate, *weights]]

    def everything():
        branch = mt.grouped_matrix_product(mt.embedding_lookup(table, indices, 2.0, 3), W, offsets)
        out = mt.gated_residual_norm(x, branch, gate, *weights)
        return [t.detach() for t in out] + list(torch.autograd.grad(out, leaves, grads))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        everything()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = everything()
    for step in range(3):
        with torch.no_grad():
            for t in leaves:
                t.mul_(1.25)
            indices.copy_((indices + 11) % 900)
        graph.replay()
        for a, b in zip(captured, everything()):
            assert torch.equal(a, b)


def test_graphs_do_not_make_streams_wait_for_one_another():
    """Two streams used in turn, on a thread that has captured many graphs, while a third is busy: no call waits for the device."""
    rt, lookup = ctypes.CDLL("libcudart.so.12"), Lookup()
    capturing, a, b = (new_stream(rt) for _ in range(3))
    graphs = [capture(rt, capturing, lookup) for _ in range(100)]
    for s in (a, b, a, b):
        lookup(s)
    torch.cuda.synchronize()
    torch.cuda._sleep(1_000_000_000)  # half a second on the default stream
    busy = torch.cuda.Event()
    busy.record()
    for s in (a, b, a, b):
        lookup(s)
    waited = busy.query()
    torch.cuda.synchronize()
    for g in graphs:
        assert rt.cudaGraphDestroy(g) == 0
    for s in (capturing, a, b):
        assert rt.cudaStreamDestroy(ctypes.c_void_p(s)) == 0
    assert not waited


def test_graphs_that_have_gone_leave_nothing_behind():
    rt, lookup = ctypes.CDLL("libcudart.so.12"), Lookup()
    stream = new_stream(rt)
    for _ in range(20):
        assert rt.cudaGraphDestroy(capture(rt, stream, lookup)) == 0
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    for _ in range(30000):  # (a few hundred bytes each where they are left behind)
        assert rt.cudaGraphDestroy(capture(rt, stream, lookup)) == 0
    assert before - torch.cuda.mem_get_info()[0] < 3 << 20
    assert rt.cudaStreamDestroy(ctypes.c_void_p(stream)) == 0


def test_words_of_a_graph_that_has_gone_serve_another():
    """Graphs alive at the same time have words of their own; what one reported is not taken for a report of the next."""
    rt, lookup = ctypes.CDLL("libcudart.so.12"), Lookup()
    stream = new_stream(rt)
    bad = torch.tensor([0, 1, 99, 2, -1], dtype=torch.int32, device="cuda")
    good = lookup.indices.clone()
    for step in range(6):
        graphs = [capture(rt, stream, lookup) for _ in range(3)]
        for g in graphs:
            run = ctypes.c_void_p()
            assert rt.cudaGraphInstantiate(ctypes.byref(run), g, ctypes.c_ulonglong(0)) == 0
            for indices in (bad, good):
                lookup.indices.copy_(indices)
                torch.cuda.synchronize()
                assert rt.cudaGraphLaunch(run, ctypes.c_void_p(stream)) == 0
                torch.cuda.synchronize()
                inside = (indices >= 0) & (indices < 10)
                assert torch.equal(lookup.out, torch.where(inside[:, None], lookup.W[indices.clamp(0, 9).long()], 0.0))
            assert rt.cudaGraphExecDestroy(run) == 0
            assert rt.cudaGraphDestroy(g) == 0
        assert torch.equal(mops_b200.embedding_lookup(lookup.W, good), lookup.W[good.long()])
    assert rt.cudaStreamDestroy(ctypes.c_void_p(stream)) == 0
