"""The scratch that the operators over the nodes of a frame keep between their kernels: calls of several host threads on one stream, on the per-thread
default streams, and calls in graphs beside larger ones outside of them, all with the bits of the same calls by themselves."""
import threading

import pytest
import torch

from test_teacher_operators import buffer, normal

# layers read once and in two passes, classes read once and by passes: scratch of a few KB to some MB
SIZES = [(300, 40, 4), (3000, 333, 8), (9001, 100, 16), (20011, 64, 32)]


def calls(nodes, frames, top, dtype=torch.float32):
    """One backward pass of layer norm and one distillation loss, both chains of kernels with scratch between them, as a function that gives what they give."""
    from binarybrain_b200 import ops
    x, dy = normal(nodes, nodes, frames), normal(nodes + 1, nodes, frames)
    mean, rstd = x.mean(0).float().cuda(), (1 / x.std(0, unbiased=False)).float().cuda()
    t, index = torch.topk(2 * normal(nodes + 2, nodes, frames), top, dim=0)
    x, dy, t, index, gamma = buffer(x, dtype), buffer(dy, dtype), buffer(t, dtype), index.to(torch.int32).cuda(), normal(nodes + 3, nodes).float().cuda()

    def run():
        dx, dgamma, dbeta = ops.layer_norm_backward(x, dy, mean, rstd, frames, gamma=gamma)
        dz, loss, buf = ops.distillation_loss(x, t, index, frames, temperature=2.0)
        return dx[:, :frames], dgamma, dbeta, dz[:, :frames], loss, buf
    return run


def same(got, want):
    return all(torch.equal(g, w) for g, w in zip(got, want))


@pytest.mark.gpu
def test_host_threads_on_one_stream():
    runs = [calls(*size) for size in SIZES]
    want = [[t.clone() for t in run()] for run in runs]
    torch.cuda.synchronize()
    stream, failed, start = torch.cuda.current_stream(), [], threading.Barrier(len(runs))

    def work(k):
        try:
            with torch.cuda.stream(stream):
                start.wait(60)
                got = [runs[k]() for _ in range(40)]
            stream.synchronize()
            failed.extend((k, i) for i, g in enumerate(got) if not same(g, want[k]))
        except Exception as e:  # noqa: BLE001 (a thread's exception is the test's)
            failed.append((k, repr(e)))
    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(runs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


@pytest.mark.gpu
def test_host_threads_on_their_default_streams():
    """The handle of the per-thread default stream (cudaStreamPerThread, 2) is the same in all threads, the streams are not."""
    from binarybrain_b200 import ops
    from binarybrain_b200.ops import _n
    cases = []
    for nodes, frames in ((9001, 100), (20011, 64), (70001, 32)):
        x, dy = (buffer(normal(s, nodes, frames), torch.float32) for s in (nodes, nodes + 1))
        mean, rstd = torch.zeros(frames, device="cuda"), torch.ones(frames, device="cuda")
        want = ops.layer_norm_backward(x, dy, mean, rstd, frames)
        outs = [[torch.empty_like(t) for t in want] for _ in range(20)]
        cases.append((x, dy, mean, rstd, nodes, frames, want, outs))
    torch.cuda.synchronize()
    failed, start = [], threading.Barrier(len(cases))

    def work(k):
        x, dy, mean, rstd, nodes, frames, want, outs = cases[k]
        try:
            start.wait(60)
            for dx, dgamma, dbeta in outs:
                _n.bbcu_fp32_LayerNormalization_Backward(x, dy, dx, None, mean, rstd, dgamma, dbeta, 0, nodes, frames, x.shape[1], dy.shape[1], dx.shape[1], 2)
        except Exception as e:  # noqa: BLE001
            failed.append((k, repr(e)))
    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed
    for *_, frames, want, outs in cases:
        for out in outs:
            assert torch.equal(out[0][:, :frames], want[0][:, :frames]) and same(out[1:], want[1:])


@pytest.mark.gpu
def test_graphs_beside_larger_calls():
    """A graph's calls keep their results when the stream that they were captured on makes larger calls afterwards, when other streams take scratch, when the
    graph runs on another stream beside both; the graph needs no call before it is captured, and gives its scratch back when it goes."""
    from binarybrain_b200 import abi
    small, large = calls(9001, 40, 4), calls(20011, 200, 40)
    want, want_large = [t.clone() for t in small()], [t.clone() for t in large()]
    torch.cuda.synchronize()
    L = abi.lib()
    L.bbcu_LocalHeap_GarbageCollect()                                    # the stream below has no scratch yet
    captured, others = torch.cuda.Stream(), [torch.cuda.Stream() for _ in range(3)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=captured):
        held = small()
        again = small()
    for s in (captured, *others):
        with torch.cuda.stream(s):
            assert same(large(), want_large)
    L.bbcu_LocalHeap_GarbageCollect()
    for turn in range(20):
        for t in (*held, *again):
            t.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(others[0]):
            graph.replay()
        got = []
        for s in (captured, others[1], others[2]):
            with torch.cuda.stream(s):
                got.append(large())
        torch.cuda.synchronize()
        assert same(held, want) and same(again, want) and all(same(g, want_large) for g in got)
    small()                                                              # (this stream's scratch, which the collection above took, is back)
    before = L.bbcu_LocalHeap_GetAllocatedSize()
    del graph, held, again
    torch.cuda.synchronize()
    for _ in range(100):                                                 # CUDA says on a thread of its own that the graph is gone
        small()
        if L.bbcu_LocalHeap_GetAllocatedSize() < before:
            break
        threading.Event().wait(0.02)
    assert L.bbcu_LocalHeap_GetAllocatedSize() < before
