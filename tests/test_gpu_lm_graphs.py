"""The language-model operators in captured CUDA graphs: replays follow their
inputs, and the workspace that a graph uses outlives larger calls."""
import ctypes

import numpy as np
import pytest
import torch

import acediar._lib as L
import acediar.tensor as T

pytestmark = pytest.mark.gpu


@pytest.fixture
def fresh(acd):
    """The package on a context of its own, whose workspace is empty."""
    device = torch.cuda.current_device()
    kept = T._ctx.pop(device, None)
    acd.context()
    yield acd
    torch.cuda.synchronize()
    L.check(acd.lib().acd_ctx_destroy(T._ctx.pop(device)))
    if kept is not None:
        T._ctx[device] = kept


def fill(t, seed):
    """New values in the same storage."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    if t.dtype == "int64":
        t.storage.copy_(torch.randint(1, 200, t.storage.shape, device="cuda", generator=g))
    elif t.dtype == "int8":
        t.storage.copy_(torch.randint(-128, 128, t.storage.shape, device="cuda", generator=g, dtype=torch.int8))
    else:
        t.storage.copy_(torch.rand(t.storage.shape, device="cuda", generator=g) + 0.1)


def calls(acd, factor=1):
    """name -> (tensors, call); each of them uses the workspace but the first two."""
    new = lambda shape, d="float": acd.empty_tensor(shape, d)  # noqa: E731
    rows, V = 300 * factor, 700
    x, tok, st = new((rows, V)), new((rows,), "int64"), new((rows,))
    D, n = 512, 400 * factor
    a, b, w = new((D, n), "float16"), new((D, n), "float16"), new((D,), "float16")
    rs = new((n,))
    # (as many columns as the blocks cannot prepare for themselves)
    K, M = 8192, 20000
    q, s, v = new((K // 2, M), "int8"), new((K // 64, M), "float16"), new((K, 10 * factor))
    return {
        "grad": ([x, tok, st], lambda: [acd.token_logprob_grad(x, tok, st, d_logprob=st, axis=2)]),
        "norm": ([a, b, w], lambda: acd.residual_norm(a, b, w, w)[:4]),
        "logprob": ([x, tok], lambda: acd.token_logprob(x, tok, axis=2, top=5)),
        "norm_grad": ([a, b, w, rs], lambda: acd.residual_norm_grad(a, b, a, b, rs, rs, w, w, w)),
        "quant4": ([q, s, v], lambda: [acd.quant4_matvec(q, s, v, 64)]),
    }


def host(out):
    return [t.as_array() for t in out]


@pytest.mark.parametrize("name", ["grad", "norm", "logprob", "norm_grad", "quant4"])
def test_replays_follow_the_inputs(fresh, name):
    tensors, call = calls(fresh)[name]
    for t in tensors:
        fill(t, 1)
    call()  # the workspace grows here
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for seed in (2, 3):
        for k, t in enumerate(tensors):
            fill(t, seed + 10 * k)
        graph.replay()
        torch.cuda.synchronize()
        got = host(out)
        for a, b in zip(got, host(call())):
            assert np.array_equal(a, b)
    graph.reset()


@pytest.mark.parametrize("name", ["logprob", "norm_grad", "quant4"])
def test_a_graph_keeps_its_workspace(fresh, name):
    """A larger call after the capture takes a new region; the old one is neither freed nor reused."""
    tensors, call = calls(fresh)[name]
    for k, t in enumerate(tensors):
        fill(t, k)
    want = host(call())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for factor in (6, 40):
        for k, t in enumerate(calls(fresh, factor)[name][0]):
            fill(t, k)
        calls(fresh, factor)[name][1]()
        for t in out:
            t.storage.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(host(out), want):
            assert np.array_equal(a, b)
    graph.reset()


@pytest.mark.parametrize("name", ["logprob", "norm_grad", "quant4"])
def test_growing_in_a_capture_is_refused(fresh, name):
    """The call says so, the capture goes on, and the call works afterwards."""
    tensors, call = calls(fresh)[name]
    for k, t in enumerate(tensors):
        fill(t, k)
    other, other_call = calls(fresh)["norm"]
    for k, t in enumerate(other):
        fill(t, k)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(L.AcdError) as e:
            call()
        out = other_call()
    assert e.value.status == 5 and "capture" in str(e.value)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(host(out), host(other_call())):
        assert np.array_equal(a, b)
    assert all(np.isfinite(v).all() for v in host(call()))
    graph.reset()


def test_a_context_with_graphs_is_destroyed(acd):
    """Regions kept for a graph are freed with their allocator."""
    alive = {}
    alloc_t = ctypes.CFUNCTYPE(ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p)
    free_t = ctypes.CFUNCTYPE(None, ctypes.c_void_p, ctypes.c_void_p)

    def alloc(n, _):
        t = torch.empty(n, dtype=torch.uint8, device="cuda")
        alive[t.data_ptr()] = t
        return t.data_ptr()

    def free(p, _):
        del alive[p]

    a, f = alloc_t(alloc), free_t(free)
    lib, device = acd.lib(), torch.cuda.current_device()
    kept = T._ctx.pop(device, None)
    try:
        c = acd.context()
        L.check(lib.acd_ctx_set_allocator(c, ctypes.cast(a, ctypes.c_void_p), ctypes.cast(f, ctypes.c_void_p), None))
        tensors, call = calls(acd)["norm_grad"]
        for k, t in enumerate(tensors):
            fill(t, k)
        call()
        assert len(alive) == 1
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        big, big_call = calls(acd, 40)["logprob"]
        for k, t in enumerate(big):
            fill(t, k)
        big_call()
        assert len(alive) == 2
        graph.replay()
        torch.cuda.synchronize()
        graph.reset()
        L.check(lib.acd_ctx_destroy(T._ctx.pop(device)))
        assert not alive
    finally:
        T._ctx.pop(device, None)
        if kept is not None:
            T._ctx[device] = kept
