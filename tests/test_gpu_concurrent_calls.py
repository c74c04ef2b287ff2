"""Calls that use a stream's scratch (attention, the norms' gradient) beside one another: host threads, streams and graphs."""
import threading

import pytest
import torch

import my_own_cnn_b200 as b2q

pytestmark = pytest.mark.gpu


def normal(seed, *shape):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda")


def gradient(seed, t=700, heads=4, d=128, dtype=torch.float32):
    """A call of the gradient."""
    q, k, dq, dk = (normal(10 * seed + i, t, heads, d).to(dtype) for i in range(4))
    w = normal(seed, d).to(dtype)
    return lambda **kw: b2q.qk_norm_rope_bprop(dq, dk, q, k, w, w, None, None, **kw)


def attention(seed, n=3000, d=128):
    """A call of attention over a sequence that several blocks share."""
    c = b2q.KV4Cache.empty(-(-n // 64), 2, 64, d)
    b2q.kv4_append(c, normal(10 * seed, n, 2, d), normal(10 * seed + 1, n, 2, d), torch.arange(n, device="cuda"))
    table, lens = torch.arange(c.pages, device="cuda").int()[None], torch.tensor([n], device="cuda").int()
    q = normal(10 * seed + 2, 1, 1, 4, d).bfloat16()
    return lambda **kw: b2q.kv4_attention(q, c, table, lens, **kw)


def same(got, want):
    got, want = (x if isinstance(x, tuple) else (x,) for x in (got, want))
    return all(torch.equal(a, b) for a, b in zip(got, want))


def in_threads(calls, times, **kw):
    """Each call by a thread of its own, again and again; which of them ever answered otherwise than alone."""
    want = [call() for call in calls]
    torch.cuda.synchronize()
    start, wrong = threading.Barrier(len(calls)), []

    def work(i):
        start.wait()
        for _ in range(times):
            got = [calls[i](**kw) for _ in range(4)]
            torch.cuda.current_stream().synchronize()
            if not all(same(x, want[i]) for x in got):
                wrong.append(i)
                return

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    return wrong


def test_threads_of_one_stream():
    """A call's launches lie together in the stream, whatever other threads put there."""
    assert in_threads([gradient(1), gradient(2), attention(3), gradient(4, t=100, dtype=torch.bfloat16), attention(5, n=9000)], 60) == []


def into(call):
    """The call with an output of its own, made here: the stream that it then runs on allocates nothing."""
    out = call()
    return lambda **kw: call(out=out, **kw)


def test_the_stream_that_each_thread_has():
    """cudaStreamPerThread is one handle for as many streams as there are threads."""
    calls = [into(attention(i, n=6000 + 500 * i)) for i in range(4)]
    want = [call().clone() for call in calls]
    torch.cuda.synchronize()
    start, wrong = threading.Barrier(4), []

    def work(i):
        start.wait()
        for _ in range(100):
            out = calls[i](stream=2)
            torch.cuda.ExternalStream(2).synchronize()
            if not torch.equal(out, want[i]):
                wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == []


def test_streams_that_come_and_go():
    """A destroyed stream's handle comes back with a new stream; the scratch of those that are gone is used again."""
    import ctypes

    cudart = ctypes.CDLL("libcudart.so.12")
    call = into(attention(1))
    want = call().clone()
    free = None
    for i in range(60):
        s = ctypes.c_void_p()
        assert cudart.cudaStreamCreateWithFlags(ctypes.byref(s), 1) == 0
        torch.cuda.synchronize()
        out = call(stream=s.value)
        assert cudart.cudaStreamDestroy(s) == 0  # its work may still run
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        if i == 20:
            free = torch.cuda.mem_get_info()[0]
    assert torch.cuda.mem_get_info()[0] > free - (64 << 20)


def captured(call, s):
    """A graph of the call on stream s, and its outputs."""
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = call()
    return g, out


def test_graphs_of_one_stream_beside_each_other_and_eager_calls():
    calls = [attention(1, n=20000), attention(2, n=30000), gradient(3, t=3000), gradient(4, t=3000), attention(5, n=25000)]
    want = [call() for call in calls]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    attention(6)(stream=s)
    torch.cuda.synchronize()
    graphs = [captured(call, s) for call in calls[:4]]
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(100):
        for (g, _), t in zip(graphs, streams):
            with torch.cuda.stream(t):
                g.replay()
        eager = [calls[4](stream=s) for _ in range(3)]
        torch.cuda.synchronize()
        assert all(same(out, x) for (_, out), x in zip(graphs, want))
        assert all(torch.equal(x, want[4]) for x in eager)


def test_streams_within_one_capture():
    """Calls on streams that fork from the captured one run beside each other in the replay."""
    calls = [attention(1, n=20000), attention(2, n=20000)]
    want = [call() for call in calls]
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    for x in (s, t):
        x.wait_stream(torch.cuda.current_stream())
        calls[0](stream=x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        t.wait_stream(s)
        outs = [calls[0](stream=s), calls[1](stream=t)]
        s.wait_stream(t)
    for _ in range(50):
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_a_graph_gives_its_scratch_back():
    call = into(attention(1))
    want = call().clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    call(stream=s)
    torch.cuda.synchronize()
    free = None
    for i in range(40):
        g, out = captured(call, s)
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        g.reset()
        del g
        if i == 10:
            free = torch.cuda.mem_get_info()[0]
    assert torch.cuda.mem_get_info()[0] > free - (48 << 20)


@pytest.mark.parametrize("mode", ["global", "thread_local", "relaxed"])
def test_eager_calls_while_another_thread_captures(mode):
    """Calls on other streams, one of them without scratch yet, leave a capture that runs in another thread as it is."""
    calls = [into(attention(i, n=8000)) for i in range(3)]
    want = [call().clone() for call in calls]
    s, old, new = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.Stream(priority=-1)
    for x in (s, old, new):
        x.wait_stream(torch.cuda.current_stream())
    calls[0](stream=s)
    calls[1](stream=old)
    torch.cuda.synchronize()
    outs = []
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s, capture_error_mode=mode):
        t = threading.Thread(target=lambda: outs.extend([calls[1](stream=old), calls[2](stream=new)]))
        t.start()
        t.join()
        out = calls[0](stream=s)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip([out] + outs, want)) and len(outs) == 2


def test_streams_that_come_and_go_while_another_thread_captures():
    """Finding scratch that destroyed streams left waits for nothing that a capture forbids."""
    import ctypes

    cudart = ctypes.CDLL("libcudart.so.12")
    calls = [into(attention(i, n=8000)) for i in range(2)]
    want = [call().clone() for call in calls]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    calls[0](stream=s)
    torch.cuda.synchronize()
    outs = []

    def churn():
        for _ in range(30):
            x = ctypes.c_void_p()
            assert cudart.cudaStreamCreateWithFlags(ctypes.byref(x), 1) == 0
            outs.append(calls[1](stream=x.value))
            assert cudart.cudaStreamDestroy(x) == 0

    for _ in range(3):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            t = threading.Thread(target=churn)
            t.start()
            out = calls[0](stream=s)
            t.join()
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(outs[-1], want[1])
        g.reset()
    assert len(outs) == 90


def test_graphs_that_come_and_go_beside_new_streams():
    """What graphs give back, on a thread of the driver's, is taken by the first calls of new streams meanwhile."""
    calls = [into(attention(i, n=8000)) for i in range(2)]
    want = [call().clone() for call in calls]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    calls[0](stream=s)
    torch.cuda.synchronize()
    wrong = []

    def eager():
        for i in range(40):
            x = torch.cuda.Stream()
            out = calls[1](stream=x)
            x.synchronize()
            if not torch.equal(out, want[1]):
                wrong.append(i)

    t = threading.Thread(target=eager)
    t.start()
    for _ in range(40):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s, capture_error_mode="relaxed"):
            out = calls[0](stream=s)
        g.replay()
        torch.cuda.current_stream().synchronize()
        assert torch.equal(out, want[0])
        del g
    t.join()
    assert wrong == []
