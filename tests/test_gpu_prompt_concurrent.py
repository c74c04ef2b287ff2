"""Prompt attention and linear_s8 from several threads, on streams of their own and on one, beside replays of graphs that hold the same calls."""
import threading

import pytest
import torch

import my_own_cnn_b200 as b2q

pytestmark = pytest.mark.gpu


def starts_of(*lens):
    return torch.tensor([0, *lens]).cumsum(0).to(torch.int32).cuda()


def work(seed, dtype, many):
    """Calls of one kind: keys in parts, whole prompts, a split product, a product on pairs of SMs."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(dtype)

    q, k, v = normal(20, 4, 64), normal(6000, 2, 64), normal(6000, 2, 64)
    few, ends = (starts_of(12, 8), starts_of(3500, 2500)), starts_of(500, 400)
    x = normal(900, 24, 128)
    rows, weight = b2q.quantize_s8(normal(2300 if many else 5, 512)), b2q.quantize_s8(normal(2600, 512))
    return [lambda s=None: b2q.prompt_attention(q, k, v, *few, stream=s),
            lambda s=None: b2q.prompt_attention(x[:, :16], x[:, 16:20], x[:, 20:], ends, stream=s),
            lambda s=None: b2q.linear_s8(rows, weight, dtype=dtype, stream=s)]


@pytest.mark.parametrize("shared", [False, True])
def test_threads_and_graphs(cuda_lib, shared):
    kinds = [work(i, t, bool(i % 2)) for i, t in enumerate((torch.float32, torch.float16, torch.bfloat16, torch.bfloat16))]
    want = [[call().clone() for call in calls] for calls in kinds]
    torch.cuda.synchronize()
    one = torch.cuda.Stream()
    streams = [one if shared else torch.cuda.Stream() for _ in kinds]
    graphs = []
    for calls in kinds[:2]:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        for call in calls:
            call(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = [call(side) for call in calls]
        graphs.append((graph, held))
    wrong = []

    def run(i):
        for _ in range(15):
            outs = [call(streams[i]) for call in kinds[i]]
            streams[i].synchronize()
            wrong.extend((i, j) for j, (a, b) in enumerate(zip(outs, want[i])) if not torch.equal(a, b))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(kinds))]
    for t in threads:
        t.start()
    for _ in range(15):
        for i, (graph, held) in enumerate(graphs):
            graph.replay()
            torch.cuda.current_stream().synchronize()
            wrong.extend(("graph", i, j) for j, (a, b) in enumerate(zip(held, want[i])) if not torch.equal(a, b))
    for t in threads:
        t.join()
    assert wrong == []
    b2q.device_error()
