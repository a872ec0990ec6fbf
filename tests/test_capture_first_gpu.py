"""A call whose shape is met for the first time while a graph is captured: what the host keeps for
that shape must be good for eager calls too, which nothing has replayed yet."""

import pytest
import torch

import attention_b200 as spa

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_contiguous_decode_with_weights():
    gen = torch.Generator(device=DEV).manual_seed(0)
    batch, length, dim = 3, 157, 64
    q = torch.randn(batch, 4, dim, generator=gen, device=DEV)
    k, v = (torch.randn(batch, 2, length, dim, generator=gen, device=DEV) for _ in range(2))
    w = torch.zeros(batch, 2, length, device=DEV)
    warm = torch.zeros(1, 2, 40, device=DEV)  # another shape: nothing is loaded during the capture
    spa.paged_decode_attention(q[:1], k[:1, :, :40].contiguous(), v[:1, :, :40].contiguous(), weights=warm)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = spa.paged_decode_attention(q, k, v, weights=w)
    eager_w = torch.zeros_like(w)
    eager = spa.paged_decode_attention(q, k, v, weights=eager_w)
    s = (q.double().view(batch, 2, 2, dim) @ k.double().transpose(2, 3)) / dim ** 0.5
    p = torch.softmax(s, -1)
    want = (p @ v.double()).flatten(1, 2)
    # fp32 scores below 2^6 (Q), 72 roundings; |v| < 6
    rel = 2 * 72 * 2.0 ** -24 * 2 ** 6
    assert ((eager.double() - want).abs() <= 6 * rel).all()
    assert ((eager_w.double() - p.sum(2)).abs() <= rel * p.sum(2) + 2.0 ** -23).all()
    graph.replay()
    assert torch.equal(captured, eager) and torch.equal(w, eager_w)
    assert spa.device_error_flags() == 0


def test_contiguous_decode_and_step():
    """The calls without weights keep the lengths of a contiguous cache, and the step its arguments."""
    gen = torch.Generator(device=DEV).manual_seed(1)
    batch, heads, dim, page, window = 2, 4, 64, 16, 32
    length = 32 + 16 * 9
    q = torch.randn(batch, heads, dim, generator=gen, device=DEV).bfloat16()
    k, v = (torch.randn(batch, heads, length, dim, generator=gen, device=DEV).bfloat16() for _ in range(2))
    summaries = torch.randn(batch, heads, 9, dim, generator=gen, device=DEV)

    def calls(n):
        kn, vn = k[:n], v[:n]
        return (spa.paged_decode_attention(q[:n], kn, vn),
                *spa.sparse_decode_step(q[:n], kn, vn, summaries[:n], top_blocks=3, local_window=window, block_size=page))

    calls(1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = calls(2)
    eager = [t.clone() for t in calls(2)]
    one = [calls(1)]
    graph.replay()
    for a, b, c in zip(captured, eager, one[0]):
        assert torch.equal(a, b) and torch.equal(b[:1], c)
    s = (q.double()[:, :, None] @ k.double().transpose(2, 3)) / dim ** 0.5
    want = (torch.softmax(s, -1) @ v.double())[:, :, 0]
    # bf16 probabilities and output: 2^-8 each of values below 6
    assert ((eager[0].double() - want).abs() <= 2 * 6 * 2.0 ** -8).all()
    assert spa.device_error_flags() == 0


@pytest.mark.parametrize("what", ["decode", "step"])
def test_graphs_replayed_side_by_side(what):
    """Two graphs captured on one stream, after eager calls on it, give what they give alone while they
    run at the same time on two streams, beside eager calls: their partial results lie apart."""
    gen = torch.Generator(device=DEV).manual_seed(2)
    heads, dim, page, pages = 2, 128, 256, 64

    def inputs():
        k, v = (torch.randn(pages, heads, page, dim, generator=gen, device=DEV).bfloat16() for _ in range(2))
        return (torch.randn(1, 8, dim, generator=gen, device=DEV).bfloat16(), k, v,
                torch.randn(1, heads, pages, dim, generator=gen, device=DEV),
                dict(page_table=torch.randperm(pages, generator=gen, device=DEV).int()[None],
                     context_lens=torch.tensor([pages * page], dtype=torch.int32, device=DEV)))

    def call(x):
        q, k, v, summaries, more = x
        if what == "decode":
            return spa.paged_decode_attention(q, k, v, **more)
        return spa.sparse_decode_step(q, k, v, summaries, top_blocks=24, local_window=page, block_size=page, **more)[0]

    sets = [inputs() for _ in range(3)]
    stream, streams, graphs = torch.cuda.Stream(), [torch.cuda.Stream() for _ in range(2)], []
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        want = [call(x).clone() for x in sets]
    torch.cuda.synchronize()
    for x in sets[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            out = [call(x) for _ in range(20)]
        graphs.append((g, out))
    torch.cuda.synchronize()
    for _ in range(10):
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(stream):
            eager = [call(sets[2]) for _ in range(20)]
        torch.cuda.synchronize()
        for (_, outs), w in zip(graphs, want):
            assert all(torch.equal(o, w) for o in outs)
        assert all(torch.equal(o, want[2]) for o in eager)
    assert spa.device_error_flags() == 0
