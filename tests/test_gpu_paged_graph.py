"""Captured calls of PagedKVCache beside later, larger calls that are not captured."""
import pytest
import torch

pytestmark = pytest.mark.gpu

D, H, G = 128, 2, 4


def cache_of(cuda, n):
    from kvquant.paged_cache import PagedKVCache
    c = PagedKVCache(1, 64, H, max_slots=2, max_tokens=1024, head_dim=D, page_tokens=32, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(5)
    c.randn = lambda *s: torch.randn(s, generator=g, device=cuda).half()
    c.extend([0], n)
    c.append(0, c.randn(n, H, D), c.randn(n, H, D), [0])
    return c


def test_larger_calls_keep_the_workspace(cuda):
    """A captured call holds the workspace's address: no later call may replace the buffer."""
    c = cache_of(cuda, 600)
    slots = torch.zeros(1, dtype=torch.int32, device=cuda)
    c.attend(0, c.randn(1, H * G, D), slots)
    at = c.workspace.buf.data_ptr()
    c.attend(0, c.randn(300, H * G, D), slots)
    c.attend(0, c.randn(12, H, D), slots)
    c.compact()
    c.extend([1], 40)
    assert c.workspace.buf.data_ptr() == at


def test_replay_after_larger_calls(cuda):
    c = cache_of(cuda, 600)
    slots = torch.zeros(1, dtype=torch.int32, device=cuda)
    q = c.randn(1, H * G, D)
    want = c.attend(0, q, slots)
    out = torch.empty_like(want)
    stream = torch.cuda.Stream(cuda)
    stream.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(stream):
        c.attend(0, q, slots, out=out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            c.attend(0, q, slots, out=out)
    torch.cuda.current_stream(cuda).wait_stream(stream)
    c.attend(0, c.randn(300, H * G, D), slots)
    held = [torch.full((5 << 20,), 7, dtype=torch.int32, device=cuda) for _ in range(4)]
    out.zero_()
    for _ in range(3):
        graph.replay()
    assert torch.equal(out, want)
    assert all(bool((x == 7).all()) for x in held)
