"""What a refused extend leaves behind: the documented loop goes on without a host
synchronisation, so the append that follows has to leave every stored token alone."""
import pytest
import torch

pytestmark = pytest.mark.gpu

D, H, PAGE = 64, 2, 32


def filled(cuda, seed=0):
    """Three pages, all taken: slot 0 holds 40 tokens, slot 1 the same pages, slot 2 30 tokens."""
    from kvquant.paged_cache import PagedKVCache
    c = PagedKVCache(1, 3, H, max_slots=4, max_tokens=128, head_dim=D, page_tokens=PAGE, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(seed)
    c.tokens = lambda n: torch.randn((2, n, H, D), generator=g, device=cuda).half().unbind(0)
    for slot, n in ((0, 40), (2, 30)):
        c.extend([slot], n)
        c.append(0, *c.tokens(n), [slot])
        if slot == 0:
            c.fork([0], [1])
    c.check()
    return c


@pytest.mark.parametrize("slots,n,why", [([1], 1, "no free pages"), ([1], 5, "no free pages"),
                                         ([0, 9], 1, "a bad slot"), ([0, 0], 1, "a bad slot")])
def test_append_after_a_refused_extend_writes_nothing(cuda, slots, n, why):
    from kvquant.kernels.cuda_ops import get_cuda_ops
    c = filled(cuda)
    before = [x.clone() for x in (c.pool, c.table, c.lengths, c.refs)]
    c.extend(slots, n)
    c.append(0, *c.tokens(n), slots[:1])
    for x, y in zip((c.pool, c.table, c.lengths, c.refs), before):
        assert torch.equal(x, y)
    with pytest.raises(RuntimeError, match="out of range"):
        get_cuda_ops().check_status(cuda)
    with pytest.raises(RuntimeError, match=why):
        c.check()


def test_siblings_of_a_refused_extend_write_nothing(cuda):
    """Both holders of the shared open page in one call; one page is missing for them."""
    from kvquant.kernels.cuda_ops import get_cuda_ops
    c = filled(cuda)
    before = c.pool.clone()
    c.extend([0, 1], 1)
    c.append(0, *c.tokens(2), [0, 1])
    assert torch.equal(c.pool, before)
    with pytest.raises(RuntimeError, match="out of range"):
        get_cuda_ops().check_status(cuda)
    with pytest.raises(RuntimeError, match="no free pages"):
        c.check()


def test_a_granted_extend_after_a_refused_one(cuda):
    """Room is made, the extend granted: the tokens go where they would have gone without the
    refusal, and the slot that shares the page keeps its own."""
    from kvquant.kernels.cuda_ops import get_cuda_ops
    ends = []
    for refused in (True, False):
        c = filled(cuda)
        new = c.tokens(3)
        if refused:
            c.extend([1], 3)
            c.append(0, *new, [1])
            with pytest.raises(RuntimeError, match="no free pages"):
                c.check()
            with pytest.raises(RuntimeError, match="out of range"):
                get_cuda_ops().check_status(cuda)
        c.free([2])
        c.extend([1], 3)
        c.append(0, *new, [1])
        c.check()
        get_cuda_ops().check_status(cuda)
        ip = torch.tensor([0, 40, 83], dtype=torch.int32, device=cuda)
        ends.append(c.read(0, None, ip, 83, [0, 1], torch.float32))
    for x, y in zip(*ends):
        assert torch.equal(x, y)
        assert torch.equal(x[:32], x[40:72])  # the shared page
        assert torch.equal(x[:32], y[:32])


def test_append_only_where_extend_granted(cuda):
    """Rows before the slot's last grant, in a slot that was only forked, and without tokens."""
    from kvquant.kernels.cuda_ops import get_cuda_ops
    c = filled(cuda)
    before = c.pool.clone()
    c.extend([2], 1)
    for slot, n in ((1, 1), (2, 2), (3, 1)):
        c.append(0, *c.tokens(n), [slot])
        with pytest.raises(RuntimeError, match="out of range"):
            get_cuda_ops().check_status(cuda)
        assert torch.equal(c.pool, before)
    c.append(0, *c.tokens(1), [2])
    get_cuda_ops().check_status(cuda)
    assert not torch.equal(c.pool, before)
    c.check()


def test_example_without_steps(cuda):
    """The example with nothing but its prompts."""
    import sys
    from pathlib import Path
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
    import paged_sampling
    assert paged_sampling.main(["--steps", "0", "--samples", "2"]) < 0.02
