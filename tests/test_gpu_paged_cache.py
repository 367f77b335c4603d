"""Append, read and the page operations of the paged 8-bit cache: equal to the oracle
byte for byte (the codes' arithmetic is fixed; the page operations are whole numbers)."""
import numpy as np
import pytest
import torch

from oracle import paged_oracle as PO
from paged_cases import DT, Cache, make_tokens, rounded

pytestmark = pytest.mark.gpu


def t(x, dev):
    return torch.from_numpy(np.ascontiguousarray(x)).to(dev)


def append_step(cuda, c, state, new, slots=None, indptr=True, xs=None, strided=False):
    """Appends `new` tokens to the slots on the GPU and in the oracle; lengths grow first."""
    from kvquant.kernels import paged_append
    from kvquant.kernels.cuda_ops import get_cuda_ops
    pool, table = state
    order = list(range(len(c.lens))) if slots is None else slots
    xs = xs or [make_tokens(c.rng, m, c.H, c.D) for m in new]
    xs = [(rounded(k, c.dtype), rounded(v, c.dtype)) for k, v in xs]
    for s, m, (k, v) in zip(order, new, xs):
        c.lengths[s] += m
        PO.append(c.pool, c.table, s, int(c.lengths[s]), k, v, c.kind)
    k, v = (t(np.concatenate(x), cuda).to(DT[c.dtype]) for x in zip(*xs))
    if strided:
        both = torch.zeros((k.shape[0], 3 * c.H, c.D), dtype=k.dtype, device=cuda)
        both[:, c.H:2 * c.H], both[:, 2 * c.H:] = k, v
        k, v = both[:, c.H:2 * c.H], both[:, 2 * c.H:]
    ip = t(np.concatenate([[0], np.cumsum(new)]).astype(np.int32), cuda) if indptr else None
    sl = None if slots is None else torch.tensor(slots, dtype=torch.int32, device=cuda)
    paged_append(k, v, pool, table, t(c.lengths, cuda), c.kind, slots=sl, indptr=ip)
    get_cuda_ops().check_status(cuda)


def roomy(lens, grow, **kw):
    """A cache whose slots have pages for `grow` more tokens."""
    c = Cache([n + grow for n in lens], fill=False, **kw)
    c.lens = lens
    c.lengths = np.zeros(len(lens), np.int32)
    return c


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 48), (128, 64)])
def test_append_in_steps(cuda, kind, dtype, D, page):
    """Prompts, then single tokens and runs across block and page ends; every byte of
    every touched record, scales and zero places included."""
    c = roomy([0] * 5, 200, H=3, D=D, page=page, kind=kind, dtype=dtype, seed=D + page)
    state = t(c.pool, cuda), t(c.table, cuda)
    for new in ([1, 16, 17, 0, 100], [1] * 5, [15, 1, 31, 3, 0], [40, 2, 1, 16, 33], [1] * 5):
        append_step(cuda, c, state, new, strided=new[0] == 15)
        np.testing.assert_array_equal(state[0].cpu().numpy(), c.pool)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_append_growing_scales(cuda, kind):
    """Each token twice as large as the one before: every append restates the block."""
    c = roomy([0, 0], 40, H=2, kind=kind, seed=3)
    state = t(c.pool, cuda), t(c.table, cuda)
    for i in range(20):
        xs = [tuple(x * np.float32(2.0 ** (i % 12) if b else 2.0 ** -(i % 12))
                    for x in make_tokens(c.rng, 1, 2, 128)) for b in range(2)]
        append_step(cuda, c, state, [1, 1], indptr=False, xs=xs)
    np.testing.assert_array_equal(state[0].cpu().numpy(), c.pool)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_append_special_values(cuda, kind, dtype):
    """Zeros, subnormals, the largest numbers, infinities and NaN; blocks of nothing else."""
    c = roomy([0] * 6, 64, H=1, kind=kind, dtype=dtype, seed=5)
    state = t(c.pool, cuda), t(c.table, cuda)
    big = 65504.0 if dtype == "fp16" else 3e38
    xs = [tuple(x.copy() for x in make_tokens(c.rng, 20, 1, 128)) for _ in range(6)]
    for k, v in xs:
        k[3, 0, 5], k[4, 0, 6], v[3, 0, 7] = np.inf, -np.inf, np.nan
    xs[1][0][:], xs[1][1][:] = 0, np.nan
    xs[2][0][:], xs[2][1][:] = np.inf, -0.0
    xs[3] = tuple(np.full_like(x, 6e-8) * np.sign(x) for x in xs[3])
    xs[4] = tuple(np.full_like(x, big) * np.sign(x) for x in xs[4])
    xs[5][0][:, :, 0] = big
    append_step(cuda, c, state, [20] * 6, xs=xs)
    np.testing.assert_array_equal(state[0].cpu().numpy(), c.pool)
    append_step(cuda, c, state, [1] * 6)
    np.testing.assert_array_equal(state[0].cpu().numpy(), c.pool)


def test_append_slots_and_many_sequences(cuda):
    c = roomy([0] * 70, 20, H=1, D=64, page=16, seed=6)
    state = t(c.pool, cuda), t(c.table, cuda)
    slots = list(c.rng.permutation(70)[:61])
    append_step(cuda, c, state, [int(x) for x in c.rng.integers(0, 20, 61)], slots=slots)
    np.testing.assert_array_equal(state[0].cpu().numpy(), c.pool)


def test_append_bad_indices_touch_nothing(cuda):
    from kvquant.kernels import paged_append
    from kvquant.kernels.cuda_ops import get_cuda_ops
    ops = get_cuda_ops()
    c = Cache([20, 30], seed=7)
    k = torch.zeros((2, 2, 128), dtype=torch.float16, device=cuda)
    for what in ("page", "length", "slot", "rows", "more rows than tokens"):
        pool, table, lengths = c.gpu(cuda)
        slots, ip = None, torch.tensor([0, 1, 1], dtype=torch.int32, device=cuda)
        if what == "page":
            table[0, 0] = -5
        elif what == "length":
            lengths[0] = 10 ** 6
        elif what == "slot":
            slots = torch.tensor([-1, 1], dtype=torch.int32, device=cuda)
        elif what == "rows":
            ip = torch.tensor([0, 3, 3], dtype=torch.int32, device=cuda)
        else:
            lengths[0] = 0
        paged_append(k, k, pool, table, lengths, "int8", slots=slots, indptr=ip)
        with pytest.raises(RuntimeError, match="out of range"):
            ops.check_status(cuda)
        assert np.array_equal(pool.cpu().numpy(), c.pool), what


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
def test_read(cuda, kind, dtype, D):
    from kvquant.kernels import paged_read
    c = Cache([0, 5, 100, 64, 33], H=3, D=D, kind=kind, seed=D)
    pool, table, lengths = c.gpu(cuda)
    slots, starts, rows = [2, 1, 4, 3, 0], [17, 0, 32, 15, 0], [70, 5, 1, 33, 0]
    ip = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    k, v = paged_read(pool, table, lengths, kind, t(np.int32(starts), cuda), t(ip, cuda), sum(rows),
                      slots=t(np.int32(slots), cuda), dtype=dtype)
    for b, s in enumerate(slots):
        for h in range(3):
            ek, ev, _ = PO.token_values(c.pool, c.table, s, starts[b] + rows[b], h, D, kind)
            for got, e in ((k, ek), (v, ev)):
                want = torch.from_numpy(e[starts[b]:].astype(np.float32)).to(dtype)
                assert torch.equal(got[ip[b]:ip[b + 1], h].cpu(), want)


def test_read_beyond_the_length_is_reported(cuda):
    from kvquant.kernels import paged_read
    from kvquant.kernels.cuda_ops import get_cuda_ops
    c = Cache([20], seed=1)
    pool, table, lengths = c.gpu(cuda)
    paged_read(pool, table, lengths, "int8", t(np.int32([10]), cuda), None, 11)
    with pytest.raises(RuntimeError, match="out of range"):
        get_cuda_ops().check_status(cuda)


# ---------------------------------------------------------------- page operations
class Both:
    """The same operations on the GPU and in the oracle, compared after each."""

    def __init__(self, cuda, lens, page=32, spare=40, extra_cols=4, layers=2, seed=0, empty=0):
        c = Cache(lens + [0] * empty, H=2, D=64, page=page, spare=spare, extra_cols=extra_cols,
                  fill=False, seed=seed)
        pool = c.rng.integers(0, 256, (layers,) + c.pool.shape, dtype=np.uint8)
        self.o = PO.Pages(c.table, c.lengths, c.refs, page, pool)
        self.pool, self.table, self.lengths, self.refs = (
            t(x, cuda) for x in (pool, c.table, c.lengths, c.refs))
        self.status = torch.zeros(1, dtype=torch.int32, device=cuda)
        self.page, self.dev = page, cuda

    def ints(self, x):
        return torch.tensor(x, dtype=torch.int32, device=self.dev)

    def check(self):
        np.testing.assert_array_equal(self.table.cpu().numpy(), self.o.table)
        np.testing.assert_array_equal(self.lengths.cpu().numpy(), self.o.lengths)
        np.testing.assert_array_equal(self.refs.cpu().numpy(), self.o.refs)
        np.testing.assert_array_equal(self.pool.cpu().numpy(), self.o.pool)
        assert int(self.status.item()) == self.o.status

    def free(self, slots):
        from kvquant.kernels import paged_free
        self.o.free(slots)
        paged_free(self.table, self.lengths, self.refs, self.ints(slots), self.page, self.status)
        self.check()

    def fork(self, src, dst):
        from kvquant.kernels import paged_fork
        self.o.fork(src, dst)
        paged_fork(self.table, self.lengths, self.refs, self.ints(src), self.ints(dst), self.page,
                   self.status)
        self.check()

    def extend(self, slots, n_new):
        from kvquant.kernels import paged_extend
        each = isinstance(n_new, list)
        self.o.extend(slots, n_new if each else [n_new] * len(slots))
        paged_extend(self.pool, self.table, self.lengths, self.refs, self.ints(slots),
                     self.ints(n_new) if each else n_new, self.status)
        self.check()

    def compact(self):
        from kvquant.kernels import paged_compact
        n = self.o.compact()
        assert int(paged_compact(self.pool, self.table, self.refs).item()) == n
        self.check()


def test_fork_extend_free_compact(cuda):
    b = Both(cuda, [0, 1, 31, 32, 33, 100], empty=8)
    b.fork([5, 5, 4, 0, 2, 1], [6, 7, 8, 9, 10, 11])
    b.extend([7, 5, 6], 1)               # all holders: the last one keeps the page
    b.extend([8, 12, 9, 2], [40, 70, 0, 1])
    b.free([5, 4, 0])
    b.compact()
    b.fork([6], [5])
    b.extend([5, 6, 3], [1, 32, 33])
    b.free([13, 7])
    b.compact()
    b.compact()                          # nothing left to move


def test_extend_single_holder_writes_in_place(cuda):
    b = Both(cuda, [20, 40])
    before = b.table.clone()
    b.extend([0, 1], 1)
    assert torch.equal(before, b.table)


def test_extend_is_all_or_nothing(cuda):
    b = Both(cuda, [20, 40, 5], spare=2, extra_cols=4)
    b.extend([0, 1], [50, 60])           # needs four pages, two are free
    assert b.o.status == 1
    b.extend([0, 1], [12, 24])
    b.extend([0, 0], 1)                  # named twice
    b.extend([0, 3], 1)                  # out of range
    b.extend([2], 10 ** 6)               # longer than a row of the table
    b.extend([2, 1], [1, -1])
    assert b.o.status == 3


def test_bad_slots_of_fork_and_free(cuda):
    b = Both(cuda, [20, 40, 5], empty=3)
    b.fork([0, 0, 1, 9, 2], [3, 3, 2, 4, -1])  # twice, holds tokens, no such slots
    b.fork([4, 0], [5, 4])                     # a src that is also a dst
    b.free([1, 1, 7, -2, 5])


@pytest.mark.parametrize("n,page", [(1, 16), (37, 64), (1500, 16)])
def test_many_slots(cuda, n, page):
    """More slots than threads of the planning block; lists longer than one scan."""
    rng = np.random.default_rng(n)
    lens = [int(x) for x in rng.integers(0, 3 * page, n)]
    b = Both(cuda, lens, page=page, spare=4 * n + 8, empty=n, layers=1, seed=n)
    b.fork(list(range(n)), list(range(n, 2 * n)))
    b.extend([int(s) for s in rng.permutation(2 * n)], [int(x) for x in rng.integers(0, page + 2, 2 * n)])
    b.free([int(s) for s in rng.permutation(2 * n)[:n]])
    b.compact()


def test_everything_live_and_nothing_live(cuda):
    b = Both(cuda, [64, 33], spare=0)
    b.compact()
    b.free([0, 1])
    b.compact()


def test_copy_between_pools(cuda):
    from kvquant.kernels import paged_copy
    from kvquant.kernels.cuda_ops import get_cuda_ops
    rng = np.random.default_rng(0)
    a = rng.integers(0, 256, (3, 11, 5, 3, 32 * 64 + 16), dtype=np.uint8)
    b = rng.integers(0, 256, (3, 7, 5, 3, 32 * 64 + 16), dtype=np.uint8)
    ga, gb = t(a, cuda), t(b, cuda)
    src, dst = [10, 0, 3, 3], [1, 6, 0, 2]
    paged_copy(ga, gb, t(np.int32(src), cuda), t(np.int32(dst), cuda))
    b[:, dst] = a[:, src]
    np.testing.assert_array_equal(gb.cpu().numpy(), b)
    paged_copy(ga, ga, t(np.int32([1, 2]), cuda), t(np.int32([9, 8]), cuda))
    a[:, [9, 8]] = a[:, [1, 2]]
    np.testing.assert_array_equal(ga.cpu().numpy(), a)
    paged_copy(ga, gb, t(np.int32([11, 2]), cuda), t(np.int32([3, 4]), cuda))
    with pytest.raises(RuntimeError, match="out of range"):
        get_cuda_ops().check_status(cuda)
    b[:, 4] = a[:, 2]
    np.testing.assert_array_equal(gb.cpu().numpy(), b)
