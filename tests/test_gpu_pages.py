"""A cache's pages against the same operations entry by entry: tables, references, lengths and
every byte of the pools equal."""
import pytest
import torch

from tests import _search_ref as R
from tilefoundry_amd._lib import TFDError
from tilefoundry_amd.pages import Pages

pytestmark = pytest.mark.gpu

BF, F32, I32 = torch.bfloat16, torch.float32, torch.int32


class Both:
    """A cache on the GPU and its definition on the CPU, compared after every call."""

    def __init__(self, dev, rows, max_pages, num_pages, shapes=((2, 16),), layers=2, seed=0):
        g = torch.Generator().manual_seed(seed)
        pools = [torch.randint(0, 100, (layers, num_pages, h, 16, d), generator=g).to(t)
                 for h, d in shapes for t in (BF, F32)]
        pools.append(torch.randint(0, 100, (num_pages, 1, 16, 16), generator=g).to(torch.uint8))
        self.dev = dev
        self.d = [p.to(dev) for p in pools]
        self.gpu = Pages(self.d, rows=rows, max_pages=max_pages)
        parts = [q for p in pools for q in (p.unbind(0) if p.dim() == 5 else [p])]
        self.pools = pools
        self.cpu = R.Cache(parts, torch.full((rows, max_pages), -1, dtype=I32),
                           torch.zeros(num_pages, dtype=I32))

    def call(self, name, *args):
        to = [a.to(self.dev) if isinstance(a, torch.Tensor) else a for a in args]
        got, want = getattr(self.gpu, name)(*to), getattr(self.cpu, name)(*args)
        if isinstance(want, torch.Tensor):
            assert torch.equal(got.cpu(), want)
        elif want is not None:
            assert got.item() == want
        self.same()
        return want

    def same(self):
        assert torch.equal(self.gpu.table.cpu(), self.cpu.table)
        assert torch.equal(self.gpu.refs.cpu(), self.cpu.refs)
        for a, b in zip(self.d, self.pools):
            assert torch.equal(a.cpu(), b)
        if self.cpu.failed:
            with pytest.raises(RuntimeError):
                self.gpu.check_errors()
            self.cpu.failed = False
        else:
            self.gpu.check_errors()


def ints(*v):
    return torch.tensor(v, dtype=I32)


def test_prompt_fork_and_writes(gpu_device):
    """A prompt in row 0, shared by all rows, which then write on their own."""
    b = Both(gpu_device, rows=4, max_pages=6, num_pages=20)
    zero = ints(0, 0, 0, 0)
    b.call("take", zero, ints(37, 0, 0, 0))
    lengths = b.call("fork", ints(0, 0, 0, 0), ints(37, 0, 0, 0))
    assert lengths.tolist() == [37] * 4
    b.call("take", lengths, 1)                       # three copies, the first row keeps the page
    assert int((b.cpu.refs == 4).sum()) == 2
    lengths = lengths + 11
    b.call("take", lengths, 1)                       # a new page each: 48 is a page's start
    b.call("fork", ints(2, 2, -1, 1), lengths)
    b.call("take", ints(48, 48, 0, 48), 1)
    b.call("free", torch.tensor([True, False, False, True]))
    live = b.call("compact")
    assert live == int((b.cpu.refs > 0).sum())


@pytest.mark.parametrize("rows,max_pages,num_pages,seed", [
    (1, 1, 1, 0), (3, 4, 9, 1), (8, 10, 60, 2), (33, 7, 150, 3), (64, 40, 1500, 4),
    (5, 300, 1400, 5)])
def test_random_walks(gpu_device, rows, max_pages, num_pages, seed):
    """Forks, writes, ends and compactions in turn, as a search makes them; some run out of pages
    or past the table."""
    b = Both(gpu_device, rows, max_pages, num_pages, seed=seed, layers=1)
    g = torch.Generator().manual_seed(seed + 100)
    lengths = torch.zeros(rows, dtype=I32)
    room = max_pages * 16
    for k in range(14):
        do = k % 7
        if do in (0, 3):
            n = torch.randint(-1, max(2, room // 3), (rows,), generator=g).to(I32)
            b.call("take", lengths, n)
            # rows that got no page are ended before they go on
            full = torch.tensor([any(int(p) < 0 for p in b.cpu.table[
                r, :-(-int(lengths[r] + max(int(n[r]), 0)) // 16)]) or
                int(lengths[r]) + int(n[r]) > room for r in range(rows)])
            lengths = torch.where(full, 0, lengths + n.clamp(min=0)).to(I32)
            b.call("free", full)
        elif do in (1, 5):
            parents = torch.randint(-1 if do == 5 else 0, rows, (rows,), generator=g).to(I32)
            lengths = b.call("fork", parents, lengths)
        elif do == 2:
            b.call("take", lengths, 1)
            full = torch.tensor([int(lengths[r]) >= room or
                                 int(b.cpu.table[r, min(int(lengths[r]) // 16, max_pages - 1)]) < 0
                                 for r in range(rows)])
            lengths = torch.where(full, 0, lengths + 1).to(I32)
            b.call("free", full)
        elif do == 4:
            which = torch.rand(rows, generator=g) < 0.4
            lengths = torch.where(which, 0, lengths).to(I32)
            b.call("free", which)
        else:
            b.call("compact")


def test_all_who_share_a_page_write(gpu_device):
    """The first row keeps it; with one that does not write, nobody does."""
    for writers in ([1, 1, 1], [1, 0, 1], [0, 0, 1], [0, 1, 1]):
        b = Both(gpu_device, rows=3, max_pages=3, num_pages=9)
        b.call("take", ints(0, 0, 0), ints(20, 0, 0))
        lengths = b.call("fork", ints(0, 0, 0), ints(20, 0, 0))
        b.call("take", lengths, torch.tensor(writers, dtype=I32) * 13)


def test_take_of_many_positions(gpu_device):
    """More entries than the threads of the block that decides."""
    b = Both(gpu_device, rows=20, max_pages=130, num_pages=5000, layers=1, shapes=((1, 16),))
    b.call("take", torch.zeros(20, dtype=I32), 2071)
    lengths = b.call("fork", torch.arange(20, dtype=I32) // 2 * 2,
                     torch.full((20,), 2071, dtype=I32))
    b.call("take", torch.full((20,), 100, dtype=I32), 1900)   # into shared pages, from 100 on
    assert lengths.tolist() == [2071] * 20


def test_too_few_pages(gpu_device):
    b = Both(gpu_device, rows=3, max_pages=4, num_pages=5)
    b.call("take", ints(0, 0, 0), ints(40, 40, 10))
    assert b.cpu.table[1].tolist()[:3] == [3, 4, -1] and b.cpu.table[2, 0] == -1
    b.call("free", torch.tensor([True, False, False]))
    b.call("take", ints(0, 32, 0), ints(0, 8, 10))


def test_what_is_out_of_range(gpu_device):
    b = Both(gpu_device, rows=3, max_pages=4, num_pages=12)
    b.call("take", ints(0, 0, 0), ints(30, 5, 17))
    b.call("fork", ints(1, 3, -2), ints(30, 5, 17))
    b.call("take", ints(5, -1, 60), ints(5, 5, 5))
    b.cpu.table[0, 1] = 99
    b.gpu.table[0, 1] = 99
    b.call("take", ints(16, 0, 0), 1)


@pytest.mark.parametrize("rows,nodes,heads,dim,seed", [
    (1, 1, 1, 16, 0), (4, 6, 2, 16, 1), (3, 33, 8, 128, 2), (2, 256, 3, 64, 3)])
def test_keep(gpu_device, rows, nodes, heads, dim, seed):
    g = torch.Generator().manual_seed(seed)
    room = 3 + (nodes + 40) // 16
    b = Both(gpu_device, rows, room, rows * room + 2, shapes=((heads, dim),), seed=seed)
    lengths = torch.randint(0, 40, (rows,), generator=g).to(I32)
    b.call("take", torch.zeros(rows, dtype=I32), lengths + nodes)
    path = torch.full((rows, nodes), -1, dtype=I32)
    counts = torch.zeros(rows, dtype=I32)
    for r in range(rows):
        n = int(torch.randint(0, nodes + 1, (), generator=g)) if r else nodes - nodes // 3
        way = torch.sort(torch.randperm(nodes, generator=g)[:n]).values
        path[r, :n], counts[r] = way.to(I32), n
    out = b.call("keep", lengths, path, counts)
    assert torch.equal(out, lengths + counts)


def test_keep_refuses_bad_paths(gpu_device):
    b = Both(gpu_device, 6, 3, 20)
    b.call("take", torch.zeros(6, dtype=I32), 40)
    path = torch.tensor([[0, 2, 1], [0, 1, 3], [-1, 1, 2], [1, 1, 2], [0, 2, -1], [0, 1, 2]],
                        dtype=I32)
    out = b.call("keep", ints(5, 5, 5, 5, 5, 46), path, ints(3, 3, 3, 3, 4, 3))
    assert out.tolist() == [5, 5, 5, 5, 5, 46]
    out = b.call("keep", ints(5, 5, 5, 5, 5, 5), path, ints(2, 2, 0, 1, 2, -1))
    assert out.tolist() == [7, 7, 5, 6, 7, 5]


def test_copy(gpu_device):
    b = Both(gpu_device, 1, 1, 12, shapes=((3, 16), (1, 2048)))
    src, dst = ints(3, 0, 7, 3), ints(1, 2, 5, 11)
    b.gpu.copy(src.to(gpu_device), dst.to(gpu_device))
    for p in b.cpu.pools:
        p[dst.long()] = p[src.long()]
    b.same()
    b.gpu.copy(ints(3, 12).to(gpu_device), ints(1, 2).to(gpu_device))
    b.cpu.failed = True
    for p in b.cpu.pools:
        p[1] = p[3]
    b.same()
    b.gpu.copy(ints().to(gpu_device), ints().to(gpu_device))
    b.same()


def test_table_and_refs_of_ones_own(gpu_device):
    pool = torch.zeros(6, 1, 16, 8, dtype=BF, device=gpu_device)
    table = torch.tensor([[0, 3, -1], [0, 1, 1]], dtype=I32, device=gpu_device)
    p = Pages([pool], table=table)
    assert p.refs.tolist() == [2, 2, 0, 1, 0, 0] and p.table is table
    p.free(torch.tensor([False, True], device=gpu_device))
    assert p.refs.tolist() == [1, 0, 0, 1, 0, 0] and table.tolist() == [[0, 3, -1], [-1] * 3]


def test_calls_in_a_graph(gpu_device):
    """A search's page work captured once and replayed beside the same calls made one by one."""
    rows = 4
    a, b = (Both(gpu_device, rows, 8, 40, seed=7) for _ in range(2))
    start = torch.full((rows,), 21, dtype=I32)
    for c in (a, b):
        c.call("take", torch.zeros(rows, dtype=I32), 21)
    lengths, parents = start.to(gpu_device), torch.arange(rows, dtype=I32, device=gpu_device)

    def step():
        new = a.gpu.fork(parents, lengths)
        a.gpu.take(new, 1)
        lengths.copy_(new + 1)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    g = torch.Generator().manual_seed(1)
    for _ in range(30):
        p = torch.randint(0, rows, (rows,), generator=g).to(I32)
        parents.copy_(p)
        graph.replay()
        torch.cuda.synchronize()
        start = b.call("fork", p, start)
        b.call("take", start, 1)
        start = start + 1
        assert torch.equal(lengths.cpu(), start)
        assert torch.equal(a.gpu.table, b.gpu.table) and torch.equal(a.gpu.refs, b.gpu.refs)
        for x, y in zip(a.d, b.d):
            assert torch.equal(x, y)
    a.gpu.check_errors()


def test_copy_of_no_page_is_reported(gpu_device):
    """-1 names no page, as any other number outside the pool: the others are copied."""
    for src, dst in (((-1, 3), (2, 1)), ((0, 3), (-1, 1)), ((-7, 3), (2, 1))):
        b = Both(gpu_device, 1, 1, 12)
        b.gpu.copy(ints(*src).to(gpu_device), ints(*dst).to(gpu_device))
        b.cpu.failed = True
        for p in b.cpu.pools:
            p[1] = p[3]
        b.same()


def test_refused_copies_leave_everything_as_it_was(gpu_device):
    """Pages too large to be copied in one call are refused before anything is decided; the calls
    after that are as ever."""
    b = Both(gpu_device, rows=3, max_pages=3, num_pages=9)
    b.call("take", ints(0, 0, 0), ints(20, 0, 18))
    lengths = b.call("fork", ints(0, 0, 2), ints(20, 0, 18))
    b.call("free", torch.tensor([True, False, False]))
    size, scratch = b.gpu._args.max_page_bytes, b.gpu._scratch.clone()
    b.gpu._args.max_page_bytes = 1 << 50
    for call in (lambda: b.gpu.take(lengths.to(gpu_device), 1), b.gpu.compact,
                 lambda: b.gpu.copy(ints(1).to(gpu_device), ints(8).to(gpu_device))):
        with pytest.raises(TFDError, match="copies"):
            call()
        b.same()
        assert torch.equal(b.gpu._scratch, scratch)
    b.gpu._args.max_page_bytes = size
    b.call("compact")
    b.call("take", lengths, 1)
