"""Pages handed out on the GPU against the host's own way (KVTileCache.register_range) and a list in Python: whole numbers, equal."""
import numpy as np
import pytest
import torch


class Host:
    """The free list and the table as the definition has them."""

    def __init__(self, beams, heads, tiles, tile, free):
        self.table = np.full((beams, heads, tiles), -1, dtype=np.int64)
        self.held, self.tile, self.free = [0] * beams, tile, list(free)

    def take(self, lengths, sizes):
        ends = [max(h, -(-(n + m) // self.tile)) for h, n, m in zip(self.held, lengths, sizes)]
        B, H, T = self.table.shape
        fits = all(e <= T for e in ends) and sum(e - h for e, h in zip(ends, self.held)) * H <= len(self.free)
        if fits:
            for b, e in enumerate(ends):
                for t in range(self.held[b], e):
                    for h in range(H):
                        self.table[b, h, t] = self.free.pop()
                self.held[b] = e
        seq = [b for b, m in enumerate(sizes) for _ in range(m)]
        pos = [n + i for n, m in zip(lengths, sizes) for i in range(m)]
        page = [[self.table[b, h, p // self.tile] if p // self.tile < T else -1 for h in range(H)] for b, p in zip(seq, pos)]
        return seq, pos, [[-1 if x < 0 else x * self.tile + p % self.tile for x in row] for row, p in zip(page, pos)]

    def release(self, lengths):
        for b in reversed(range(len(lengths))):
            keep = min(self.held[b], -(-lengths[b] // self.tile))
            for t in reversed(range(keep, self.held[b])):
                for h in reversed(range(self.table.shape[1])):
                    self.free.append(self.table[b, h, t])
                    self.table[b, h, t] = -1
            self.held[b] = keep

    def same(self, pages):
        return np.array_equal(pages.table.device_data().cpu().numpy().reshape(self.table.shape), self.table) and pages.free_pages() == len(self.free) and \
            pages._free[:len(self.free)].tolist() == [int(x) for x in self.free] and pages._held.tolist() == self.held


def start_of(sizes):
    return torch.tensor(np.concatenate([[0], np.cumsum(sizes)]), dtype=torch.int32, device="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("seed,beams,heads,tiles,tile,most", [(0, 1, 1, 8, 16, 9), (1, 5, 3, 9, 16, 40), (2, 700, 2, 6, 4, 5), (3, 16, 12, 70, 32, 1000), (4, 3, 1, 4000, 1, 1500),
                                                              (5, 2, 32, 600, 16, 4000)])
def test_against_a_list(seed, beams, heads, tiles, tile, most):
    import llm_decoder as ld
    rng = np.random.default_rng(seed)
    total = max(heads, int(beams * heads * tiles * 0.8))
    free = rng.permutation(total)
    pt = ld.PageTable()
    pt.init(beams, heads, tiles)
    pages, host = ld.DevicePages(pt, total, tile, free=free.tolist()), Host(beams, heads, tiles, tile, free)
    refused = 0
    lengths = [0] * beams
    for step in range(12):
        B = beams if step % 3 else int(rng.integers(1, beams + 1))
        sizes = [0 if rng.random() < 0.3 else int(rng.integers(0, most + 1)) for _ in range(B)]
        before = sum(host.held)
        seq, pos, slots = host.take(lengths[:B], sizes)
        refused += sum(host.held) == before and any(-(-(n + m) // tile) > h for n, m, h in zip(lengths, sizes, host.held))
        new = pages.take(lengths[:B], start_of(sizes), sum(sizes))
        assert new.row_seq.tolist() == seq and new.positions.tolist() == pos and new.slots.tolist() == slots and host.same(pages), step
        lengths[:B] = [n + int(rng.integers(0, m + 1)) if -(-(n + m) // tile) <= tiles and rng.random() < 0.8 else int(rng.integers(0, n + 1)) for n, m in zip(lengths, sizes)]
        host.release(lengths)
        pages.release(torch.tensor(lengths, dtype=torch.int32, device="cuda"))
        assert host.same(pages), step
    if refused:
        with pytest.raises(RuntimeError):
            pages.check()
    pages.check()


@pytest.mark.gpu
def test_taken_pages_are_those_of_the_host(tmp_path):
    """A cache whose pages the host has handed out so far goes on on the GPU, in the same order, and back."""
    import llm_decoder as ld

    def cache():
        kv = ld.KVTileCache("f16")
        kv.init(60, 16, 64)
        kv.configure_table(3, 2, 10)
        kv.register_range(0, 0, 3)
        kv.register_range(2, 0, 1)
        return kv
    a, b = cache(), cache()
    pages = a.pages_on_device()
    pages.take([40, 0, 16], start_of([30, 20, 1]), 51)
    b.register_range(0, 3, 5)
    b.register_range(1, 0, 2)
    b.register_range(2, 1, 2)
    assert torch.equal(a.page_table_.device_data(), b.page_table_.device_data())
    for call in (lambda: a.register_tile(0, 0, 9), lambda: a.register_range(0, 9, 10), lambda: a.release_beam(0), lambda: a.fork_beam(0, 1), lambda: a.free_pages(),
                 lambda: a.append_cow(None, None, [0]), lambda: a.save_tiles_cpu_format(str(tmp_path / "x")), lambda: a.page_table_.assign(0, 0, 0, 1),
                 lambda: a.page_table_.remove(0, 0, 0), lambda: a.page_table_.lookup(0, 0, 0), lambda: a.sync_page_table_to_gpu(),
                 lambda: a.page_table_.load_host_table(np.zeros(60)), lambda: a.page_table_.assign_many([0], [1]), lambda: a.pages_on_device()):
        with pytest.raises(RuntimeError):
            call()
    pages.release([40, 20, 16])
    pages.to_host()
    with pytest.raises(RuntimeError):
        pages.take([0], start_of([1]), 1)
    assert a.free_pages() == 60 - 2 * (3 + 2 + 1) and a.page_table_.lookup(1, 1, 1) == b.page_table_.lookup(1, 1, 1)
    assert a.release_beam(1) == 4 and a.free_pages() == 60 - 2 * 4
    assert a.register_tile(1, 0, 0) not in [a.page_table_.lookup(r, h, t) for r, h, t in ((0, 0, 0), (0, 1, 2), (2, 0, 0))]


@pytest.mark.gpu
@pytest.mark.parametrize("pool,dtype", [("f32", torch.float32), ("f16", torch.float32), ("f16", torch.float16), ("bf16", torch.bfloat16), ("i8", torch.float32)])
def test_append_by_slots(pool, dtype):
    """Rows that go by slots lie where those that go by positions lie; those at -1, of a call that found too few pages, lie nowhere."""
    import llm_decoder as ld

    def cache():
        kv = ld.KVTileCache(pool)
        kv.init(24, 16, 64)
        kv.configure_table(2, 3, 6)
        return kv
    g = torch.Generator(device="cuda").manual_seed(1)
    one, other = cache(), cache()
    for kv, by_slots in ((one, False), (other, True)):
        g.manual_seed(1)
        pages = kv.pages_on_device()
        for lengths, sizes in (([0, 0], [5, 33]), ([5, 33], [14, 1]), ([19, 34], [90, 0])):
            new = pages.take(lengths, start_of(sizes), sum(sizes))
            k, v = (torch.randn(sum(sizes), 3, 64, device="cuda", generator=g).to(dtype) for _ in "kv")
            if by_slots:
                kv.append(k, v, slots=new.slots)
            else:
                kv.append(k, v, new.positions, new.row_seq)
        with pytest.raises(RuntimeError):
            pages.check()
    for name in ("key_buffer_", "value_buffer_", "k_scales_", "v_scales_"):
        a, b = getattr(one, name), getattr(other, name)
        assert (a is None) == (b is None) and (a is None or torch.equal(a, b))
    assert float(one.key_buffer_.float().abs().sum()) > 0
    k = torch.zeros(2, 3, 64, device="cuda", dtype=dtype)
    slots = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    for kw in (dict(), dict(positions=slots[:, 0].contiguous(), slots=slots), dict(slots=slots, beam_ids=slots[:, 0]), dict(slots=slots[:1]), dict(slots=slots.long()),
               dict(slots=slots.cpu()), dict(slots=slots.t())):
        with pytest.raises(ValueError):
            one.append(k, k, **kw)


@pytest.mark.gpu
def test_refusals_and_replays():
    import llm_decoder as ld
    pt = ld.PageTable()
    pt.init(2, 2, 4)
    for kw in (dict(total_pages=0, tile_size=16), dict(total_pages=2 ** 27, tile_size=16), dict(total_pages=8, tile_size=16, free=[0, 0]),
               dict(total_pages=8, tile_size=16, free=[8]), dict(total_pages=8, tile_size=16, free=[-1])):
        with pytest.raises(ValueError):
            ld.DevicePages(pt, **kw)
    for table in ([[0, 1, -1, -1], [2, -1, -1, -1]], [[0, -1, 1, -1], [2, -1, 3, -1]], [[0, 1, -1, -1], [1, 0, -1, -1]], [[0, -1, -1, -1], [9, -1, -1, -1]]):
        pt.load_host_table(np.array([table, [[-1] * 4] * 2]))
        with pytest.raises(ValueError):
            ld.DevicePages(pt, 8, 16)
    with pytest.raises(ValueError):
        ld.DevicePages(ld.PageTable(), 8, 16)
    pt.load_host_table(np.array([[[5, 1, -1, -1], [3, 2, -1, -1]], [[-1] * 4] * 2]))
    pages = ld.DevicePages(pt, 9, 16)
    for args in (([0, 0, 0], start_of([1, 1, 1]), 3), ([0, 0], start_of([1]), 1), ([0], start_of([1]), -1), ([], start_of([]), 1),
                 (torch.zeros(2, device="cuda"), start_of([1, 1]), 2), (torch.zeros(2, dtype=torch.int32), start_of([1, 1]), 2)):
        with pytest.raises(ValueError):
            pages.take(*args)
    with pytest.raises(ValueError):
        pages.release([0, 0, 0])
    assert pages.take([], [0], 0).slots.shape == (0, 2)
    # a step that grows and shrinks, replayed
    lengths, start = torch.tensor([20, 0], dtype=torch.int32, device="cuda"), start_of([3, 4])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pages.release(lengths)
        new = pages.take(lengths, start, 7)
    host = Host(2, 2, 4, 16, [8, 7, 6, 4, 0])
    host.table[0, :, :2], host.held = [[5, 1], [3, 2]], [2, 0]
    for now in ([20, 0], [30, 1], [14, 17], [60, 0], [17, 3]):
        lengths.copy_(torch.tensor(now))
        graph.replay()
        host.release(now)
        want = host.take(now, [3, 4])
        assert (new.row_seq.tolist(), new.positions.tolist(), new.slots.tolist()) == want and host.same(pages), now
    with pytest.raises(RuntimeError):
        pages.check()


def test_refused_on_the_host():
    from llm_decoder import _cabi
    lib = _cabi.lib()
    good = (0x1000, 2, 2, 4, 16, 8, 0x2000, 0x3000, 0x4000)
    assert lib.pa_take_pages(*good, 0x5000, 0x6000, 3, 1, 0x7000, 0x8000, 0x9000, None) == -1             # more sequences than table rows
    assert lib.pa_take_pages(*good, 0x5000, None, 2, 1, 0x7000, 0x8000, 0x9000, None) == -1
    assert lib.pa_take_pages(*good, 0x5000, 0x6000, 2, 1, 0x7000, None, 0x9000, None) == -1
    assert lib.pa_take_pages(*good, 0x5000, 0x6000, 2, 2 ** 30 + 1, 0x7000, 0x8000, 0x9000, None) == -1
    assert lib.pa_take_pages(*good, 0x5000, 0x6000, 0, 1, 0x7000, 0x8000, 0x9000, None) == -1
    assert lib.pa_take_pages(*good, 0x5000, 0x6000, 0, 0, None, None, None, None) == 0
    assert lib.pa_take_pages(None, *good[1:], 0x5000, 0x6000, 2, 1, 0x7000, 0x8000, 0x9000, None) == -1
    assert lib.pa_take_pages(0x1000, 2, 2, 4, 16, 2 ** 27, *good[6:], 0x5000, 0x6000, 2, 1, 0x7000, 0x8000, 0x9000, None) == -1
    assert lib.pa_take_pages(0x1000, 40000, *good[2:], 0x5000, 0x6000, 20000, 1, 0x7000, 0x8000, 0x9000, None) == -2
    assert lib.pa_release_pages(*good, 0x5000, 3, None) == -1
    assert lib.pa_release_pages(*good, None, 2, None) == -1
    assert lib.pa_release_pages(*good, None, 0, None) == 0


def test_pools_do_not_change_under_pages_on_the_gpu():
    """While a DevicePages hands out a cache's pages, the cache takes no other buffers and no other cache's pages: to_host would give its free list pages of the
    pool it had, or write the other cache's."""
    import llm_decoder as ld
    a, b = ld.KVTileCache("f16"), ld.KVTileCache("f16")
    pool = torch.zeros(4, 16, 64, dtype=torch.float16)
    for kv in (a, b):
        kv.adopt_buffers(pool, pool)
    a.page_table_.device_pages_ = object()
    free, table = a._free, a.page_table_
    for call in (lambda: a.adopt_buffers(pool[:2], pool[:2]), lambda: a.share_pages(b)):
        with pytest.raises(RuntimeError, match="to_host"):
            call()
    assert a.total_pages_ == 4 and a._free is free and a.page_table_ is table
    for _ in range(2):
        b.share_pages(a)        # (the other way: one set of pages, handed out on the GPU)
        assert b.page_table_ is table


def test_rows_go_to_the_stream_of_their_device(monkeypatch):
    """append and what it allocates belong to the pools' device, whichever is current: the stream is asked for where that device is."""
    import contextlib

    from llm_decoder import KVTileCache, _cabi

    class OnGpu(torch.Tensor):          # (nothing is launched here)
        is_cuda = property(lambda self: True)
    here, asked = [], []

    @contextlib.contextmanager
    def on_device(device):
        here.append(device)
        yield
        here.pop()

    class Library:
        def __getattr__(self, name):
            return lambda *args: 0
    monkeypatch.setattr(_cabi, "on_device", on_device)
    monkeypatch.setattr(_cabi, "stream", lambda: asked.append(bool(here)) or 0)
    monkeypatch.setattr(_cabi, "lib", lambda: Library())
    kv, k = KVTileCache("f16"), torch.zeros(3, 2, 64, dtype=torch.float16).as_subclass(OnGpu)
    kv.adopt_buffers(torch.zeros(4, 16, 64, dtype=torch.float16), torch.zeros(4, 16, 64, dtype=torch.float16))
    monkeypatch.setattr(kv.page_table_, "num_heads_", 2)
    monkeypatch.setattr(kv.page_table_, "d_table_", torch.zeros(8, dtype=torch.int32))
    kv.append(k, k, torch.zeros(3, dtype=torch.int32))
    kv.append(k, k, slots=torch.zeros(3, 2, dtype=torch.int32))
    assert asked == [True, True]


@pytest.mark.gpu
def test_captured_calls_take_tensors():
    """Numbers of the host are copied once, by way of a buffer that others use next: a captured call is refused them, and what was captured before replays."""
    import llm_decoder as ld
    pt = ld.PageTable()
    pt.init(2, 2, 4)
    pages = ld.DevicePages(pt, 16, 16)
    lengths, start = torch.tensor([20, 0], dtype=torch.int32, device="cuda"), start_of([3, 4])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: pages.take([20, 0], start, 7), lambda: pages.take(lengths, [0, 3, 7], 7), lambda: pages.release([20, 0])):
            with pytest.raises(RuntimeError, match="captured"):
                call()
        new = pages.take(lengths, start, 7)
    graph.replay()
    assert new.positions.tolist() == [20, 21, 22, 0, 1, 2, 3] and pages.free_pages() == 16 - 2 * 3
    assert pages.take([20, 0], [0, 3, 7], 7).slots.tolist() == new.slots.tolist()
