"""Trees of drafted tokens: DraftTree on the CPU, paged_tree_attention and tree_accept against plain forms (float64, integers).

Bounds of the attention.  A score is off by at most 2^-20 of sum |q| |k| / T (float or two-term products, float sums) and the
result then by 2 max|v| times that; softmax weights of float queries are good to 2^-18, those of 16-bit queries are rounded to that type and the
result is too, which takes at most 2^-8 (bfloat16) or 2^-11 (half) of a number each; 1.1 times the sum is asked."""
import math

import numpy as np
import pytest
import torch

T16 = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
UNIT = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def random_parents(rng, n, back=5):
    return [int(rng.integers(max(0, i - back), i)) if i else -1 for i in range(n)]


def path_of(parents, i):
    out = []
    while i >= 0:
        out.append(i)
        i = parents[i]
    return out[::-1]


# --------------------------------------------------------------------------------------------------------------- on the CPU
def test_tree_arrays():
    import llm_decoder as ld
    rng = np.random.default_rng(3)
    parents = [random_parents(rng, n) for n in (1, 40, 0, 7, 33)]
    tokens = [list(range(100 * b, 100 * b + len(p))) for b, p in enumerate(parents)]
    t = ld.DraftTree(parents, tokens, device="cpu")
    assert (t.rows, t.num_seqs, t.most) == (81, 5, 40) and t.node_start.tolist() == [0, 1, 41, 41, 48, 81]
    assert t.tokens.tolist() == [x for s in tokens for x in s] and t.mask.shape == (81, 2)
    words = t.mask.numpy().view(np.uint32)
    r = 0
    for b, p in enumerate(parents):
        for i in range(len(p)):
            path = path_of(p, i)
            assert int(t.row_seq[r]) == b and int(t.nodes[r]) == i and int(t.parents[r]) == p[i] and int(t.depths[r]) == len(path) - 1
            assert [j for j in range(64) if (int(words[r][j // 32]) >> (j % 32)) & 1] == path
            r += 1
    assert t.depth == max(len(path_of(p, i)) for p in parents for i in range(len(p)))
    assert t.positions(torch.tensor([5, 0, 9, 2, 100], dtype=torch.int32)).tolist()[:3] == [5, 0, 1]
    empty = ld.DraftTree([[], []], device="cpu")
    assert empty.rows == 0 and empty.depth == 0 and empty.tokens is None


@pytest.mark.parametrize("parents", [[[0]], [[-1, -1]], [[-1, 1]], [[-1, 2, 0]], [[-1] + [0] * 1024]])
def test_tree_refusals(parents):
    import llm_decoder as ld
    with pytest.raises(ValueError):
        ld.DraftTree(parents, device="cpu")
    with pytest.raises(ValueError):
        ld.DraftTree([[-1, 0]], tokens=[[4]], device="cpu")


def test_argument_rules_need_no_gpu():
    from llm_decoder import _cabi
    lib = _cabi.lib()
    x = 0x1000

    def att(q=x, qt=0, kt=1, ks=None, beams=1, kvh=2, rows=4, most=4, heads=4, dim=64, words=1, temp=1.0, stride=256):
        return lib.pa_tree_attention(q, stride, qt, x, x, x, ks, ks, kt, x, beams, kvh, 4, 8, None, x, x, x, words, rows, 1, most, heads, dim, 16,
                                     temp, None, 0, None)
    assert att(q=None) == -1 and att(heads=3) == -1 and att(temp=0.0) == -1 and att(most=40) == -1 and att(stride=255) == -1
    assert att(kt=3) == -1 and att(ks=x) == -1 and att(beams=0) == -1              # int8 pages with scales, others without
    assert att(most=2000, words=64) == -2 and att(qt=2, kt=1) == -2 and att(qt=2, kt=0) == -2 and att(dim=300, stride=1200) == -2
    assert att(rows=0) == 0
    assert lib.pa_tree_accept(x, x, x, x, 1, 4, 2, x, None, 1, 1, 1, 1, 16, 128, 128, 1, None, x, x, x, x, None) == -1
    assert lib.pa_tree_accept(x, x, x, x, 1, 2000, 2, x, None, 0, 0, 0, 0, 0, 0, 0, 0, None, x, x, x, x, None) == -2
    assert lib.pa_tree_accept(x, x, x, None, 1, 4, 2, x, None, 0, 0, 0, 0, 0, 0, 0, 0, None, x, x, x, x, None) == -1
    assert lib.pa_tree_accept(None, None, None, None, 0, 0, 0, None, None, 0, 0, 0, 0, 0, 0, 0, 0, None, None, None, None, None, None) == 0


# ---------------------------------------------------------------------------------------------------------------- attention
class Case:
    """Pages in random order, rows that nobody may see hold NaN (int8: scales of 0)."""

    def __init__(self, seed, pool, q, heads, kv_heads, dim, ctx, sizes, tile=16, spare_rows=1):
        import llm_decoder as ld
        rng = np.random.default_rng(seed)
        g = torch.Generator().manual_seed(seed)
        self.ctx, self.parents = ctx, [random_parents(rng, n) for n in sizes]
        self.heads, self.kvh, self.dim, self.tile = heads, kv_heads, dim, tile
        B, beams = len(ctx), len(ctx) + spare_rows
        self.beams = rng.permutation(beams)[:B].astype(np.int32)
        tiles = max(1, max(-(-(c + n) // tile) for c, n in zip(ctx, sizes)) + 1)
        pages = beams * kv_heads * tiles
        table = rng.permutation(pages).astype(np.int32).reshape(beams, kv_heads, tiles)
        self.table = table
        k, v = (torch.full((pages, tile, dim), float("nan")) for _ in range(2))
        self.scales = None
        for b, c in enumerate(ctx):
            used = c + sizes[b]
            for h in range(kv_heads):
                for t in range(-(-used // tile)):
                    n = min(tile, used - t * tile)
                    for x in (k, v):
                        x[table[self.beams[b], h, t], :n] = torch.randn(n, dim, generator=g)
        kv = ld.KVTileCache(pool)
        if pool == "i8":
            ks, vs = (127.0 / x.abs().amax(-1).nan_to_num(0.0).clamp(min=1e-6) for x in (k, v))
            ks[k[..., 0].isnan()] = 0.0
            vs[v[..., 0].isnan()] = 0.0
            k8, v8 = ((x * s[..., None]).nan_to_num(77.0).round().clamp(-128, 127).to(torch.int8) for x, s in ((k, ks), (v, vs)))
            self.k, self.v = k8.double() / ks.double()[..., None], v8.double() / vs.double()[..., None]
            kv.adopt_buffers(k8.cuda(), v8.cuda(), ks.cuda(), vs.cuda())
        else:
            k, v = k.to(T16[pool]), v.to(T16[pool])
            self.k, self.v = k.double(), v.double()
            kv.adopt_buffers(k.cuda(), v.cuda())
        kv.configure_table(beams, kv_heads, tiles)
        self.cache = kv
        self.tree = ld.DraftTree(self.parents, device="cuda")
        self.q = torch.randn(self.tree.rows, heads, dim, generator=g).to(T16[q])
        self.qt, self.temp = q, math.sqrt(dim) * 0.7
        self.load()

    def load(self):
        self.cache.page_table_.load_host_table(self.table)

    def run(self, q=None, **kw):
        import llm_decoder as ld
        q = self.q.cuda() if q is None else q
        return ld.paged_tree_attention(q, self.cache, self.tree, self.ctx, self.temp, beam_ids=self.beams, **kw)

    def check(self, got, mask=None):
        words = (self.tree.mask.cpu().numpy() if mask is None else mask).view(np.uint32)
        got, r = got.double().cpu(), 0
        for b, c in enumerate(self.ctx):
            n = len(self.parents[b])
            t = np.arange(c + n)
            for i in range(n):
                for h in range(self.heads):
                    pages = self.table[self.beams[b], h * self.kvh // self.heads][t // self.tile]
                    see = np.array([0 <= p < self.cache.total_pages_ and (x < c or (int(words[r][(x - c) // 32]) >> ((x - c) % 32)) & 1) for x, p in zip(t, pages)], dtype=bool)
                    at, off = pages[see], t[see] % self.tile
                    if not len(at):
                        assert bool((got[r, h] == 0).all())
                        continue
                    k, v, q = self.k[at, off], self.v[at, off], self.q[r, h].double()
                    s = k @ q / self.temp
                    e = (s - s.max()).exp()
                    want = (e @ v) / (e.sum() + 1e-6)
                    size = float((k.abs() @ q.abs()).max()) / self.temp
                    bound = 1.1 * float(v.abs().max()) * (2 * 2.0 ** -20 * size + 2.0 ** -18 + 2 * UNIT[self.qt])
                    err = float((got[r, h] - want).abs().max())
                    assert err <= bound, (b, i, h, err, bound)
                r += 1


PAIRS = [("f16", "f32"), ("i8", "f32"), ("f32", "f32"), ("f16", "f16"), ("i8", "f16"), ("bf16", "bf16")]


@pytest.mark.gpu
@pytest.mark.parametrize("pool,q", PAIRS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 64), (8, 2, 128), (6, 1, 128), (2, 2, 96)])
def test_attention(pool, q, heads, kv_heads, dim):
    """Contexts that end on, before and behind tiles and units of 64 keys, none, and some hundred; trees from no node to more than 32."""
    c = Case(heads + dim, pool, q, heads, kv_heads, dim, [0, 1, 15, 16, 17, 63, 64, 130, 300, 5, 0], [1, 3, 8, 1, 2, 40, 4, 7, 16, 0, 33])
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("pool,q", PAIRS)
def test_attention_splits_long_contexts(pool, q):
    """One sequence of some thousand keys beside short ones: its keys are shared out and joined."""
    c = Case(5, pool, q, 4, 2, 128 if pool != "f32" else 64, [5000, 3, 700], [9, 2, 5])
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("tile", [16, 48, 5, 1])
def test_attention_page_sizes(tile):
    c = Case(tile, "f16", "f32", 4, 2, 64, [100, 0, 33], [5, 3, 20], tile=tile)
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,nodes", [(8, 1, 70), (16, 1, 40), (3, 1, 200), (2, 2, 300)])
def test_attention_wide_trees(heads, kv_heads, nodes):
    """More (node, head) rows of a kv head than a tile of queries holds, and trees that fill several units of keys."""
    c = Case(nodes, "bf16", "bf16", heads, kv_heads, 64, [90, 17], [nodes, 3])
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("pool,q", PAIRS)
def test_attention_views_masks_and_missing_pages(pool, q):
    c = Case(11, pool, q, 4, 2, 128, [70, 40, 0], [6, 35, 2])
    wide = torch.full((c.tree.rows, 3, 4, 128), float("nan"), dtype=T16[q], device="cuda")
    wide[:, 1] = c.q.cuda()
    out = torch.empty(c.tree.rows, 4, 128, dtype=T16[q], device="cuda")
    assert c.run(wide[:, 1], out=out) is out                    # queries as columns of a wider projection
    c.check(out)
    c.table[c.beams[0], 0, 1] = -1                              # pages that are not there, one of them behind the pool
    c.table[c.beams[1], 1, 0] = c.cache.total_pages_ + 3
    c.table[c.beams[2]] = -1                                    # nothing is visible
    c.load()
    c.check(c.run())
    mask = c.tree.mask.cpu().numpy().copy()
    mask[2:9] = 0                                               # rows that see the context only; in the last sequence nothing
    mask[-1] = -1                                               # bits of nodes that are not there
    c.tree.mask.copy_(torch.from_numpy(mask))
    c.check(c.run(), mask)


@pytest.mark.gpu
@pytest.mark.parametrize("pool,q", [("f16", "f32"), ("f16", "f16"), ("bf16", "bf16")])
def test_attention_hidden_rows_may_hold_anything(pool, q):
    """A branch whose rows are not finite changes nothing for the rows that do not see it."""
    c = Case(21, pool, q, 4, 2, 128, [37, 64], [12, 30])
    c.parents = [[-1] + [0] * 11, [-1] + [0] * 29]
    import llm_decoder as ld
    c.tree = ld.DraftTree(c.parents, device="cuda")
    want = c.run()
    for b, node in ((0, 5), (1, 20)):
        pos = c.ctx[b] + node
        for h in range(2):
            page = int(c.table[c.beams[b], h, pos // 16])
            c.cache.key_buffer_[page, pos % 16, 3] = float("nan")
            c.cache.value_buffer_[page, pos % 16, 7] = float("inf")
    got = c.run()
    hit = torch.zeros(c.tree.rows, dtype=torch.bool)
    hit[5] = hit[12 + 20] = True
    assert bool(got[~hit].isfinite().all()) and not bool(got[hit].isfinite().any(-1).all())
    c.check(torch.where(hit[:, None, None].cuda(), want, got))


@pytest.mark.gpu
def test_attention_repeats_its_bits_and_serves_streams():
    c = Case(31, "bf16", "bf16", 16, 4, 128, [3000, 900, 1, 0], [17, 30, 64, 1])
    a = c.run()
    side = torch.cuda.Stream()
    q = c.q.cuda()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        outs = [c.run(q) for _ in range(4)]
    here = [c.run(q) for _ in range(4)]
    torch.cuda.synchronize()
    for o in outs + here:
        assert torch.equal(o, a)


@pytest.mark.gpu
def test_attention_refusals():
    import llm_decoder as ld
    c = Case(41, "f16", "f32", 4, 2, 64, [10], [3])
    q = c.q.cuda()
    for bad in (q[:2], q[:, :3], q[..., :32], q.to(torch.bfloat16), q.cpu(), q[0]):
        with pytest.raises(ValueError):
            c.run(bad)
    for kw in (dict(out=torch.empty(3, 4, 32, device="cuda")), dict(out=torch.empty(3, 4, 64, dtype=torch.float16, device="cuda"))):
        with pytest.raises(ValueError):
            c.run(q, **kw)
    with pytest.raises(ValueError):
        ld.paged_tree_attention(q, c.cache, c.tree, [1, 2])
    with pytest.raises(ValueError):
        ld.paged_tree_attention(q, c.cache, c.tree, [10], temperature=0.0)
    empty = ld.DraftTree([[], []], device="cuda")
    assert ld.paged_tree_attention(q[:0], c.cache, empty, [0, 0]).shape == (0, 4, 64)


# ------------------------------------------------------------------------------------------------------------------- accept
@pytest.mark.gpu
@pytest.mark.parametrize("pool,dim,tile,layers,shared", [("f16", 64, 16, 3, True), ("i8", 128, 16, 2, False), ("bf16", 40, 5, 1, False),
                                                         ("i8", 33, 7, 2, True), ("f32", 64, 16, 70, True)])
def test_accept(pool, dim, tile, layers, shared):
    import llm_decoder as ld
    rng = np.random.default_rng(dim)
    sizes, ctx = [9, 1, 0, 40, 70, 33], [30, 0, 4, 15, 1, 64]
    parents = [random_parents(rng, n, 3) for n in sizes]
    B, KVH = len(sizes), 2
    tokens = [rng.integers(0, 2, n).tolist() for n in sizes]             # few tokens: siblings often share theirs
    ids = [[tokens[b][rng.choice([j for j in range(n) if parents[b][j] == i] or [0])] for i in range(n)] for b, n in enumerate(sizes)]
    tree = ld.DraftTree(parents, tokens, device="cuda")
    tiles = max(-(-(c + n) // tile) for c, n in zip(ctx, sizes))
    beams = rng.permutation(B + 1)[:B].astype(np.int32)
    pages = (B + 1) * KVH * tiles
    caches, want, tables = [], [], []
    for layer in range(layers):
        if layer == 0 or not shared:
            table = rng.permutation(pages).astype(np.int32).reshape(B + 1, KVH, tiles)
            table[beams[3], 1, 1] = -1                                   # rows there stay
        pools = [torch.from_numpy(rng.integers(-100, 100, (pages, tile, dim)).astype(np.float32)).to(ld.kv_tile_cache._DTYPES[pool]) for _ in "kv"]
        scales = [torch.from_numpy(rng.random((pages, tile)).astype(np.float32)) for _ in "kv"] if pool == "i8" else [None, None]
        kv = ld.KVTileCache(pool)
        kv.adopt_buffers(*(x.cuda() for x in pools), *(None if s is None else s.cuda() for s in scales))
        if layer and shared:
            kv.share_pages(caches[0])
        else:
            kv.configure_table(B + 1, KVH, tiles)
            kv.page_table_.load_host_table(table)
        caches.append(kv)
        want.append([x.clone() for x in pools + scales if x is not None])
        tables.append(table)
    paths = []
    for b, p in enumerate(parents):
        path, cur = [], 0 if p else -1
        while cur >= 0:
            path.append(cur)
            cur = next((j for j in range(len(p)) if p[j] == cur and tokens[b][j] == ids[b][cur]), -1)
        paths.append(path)
        for table, xs in zip(tables, want):
            for x in xs:
                for h in range(KVH):
                    at = lambda pos: (int(table[beams[b], h, pos // tile]), pos % tile)  # noqa: E731, B023
                    rows = [x[at(ctx[b] + i)].clone() if at(ctx[b] + i)[0] >= 0 else None for i in path]
                    for d, row in enumerate(rows):
                        if row is not None and at(ctx[b] + d)[0] >= 0:
                            x[at(ctx[b] + d)] = row
    assert max(len(p) for p in paths) >= 3 and any(any(i != d for d, i in enumerate(p)) for p in paths)
    got = ld.tree_accept(torch.tensor([x for s in ids for x in s], dtype=torch.int32, device="cuda"), tree, ld.TreeCaches(caches), ctx, beam_ids=beams)
    assert got.counts.tolist() == [len(p) for p in paths] and got.ctx_lens.tolist() == [c + len(p) for c, p in zip(ctx, paths)]
    pad = lambda x: x + [-1] * (tree.depth - len(x))  # noqa: E731
    assert got.nodes.tolist() == [pad(p) for p in paths]
    assert got.tokens.tolist() == [pad([ids[b][i] for i in p]) for b, p in enumerate(paths)]
    for kv, xs in zip(caches, want):
        have = [kv.key_buffer_, kv.value_buffer_] + ([kv.k_scales_, kv.v_scales_] if pool == "i8" else [])
        for a, x in zip(have, xs):
            assert torch.equal(a.cpu(), x)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [2, 33, 500])
def test_accept_long_paths(n):
    """A path of every second node: each place that a row goes to held the row of an earlier one, or nobody's."""
    import llm_decoder as ld
    parents = [-1] + [max(0, 2 * ((i - 1) // 2) - 1) if i > 1 else 0 for i in range(1, n)]       # node 2k + 1 and a leaf below node 2k - 1
    tokens = list(range(n))
    path = path_of(parents, n - 1 if n % 2 == 0 else n - 2)
    ids = [-5] * n
    for a, b in zip(path, path[1:]):
        ids[a] = b
    kv = ld.KVTileCache("f32")
    k = torch.arange(40 * 16 * 4, dtype=torch.float32, device="cuda").view(40, 16, 4)
    kv.adopt_buffers(k.clone(), k.clone() + 0.5)
    kv.configure_table(1, 1, 40)
    kv.page_table_.load_host_table(np.arange(39, -1, -1, dtype=np.int32))
    a = ld.tree_accept(torch.tensor(ids, dtype=torch.int32, device="cuda"), ld.DraftTree([parents], [tokens], device="cuda"), [kv], [100])
    assert a.counts.tolist() == [len(path)] and a.nodes[0, :len(path)].tolist() == path
    flat = k.flip(0).reshape(-1, 4)                                                     # by position
    want = flat.clone()
    want[100:100 + len(path)] = flat[torch.tensor(path, device="cuda") + 100]
    assert torch.equal(kv.key_buffer_.flip(0).reshape(-1, 4), want) and torch.equal(kv.value_buffer_.flip(0).reshape(-1, 4), want + 0.5)


@pytest.mark.gpu
def test_accept_without_caches_and_refusals():
    import llm_decoder as ld
    tree = ld.DraftTree([[-1, 0, 0, 2], []], [[9, 4, 5, 6], []], device="cuda")
    ids = torch.tensor([5, 1, 6, 7], dtype=torch.int32, device="cuda")
    a = ld.tree_accept(ids, tree, [], [3, 8])
    assert a.counts.tolist() == [3, 0] and a.tokens.tolist() == [[5, 6, 7], [-1] * 3] and a.ctx_lens.tolist() == [6, 8]
    for bad in (ids[:3], ids.long(), ids.cpu()):
        with pytest.raises(ValueError):
            ld.tree_accept(bad, tree, [], [3, 8])
    with pytest.raises(ValueError):
        ld.tree_accept(ids, ld.DraftTree([[-1, 0, 0, 2]], device="cuda"), [], [3])
    kv = [ld.KVTileCache("f16", device="cuda:0") for _ in range(2)]
    for k, d in zip(kv, (64, 128)):
        k.init(4, 16, d)
        k.configure_table(1, 1, 4)
    with pytest.raises(ValueError):
        ld.TreeCaches(kv)
    nothing = ld.tree_accept(ids[:0], ld.DraftTree([[], []], [[], []], device="cuda"), [], [3, 8])
    assert nothing.counts.tolist() == [0, 0] and nothing.ctx_lens.tolist() == [3, 8] and nothing.tokens.shape == (2, 0)
