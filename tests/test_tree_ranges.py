"""paged_tree_attention over the range of what pages hold: values of any size, of sizes that differ from row to row, drafted rows that some
rows do not see and that hold anything.

Bounds.  A score is off by at most 2^-20 of sum |q| |k| / T, softmax weights of float queries are good to 2^-18 of each, those of 16-bit
queries are rounded to that type (2^-11 half, 2^-8 bfloat16) and so is the result.  All of these are relative errors of one key's share p |v| of the
result, so the bound is their sum times sum p max|v| over the keys that the row sees, whatever the size of other rows' keys; 1.1
times that is asked, and half of the smallest half where results are halves."""
import numpy as np
import pytest
import torch

from test_draft_trees import UNIT, Case


def check(c, got, skip=()):
    """Every row but those of `skip` (sequence, node) against float64."""
    words, r = c.tree.mask.cpu().numpy().view(np.uint32), 0
    got = got.double().cpu()
    for b, ctx in enumerate(c.ctx):
        n = len(c.parents[b])
        t = np.arange(ctx + n)
        for i in range(n):
            see = np.array([x < ctx or (int(words[r][(x - ctx) // 32]) >> ((x - ctx) % 32)) & 1 for x in t], dtype=bool)
            for h in range(c.heads) if (b, i) not in skip else ():
                pages = c.table[c.beams[b], h * c.kvh // c.heads][t // c.tile]
                k, v, q = c.k[pages[see], t[see] % c.tile], c.v[pages[see], t[see] % c.tile], c.q[r, h].double()
                s = k @ q / c.temp
                e = (s - s.max()).exp()
                p = e / (e.sum() + 1e-6)
                size = float((k.abs() @ q.abs()).max()) / abs(c.temp)
                bound = 1.1 * float(p @ v.abs().amax(-1)) * (2 * 2.0 ** -20 * size + 2.0 ** -18 + 2 * UNIT[c.qt]) + (2.0 ** -25 if c.qt == "f16" else 0.0)
                err = float((got[r, h] - p @ v).abs().max())
                assert err <= bound, (b, i, h, err, bound)
            r += 1


def scale_values(c, by):
    """Int8 values times by [pages, tile]."""
    by = torch.as_tensor(by, dtype=torch.float32).expand(c.cache.v_scales_.shape)
    c.cache.v_scales_.div_(by.cuda())
    c.v = torch.where(c.cache.v_scales_.cpu()[..., None] > 0, torch.nan_to_num(c.cache.value_buffer_.cpu().double() / c.cache.v_scales_.cpu().double()[..., None]), c.v)


SHAPES = [(4, 4, 64, 8), (4, 4, 128, 8), (4, 2, 128, 24), (6, 2, 64, 24), (2, 2, 96, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("q,size", [("f32", 1e-5), ("f32", 1e-3), ("f32", 30.0), ("f32", 300.0), ("f32", 1e3), ("f32", 1e5), ("f16", 1e-3), ("f16", 300.0), ("f16", 1e4)])
@pytest.mark.parametrize("heads,kv_heads,dim,nodes", SHAPES)
def test_int8_values_of_any_size(heads, kv_heads, dim, nodes, q, size):
    """Scores of some spread, so that the largest so far is passed again and again along the context."""
    c = Case(77, "i8", q, heads, kv_heads, dim, [500, 40], [nodes, 3])
    c.temp = dim ** 0.5 * 0.33
    scale_values(c, size)
    check(c, c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("q", ["f32", "f16"])
@pytest.mark.parametrize("heads,kv_heads,dim,nodes", SHAPES)
def test_int8_values_of_sizes_that_differ(heads, kv_heads, dim, nodes, q):
    """Rows from a thousandth to a thousand, some of zeros."""
    c = Case(78, "i8", q, heads, kv_heads, dim, [3000, 200, 17], [nodes, 3, 5])
    rng = np.random.default_rng(5)
    by = 10.0 ** rng.uniform(-3, 3, tuple(c.cache.v_scales_.shape))
    scale_values(c, by)
    none = torch.from_numpy(rng.random(by.shape) < 0.05) & (c.cache.v_scales_.cpu() > 0)
    c.cache.value_buffer_[none.cuda()] = 0
    c.cache.v_scales_[none.cuda()] = 127.0 / 1e-6               # as an appended row of zeros
    c.v[none] = 0.0
    check(c, c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("q", ["f32", "f16"])
@pytest.mark.parametrize("heads,kv_heads,dim,nodes", SHAPES)
def test_int8_values_that_weigh_nothing(heads, kv_heads, dim, nodes, q):
    """Keys that every row scores far below the others, with values ten thousand times as large: no row loses bits to them."""
    c = Case(81, "i8", q, heads, kv_heads, dim, [700, 90], [nodes, 3])
    g = torch.Generator().manual_seed(3)
    way = torch.sign(torch.randn(dim, generator=g))
    c.q = (way + 0.1 * torch.randn(c.q.shape, generator=g)).to(c.q.dtype)       # every query along `way`
    k = torch.randn(c.cache.key_buffer_.shape, generator=g) * 20
    k -= (k @ way / dim)[..., None] * way                                       # keys across it
    far = torch.rand(k.shape[:2], generator=g) < 0.02
    far[:, 0] = False
    k[far] = -way * 120                                                         # some against it
    k = k.round().clamp(-128, 127)
    used = c.cache.v_scales_.cpu() > 0
    c.cache.key_buffer_.copy_(k.to(torch.int8))
    c.cache.k_scales_.fill_(40.0)
    c.k = k.double() / 40.0
    c.temp = dim * 3.0 / 60.0                                                   # -60 for those, some tenths for the others
    by = torch.ones(used.shape)
    by[far] = 1e4
    scale_values(c, by)
    check(c, c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("pool,q", [("i8", "f32"), ("i8", "f16"), ("f16", "f32"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("heads,kv_heads,dim,nodes", SHAPES)
@pytest.mark.parametrize("what", ["scale 0", "not a number", "huge"])
def test_hidden_rows_may_hold_anything(pool, q, heads, kv_heads, dim, nodes, what):
    """A drafted row of anything changes nothing for rows that do not see it, in pieces that are joined and in whole items."""
    c = Case(79, pool, q, heads, kv_heads, dim, [2500, 37], [nodes, nodes + 1])
    import llm_decoder as ld
    c.parents = [[-1] + [0] * (nodes - 1), [-1] + [0] * nodes]
    c.tree = ld.DraftTree(c.parents, device="cuda")
    for b, node in ((0, 5), (1, nodes - 2)):
        pos = c.ctx[b] + node
        for h in range(kv_heads):
            at = (int(c.table[c.beams[b], h, pos // 16]), pos % 16)
            if pool == "i8":
                x = {"scale 0": 0.0, "not a number": float("nan"), "huge": 1e-30}[what]
                c.cache.v_scales_[at] = x
                if what != "huge":
                    c.cache.k_scales_[at] = x
                c.v[at] = c.cache.value_buffer_[at].cpu().double() / float(np.float32(x)) if x else float("nan")
            else:
                x = {"scale 0": float("inf"), "not a number": float("nan"), "huge": 60000.0}[what]
                c.cache.value_buffer_[at][7] = x
                c.cache.key_buffer_[at][3] = 1.0 if what == "huge" else x
                c.k[at], c.v[at] = c.cache.key_buffer_[at].cpu().double(), c.cache.value_buffer_[at].cpu().double()
    got = c.run()
    hit = [(0, 5), (1, nodes - 2)]
    check(c, got, hit if what != "huge" or q == "f16" else ())
    rows = got[[5, nodes + nodes - 2]]
    if what != "huge":
        assert not bool(rows.isfinite().all())
