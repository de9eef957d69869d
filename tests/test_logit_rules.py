"""adjust_logits and adjusted_argmax against the same rules in float64, token by token.

Bound: five operations, each rounded to 2^-24 of the largest number on the way; 16-bit logits give what the same logits as floats give,
rounded once, bit for bit.  Ids are compared where the float64 maximum leads by more than the bound, and against the
adjusted float logits themselves always."""
import math

import numpy as np
import pytest
import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def bits_of(rows, words_per_row, allow):
    out = np.zeros((rows, words_per_row), dtype=np.uint32)
    for r in range(rows):
        for v in allow[r]:
            out[r, v >> 5] |= np.uint32(1 << (v & 31))
    return torch.from_numpy(out.view(np.int32))


class Case:
    def __init__(self, seed, kind, seqs, V, hist, bias=0, masked=False, nodes=None, pad=0, shared=False):
        import llm_decoder as ld
        rng = np.random.default_rng(seed)
        self.kind, self.V = kind, V
        parents = [[-1] + [int(rng.integers(max(0, i - 3), i)) for i in range(1, n)] if n else [] for n in nodes] if nodes else None
        self.row_seq = [b for b, p in enumerate(parents) for _ in p] if parents else list(range(seqs))
        R = len(self.row_seq)
        store = torch.from_numpy((rng.standard_normal((max(R, 1), V + pad)) * 4).astype(np.float32)).to(TYPES[kind])
        store[0, V // 2] = 0.0
        self.logits = store[:R, :V]
        self.dev = store.cuda()[:R, :V]
        lens = [hist[b % len(hist)] for b in range(seqs)]
        self.hist = [rng.integers(0, min(V, 1 + n), n).tolist() for n in lens]
        for h in self.hist[1::2]:
            h += [-1, V, V + 5]                     # no tokens of the vocabulary
        self.rep, self.pres, self.freq = (rng.random(seqs).astype(np.float32) * s + o for s, o in ((1.0, 0.6), (1.5, -0.2), (0.4, -0.1)))
        self.bias = [[(int(rng.integers(0, V)), float(np.float32(rng.standard_normal()))) for _ in range(bias)] for _ in range(seqs)]
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        starts = lambda xs: i32(np.concatenate([[0], np.cumsum([len(x) for x in xs])]).tolist())  # noqa: E731
        flat = lambda xs: [y for x in xs for y in x]  # noqa: E731
        self.kw = dict(history=i32(flat(self.hist)), history_start=starts(self.hist),
                       repetition=torch.from_numpy(self.rep).cuda(), presence=torch.from_numpy(self.pres).cuda(), frequency=torch.from_numpy(self.freq).cuda())
        if bias:
            self.kw["bias"] = (i32([v for v, _x in flat(self.bias)]), torch.tensor([x for _v, x in flat(self.bias)], device="cuda"), starts(self.bias))
        self.allow = [set(range(V))] * R
        if masked:
            few = [sorted({int(x) for x in rng.integers(0, V, max(1, V // 7))}) for _ in range(R)]
            few[0] = []                             # a row with nothing left
            words = (V + 31) // 32
            if shared:                              # masks by number, some rows without one
                index = [int(rng.integers(-1, R)) for _ in range(R)]
                self.allow = [set(few[i]) if i >= 0 else set(range(V)) for i in index]
                self.kw["allowed_rows"] = i32(index)
            else:
                self.allow = [set(x) for x in few]
            self.kw["allowed"] = bits_of(R, words + 1, few).cuda()[:, :words]
        self.way = [[] for _ in range(R)]
        if parents:
            tokens = [rng.integers(0, V, len(p)).tolist() for p in parents]
            first = np.concatenate([[0], np.cumsum([len(p) for p in parents])])
            for b, p in enumerate(parents):
                for i in range(len(p)):
                    j = i
                    while j >= 0:
                        self.way[first[b] + i].append(tokens[b][j])
                        j = p[j]
            self.kw["tree"] = ld.DraftTree(parents, tokens, device="cuda")

    def want(self):
        out, size = self.logits.double().numpy().copy(), np.zeros(self.logits.shape)
        for r, b in enumerate(self.row_seq):
            c = np.zeros(self.V)
            for v in self.hist[b] + self.way[r]:
                if 0 <= v < self.V:
                    c[v] += 1
            x, on = out[r], c > 0
            size[r] = np.abs(x) * np.maximum(1, np.maximum(self.rep[b], 1 / self.rep[b])) + np.abs(self.pres[b]) + np.abs(self.freq[b]) * c
            x[on] = np.where(x[on] > 0, x[on] / self.rep[b], x[on] * self.rep[b]) - self.pres[b] - float(self.freq[b]) * c[on]
            for v, val in dict(self.bias[b]).items():
                x[v] += val
                size[r, v] += abs(val)
            x[[v for v in range(self.V) if v not in self.allow[r]]] = -math.inf
        return out, size

    def check(self, got=None, ids=None):
        want, size = self.want()
        if got is not None:
            if self.kind != "f32":
                from llm_decoder import sampling
                wide = sampling.adjust_logits(self.dev.float(), **self.kw)
                assert got.dtype == self.dev.dtype and torch.equal(wide.to(got.dtype), got)
                got = wide
            if ids is not None:
                assert ids.tolist() == [int(np.argmax(x)) for x in got.cpu().numpy()]       # the first of the largest
            got = got.double().cpu().numpy()
            assert np.array_equal(np.isinf(got), np.isinf(want))
            fine = np.isfinite(want)
            assert np.all(np.abs(got[fine] - want[fine]) <= 1.1 * 5 * 2.0 ** -24 * size[fine])
        if ids is not None:
            for r, i in enumerate(ids.tolist()):
                top = want[r].max()
                if np.isinf(top):
                    assert i == 0
                    continue
                assert 0 <= i < self.V and want[r, i] >= top - 2 * 1.1 * 5 * 2.0 ** -24 * size[r].max()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V,pad", [(1, 0), (31, 1), (1000, 24), (50257, 0), (33333, 3), (70000, 8)])
def test_rules(kind, V, pad):
    from llm_decoder import sampling
    c = Case(V, kind, 5, V, [0, 1, 300, 17, 2000], bias=min(V, 40), masked=V > 1, pad=pad)
    got, ids = sampling.adjust_logits(c.dev, ids=True, **c.kw)
    c.check(got, ids)
    assert torch.equal(sampling.adjusted_argmax(c.dev, **c.kw), ids)
    assert torch.equal(sampling.adjust_logits(c.dev, **c.kw), got)
    store = torch.full((5, V + 7), 9.0, dtype=c.dev.dtype, device="cuda")
    store[:, :V] = c.dev                            # in place, in rows of a wider buffer
    assert torch.equal(sampling.adjust_logits(store[:, :V], out=store[:, :V], **c.kw), got) and bool((store[:, V:] == 9.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("nodes", [[1], [12, 0, 1, 70], [40] * 9])
def test_rules_of_trees(kind, nodes):
    from llm_decoder import sampling
    c = Case(len(nodes), kind, len(nodes), 5003, [50, 0, 700], bias=9, masked=True, nodes=nodes)
    got, ids = sampling.adjust_logits(c.dev, ids=True, **c.kw)
    c.check(got, ids)
    assert torch.equal(sampling.adjusted_argmax(c.dev, **c.kw), ids)


@pytest.mark.gpu
def test_each_rule_alone_and_none():
    from llm_decoder import sampling
    c = Case(77, "f32", 4, 3001, [64, 0, 9], bias=5, masked=True, shared=True)
    assert torch.equal(sampling.adjust_logits(c.dev), c.dev)
    base = c.kw
    for names, keep in ((("repetition",), "rep"), (("presence",), "pres"), (("frequency",), "freq"), (("bias",), "bias"), (("allowed", "allowed_rows"), "allow")):
        d = Case(77, "f32", 4, 3001, [64, 0, 9], bias=5, masked=True, shared=True)
        for attr, neutral in (("rep", np.ones(4, np.float32)), ("pres", np.zeros(4, np.float32)), ("freq", np.zeros(4, np.float32)),
                              ("bias", [[]] * 4), ("allow", [set(range(3001))] * 4)):
            if attr != keep:
                setattr(d, attr, neutral)
        kw = {k: base[k] for k in names}
        if keep in ("rep", "pres", "freq"):
            kw.update(history=base["history"], history_start=base["history_start"])
        d.check(sampling.adjust_logits(d.dev, **kw))
    one = Case(78, "f32", 4, 3001, [64, 0, 9])
    one.rep[:], one.pres[:], one.freq[:] = 1.25, 0.5, 0.125
    one.check(sampling.adjust_logits(one.dev, one.kw["history"], one.kw["history_start"], 1.25, 0.5, 0.125))
    seq = torch.tensor([2, 0, 0, 2], dtype=torch.int32, device="cuda")
    one.row_seq = seq.tolist()
    one.check(sampling.adjust_logits(one.dev, one.kw["history"], one.kw["history_start"], 1.25, 0.5, 0.125, row_seq=seq))


@pytest.mark.gpu
def test_ties_infinities_and_nan():
    from llm_decoder import sampling
    x = torch.zeros(6, 40000, device="cuda")
    x[1, 7:] = 3.0
    x[2] = -math.inf
    x[3, 0], x[3, 39999] = math.nan, 1.0
    x[4, 123], x[4, 30000] = math.inf, math.inf
    x[5], x[5, 9000] = -0.0, 0.0
    assert sampling.adjusted_argmax(x).tolist() == [0, 7, 0, 39999, 123, 0]
    got, ids = sampling.adjust_logits(x, repetition=2.0, history=torch.tensor([123, 9000], dtype=torch.int32, device="cuda").repeat(6),
                                      history_start=torch.arange(0, 14, 2, dtype=torch.int32, device="cuda"), ids=True)
    assert ids.tolist() == [0, 7, 0, 39999, 123, 0] and math.isnan(float(got[3, 0])) and float(got[4, 123]) == math.inf


@pytest.mark.gpu
def test_long_histories():
    """Counts above 16 bits, and a history much longer than the vocabulary."""
    from llm_decoder import sampling
    hist = torch.full((200000,), 11, dtype=torch.int32, device="cuda")
    hist[::1000] = torch.arange(200, dtype=torch.int32, device="cuda")
    x = torch.zeros(1, 300, device="cuda")
    got = sampling.adjust_logits(x, hist, torch.tensor([0, 200000], dtype=torch.int32, device="cuda"), frequency=1.0)
    want = -torch.bincount(hist.long(), minlength=300).float()
    assert float(want.min()) < -65536 and torch.equal(got[0], want)


@pytest.mark.gpu
def test_refusals():
    from llm_decoder import sampling
    import llm_decoder as ld
    x = torch.zeros(3, 64, device="cuda")
    h, hs = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.tensor([0, 1, 2, 4], dtype=torch.int32, device="cuda")
    assert sampling.adjust_logits(x[:0]).shape == (0, 64) and sampling.adjusted_argmax(x[:0]).shape == (0,)
    for bad in (dict(history=h), dict(history_start=hs), dict(history=h.long(), history_start=hs), dict(history=h, history_start=hs[:3]),
                dict(history=h.cpu(), history_start=hs), dict(repetition=0.0), dict(repetition=-1.0), dict(repetition=float("nan")),
                dict(repetition=torch.ones(2, device="cuda")), dict(presence=torch.ones(3)), dict(bias=(h, h, hs)), dict(bias=(h, x[0, :3], hs)),
                dict(allowed=torch.zeros(3, 1, dtype=torch.int32, device="cuda")), dict(allowed=torch.zeros(2, 2, dtype=torch.int32, device="cuda")),
                dict(allowed=torch.zeros(3, 2, device="cuda")), dict(row_seq=h), dict(tree=ld.DraftTree([[-1, 0, 0]], device="cuda")),
                dict(tree=ld.DraftTree([[-1]], [[2]], device="cuda")), dict(out=x.half()), dict(out=x[:, :32])):
        with pytest.raises(ValueError):
            sampling.adjust_logits(x, **bad)
    for bad in (x.double(), x[0], x.cpu(), x.t(), x[:1].expand(3, 64)):
        with pytest.raises(ValueError):
            sampling.adjust_logits(bad)


@pytest.mark.gpu
def test_numbers_outside_the_arrays_read_nothing():
    """Rows of sequences that the call has not, mask rows that there are not and starts behind the lists: as without the rule."""
    import llm_decoder as ld
    V = 500
    x = torch.from_numpy(np.random.default_rng(14).standard_normal((6, V)).astype(np.float32)).cuda()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    history, start = i32([3, 4, 5, 6]), i32([0, 2, 900])
    rep = torch.tensor([2.0, 2.0], device="cuda")
    masks = torch.zeros((2, 16), dtype=torch.int32, device="cuda")
    seq, rows = i32([0, 1, 2, -1, 1 << 30, 0]), i32([-1, 2, 1 << 30, -(1 << 31), 5, 0])
    bias = (i32([7, 8]), torch.tensor([1.5, -2.5], device="cuda"), i32([0, 1, 1 << 20]))
    got = ld.sampling.adjust_logits(x, history, start, rep, 0.25, 0.0, bias=bias, allowed=masks, allowed_rows=rows, row_seq=seq)
    want = x.clone()
    for r, (tokens, b) in enumerate([([3, 4], (7, 1.5)), ([5, 6], (8, -2.5)), ([], None), ([], None), ([], None)]):
        for t in tokens:
            want[r, t] = (want[r, t] / 2 if want[r, t] > 0 else want[r, t] * 2) - 0.25
        if b:
            want[r, b[0]] += b[1]
    want[5] = -math.inf
    assert torch.equal(got, want)
