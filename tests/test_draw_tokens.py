"""truncated_softmax, draw_tokens and verify_drafts against their definitions in float64, row by row.

Bounds.  A weight is off by 1.3e-12 of itself (the polynomial's end; 64-bit rounding is far below), so that a border of the cumulative sums is off by
at most 2.6e-12 of the sum: an id is right where its number lies within 4e-12 of the id's own stretch.  A probability is rounded once to a float
(2^-24), next to 2.6e-12 and, where it is below the normal floats, half of the smallest one; a log probability likewise, on
top of 2.6e-12 of its argument."""
import math

import numpy as np
import pytest
import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 4e-12


def kept_weights(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, most=np.inf):
    """Weights of one row by the definition, 0 where a rule leaves the token out."""
    x = np.where(np.isnan(x), -np.inf, np.minimum(x.astype(np.float64), most))
    w = np.zeros(len(x))
    if x.max() == -np.inf:
        return w
    if not temperature > 0:
        w[int(np.argmax(x))] = 1.0
        return w
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x == -np.inf, 0.0, np.exp((x - x.max()) / np.float64(temperature)))
    alive = x > -np.inf
    values, group, size = np.unique(x, return_inverse=True, return_counts=True)
    above = np.concatenate([np.cumsum(size[::-1])[::-1][1:], [0]])[group]
    if 0 < top_k < len(x):
        alive &= above < top_k
    if top_p < 1:
        mass = np.bincount(group, np.where(alive, w, 0.0), len(values))
        before = np.concatenate([np.cumsum(mass[::-1])[::-1][1:], [0.0]])[group]
        alive &= (before < np.float64(top_p) * mass.sum()) | (x == x.max())
    alive &= (w >= min(min_p, 1.0)) if min_p > 0 else True
    return np.where(alive, w, 0.0)


def is_drawn(w, token, number):
    """Whether `number` (in [0, 1)) draws the token, up to the bound."""
    if w.sum() == 0:
        return token == -1
    cum = np.cumsum(w)
    target, eps = np.float64(number) * cum[-1], EPS * cum[-1]
    return 0 <= token < len(w) and w[token] > 0 and cum[token] - w[token] - eps <= target < cum[token] + eps


def near_float(got, want):
    return np.all(np.abs(got - want) <= np.abs(want) * (2.0 ** -24 + 3e-12) + 2.0 ** -150)


class Case:
    """Logits on the GPU as rows of a wider, odd allocation, and what each row's request asks for."""

    def __init__(self, seed, kind, rows, V, rules="mixed", pad=0, shift=0, spread=3.0, odd=False):
        rng = np.random.default_rng(seed)
        x = rng.standard_normal((rows, V)) * spread
        if odd:             # masks, infinities, not-a-numbers, lowest values, ties
            x[rng.random((rows, V)) < 0.3] = -np.inf
            x[rng.random((rows, V)) < 0.02] = np.nan
            x[::5][rng.random((len(x[::5]), V)) < 0.02] = np.inf
            x[1::5] = np.round(x[1::5])
            x[2::5] = -np.inf
            x[3::5][rng.random((len(x[3::5]), V)) < 0.5] = float(torch.finfo(TYPES[kind]).min)
            if rows > 6:
                x[6] = float(torch.finfo(TYPES[kind]).min)
        store = torch.from_numpy(x.astype(np.float32)).to(TYPES[kind])
        wide = torch.full((rows * (V + pad) + shift,), float("nan"), dtype=TYPES[kind]).cuda()
        self.dev = wide[shift:].view(rows, V + pad)[:, :V]
        self.dev.copy_(store)
        self.x, self.rows, self.V, self.most = store.float().numpy(), rows, V, float(torch.finfo(TYPES[kind]).max)
        u = rng.random((4, rows)).astype(np.float32)
        on = rng.random((4, rows)) < 0.6
        if rules == "mixed":
            self.rules = dict(temperature=np.where(on[0], 0.2 + 2 * u[0], np.where(u[0] < 0.3, 0, 1)).astype(np.float32),
                              top_k=np.where(on[1], 1 + (u[1] ** 2 * 1.2 * V).astype(np.int32), 0).astype(np.int32),
                              top_p=np.where(on[2], u[2], 1).astype(np.float32), min_p=np.where(on[3], u[3] ** 4, 0).astype(np.float32))
            self.kw = {k: torch.from_numpy(v).cuda() for k, v in self.rules.items()}
        else:
            self.kw = rules
            self.rules = {k: np.full(rows, v, dtype=np.int32 if k == "top_k" else np.float64) for k, v in rules.items()}
        self.numbers = rng.random((rows, 8)).astype(np.float32)

    def weights(self, r, seq=None):
        return kept_weights(self.x[r], most=self.most, **{k: v[r if seq is None else seq] for k, v in self.rules.items()})


CASES = [(0, "f32", 9, 1000, "mixed", 3, 1), (1, "f32", 3, 50257, "mixed", 0, 0), (2, "bf16", 12, 1003, "mixed", 1, 3), (3, "f16", 12, 4097, "mixed", 0, 5),
         (4, "f32", 5, 1, "mixed", 2, 1), (5, "f32", 40, 2, "mixed", 0, 0), (6, "bf16", 40, 7, "mixed", 0, 1), (7, "f32", 21, 33, "mixed", 1, 0),
         (8, "f32", 2, 128000, dict(top_p=0.9), 0, 0), (9, "bf16", 2, 128001, dict(top_k=50, top_p=0.95), 0, 1), (10, "f32", 3, 20000, dict(), 5, 2),
         (11, "f32", 2, 375000, dict(top_p=0.999, temperature=2.0), 0, 0), (12, "f16", 160, 3000, "mixed", 0, 0), (13, "f32", 300, 517, "mixed", 0, 0),
         (14, "f32", 4, 9000, dict(top_k=8999), 0, 0), (15, "f32", 4, 9000, dict(temperature=1e-30, top_p=0.5), 0, 3), (16, "f32", 4, 9000, dict(temperature=math.inf, top_p=0.4), 0, 0),
         (17, "bf16", 4, 9000, dict(top_p=0.0), 0, 0), (18, "f32", 4, 9000, dict(min_p=1.0), 0, 0), (19, "f32", 6, 30000, dict(top_p=0.9999999), 1, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("spread", [3.0, 0.01, 30.0])
@pytest.mark.parametrize("seed,kind,rows,V,rules,pad,shift", CASES)
def test_probabilities_and_draws(seed, kind, rows, V, rules, pad, shift, spread, odd):
    from llm_decoder import sampling
    c = Case(seed, kind, rows, V, rules, pad, shift, spread, odd)
    probs = sampling.truncated_softmax(c.dev, **c.kw).double().cpu().numpy()
    one, logs = sampling.draw_tokens(c.dev, torch.from_numpy(c.numbers[:, 0].copy()).cuda(), logprobs=True, **c.kw)
    some, more = sampling.draw_tokens(c.dev, torch.from_numpy(c.numbers).cuda(), logprobs=True, **c.kw)
    one, logs, some, more = (t.cpu().numpy() for t in (one, logs, some, more))
    assert probs.shape == (rows, V) and one.shape == (rows,) and some.shape == more.shape == (rows, 8)
    for r in range(rows):
        w = c.weights(r)
        p = w / w.sum() if w.sum() else w
        assert np.array_equal(probs[r] > 0, p.astype(np.float32) > 0) and near_float(probs[r], p)
        assert is_drawn(w, one[r], c.numbers[r, 0])
        for i, t in enumerate(some[r]):
            assert is_drawn(w, t, c.numbers[r, i]), (r, i)
            lp = math.log(p[t]) if t >= 0 else -math.inf
            assert more[r, i] == lp or abs(more[r, i] - lp) <= abs(lp) * 2.0 ** -24 + 3e-12
            if t >= 0:
                w = w.copy()
                w[t] = 0
        assert some[r, 0] == one[r] and more[r, 0] == logs[r]


@pytest.mark.gpu
def test_numbers_at_the_ends():
    """0 draws the first token that stays, what is not below 1 the last one, what is below 0 or no number the first."""
    from llm_decoder import sampling
    x = torch.full((6, 700), -math.inf, device="cuda")
    x[:, 5], x[:, 30], x[:, 600] = 0.0, 1.0, 0.5
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 7.0, -3.0, math.nan], device="cuda")
    assert sampling.draw_tokens(x, u).tolist() == [5, 600, 600, 600, 5, 5]
    ids, logs = sampling.draw_tokens(x[:1], torch.zeros(1, 5, device="cuda"), logprobs=True)
    assert ids.tolist() == [[5, 30, 600, -1, -1]] and logs[0, 3:].tolist() == [-math.inf] * 2
    assert sampling.draw_tokens(x, u, temperature=0.0).tolist() == [30] * 6
    assert sampling.draw_tokens(x[:1], torch.zeros(1, 2, device="cuda"), temperature=0.0).tolist() == [[30, -1]]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_masks_that_leave_a_few(kind):
    """Rows of many chunks of which a mask leaves three tokens, with rules per sequence that leave nothing out: these, and then none."""
    from llm_decoder import sampling
    x = torch.full((3, 60000), -math.inf, device="cuda", dtype=TYPES[kind])
    for r, kept in enumerate(([5, 30, 600], [100, 30000, 59999], [41000, 41001, 50000])):
        x[r, kept] = torch.tensor([0.0, 1.0, 0.5], device="cuda", dtype=TYPES[kind])
    zero, u = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(3, 5, device="cuda")
    for kw in (dict(), dict(top_k=zero), dict(min_p=zero.float()), dict(top_k=zero, top_p=zero.float() + 1, temperature=zero.float() + 0.01)):
        ids = sampling.draw_tokens(x, u, **kw)
        assert [sorted(i[:3]) for i in ids.tolist()] == [[5, 30, 600], [100, 30000, 59999], [41000, 41001, 50000]] and (ids[:, 3:] == -1).all()
        assert sampling.draw_tokens(x, u[:, 0] + 1, **kw).tolist() == [600, 59999, 50000]


@pytest.mark.gpu
def test_rows_by_sequence_and_other_streams():
    """Rows name their sequences (or none: nothing is left out), calls run on the stream that is current, captured calls follow their inputs."""
    from llm_decoder import DraftTree, sampling
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(5, 999, device="cuda", generator=g)
    k = torch.tensor([1, 3], dtype=torch.int32, device="cuda")
    row_seq = torch.tensor([1, 0, 1, 2, -1], dtype=torch.int32, device="cuda")
    kept = (sampling.truncated_softmax(x, top_k=k, row_seq=row_seq) > 0).sum(1).tolist()
    assert kept == [3, 1, 3, 999, 999]
    assert (sampling.truncated_softmax(x, top_k=2, row_seq=row_seq) > 0).sum(1).tolist()[:4] == [2, 2, 2, 2]
    tree = DraftTree([[-1, 0], [], [-1, 0, 0]], device="cuda")
    kept = (sampling.truncated_softmax(x, top_k=torch.tensor([4, 5, 6], dtype=torch.int32, device="cuda"), tree=tree) > 0).sum(1).tolist()
    assert kept == [4, 4, 6, 6, 6]
    u = torch.rand(5, device="cuda", generator=g)
    want = sampling.draw_tokens(x, u, top_p=0.8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sampling.draw_tokens(x, u, top_p=0.8)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ids = sampling.draw_tokens(x, u, top_p=0.8)
        probs = sampling.truncated_softmax(x, top_p=0.8)
    x.copy_(torch.randn(5, 999, device="cuda", generator=g))
    graph.replay()
    assert torch.equal(ids, sampling.draw_tokens(x, u, top_p=0.8)) and torch.equal(probs, sampling.truncated_softmax(x, top_p=0.8))
    out = torch.zeros(5, 1203, device="cuda")
    sampling.truncated_softmax(x, top_p=0.8, out=out[:, 2:1001])
    assert torch.equal(out[:, 2:1001], probs) and not out[:, :2].any() and not out[:, 1001:].any()


# ------------------------------------------------------------------------------------------------------------ verification
def verified(w, children, tokens, q, numbers, draws, distinct):
    """(kept child's token, or None; the weights that are drawn from; whether every test is clear of the bound) at one node."""
    p = w / w.sum()
    left, gone, clear = p, [], True
    for c in children:
        t = tokens[c]
        if not 0 <= t < len(w):
            continue
        was = q.copy()
        if distinct and gone:
            was[gone] = 0
            was = was / max(1 - q[gone].sum(), 1e-18)
        clear &= abs(numbers[c] * was[t] - left[t]) > 1e-9 * (was[t] + left[t]) or was[t] == left[t] == 0
        if numbers[c] * was[t] < left[t]:
            return t, p, clear
        rest = np.maximum(left - was, 0)
        gone.append(t)
        left = rest / rest.sum() if rest.sum() > 1e-300 else np.zeros_like(rest)
    return None, (left if left.sum() else p), clear


def tree_of(rng, n, most):
    parents, children = [-1], [0]
    for i in range(1, n):
        p = int(rng.choice([j for j in range(i) if children[j] < most]))
        parents.append(p)
        children[p] += 1
        children.append(0)
    return parents


@pytest.mark.gpu
@pytest.mark.parametrize("distinct", [False, True])
@pytest.mark.parametrize("seed,kind,draft,sizes,V,most,rules,pad", [
    (0, "f32", "f32", [6], 50257, 1, dict(top_p=0.9), 0), (1, "bf16", "bf16", [5, 0, 9, 1], 1003, 3, "mixed", 1), (2, "f16", "f32", [12, 7], 4097, 4, dict(), 3),
    (3, "f32", "f16", [40] * 4, 300, 5, "mixed", 0), (4, "f32", "f32", [30, 30], 8, 6, dict(), 1), (5, "bf16", "f32", [3] * 60, 2000, 2, dict(temperature=0.7), 0),
    (6, "f32", "bf16", [200], 64, 20, dict(top_k=20), 0), (7, "f32", "f32", [8, 8], 128000, 2, "mixed", 0), (8, "f32", "f32", [5], 40, 4, dict(temperature=0.0), 0)])
def test_verification(seed, kind, draft, sizes, V, most, rules, pad, distinct):
    from llm_decoder import DraftTree, sampling
    rng = np.random.default_rng(seed)
    parents = [tree_of(rng, n, min(most, V - 1)) if n else [] for n in sizes]
    R = sum(sizes)
    c = Case(seed, kind, R, V, rules, pad)
    seq = [b for b, n in enumerate(sizes) for _ in range(n)]
    first = np.concatenate([[0], np.cumsum(sizes)])
    near = c.x.astype(np.float64) + rng.standard_normal((R, V)) * 0.8
    q = np.exp(near - near.max(1, keepdims=True))
    q /= q.sum(1, keepdims=True)
    qd = torch.from_numpy(q.astype(np.float32)).to(TYPES[draft])
    q = qd.double().numpy()
    kids = [[int(first[b]) + i for i, p in enumerate(parents[b]) if p == r - first[b]] for r, b in enumerate(seq)]
    tokens = rng.integers(0, V, R)
    for r in range(R):
        if kids[r]:
            pool = q[r] / q[r].sum()
            some = rng.choice(V, len(kids[r]), replace=not distinct or np.count_nonzero(pool) < len(kids[r]), p=pool)
            tokens[kids[r]] = some
    if R > 20:
        tokens[R - 1] = V + 3           # no token of the vocabulary
    # every second node's distribution at another place, some nodes' children not by chance
    rank = np.array([r if rng.random() < 0.9 else rng.choice([-1, R + 5]) for r in range(R)], dtype=np.int32)
    order = rng.permutation(R)
    where = np.empty(R, dtype=np.int32)
    where[order] = np.arange(R)
    rows = np.where((rank >= 0) & (rank < R), where[np.clip(rank, 0, R - 1)], rank).astype(np.int32)
    numbers = rng.random((R, 2)).astype(np.float32)
    tree = DraftTree(parents, [tokens[first[b]:first[b + 1]].tolist() for b in range(len(sizes))], "cuda")
    wide = torch.full((R, V + pad), float("nan"), dtype=qd.dtype).cuda()
    wide[:, :V] = qd[torch.from_numpy(order)].cuda()
    kw = {k: (v[:len(sizes)].contiguous() if isinstance(v, torch.Tensor) else v) for k, v in c.kw.items()}
    ids, logs = sampling.verify_drafts(c.dev, tree, torch.from_numpy(numbers).cuda(), wide[:, :V], draft_rows=torch.from_numpy(rows).cuda(), distinct=distinct,
                                       logprobs=True, **kw)
    again = sampling.verify_drafts(c.dev, tree, torch.from_numpy(numbers).cuda(), wide[:, :V], draft_rows=torch.from_numpy(rows).cuda(), distinct=distinct, **kw)
    assert torch.equal(ids, again)
    plain = sampling.draw_tokens(c.dev, torch.from_numpy(numbers[:, 1].copy()).cuda(), tree=tree, **kw).cpu().numpy()
    ids, logs, unclear = ids.cpu().numpy(), logs.cpu().numpy(), 0
    for r in range(R):
        w = c.weights(r, seq[r])
        chance = 0 <= rank[r] < R
        token, rest, clear = verified(w, kids[r] if chance else [], tokens, q[r], numbers[:, 0], numbers[:, 1], distinct)
        if not clear:
            unclear += 1
            continue
        if token is not None:
            assert ids[r] == token
        else:               # what is left may be small: its sums are off by the bound of what it was
            cum, at = np.cumsum(rest), ids[r]
            target, eps = numbers[r, 1] * cum[-1], 1e-9 * cum[-1]
            assert rest[at] > -eps and cum[at] - rest[at] - eps <= target < cum[at] + eps
        if not chance or not kids[r]:
            assert ids[r] == plain[r]
        lp = math.log(w[ids[r]] / w.sum())
        assert abs(logs[r] - lp) <= abs(lp) * 2.0 ** -24 + 3e-12
    assert unclear <= R // 20


@pytest.mark.gpu
@pytest.mark.parametrize("distinct,most", [(False, 1), (False, 3), (True, 3)])
def test_ids_are_distributed_as_the_model(distinct, most):
    """40000 sequences with one root, whose children are drawn from q: the roots' ids follow p.  A share of 40000 draws is off by more than six of its
    deviations once in 5e8."""
    from llm_decoder import DraftTree, sampling
    n, V = 40000, 9
    rng = np.random.default_rng(5)
    x = rng.standard_normal(V).astype(np.float32) * 1.5
    q = rng.dirichlet(np.ones(V)).astype(np.float32)
    g = torch.Generator(device="cuda").manual_seed(7)
    logits = torch.from_numpy(np.log(q)).cuda().expand(n, V).contiguous()
    kids = sampling.draw_tokens(logits, torch.rand(n, most, device="cuda", generator=g)) if distinct else \
        torch.stack([sampling.draw_tokens(logits, torch.rand(n, device="cuda", generator=g)) for _ in range(most)], 1)
    kids = kids.cpu().numpy()
    if distinct:
        assert all(len(set(k)) == most for k in kids.tolist())
    tree = DraftTree([[-1] + [0] * most] * n, [[0, *k] for k in kids.tolist()], "cuda")
    target = torch.from_numpy(x).cuda().expand(tree.rows, V).contiguous()
    rows = torch.full((tree.rows,), -1, dtype=torch.int32, device="cuda")
    rows[::most + 1] = 0
    ids = sampling.verify_drafts(target, tree, torch.rand(tree.rows, 2, device="cuda", generator=g), torch.from_numpy(q).cuda()[None], draft_rows=rows,
                                 distinct=distinct, top_k=7)[::most + 1]
    w = kept_weights(x, top_k=7)
    p = w / w.sum()
    share = np.bincount(ids.cpu().numpy(), minlength=V) / n
    assert np.all(np.abs(share - p) <= 6 * np.sqrt(p * (1 - p) / n)) and np.all(share[p == 0] == 0)


# ---------------------------------------------------------------------------------------------------------------- refusals
def test_refused_on_the_host():
    from llm_decoder import _cabi, sampling
    x = torch.zeros(3, 10)
    for call in (lambda: sampling.truncated_softmax(x), lambda: sampling.draw_tokens(x, torch.zeros(3))):
        with pytest.raises(ValueError):
            call()
    lib, ref = _cabi.lib(), __import__("ctypes").byref
    rules, ws = _cabi.DrawRules(num_seqs=4, temperature=1.0, top_p=1.0), (0x10000, 1 << 30)
    assert lib.pa_draw_workspace_bytes(0, 4, 8, 0) > 0 and lib.pa_draw_workspace_bytes(0, 0, 8, 0) == lib.pa_draw_workspace_bytes(3, 4, 8, 0) == 0
    assert lib.pa_truncated_softmax(None, 0, 8, 4, 8, ref(rules), 0x1000, 8, *ws, None) == -1
    assert lib.pa_truncated_softmax(0x1000, 0, 7, 4, 8, ref(rules), 0x9000, 8, *ws, None) == -1
    assert lib.pa_truncated_softmax(0x1000, 0, 8, 4, 8, ref(rules), 0x9000, 7, *ws, None) == -1
    assert lib.pa_draw_tokens(0x1000, 0, 8, 2 ** 30 + 1, 8, ref(rules), 0x8000, 1, 0x9000, None, *ws, None) == -1
    assert lib.pa_truncated_softmax(0x1000, 0, 8, 4, 8, ref(rules), 0x1040, 8, *ws, None) == -1          # overlaps
    assert lib.pa_truncated_softmax(0x1002, 0, 8, 4, 8, ref(rules), 0x9000, 8, *ws, None) == -1          # no address of a float
    assert lib.pa_truncated_softmax(0x1000, 0, 8, 4, 8, None, 0x9000, 8, *ws, None) == -1
    assert lib.pa_truncated_softmax(0x1000, 0, 8, 0, 8, ref(rules), None, 8, *ws, None) == 0
    assert lib.pa_truncated_softmax(0x1000, 3, 8, 4, 8, ref(rules), 0x9000, 8, *ws, None) == -2
    assert lib.pa_draw_tokens(0x1000, 0, 8, 4, 8, ref(rules), None, 1, 0x9000, None, *ws, None) == -1
    assert lib.pa_draw_tokens(0x1000, 0, 8, 4, 8, ref(rules), 0x8000, 0, 0x9000, None, *ws, None) == -1
    assert lib.pa_draw_tokens(0x1000, 0, 8, 4, 0, ref(rules), 0x8000, 1, 0x9000, None, *ws, None) == -1
    assert lib.pa_draw_tokens(0x1000, 0, 8, 4, 8, ref(rules), 0x8000, 1, 0x9000, None, 0x10000, 8, None) == -3
    assert lib.pa_draw_tokens(0x1000, 0, 8, 4, 8, ref(rules), 0x8000, 1, 0x9000, None, None, 1 << 30, None) == -3
    tree = (0x2000, 0x3000, 0x4000)
    assert lib.pa_verify_drafts(0x1000, 0, 8, 4, 8, ref(rules), 0x8000, *tree, 2, 0x5000, 0, 8, 4, None, 0, 0x9000, None, *ws, None) == -1      # no row_seq
    rules.row_seq = 0x6000
    assert lib.pa_verify_drafts(0x1000, 0, 8, 4, 8, ref(rules), 0x8000, *tree, 2, 0x5000, 0, 8, 3, None, 0, 0x9000, None, *ws, None) == -1      # rows without one
    assert lib.pa_verify_drafts(0x1000, 0, 8, 4, 8, ref(rules), 0x8000, *tree, 2, 0x5000, 0, 7, 4, None, 0, 0x9000, None, *ws, None) == -1
    assert lib.pa_verify_drafts(0x1000, 0, 8, 4, 8, ref(rules), 0x8000, *tree, 2, 0x5000, 3, 8, 4, None, 0, 0x9000, None, *ws, None) == -2
    assert lib.pa_verify_drafts(0x1000, 0, 8, 4, 8, ref(rules), 0x8000, *tree, 2, 0x5002, 0, 8, 4, None, 0, 0x9000, None, *ws, None) == -1      # no address of a float
    assert lib.pa_draw_workspace_bytes(0, 1, 375001, 0) == lib.pa_draw_workspace_bytes(1, 1, 2 ** 31 - 1, 0) == 0
    assert lib.pa_draw_tokens(0x1000, 0, 375001, 1, 375001, ref(rules), 0x8000, 1, 0x9000, None, *ws, None) == -2


@pytest.mark.gpu
def test_refused_tensors():
    from llm_decoder import DraftTree, sampling
    x, u = torch.zeros(3, 10, device="cuda"), torch.zeros(3, device="cuda")
    f, i = torch.float32, torch.int32
    of = lambda n, t: torch.ones(n, dtype=t, device="cuda")  # noqa: E731
    tree = DraftTree([[-1, 0], [-1]], [[1, 2], [3]], "cuda")
    bad = [dict(temperature=-1.0), dict(top_k=-1), dict(top_p=float("nan")), dict(min_p=1.5), dict(temperature=of(2, f)), dict(top_k=of(3, f)),
           dict(top_p=of(3, f).cpu()), dict(row_seq=of(2, i)), dict(row_seq=of(3, f)), dict(tree=DraftTree([[-1]], device="cuda")), dict(tree=tree, row_seq=of(3, i)),
           dict(temperature=of(2, f), top_p=of(3, f), row_seq=of(3, i))]
    for kw in bad:
        for call in (sampling.truncated_softmax, lambda x, **kw: sampling.draw_tokens(x, u, **kw)):
            with pytest.raises(ValueError):
                call(x, **kw)
    for logits in (x.double(), x[0], x.t(), torch.zeros(2, 3, 4, device="cuda"), torch.zeros(1, 400000, device="cuda"), torch.zeros(1, 10, device="cuda").expand(3, 10)):
        with pytest.raises(ValueError):
            sampling.truncated_softmax(logits)
    for numbers in (u.double(), u[:2], u.cpu(), torch.zeros(3, 2, 2, device="cuda"), torch.zeros(3, 4, device="cuda")[:, :2]):
        with pytest.raises(ValueError):
            sampling.draw_tokens(x, numbers)
    for out in (x.half(), x[:2], torch.zeros(10, 3, device="cuda").t()):
        with pytest.raises(ValueError):
            sampling.truncated_softmax(x, out=out)
    with pytest.raises(Exception):
        sampling.truncated_softmax(x, out=x)
    pair, q = torch.zeros(3, 2, device="cuda"), torch.full((3, 10), 0.1, device="cuda")
    assert sampling.verify_drafts(x, tree, pair, q).shape == (3,)
    for args in ((x, DraftTree([[-1, 0], [-1]], device="cuda"), pair, q), (x, tree, u, q), (x, tree, pair, q[:2]), (x, tree, pair, q[:, :9]), (x, tree, pair, q.double()),
                 (x, tree, pair, q.cpu()), (x[:2], tree, pair, q)):
        with pytest.raises(ValueError):
            sampling.verify_drafts(*args)
    for rows in (of(2, i), of(3, f), of(3, i).cpu()):
        with pytest.raises(ValueError):
            sampling.verify_drafts(x, tree, pair, q, draft_rows=rows)
    empty = torch.zeros(0, 10, device="cuda")
    assert sampling.truncated_softmax(empty).shape == (0, 10) and sampling.draw_tokens(empty, torch.zeros(0, device="cuda")).shape == (0,)
    assert sampling.draw_tokens(x, torch.zeros(3, 0, device="cuda")).shape == (3, 0)


@pytest.mark.gpu
def test_more_children_than_said():
    """Children beyond the number that the call was told count as not there."""
    from llm_decoder import DraftTree, _cabi, sampling
    g = torch.Generator(device="cuda").manual_seed(4)
    n, V = 200, 50
    x, q = torch.randn(3 * n, V, device="cuda", generator=g), torch.rand(3 * n, V, device="cuda", generator=g)
    q /= q.sum(1, keepdim=True)
    u, tokens = torch.rand(3 * n, 2, device="cuda", generator=g), np.random.default_rng(1).integers(0, V, (n, 2)).tolist()
    tree = DraftTree([[-1, 0, 0]] * n, [[0, *t] for t in tokens], "cuda")
    ids, ws = torch.full((3 * n,), -7, dtype=torch.int32, device="cuda"), torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    rules = _cabi.DrawRules(num_seqs=n, temperature=1.0, top_p=1.0)
    rules.row_seq = tree.row_seq.data_ptr()
    _cabi.check(_cabi.lib().pa_verify_drafts(x.data_ptr(), 0, V, 3 * n, V, __import__("ctypes").byref(rules), u.data_ptr(), tree.tokens.data_ptr(), tree.parents.data_ptr(),
                                             tree.node_start.data_ptr(), 1, q.data_ptr(), 0, V, 3 * n, None, 0, ids.data_ptr(), None, ws.data_ptr(), ws.numel(),
                                             _cabi.stream()), "pa_verify_drafts")
    keep = torch.arange(3 * n, device="cuda").view(n, 3)[:, :2].reshape(-1)
    fewer = DraftTree([[-1, 0]] * n, [[0, t[0]] for t in tokens], "cuda")
    want = sampling.verify_drafts(x[keep].contiguous(), fewer, u[keep].contiguous(), q[keep].contiguous())
    assert torch.equal(ids[keep], want) and int(ids.min()) >= 0


@pytest.mark.gpu
def test_two_calls_at_once():
    """Calls of several host threads on streams of their own, and captured calls that are replayed beside each other, give what each gives alone."""
    import threading

    from llm_decoder import sampling
    g = torch.Generator(device="cuda").manual_seed(11)
    cases = [(torch.randn(n, v, device="cuda", generator=g) * 2, torch.rand(n, 2, device="cuda", generator=g), kw)
             for n, v, kw in ((70, 30011, dict(top_p=0.9)), (3, 128000, dict(top_k=300)), (150, 9000, dict(temperature=0.5)), (33, 50257, dict(top_k=40, top_p=0.8)))]
    want = [(sampling.draw_tokens(x, u, **kw), sampling.truncated_softmax(x, **kw)) for x, u, kw in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        x, u, kw = cases[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                ids, probs = sampling.draw_tokens(x, u, **kw), sampling.truncated_softmax(x, **kw)
                if not torch.equal(ids, want[i][0]) or not torch.equal(probs, want[i][1]):
                    wrong.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    graphs, got, streams = [], [], [torch.cuda.Stream() for _ in range(4)]
    for x, u, kw in cases:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append((sampling.draw_tokens(x, u, **kw), sampling.truncated_softmax(x, **kw)))
    torch.cuda.synchronize()
    for _ in range(10):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


# ---------------------------------------------------------------------------------- rows with thousands of tokens next to the border
def steps_of(x, temperature):
    """Which step of 1/32 (of log2 w, or of a logit where these are smaller) every token of a row lies in, counted from the largest."""
    fine = np.float32(max(1.4426950408889634 / temperature * 32, 32.0)) * np.float32(16)
    part = np.rint(x.astype(np.float64) * np.float64(fine)).astype(np.int64)
    return ((part.max() | 15) - part) // 16


@pytest.mark.gpu
@pytest.mark.parametrize("seed,kind,V,spread,rules", [
    (0, "f32", 128000, 0.3, dict(top_p=0.9)), (1, "f32", 128000, 0.4, dict(top_p=0.7, temperature=0.8)), (2, "f32", 250001, 0.9, dict(top_p=0.88, temperature=2.0)),
    (3, "f32", 300001, 1.5, dict(top_p=0.9, temperature=1.5)), (4, "f32", 128000, 0.5, dict(top_k=60000)), (5, "f32", 200003, 0.6, dict(top_k=90000, min_p=0.001)),
    (6, "f32", 128000, 0.3, dict(top_k=64000)), (7, "f16", 128000, 0.3, dict(top_p=0.9)), (8, "f16", 250001, 0.7, dict(top_k=100000)),
    (9, "bf16", 160000, 0.35, dict(top_p=0.85)), (10, "bf16", 128000, 0.5, dict(top_k=70000))])
def test_many_tokens_next_to_the_border(seed, kind, V, spread, rules):
    """More than 2048 tokens of a row in the border's step, at most 1024 of any 8192 neighbours: narrowed down among themselves, counted or weighed, and
    summed from their list.  The same each time."""
    from llm_decoder import sampling
    c = Case(seed, kind, 3, V, rules, spread=spread)
    u = torch.from_numpy(c.numbers[:, 0].copy()).cuda()
    t = c.rules.get("temperature", np.ones(3))
    probs, (ids, logs) = sampling.truncated_softmax(c.dev, **rules), sampling.draw_tokens(c.dev, u, logprobs=True, **rules)
    for _ in range(20):
        again = sampling.draw_tokens(c.dev, u, logprobs=True, **rules)
        assert torch.equal(again[0], ids) and torch.equal(again[1], logs) and torch.equal(sampling.truncated_softmax(c.dev, **rules), probs)
    probs, ids = probs.double().cpu().numpy(), ids.tolist()
    for r in range(3):
        w, step = c.weights(r), steps_of(c.x[r], t[r])
        near = step == step[w > 0].max()
        assert near.sum() > 2048
        for s in (near, np.isin(step, step[w > 0].max() + np.array([-1, 0, 1]))):
            assert max(s[i:i + 8192].sum() for i in range(0, V, 1024)) <= 1024
        p = w / w.sum()
        assert np.array_equal(probs[r] > 0, p > 0) and near_float(probs[r], p)
        assert is_drawn(w, ids[r], c.numbers[r, 0])


# -------------------------------------------------------------------------------------------------------- temperatures next to 0
SMALL = [1e-3, 1e-6, 1e-8, 1e-10, 1e-12, 1e-14, 1e-16, 1e-17, 1e-18, 1e-20, 1e-22, 1e-24, 1e-40, 1e-310, 5e-324]


@pytest.mark.gpu
@pytest.mark.parametrize("top_p", [1.0, 0.9])
@pytest.mark.parametrize("at", [3.3, 28.7, -1e10])
def test_every_id_is_written(at, top_p):
    """Ids in memory that holds something else before the call are tokens or -1 after it."""
    import ctypes

    from llm_decoder import DraftTree, _cabi
    V, rows = 9001, 12
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn(rows, V, device="cuda", generator=g) + at - 3.3
    x[::2, 77] = at + 1
    q = torch.softmax(x + torch.randn(rows, V, device="cuda", generator=g), 1)
    u, ws = torch.rand(rows, 3, device="cuda", generator=g), torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    tree = DraftTree([[-1, 0, 0, 1]] * 3, [[0, 77, 5, 9]] * 3, "cuda")
    lib = _cabi.lib()
    for t in SMALL:
        ids, one = (torch.full(s, -7, dtype=torch.int32, device="cuda") for s in ((rows, 3), (rows,)))
        rules = _cabi.DrawRules(num_seqs=rows, temperature=t, top_p=top_p)
        _cabi.check(lib.pa_draw_tokens(x.data_ptr(), 0, V, rows, V, ctypes.byref(rules), u.data_ptr(), 3, ids.data_ptr(), None, ws.data_ptr(), ws.numel(),
                                       _cabi.stream()), "pa_draw_tokens")
        rules.row_seq = tree.row_seq.data_ptr()
        _cabi.check(lib.pa_verify_drafts(x.data_ptr(), 0, V, rows, V, ctypes.byref(rules), u.data_ptr(), tree.tokens.data_ptr(), tree.parents.data_ptr(),
                                         tree.node_start.data_ptr(), 2, q.data_ptr(), 0, V, rows, None, 0, one.data_ptr(), None, ws.data_ptr(), ws.numel(),
                                         _cabi.stream()), "pa_verify_drafts")
        for got in (ids, one):
            assert int(got.min()) >= -1 and int(got.max()) < V, t


@pytest.mark.gpu
@pytest.mark.parametrize("rules", [dict(), dict(top_p=0.9), dict(top_k=5), dict(min_p=0.2), dict(top_k=400, top_p=0.7)])
@pytest.mark.parametrize("kind,at", [("f32", 3.3), ("f32", 28.7), ("f32", 1e4), ("f32", -1e10), ("f32", 1e20), ("f32", -3e38), ("bf16", 28.7), ("bf16", 1e20),
                                     ("f16", -1e4)])
def test_small_temperatures_and_large_logits(kind, at, rules):
    """Weights are those of the differences from the largest logit, however small the temperature or large the logits: as numbers and per sequence, with rules
    and without.  (Where what is left weighs less than 2^-960 of all, a float64 of the definition has no full precision: not looked at.)"""
    from llm_decoder import DraftTree, sampling
    rows, V = 6, 20001
    c = Case(17, kind, rows, V, dict(rules), 1, 1)
    x = torch.from_numpy(c.x) / 3 * (3 if abs(at) < 100 else abs(at) * (1e-6 if kind == "f32" else 0.01)) + at
    c.dev.copy_(x.clamp(-c.most, c.most).to(TYPES[kind]))
    c.x = c.dev.float().cpu().numpy()
    u = torch.from_numpy(c.numbers[:, :3].copy()).cuda()
    q = np.full((rows, V), 0.5 / V)
    q[:, 11] += 0.25
    q[np.arange(rows), np.argmax(c.x, 1)] += 0.25
    qd = torch.from_numpy(q.astype(np.float32)).cuda()
    q = qd.double().cpu().numpy()
    parents, tokens = [-1, 0, 0, 1, 1, 2], [0, 11, int(np.argmax(c.x[0])), int(np.argmax(c.x[1])), 11, 300]
    tree, kids = DraftTree([parents], [tokens], "cuda"), [[1, 2], [3, 4], [5], [], [], []]
    pair = torch.from_numpy(c.numbers[:, 3:5].copy()).cuda()
    some = [1.0, abs(at) * 1e-6, abs(at) * 1e-8, *SMALL]
    for form in ("number", "each"):
        temperatures = [float(np.float32(t)) for t in some if np.float32(t) > 0] if form == "each" else some
        for i, t in enumerate(temperatures):
            each = np.full(rows, t)
            kw = dict(rules, temperature=t)
            if form == "each":
                each = np.roll(np.array(temperatures), -i)[:rows].astype(np.float32)
                kw["temperature"] = torch.from_numpy(each).cuda()
            c.rules["temperature"] = each
            probs = sampling.truncated_softmax(c.dev, **kw).double().cpu().numpy()
            ids, logs = (y.cpu().numpy() for y in sampling.draw_tokens(c.dev, u, logprobs=True, **kw))
            for r in range(rows):
                w = c.weights(r)
                p = w / w.sum()
                assert near_float(probs[r], p), (t, r)
                for k, token in enumerate(ids[r]):
                    if w.sum() < 2.0 ** -960 * p.max():
                        break
                    assert is_drawn(w, token, c.numbers[r, k]), (t, r, k)
                    assert abs(float(logs[r, k]) - math.log(p[token])) <= abs(math.log(p[token])) * 2.0 ** -24 + 3e-12
                    w = w.copy()
                    w[token] = 0
            if form == "each":
                kw["temperature"] = kw["temperature"][:1].contiguous()
            got = sampling.verify_drafts(c.dev, tree, pair, qd, **kw).tolist()
            for r in range(rows):
                w = kept_weights(c.x[r], most=c.most, temperature=each[0], **rules)
                token, rest, clear = verified(w, kids[r], tokens, q[r], c.numbers[:, 3], c.numbers[:, 4], False)
                if clear and token is not None:
                    assert got[r] == token, (t, r)
                elif clear:
                    at_id, cum = got[r], np.cumsum(rest)
                    target, eps = np.float64(c.numbers[r, 4]) * cum[-1], 1e-9 * cum[-1]
                    assert rest[at_id] > 0 and cum[at_id] - rest[at_id] - eps <= target < cum[at_id] + eps, (t, r)


def test_logits_of_no_rows_are_refused():
    """Logits that are no matrix raise what other wrong arguments raise, with `out` and without."""
    from llm_decoder import sampling
    for shape in ((10,), (), (2, 3, 4)):
        x = torch.zeros(shape)
        for call in (lambda: sampling.truncated_softmax(x), lambda: sampling.truncated_softmax(x, out=torch.zeros(shape)), lambda: sampling.draw_tokens(x, torch.zeros(10)),
                     lambda: sampling.verify_drafts(x, None, torch.zeros(10, 2), torch.zeros(10, 10))):
            with pytest.raises(ValueError):
                call()


@pytest.mark.gpu
@pytest.mark.parametrize("distinct", [False, True])
@pytest.mark.parametrize("seed,kind,V,rules", [(0, "f32", 5001, dict(top_k=30)), (1, "bf16", 20000, dict(top_p=0.8, temperature=1.3)), (2, "f16", 300, dict(min_p=0.05)),
                                               (3, "f32", 60001, dict(top_k=400, top_p=0.9)), (4, "f32", 12, dict())])
def test_replacements_are_what_refused_children_leave(seed, kind, V, rules, distinct):
    """Where every child is refused, the id has weight by the rules and in what the children have left: none that the rules leave out, and none of which
    the draft gave more than the model does."""
    from llm_decoder import DraftTree, sampling
    rng = np.random.default_rng(seed)
    B, kids = 40, 3
    c = Case(seed, kind, B * (kids + 1), V, rules)
    roots = np.arange(B) * (kids + 1)
    q, tokens = np.zeros((B, V)), np.zeros((B, kids + 1), dtype=np.int64)
    for b, r in enumerate(roots):       # drafts that like what the model likes less: many children are refused
        w = c.weights(r)
        some = rng.permutation(V)[:min(V, 6)]
        q[b, some] = rng.random(len(some)) + 0.1
        q[b, rng.choice(np.flatnonzero(w > 0), 3)] += rng.random(3)
        q[b] /= q[b].sum()
        tokens[b, 1:] = rng.choice(V, kids, replace=False, p=q[b])
    qd = torch.from_numpy(q.astype(np.float32)).cuda()
    q = qd.double().cpu().numpy()
    rows = torch.full((len(c.x),), -1, dtype=torch.int32)
    rows[::kids + 1] = torch.arange(B, dtype=torch.int32)
    numbers = np.concatenate([rng.random((len(c.x), 1)) ** 0.25, rng.random((len(c.x), 1))], 1).astype(np.float32)
    tree = DraftTree([[-1, 0, 0, 0]] * B, tokens.tolist(), "cuda")
    ids = sampling.verify_drafts(c.dev, tree, torch.from_numpy(numbers).cuda(), qd, draft_rows=rows.cuda(), distinct=distinct, **rules).tolist()
    replaced = 0
    for b, r in enumerate(roots):
        w = c.weights(r)
        token, rest, clear = verified(w, list(range(r + 1, r + kids + 1)), tokens.reshape(-1), q[b], numbers[:, 0], numbers[:, 1], distinct)
        if clear and token is None:
            replaced += 1
            cum, at = np.cumsum(rest), ids[r]
            target, eps = numbers[r, 1] * cum[-1], 1e-9 * cum[-1]
            assert w[at] > 0 and rest[at] > 0 and cum[at] - rest[at] - eps <= target < cum[at] + eps
        elif clear:
            assert ids[r] == token
    assert replaced >= B // 4


@pytest.mark.gpu
@pytest.mark.parametrize("top_p", [0.3, 0.9, 0.99])
@pytest.mark.parametrize("kind,at,V", [("f16", 1000, 300), ("f16", 1000, 30001), ("f16", -1000, 5000), ("f16", 30000, 7), ("f16", -60000, 20000), ("bf16", 100, 30001),
                                       ("bf16", 1000, 9000), ("bf16", -1e4, 500), ("bf16", 1e6, 40000), ("f32", 1e6, 9000)])
def test_coarse_logits_far_from_zero(kind, at, V, top_p):
    """Logits with a common offset, next to which their type has few values: a share of them is that of the definition where the least value with a weight is
    none of the type.  Temperatures from half a step of the type to 30 of them."""
    from llm_decoder import sampling
    rows = 40
    step = 2.0 ** (math.floor(math.log2(abs(at))) + 1) * {"f32": 2.0 ** -23, "f16": 2.0 ** -10, "bf16": 2.0 ** -7}[kind] / 2
    c = Case(23, kind, rows, V, dict(top_p=top_p))
    g = torch.from_numpy(np.random.default_rng(2).standard_normal((rows, V)) * step * 2 + at)
    c.dev.copy_(g.clamp(-c.most, c.most).float().to(TYPES[kind]))
    c.x = c.dev.float().cpu().numpy()
    c.rules["temperature"] = np.exp(np.linspace(math.log(step / 2), math.log(step * 30), rows)).astype(np.float32)
    kw = dict(top_p=top_p, temperature=torch.from_numpy(c.rules["temperature"]).cuda())
    probs = sampling.truncated_softmax(c.dev, **kw).double().cpu().numpy()
    ids = sampling.draw_tokens(c.dev, torch.from_numpy(c.numbers[:, 0].copy()).cuda(), **kw).tolist()
    for r in range(rows):
        w = c.weights(r)
        p = w / w.sum()
        assert np.array_equal(probs[r] > 0, p > 0) and near_float(probs[r], p), r
        assert is_drawn(w, ids[r], c.numbers[r, 0]), r


def test_limits_are_those_of_the_library():
    """Where Python refuses, the library does."""
    from llm_decoder import _cabi, device_pages, sampling
    lib, most = _cabi.lib(), sampling._MOST_ROW_BYTES
    for kind, size in ((0, 4), (1, 2), (2, 2)):
        assert lib.pa_draw_workspace_bytes(kind, 1, most // size, 0) > 0 and lib.pa_draw_workspace_bytes(kind, 1, most // size + 1, 0) == 0
    n = device_pages.MOST_SEQS + 1
    table = (0x1000, n, 2, 4, 16, 8, 0x2000, 0x3000, 0x4000)
    assert lib.pa_take_pages(*table, 0x5000, 0x6000, n, 1, 0x7000, 0x8000, 0x9000, None) == lib.pa_release_pages(*table, 0x5000, n, None) == -2
