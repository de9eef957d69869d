"""Generation with drafted trees whose tokens are drawn by chance: rows, attention, logits, draws, verification, acceptance and pages together."""
import json

import numpy as np
import pytest
import torch

from test_draw_tokens import EPS, kept_weights
from test_generate_drafted import TOL, decoder, one_by_one


def numbers_of(seed, batch, n):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.rand((batch, n), device="cuda", generator=g).cpu().numpy()


def check_drawn(dec, got, n, seed, temperature, **kw):
    """Every token is drawn by its number from the logits that its own predecessors give, one by one, up to their rounding: a logit that is off by
    d moves every weight, and the sum, by at most 2 d / temperature of itself, and a border of the cumulative sums by twice that (of kept sets alone:
    where a border of the truncation lies as near, the token next to it may be in or out)."""
    logits = one_by_one(dec, got, n)
    u = numbers_of(seed, len(got), len(got[0]) - n)
    tol, t = TOL[type(dec).__name__], temperature if dec.ARGMAX_DIVIDE else 1 / temperature
    misses = 0
    for b, (s, rows) in enumerate(zip(got, logits)):
        for i, (token, row) in enumerate(zip(s[n:], rows)):
            w = kept_weights(row, temperature=t, **kw)
            cum = np.cumsum(w) / w.sum()
            near = EPS + 8 * tol * np.abs(row[np.isfinite(row)]).max() / t
            if w[token] == 0 or not cum[token] - w[token] / w.sum() - near <= u[b, i] < cum[token] + near:
                misses += 1
    assert misses <= (0 if not kw else len(got) * len(got[0]) // 50)


@pytest.mark.gpu
@pytest.mark.parametrize("cls,batch,kv_tokens", [("CUDADecoder", 3, None), ("CUDADecoder", 10, 10 * 64), ("INT8Decoder", 2, 128), ("INT8Decoder", 9, None)])
def test_tokens_are_drawn_whatever_is_guessed(tmp_path, cls, batch, kv_tokens):
    rng = np.random.default_rng(batch)
    dec = decoder(cls, tmp_path, 5, 97, 2, 64, batch_size=batch, kv_tokens=kv_tokens)
    prompts = rng.integers(0, 97, (batch, 6)).tolist()
    for kw in (dict(temperature=0.7), dict(temperature=1.3, top_p=0.8), dict(temperature=1.0, top_k=9, min_p=0.02)):
        for more in (dict(drafts=0), dict(drafts=20, branches=4)):
            got = dec.generate_drafted(prompts, 40, seed=11, **kw, **more)
            assert [s[:6] for s in got] == prompts and all(len(s) == 46 for s in got) and dec.drafted_steps_ <= 40
            check_drawn(dec, got, 6, 11, **kw)
    greedy = dec.generate_drafted(prompts, 40)
    assert dec.ARGMAX_DIVIDE == 0 or greedy == dec.generate_drafted(prompts, 40, temperature=0.0)
    assert dec.generate_drafted(prompts, 12, seed=3, temperature=0.9) != dec.generate_drafted(prompts, 12, seed=4, temperature=0.9)


@pytest.mark.gpu
@pytest.mark.parametrize("distinct", [False, True])
def test_a_draft_model(tmp_path, distinct):
    """Guesses drawn from a distribution that knows the tokens' own, more or less: many of them are kept, and what comes is possible."""
    from llm_decoder import sampling
    V, n = 61, 4
    dec = decoder("CUDADecoder", tmp_path, 6, V, 2, 64, batch_size=2)
    g = torch.Generator(device="cuda").manual_seed(2)
    prompts = [[1, 2, 3, 4], [9, 8, 7, 6]]
    q = torch.softmax(torch.randn(V, device="cuda", generator=g), 0)

    def draft(tokens, most, depth):
        parents, out, level = [-1], [int(tokens[-1])], [0]
        for _ in range(min(depth - 1, 3)):
            here = []
            for node in level:
                kids = 2 if len(out) + 2 <= most else 0
                if kids:
                    u = torch.rand(1, kids, device="cuda", generator=g)
                    x = q.log().expand(1, V).contiguous()
                    drawn = sampling.draw_tokens(x, u)[0] if distinct else torch.stack([sampling.draw_tokens(x, u[:, i].contiguous())[0] for i in range(kids)])
                    for t in drawn.tolist():
                        here.append(len(out))
                        parents.append(node)
                        out.append(t)
            level = here
        return parents, out, q.expand(len(out), V)
    got = dec.generate_drafted(prompts, 60, drafts=14, draft=draft, temperature=2.0, top_k=30, seed=1, distinct=distinct)
    assert all(len(s) == n + 60 for s in got) and dec.drafted_steps_ < 60
    logits = one_by_one(dec, got, n)
    for s, rows in zip(got, logits):            # no token that the rules leave out (but within the rounding of the logits)
        for token, row in zip(s[n:], rows):
            assert row[token] >= np.sort(row)[-30] - TOL["CUDADecoder"] * np.abs(row).max()
    for bad in (lambda t, m, d: ([-1], [int(t[-1])], q[None, :-1]), lambda t, m, d: ([-1], [int(t[-1])], None)):
        with pytest.raises(ValueError):
            dec.generate_drafted(prompts, 5, draft=bad, temperature=1.0)
    with pytest.raises(ValueError):
        dec.generate_drafted(prompts, 5, draft=lambda t, m, d: ([-1], [int(t[-1])], q[None]))
    with pytest.raises(ValueError):
        dec.generate_drafted(prompts, 5, top_p=0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("cls", ["CUDADecoder", "INT8Decoder"])
def test_pools_for_fewer_tokens(tmp_path, cls):
    """Pages handed out on the GPU: the same tokens as with pages for every tile, in captured steps too; too few raise, and the next call is as before."""
    whole = decoder(cls, tmp_path, 7, 97, 2, 64, batch_size=2)
    few = decoder(cls, tmp_path, 7, 97, 2, 64, batch_size=2, kv_tokens=2 * 64)
    assert few.kv_caches[0].total_pages_ == 2 * 8 and whole.kv_caches[0].total_pages_ > 16
    prompts = [[3, 5, 7, 11, 13], [2, 4, 6, 8, 10]]
    want = whole.generate_batch(prompts, 50)
    for _ in range(2):
        assert few.generate_batch(prompts, 50) == want
    few.use_prefill = whole.use_prefill = False
    assert few.generate_batch(prompts, 50) == whole.generate_batch(prompts, 50)
    few.use_prefill = whole.use_prefill = True
    assert few.generate_drafted(prompts, 50) == whole.generate_drafted(prompts, 50)
    for call in (lambda: few.generate_batch(prompts, 100), lambda: few.generate_drafted(prompts, 100)):
        with pytest.raises(RuntimeError):
            call()
        assert few.generate_batch(prompts, 50) == want
    few.reset()
    assert few.pages.free_pages() == 16
    with pytest.raises(ValueError):
        decoder(cls, tmp_path, 7, 97, 2, 64, kv_tokens=0)


@pytest.mark.gpu
def test_rules_masks_and_chance(tmp_path):
    """Penalties, biases and masks apply to what is drawn from; a mask that leaves nothing is an error, not a token."""
    dec = decoder("CUDADecoder", tmp_path, 8, 97, 2, 64, batch_size=2)
    prompts = [[3, 5, 7], [2, 4, 6]]
    ok = np.zeros((2, 4), dtype=np.int32)
    ok[0, 0], ok[1, 1] = 0b11110, 0b110
    got = dec.generate_drafted(prompts, 30, temperature=1.5, allowed=ok, repetition=1.2, seed=5)
    assert {t for t in got[0][3:]} <= {1, 2, 3, 4} and {t for t in got[1][3:]} <= {33, 34}
    assert got == dec.generate_drafted(prompts, 30, temperature=1.5, allowed=ok, repetition=1.2, seed=5, drafts=0)
    ok[1] = 0
    with pytest.raises(RuntimeError):
        dec.generate_drafted(prompts, 30, temperature=1.5, allowed=ok)


@pytest.mark.gpu
def test_a_step_that_needs_no_host(tmp_path):
    """Room for drafted rows, their K/V, attention, draws, acceptance and the pages that go back, captured once and replayed: what the same calls give one by
    one, for lengths that only the GPU knows."""
    import llm_decoder as ld
    H, D, V, tiles, parents = 2, 64, 101, 6, [[-1, 0, 1, 1], [-1, 0, 0, 2]]

    def run(captured):
        kv = ld.KVTileCache("f16")
        kv.init(2 * H * tiles, 16, D)
        kv.configure_table(2, H, tiles)
        pages = kv.pages_on_device()
        g = torch.Generator(device="cuda").manual_seed(9)
        ctx = torch.tensor([3, 20], dtype=torch.int32, device="cuda")
        pages.take([0, 0], torch.tensor([0, 3, 23], dtype=torch.int32, device="cuda"), 23)
        tree = ld.DraftTree(parents, [[1, 2, 3, 4], [5, 6, 7, 8]], "cuda")
        head = torch.randn(H * D, V, device="cuda", generator=g) * 0.3
        q, k, v = (torch.empty(8, H, D, device="cuda") for _ in range(3))
        u, caches, out = torch.empty(8, device="cuda"), ld.TreeCaches([kv]), []

        def step():
            new = pages.take(ctx, tree.node_start, tree.rows)
            kv.append(k, v, slots=new.slots)
            o = ld.paged_tree_attention(q, kv, tree, ctx, 8.0)
            ids = ld.sampling.draw_tokens((o.view(8, H * D) @ head), u, top_p=0.9, tree=tree)
            done = ld.tree_accept(ids, tree, caches, ctx)
            ctx.copy_(done.ctx_lens)
            pages.release(ctx)
            return done.tokens, new.slots

        def fill():
            for x in (q, k, v):
                x.copy_(torch.randn(8, H, D, device="cuda", generator=g))
            u.copy_(torch.rand(8, device="cuda", generator=g))
        fill()
        out.append([x.tolist() for x in step()])
        if captured:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                res = step()
        for _ in range(12):
            fill()
            if captured:
                graph.replay()
            else:
                res = step()
            out.append([x.tolist() for x in res] + [ctx.tolist(), kv.page_table_.device_data().tolist()])
        pages.check()
        return out
    assert run(True) == run(False)


@pytest.mark.gpu
@pytest.mark.parametrize("cls", ["CUDADecoder", "INT8Decoder"])
def test_the_command_samples(tmp_path, capsys, cls):
    from llm_decoder import cli
    dec = decoder(cls, tmp_path, 13, 97, 2, 64, max_len=128)
    config = dict(architecture=cls, num_layers=2, num_heads=2, head_dim=64, hidden_dim=128, vocab_size=97, max_seq_len=128,
                  weights="q" if cls == "INT8Decoder" else "w")
    (tmp_path / "config.json").write_text(json.dumps(config))

    def run(*args):
        assert cli.main(["generate", "--model", str(tmp_path), "--prompt", "5,17,3", "--max-new-tokens", "20", *args]) == 0
        return [[int(t) for t in line.split(",")] for line in capsys.readouterr().out.splitlines() if line[:1].isdigit()]
    want = dec.generate_drafted([[5, 17, 3]], 20, drafts=8, temperature=0.8, top_k=20, top_p=0.9, min_p=0.01, seed=6)
    assert run("--sample", "--drafts", "8", "--temperature", "0.8", "--top-k", "20", "--top-p", "0.9", "--min-p", "0.01", "--seed", "6") == want
    with pytest.raises(SystemExit):
        run("--min-p", "0.1")


@pytest.mark.gpu
@pytest.mark.parametrize("cls", ["CUDADecoder", "INT8Decoder"])
def test_what_is_wrong_is_what_is_raised(tmp_path, monkeypatch, cls):
    """Logits from which nothing can be drawn, in a call that found too few pages or whose kernels gave up on a wait: that is what the error says, and "no token"
    only where neither happened."""
    from llm_decoder import _cabi
    dec = decoder(cls, tmp_path, 7, 97, 2, 64, batch_size=2, kv_tokens=64)
    nothing = np.zeros((2, 4), dtype=np.int32)
    for n, what in ((50, "too few pages"), (5, "no token is allowed")):
        with pytest.raises(RuntimeError, match=what):
            dec.generate_drafted([[3] * n, [4] * n], 20, temperature=0.8, allowed=nothing)
    assert len(dec.generate_drafted([[3] * 5, [4] * 5], 6, temperature=0.8)[0]) == 11
    counts = iter(range(9))
    monkeypatch.setattr(_cabi, "lost_waits", lambda: next(counts))
    with pytest.raises(RuntimeError, match="gave up on a wait"):
        dec.generate_drafted([[3] * 5, [4] * 5], 20, temperature=0.8, allowed=nothing)


@pytest.mark.gpu
@pytest.mark.parametrize("cls", ["CUDADecoder", "INT8Decoder"])
def test_numbers_of_numpy_are_numbers(tmp_path, cls):
    """Rules given as numpy's scalars, and per sequence, draw what they draw as Python's numbers."""
    dec = decoder(cls, tmp_path, 7, 97, 2, 64, batch_size=2)
    prompts, rules = [[3, 5, 7], [2, 4, 6]], dict(temperature=0.75, top_k=20, top_p=0.875, min_p=0.0625, repetition=1.25)
    want = dec.generate_drafted(prompts, 20, seed=2, **rules)
    assert dec.generate_drafted(prompts, 20, seed=2, **{k: (np.int64 if k == "top_k" else np.float32)(v) for k, v in rules.items()}) == want
    assert dec.generate_drafted(prompts, 20, seed=2, **{k: [v, v] for k, v in rules.items()}) == want


@pytest.mark.gpu
@pytest.mark.parametrize("cls", ["CUDADecoder", "INT8Decoder"])
@pytest.mark.parametrize("rules", [dict(temperature=0.7), dict(temperature=1.3, top_p=0.8), dict(temperature=1.0, top_k=9, min_p=0.02)])
def test_tokens_are_those_of_the_logits_of_their_step(tmp_path, monkeypatch, cls, rules):
    """Every node's id is drawn by its number from the very logits of its row, to the draws' own bound, and the tokens of a sequence are the ids along the paths
    that were taken, each drawn by the number of its place."""
    from test_draw_tokens import is_drawn

    from llm_decoder import sampling
    dec, n, more, seed = decoder(cls, tmp_path, 5, 97, 2, 64, batch_size=2), 6, 30, 11
    plain, calls = sampling.draw_tokens, []

    def draw_tokens(logits, u, tree, **kw):
        ids = plain(logits, u, tree=tree, **kw)
        calls.append((logits.float().cpu().numpy(), u.cpu().numpy(), kw, tree, ids.cpu().numpy()))
        return ids
    monkeypatch.setattr(sampling, "draw_tokens", draw_tokens)
    prompts = np.random.default_rng(3).integers(0, 97, (2, n)).tolist()
    got = dec.generate_drafted(prompts, more, drafts=10, branches=3, seed=seed, **rules)
    given, at = numbers_of(seed, 2, more), [n, n]
    for logits, u, kw, tree, ids in calls:
        for row, number, token in zip(logits, u, ids):
            w = kept_weights(row, **kw)
            assert is_drawn(w, token, number)
        first = np.concatenate([[0], np.cumsum(tree.sizes)])
        parents, tokens = tree.parents.cpu().numpy(), tree.tokens.cpu().numpy()
        for b in range(2):
            node = 0 if tree.sizes[b] else None
            while node is not None and at[b] < n + more:
                r = first[b] + node
                assert u[r] == given[b, at[b] - n] and got[b][at[b]] == ids[r]
                at[b] += 1
                node = next((k for k in range(node + 1, tree.sizes[b]) if parents[first[b] + k] == node and tokens[first[b] + k] == ids[r]), None)
    assert at == [n + more] * 2
