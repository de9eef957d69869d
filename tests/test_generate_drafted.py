"""Generation with drafted trees (decoders.generate_drafted): the tokens of one-by-one generation, in fewer steps.

Both ways compute a logit from the same weights and cached rows, in sums of another order.  Where they choose another token, the
one-by-one logits of the two tokens have to lie within TOL of the largest of their row: for float weights 2^-24 times a
thousand additions of a value that passes a handful of layers (1e-3); for int8 weights a rounding to int8 may fall the other way, which moves one of
a row's 128 or more terms by 1/127 of its largest (2e-2)."""
import numpy as np
import pytest
import torch

from test_decoders import make_weights, write_fp32_tree

TOL = {"CUDADecoder": 1e-3, "INT8Decoder": 2e-2}


def test_lookup_drafts():
    from llm_decoder import lookup_drafts
    # the last three tokens came up twice: the later continuation first, then the other one; then those of the last two
    assert lookup_drafts([1, 2, 3, 4, 1, 2, 3, 5, 1, 2, 3], 8, 4) == ([-1, 0, 1, 2, 0, 4, 5], [3, 5, 1, 2, 4, 1, 2])
    assert lookup_drafts([1, 2, 3, 4, 1, 2, 3, 5, 1, 2, 3], 4, 4) == ([-1, 0, 1, 2], [3, 5, 1, 2])
    assert lookup_drafts([1, 2, 3, 4, 1, 2, 3, 5, 1, 2, 3], 8, 2) == ([-1, 0, 0], [3, 5, 4])
    assert lookup_drafts([1, 2, 3, 4, 1, 2, 3, 5, 1, 2, 3], 8, 1) == ([-1], [3])
    assert lookup_drafts([1, 2, 3, 4, 1, 2, 3, 5, 1, 2, 3], 8, 3, branches=1) == ([-1, 0, 1], [3, 5, 1])
    assert lookup_drafts([1, 5, 2, 5], 8, 3) == ([-1, 0, 1], [5, 2, 5])
    for tokens in ([7], [7, 8], [1, 2, 3]):
        assert lookup_drafts(tokens, 8, 4) == ([-1], tokens[-1:])


def decoder(cls, tmp_path, seed, vocab, heads, dim, attn=False, max_len=200, **kw):
    import llm_decoder as ld
    hid = heads * dim
    w = make_weights(np.random.default_rng(seed), 2, hid, vocab, attn=attn)
    write_fp32_tree(w, str(tmp_path / "w"), False)
    dec = getattr(ld, cls)(2, heads, dim, hid, vocab, max_len, **kw)
    if cls == "INT8Decoder":
        dec.quantize_weights(str(tmp_path / "w"), str(tmp_path / "q"))
        dec.load_quantized_weights(str(tmp_path / "q"))
    else:
        dec.load_weights(str(tmp_path / "w"))
    return dec


def one_by_one(dec, seqs, n, rules=None):
    """The logits behind every token of seqs from place n on, [B, tokens, vocab] in float64, changed by rules(sequence, its logits)."""
    dec.reset()
    out = []
    for t in range(len(seqs[0]) - 1):
        x = dec.forward_tokens([s[t] for s in seqs]).double().cpu().numpy()
        if t + 1 >= n:
            out.append([rules(b, s[:t + 1], r.copy()) if rules else r for b, (s, r) in enumerate(zip(seqs, x))])
    return np.array(out).transpose(1, 0, 2)


def check(dec, got, n, rules=None):
    """Every token is the largest of the one-by-one logits that its own predecessors give, or as good as that."""
    logits = one_by_one(dec, got, n, rules)
    tol = TOL[type(dec).__name__]
    for s, rows in zip(got, logits):
        for t, row in zip(s[n:], rows):
            assert row.max() - row[t] <= tol * np.abs(row[np.isfinite(row)]).max()


@pytest.mark.gpu
@pytest.mark.parametrize("cls,heads,dim,attn", [("CUDADecoder", 2, 64, False), ("CUDADecoder", 3, 128, True), ("INT8Decoder", 2, 128, False),
                                                ("INT8Decoder", 3, 64, True)])
@pytest.mark.parametrize("batch,n", [(1, 1), (3, 7), (10, 33)])
def test_tokens_are_those_of_single_steps(tmp_path, cls, heads, dim, attn, batch, n):
    rng = np.random.default_rng(batch)
    dec = decoder(cls, tmp_path, 5, 97, heads, dim, attn, batch_size=batch)
    prompts = rng.integers(0, 97, (batch, n)).tolist()
    plain = dec.generate_batch(prompts, 40)
    for kw in (dict(drafts=0), dict(), dict(drafts=70, branches=5)):
        got = dec.generate_drafted(prompts, 40, **kw)
        assert [s[:n] for s in got] == prompts and all(len(s) == n + 40 for s in got)
        check(dec, got, n)
        assert dec.drafted_steps_ <= 40
    assert plain == dec.generate_batch(prompts, 40)         # and what it leaves behind is nothing to the next call


@pytest.mark.gpu
@pytest.mark.parametrize("cls", ["CUDADecoder", "INT8Decoder"])
def test_right_guesses_save_steps(tmp_path, cls):
    """Guesses taken from what the model gives, next to wrong ones: k of them in every step, so tokens / (k + 1) steps."""
    dec = decoder(cls, tmp_path, 6, 211, 2, 64)
    prompt, n, k = [3, 14, 15, 92, 6], 5, 4
    want = dec.generate_drafted([prompt], 60, drafts=0)[0]
    assert dec.drafted_steps_ == 60

    def draft(tokens, most, depth):
        at = len(tokens)
        right = want[at:at + min(k, depth - 1)]
        parents, out, node = [-1], [int(tokens[-1])], 0
        for t in right:                                     # a wrong sibling first, then the right one
            parents += [node, node]
            out += [(t + 1) % 211, t]
            node = len(out) - 1
        return parents, out
    got = dec.generate_drafted([prompt], 60, drafts=16, draft=draft)[0]
    check(dec, [got], n)
    if got == want:
        assert dec.drafted_steps_ == 60 // (k + 1)
    # the cache is filled up to the last row: what does not fit is not drafted
    long = dec.generate_drafted([prompt], 196, drafts=64, branches=8)[0]
    assert len(long) == 201
    check(dec, [long], n)


@pytest.mark.gpu
@pytest.mark.parametrize("cls,batch", [("CUDADecoder", 2), ("INT8Decoder", 9)])
def test_penalties_biases_and_masks(tmp_path, cls, batch):
    rng = np.random.default_rng(8)
    V, n = 97, 6
    dec = decoder(cls, tmp_path, 7, V, 2, 64, batch_size=batch)
    prompts = rng.integers(0, V, (batch, n)).tolist()
    rep = (1 + rng.random(batch)).astype(np.float32)
    freq = (rng.random(batch) * 2).astype(np.float32)
    b_ids, b_val = rng.integers(0, V, 2 * batch).astype(np.int32), rng.standard_normal(2 * batch).astype(np.float32)
    b_start = np.arange(0, 2 * batch + 1, 2, dtype=np.int32)
    b_ids[1::2] = (b_ids[::2] + 1) % V                      # a token once
    ok = rng.random((batch, 128)) < 0.5
    words = np.packbits(ok, axis=1, bitorder="little").view(np.int32)
    got = dec.generate_drafted(prompts, 50, drafts=12, repetition=rep, presence=0.25, frequency=freq, bias=(b_ids, b_val, b_start),
                               allowed=words)

    def rules(b, seq, x):
        tokens, counts = np.unique(seq, return_counts=True)
        x[tokens] = np.where(x[tokens] > 0, x[tokens] / rep[b], x[tokens] * rep[b]) - 0.25 - freq[b] * counts
        for i in range(b_start[b], b_start[b + 1]):
            x[b_ids[i]] += b_val[i]
        x[~ok[b, :V]] = -np.inf
        return x
    check(dec, got, n, rules)
    assert all(ok[b, t] for b, s in enumerate(got) for t in s[n:])


@pytest.mark.gpu
def test_refusals(tmp_path):
    dec = decoder("CUDADecoder", tmp_path, 9, 50, 2, 64, max_len=32)
    for args, kw in ((([[]], 4), {}), (([[1], [1, 2]], 4), {}), (([[1, 2, 3]], 31), {}), (([[1, 2, 3]], 4), dict(drafts=-1)),
                     (([[1, 2, 3]], 4), dict(draft=lambda tokens, most, depth: ([], []))),
                     (([[1, 2, 3]], 4), dict(draft=lambda tokens, most, depth: ([-1, 0], [9, 9]))),
                     (([[1, 2, 3]], 4), dict(drafts=1, draft=lambda tokens, most, depth: ([-1, 0, 1], [3, 9, 9]))),
                     (([[1, 2, 3]], 4), dict(repetition=0.0))):
        with pytest.raises(ValueError):
            dec.generate_drafted(*args, **kw)
    assert dec.generate_drafted([[1, 2, 3]], 0) == [[1, 2, 3]]
    assert dec.generate_drafted([[1, 2, 3]], 30) == dec.generate_drafted([[1, 2, 3]], 30, drafts=0)


@pytest.mark.gpu
@pytest.mark.parametrize("pool", ["f16", "i8"])
def test_the_step_replays_as_a_graph(pool):
    """Attention, rules and acceptance in a graph, replayed next to launched calls on the stream of the capture: equal bits."""
    import llm_decoder as ld
    rng = np.random.default_rng(12)
    B, H, D, V, tile = 3, 4, 128, 1000, 16
    dev = torch.device("cuda", torch.cuda.current_device())
    kv = ld.KVTileCache(pool, device=dev)
    kv.init(B * H * 40, tile, D)
    kv.configure_table(B, H, 40)
    kv.page_table_.load_host_table(rng.permutation(B * H * 40).astype(np.int32).reshape(B, H, 40))
    lens = [600, 30, 0]
    for b, n in enumerate(lens):
        x = torch.from_numpy(rng.standard_normal((max(n, 1) + 20, H, D)).astype(np.float32)).to(dev)
        kv.append(x, -x, torch.arange(len(x), dtype=torch.int32, device=dev), torch.full((len(x),), b, dtype=torch.int32, device=dev))
    tokens = [rng.integers(0, V, n).tolist() for n in (18, 5, 20)]
    tree = ld.DraftTree([[-1] + [int(rng.integers(0, i)) for i in range(1, len(t))] for t in tokens], tokens, dev)
    ctx = torch.tensor(lens, dtype=torch.int32, device=dev)
    q = torch.from_numpy(rng.standard_normal((tree.rows, H, D)).astype(np.float32)).to(dev)
    logits = torch.from_numpy(rng.standard_normal((tree.rows, V)).astype(np.float32)).to(dev)
    history = torch.from_numpy(rng.integers(0, V, 90).astype(np.int32)).to(dev)
    start = torch.tensor([0, 40, 40, 90], dtype=torch.int32, device=dev)

    def step():
        return (ld.paged_tree_attention(q, kv, tree, ctx), ld.sampling.adjusted_argmax(logits, history, start, 1.3, 0.2, 0.1, tree=tree))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        want = [x.clone() for x in step()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step()
    for _ in range(3):
        graph.replay()
        with torch.cuda.stream(side):
            launched = step()
        torch.cuda.synchronize()
        for w, g, x in zip(want, got, launched):
            assert torch.equal(w, g) and torch.equal(w, x)
            g.zero_()
