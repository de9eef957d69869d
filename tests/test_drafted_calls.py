"""What generation with drafted trees refuses, and what it does when something under it goes wrong."""
import weakref

import numpy as np
import pytest
import torch

from test_generate_drafted import decoder


def test_longest_path():
    from llm_decoder.draft_tree import longest_path
    assert [longest_path(p) for p in ([], [-1], [-1, 0, 0], [-1, 0, 1, 0, 3, 4], [-1, 0, 1, 2])] == [0, 1, 2, 4, 4]


@pytest.mark.gpu
def test_paths_that_are_too_long_are_refused(tmp_path):
    """A path of right guesses that goes on past the tokens asked for would leave more rows behind than tokens."""
    dec = decoder("CUDADecoder", tmp_path, 11, 60, 2, 64, max_len=100)
    prompt, n = [3, 14, 15], 12
    want = dec.generate_drafted([prompt], 40, drafts=0)[0]

    def draft(tokens, most, depth, more):
        out = [int(t) for t in want[len(tokens) - 1:len(tokens) - 1 + min(most, depth + more)]]
        return [-1] + list(range(len(out) - 1)), out
    got = dec.generate_drafted([prompt], n, draft=lambda *a: draft(*a, 0))[0]
    assert len(got) == len(prompt) + n and dec.positions.tolist() == [len(prompt) + n - 1]
    with pytest.raises(ValueError):
        dec.generate_drafted([prompt], n, draft=lambda *a: draft(*a, 1))


@pytest.mark.gpu
def test_no_tokens_where_a_wait_ran_out(tmp_path, monkeypatch):
    from llm_decoder import decoders
    dec = decoder("CUDADecoder", tmp_path, 12, 60, 2, 64, max_len=64)
    assert len(dec.generate_drafted([[1, 2]], 5)[0]) == 7
    counts = [3, 4]
    monkeypatch.setattr(decoders._cabi, "lost_waits", lambda: counts.pop(0))
    with pytest.raises(RuntimeError):
        dec.generate_drafted([[1, 2]], 5)


@pytest.mark.gpu
@pytest.mark.parametrize("pool,dtype", [("f32", torch.float32), ("f16", torch.float32), ("f16", torch.float16), ("bf16", torch.bfloat16), ("i8", torch.float32)])
def test_a_step_as_it_is_written_down(pool, dtype):
    """Rows of all nodes by append, attention, acceptance, for every type of pages: the rows are where they should be."""
    import llm_decoder as ld
    rng = np.random.default_rng(4)
    B, H, D, tiles = 2, 3, 64, 6
    kv = ld.KVTileCache(pool)
    kv.init(B * H * tiles, 16, D)
    kv.configure_table(B, H, tiles)
    table = rng.permutation(B * H * tiles).astype(np.int32).reshape(B, H, tiles)
    kv.page_table_.load_host_table(table)
    kv.key_buffer_.zero_()
    kv.value_buffer_.zero_()
    tree = ld.DraftTree([[-1, 0, 0, 2], [-1, 0]], [[5, 6, 7, 8], [9, 1]], "cuda")
    ctx = torch.tensor([14, 40], dtype=torch.int32, device="cuda")
    k, v = (torch.from_numpy(rng.standard_normal((tree.rows, H, D)).astype(np.float32)).to(dtype).cuda() for _ in "kv")
    kv.append(k, v, tree.positions(ctx), tree.row_seq)

    def row(x, b, h, pos):
        x, s = (kv.key_buffer_, kv.k_scales_) if x == "k" else (kv.value_buffer_, kv.v_scales_)
        at = int(table[b, h, pos // 16]), pos % 16
        return x[at].float() if s is None else x[at].float() / s[at]
    near = {"f32": 0.0, "f16": 2.0 ** -11 if dtype is torch.float32 else 0.0, "bf16": 0.0, "i8": 0.5 / 127 * 1.01}[pool]       # rounding to the pool's type
    place = [(0, 14 + i) for i in range(4)] + [(1, 40), (1, 41)]
    for x, new in (("k", k), ("v", v)):
        for r, (b, pos) in enumerate(place):
            for h in range(H):
                assert float((row(x, b, h, pos) - new[r, h].float()).abs().max()) <= near * float(new[r, h].abs().max())
    q = torch.randn(tree.rows, H, D, device="cuda").to({"f16": torch.float32, "i8": torch.float32}.get(pool, dtype))
    assert bool(ld.paged_tree_attention(q, kv, tree, ctx, 8.0).isfinite().all())
    want = row("k", 0, 1, 17)
    done = ld.tree_accept(torch.tensor([7, 1, 8, 3, 2, 1], dtype=torch.int32, device="cuda"), tree, [kv], ctx)
    assert done.counts.tolist() == [3, 1] and torch.equal(row("k", 0, 1, 16), want)


@pytest.mark.gpu
@pytest.mark.parametrize("cls", ["CUDADecoder", "INT8Decoder"])
def test_the_command(tmp_path, capsys, cls):
    """bin/generate with drafts and penalties: what generate_drafted gives; without them what it gave before."""
    import json

    from llm_decoder import cli
    dec = decoder(cls, tmp_path, 13, 97, 2, 64, max_len=128)
    config = dict(architecture=cls, num_layers=2, num_heads=2, head_dim=64, hidden_dim=128, vocab_size=97, max_seq_len=128,
                  weights="q" if cls == "INT8Decoder" else "w")
    (tmp_path / "config.json").write_text(json.dumps(config))

    def run(*args):
        assert cli.main(["generate", "--model", str(tmp_path), "--prompt", "5,17,3", "--prompt", "9,9", "--max-new-tokens", "30", *args]) == 0
        return [[int(t) for t in line.split(",")] for line in capsys.readouterr().out.splitlines() if line[:1].isdigit()]
    prompts = [[5, 17, 3], [9, 9]]
    assert run("--drafts", "12") == [dec.generate_drafted([p], 30, drafts=12)[0] for p in prompts]
    rules = dict(repetition=1.3, presence=0.2, frequency=0.1)
    want = [dec.generate_drafted([p], 30, drafts=4, **rules)[0] for p in prompts]
    assert run("--drafts", "4", "--repetition-penalty", "1.3", "--presence-penalty", "0.2", "--frequency-penalty", "0.1") == want
    assert run("--repetition-penalty", "1.3") == [dec.generate_drafted([p], 30, drafts=0, repetition=1.3)[0] for p in prompts]
    assert run() == [dec.generate(p, 30) for p in prompts]
    for args in (["--drafts", "4", "--temperature", "0.7"], ["--presence-penalty", "1", "--top-k", "3"], ["--drafts", "4", "--top-p", "0.5"]):
        with pytest.raises(SystemExit):
            run(*args)


@pytest.mark.gpu
def test_steps_of_other_sizes_share_their_scratch(tmp_path):
    from llm_decoder.decoders import _Bufs
    dec = decoder("INT8Decoder", tmp_path, 14, 97, 2, 64, attn=True, batch_size=10)
    bufs = _Bufs(12, 128, 512, dec.device)
    few, fewer = bufs.first(9), bufs.first(4)
    assert dec._scratch(few, 1000) == dec._scratch(fewer, 900) == dec._scratch(bufs, 1000)
    made = [b.on_demand("lq", lambda rows: torch.empty((rows, 128), dtype=torch.int8, device=dec.device)) for b in (few, fewer, bufs, bufs.first(7))]
    assert [len(x) for x in made] == [9, 4, 12, 7] and len({x.data_ptr() for x in made}) == 1
    gone = weakref.ref(bufs)
    del bufs, few, fewer, made
    assert gone() is None           # and it goes with the buffers, at once
