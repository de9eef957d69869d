"""What generation with drafted trees refuses, and what it does when something under it goes wrong."""
import pytest

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
