"""Where adjust_logits may write: anywhere that is not read, or in place."""
import pytest
import torch


def call(out, stride, out_stride, rows=4, vocab=100, type=0, logits=0x10000):
    """The argument rules of pa_adjust_logits alone: ids are asked for without a workspace, which is looked at last."""
    from llm_decoder import _cabi
    return _cabi.lib().pa_adjust_logits(logits, type, stride, rows, vocab, out, out_stride, 0x100, None, rows, None, 0, None, None, None, None, 1.0, 0.0,
                                        0.0, None, None, 0, None, None, 0, 0, None, None, None, 0, None, None, 0, None)


def test_overlapping_rows_are_refused():
    fine, bad, at = -3, -1, 0x10000
    assert call(at, 100, 100) == fine and call(None, 100, 100) == fine              # in place; ids alone
    assert call(at, 100, 200) == bad and call(at, 200, 100) == bad                  # other rows from the same place
    assert call(at, 100, 200, rows=1) == fine
    assert call(at + 4, 100, 100) == bad and call(at - 4, 100, 100) == bad
    assert call(at + 4 * 100, 100, 100) == bad                                      # row r of one is row r + 1 of the other
    assert call(at + 4 * 400, 100, 100) == fine and call(at - 4 * 400, 100, 100) == fine
    assert call(at + 4 * 399, 100, 100) == bad and call(at - 4 * 399, 100, 100) == bad
    assert call(at + 4 * 100, 200, 200) == fine and call(at + 4 * 99, 200, 200) == bad      # columns of one tensor
    assert call(at + 4 * 101, 200, 200) == bad and call(at - 4 * 100, 200, 200) == fine
    assert call(at + 4 * 100, 300, 200) == bad and call(at + 4 * 100, 200, 400) == fine      # rows that meet later on, and rows that do not
    assert call(at + 2 * 100, 200, 200, type=1) == fine and call(at + 2 * 99, 200, 200, type=2) == bad


@pytest.mark.gpu
def test_views_of_one_tensor():
    from llm_decoder import sampling
    g = torch.Generator(device="cuda").manual_seed(1)
    store = torch.randn(5, 3000, device="cuda", generator=g)
    history, start = torch.arange(0, 900, dtype=torch.int32, device="cuda"), torch.tensor([0, 900] + [900] * 4, dtype=torch.int32, device="cuda")
    want = sampling.adjust_logits(store[:, :1500].clone(), history, start, 1.5, 0.25, 0.5)
    keep = store[:, :1500].clone()
    for out in (store[:, 1:1501], store[:, 1499:2999]):
        with pytest.raises(Exception):
            sampling.adjust_logits(store[:, :1500], history, start, 1.5, 0.25, 0.5, out=out)
    assert torch.equal(store[:, :1500], keep)
    assert torch.equal(sampling.adjust_logits(store[:, :1500], history, start, 1.5, 0.25, 0.5, out=store[:, 1500:]), want)
    assert torch.equal(sampling.adjust_logits(store[:, :1500], history, start, 1.5, 0.25, 0.5, out=store[:, :1500]), want)
