"""Biases for most of a vocabulary, more to a stretch of it than the kernel lists."""
import pytest
import torch

from test_logit_rules import Case


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V,bias,nodes", [(1000, 700, None), (5003, 12000, None), (9001, 5000, [4, 0, 9])])
def test_many_biases(kind, V, bias, nodes):
    """Some tokens several times: the last entry counts."""
    from llm_decoder import sampling
    c = Case(V + bias, kind, 3, V, [100, 0, 2000], bias=bias, masked=True, nodes=nodes)
    got, ids = sampling.adjust_logits(c.dev, ids=True, **c.kw)
    c.check(got, ids)
    assert torch.equal(sampling.adjusted_argmax(c.dev, **c.kw), ids)


@pytest.mark.gpu
def test_many_biases_take_no_time_of_their_square():
    from llm_decoder import sampling
    R, V = 16, 128000
    x, out, times = torch.randn(R, V, device="cuda"), torch.empty(R, V, device="cuda"), {}
    for n in (64, V):
        ids = torch.stack([torch.randperm(V, device="cuda")[:n] for _ in range(R)]).to(torch.int32).reshape(-1)
        bias = (ids, torch.randn(R * n, device="cuda"), (torch.arange(R + 1, device="cuda") * n).to(torch.int32))
        sampling.adjust_logits(x, bias=bias, out=out)
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        for _ in range(3):
            sampling.adjust_logits(x, bias=bias, out=out)
        end.record()
        torch.cuda.synchronize()
        times[n] = begin.elapsed_time(end)
    assert times[V] < 200 * times[64]           # 2000 times the entries; their square took 4000 times as long
