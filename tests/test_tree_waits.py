"""Kernels of drafted trees and logit rules whose waits run out (the limit of a wait is an argument; with 0 nothing is requested, so that all run
out): the call returns, its rows are NaN and never plausible numbers, ids are -1, the count of waits that ran out goes up, and the next call
is served.  In processes of their own, since other tests ask for a count of zero."""
import os
import subprocess
import sys

import pytest
import torch

MOST = 1 << 25


def _count(lib):
    import ctypes
    n = ctypes.c_int(-1)
    assert lib.pa_attention_tc_errors(ctypes.byref(n)) == 0
    return n.value


def rules():
    """Rows with tokens that a rule touches (the CTA's threads share what they do) and without, of every type; logits, ids or both."""
    from llm_decoder import _cabi
    lib, dev, R, V = _cabi.lib(), torch.device("cuda"), 5, 9001
    g = torch.Generator().manual_seed(1)
    history = torch.randint(0, V, (300,), generator=g).to(torch.int32).to(dev)
    start = torch.tensor([0, 300, 300, 300, 300, 300], dtype=torch.int32, device=dev)      # the first row alone has one
    ws = torch.zeros(R * 8, dtype=torch.uint8, device=dev)
    for kind, dtype in enumerate((torch.float32, torch.float16, torch.bfloat16)):
        x = torch.randn(R, V, generator=g).to(dtype).to(dev)
        for logits, ids in ((True, True), (True, False), (False, True)):
            for polls in (0, MOST):
                out, chosen, before = torch.zeros_like(x), torch.full((R,), 7, dtype=torch.int32, device=dev), _count(lib)
                assert lib.pa_adjust_logits_polls(
                    x.data_ptr(), kind, V, R, V, out.data_ptr() if logits else None, V, chosen.data_ptr() if ids else None, None, R,
                    history.data_ptr(), 300, start.data_ptr(), None, None, None, 1.5, 0.5, 0.1, None, None, 0, None, None, 0, 0, None, None, None, 0,
                    None, ws.data_ptr(), ws.numel(), polls, _cabi.stream()) == 0
                ran_out = _count(lib) - before
                assert ran_out > 0 if polls == 0 else ran_out == 0
                assert not bool(ws.any())
                if logits:
                    assert bool(out.isnan().all() if polls == 0 else out.isfinite().all())
                if ids:
                    assert bool((chosen == -1).all() if polls == 0 else ((chosen >= 0) & (chosen < V)).all())
    assert lib.pa_adjust_logits_polls(x.data_ptr(), 2, V, R, V, out.data_ptr(), V, None, None, R, None, 0, None, *[None] * 3, 1.0, 0.0, 0.0, None, None, 0,
                                      None, None, 0, 0, None, None, None, 0, None, None, 0, -1, _cabi.stream()) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("case", ["rules"])
def test_rows_of_waits_that_run_out(case):
    r = subprocess.run([sys.executable, os.path.abspath(__file__), case], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("done"), r.stdout + r.stderr


if __name__ == "__main__":
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    sys.path.insert(0, os.path.join(root, "pagedattention-based-transformer-decoder-inference-framework_b200"))
    globals()[sys.argv[1]]()
    torch.cuda.synchronize()
    print("done")
