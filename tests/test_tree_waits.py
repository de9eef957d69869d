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


def attention(pool, q_type, heads, kv_heads, dim, nodes):
    """More items than workers and items that are cut; a workspace with the notes of a call over other contexts."""
    import llm_decoder as ld
    from llm_decoder import _cabi
    lib, dev, B, tiles = _cabi.lib(), torch.device("cuda", torch.cuda.current_device()), 40, 64
    kv = ld.KVTileCache(pool)
    kv.init(B * kv_heads * tiles, 16, dim)
    kv.configure_table(B, kv_heads, tiles)
    import numpy as np
    kv.page_table_.load_host_table(np.arange(B * kv_heads * tiles, dtype=np.int32).reshape(B, kv_heads, tiles))
    if pool == "i8":
        for x, s in ((kv.key_buffer_, kv.k_scales_), (kv.value_buffer_, kv.v_scales_)):
            x.random_(-127, 128)
            s.fill_(40.0)
    else:
        kv.key_buffer_.normal_()
        kv.value_buffer_.normal_()
    rng = np.random.default_rng(3)
    sizes = [nodes if b % 3 else 1 + nodes // 2 for b in range(B)]
    tree = ld.DraftTree([[-1] + list(range(n - 1)) for n in sizes], device=dev)
    ctx = [torch.from_numpy(rng.integers(1, 16 * tiles - nodes, B).astype(np.int32)).to(dev) for _ in range(2)]
    q = torch.randn(tree.rows, heads, dim, device=dev).to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[q_type])
    types = ld.draft_tree.TYPES
    ws = torch.zeros(lib.pa_tree_attention_workspace_bytes(tree.rows, B, tree.most, heads, kv_heads, dim), dtype=torch.uint8, device=dev)

    def call(ctx, polls):
        out, before, pt = torch.zeros_like(q), _count(lib), kv.page_table_
        assert lib.pa_tree_attention_polls(
            q.data_ptr(), heads * dim, types[q.dtype], out.data_ptr(), kv.key_buffer_.data_ptr(), kv.value_buffer_.data_ptr(), _cabi.ptr(kv.k_scales_),
            _cabi.ptr(kv.v_scales_), types[kv.key_buffer_.dtype], pt.device_data().data_ptr(), B, kv_heads, tiles, kv.total_pages_, None, ctx.data_ptr(),
            tree.node_start.data_ptr(), tree.mask.data_ptr(), tree.mask.shape[1], tree.rows, B, tree.most, heads, dim, 16, 8.0, ws.data_ptr(),
            ws.numel(), polls, _cabi.stream()) == 0
        return out, _count(lib) - before
    for first, second in ((ctx[0], ctx[1]), (ctx[1], ctx[0])):
        want, ran_out = call(first, MOST)
        assert ran_out == 0 and bool(want.isfinite().all())
        lost, ran_out = call(second, 0)
        assert ran_out > 0 and bool(lost.isnan().all())
        again, ran_out = call(first, MOST)
        assert ran_out == 0 and torch.equal(want, again)
    assert lib.pa_tree_attention_polls(q.data_ptr(), heads * dim, types[q.dtype], *[q.data_ptr()] * 5, 0, q.data_ptr(), B, kv_heads, tiles, 1, None,
                                       *[q.data_ptr()] * 3, 1, 1, 1, 1, heads, dim, 16, 1.0, None, 0, -1, _cabi.stream()) == -1


def stream_float():
    attention("f16", "f32", 8, 8, 64, 8)


def stream_16_bits():
    attention("bf16", "bf16", 8, 8, 128, 8)
    attention("f16", "f16", 16, 8, 64, 8)


def stream_int8():
    attention("i8", "f32", 8, 8, 64, 12)
    attention("i8", "f16", 16, 8, 64, 12)


def tiles_of_rows():
    attention("bf16", "bf16", 32, 8, 128, 20)
    attention("f16", "f16", 32, 8, 64, 50)          # 200 rows a kv head
    attention("bf16", "bf16", 24, 8, 128, 20)       # queries without boxes


def tiles_of_terms():
    attention("f16", "f32", 8, 8, 128, 30)
    attention("f16", "f32", 16, 8, 64, 30)


def tiles_of_digits():
    attention("i8", "f32", 8, 8, 128, 12)
    attention("i8", "f16", 16, 8, 128, 20)


@pytest.mark.gpu
@pytest.mark.parametrize("case", ["rules", "stream_float", "stream_16_bits", "stream_int8", "tiles_of_rows", "tiles_of_terms", "tiles_of_digits"])
def test_rows_of_waits_that_run_out(case):
    r = subprocess.run([sys.executable, os.path.abspath(__file__), case], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("done"), r.stdout + r.stderr


if __name__ == "__main__":
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    sys.path.insert(0, os.path.join(root, "pagedattention-based-transformer-decoder-inference-framework_b200"))
    globals()[sys.argv[1]]()
    torch.cuda.synchronize()
    print("done")
