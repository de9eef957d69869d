"""Operators of drafted trees called from two host threads: the library is called without the interpreter's lock, so that two calls may be
issued at the same time, on one stream too.  Where a case would be a matter of luck, a stand-in for the library holds both calls until the other
one is under way."""
import threading

import numpy as np
import pytest
import torch


class Library:
    """The library, with calls of `name` answered by `answer`."""

    def __init__(self, real, name, answer):
        self.__dict__.update(real=real, name=name, answer=answer)

    def __getattr__(self, name):
        return self.answer if name == self.name else getattr(self.real, name)


def in_threads(n, work):
    out, errors = [None] * n, []

    def run(i):
        try:
            out[i] = work(i)
        except BaseException as e:      # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=run, args=(i,)) for i in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    return out


@pytest.mark.gpu
def test_rules_in_two_threads_have_words_of_their_own(monkeypatch):
    from llm_decoder import _cabi, sampling
    real, gate, words = _cabi.lib(), threading.Barrier(2, timeout=60), []

    def answer(*args):
        gate.wait()
        words.append(args[-3])
        return 0
    logits = torch.zeros(3, 100, device="cuda")
    monkeypatch.setattr(_cabi, "lib", lambda: Library(real, "pa_adjust_logits", answer))
    in_threads(2, lambda i: sampling.adjusted_argmax(logits))
    assert len(set(words)) == 2 and None not in words


@pytest.mark.gpu
def test_rules_in_threads_give_their_own_ids():
    from llm_decoder import sampling
    g = torch.Generator(device="cuda").manual_seed(1)
    logits = [torch.randn(40, 5000, device="cuda", generator=g) for _ in range(4)]
    want = [x.argmax(1).to(torch.int32) for x in logits]
    torch.cuda.synchronize()
    got = in_threads(4, lambda i: [sampling.adjusted_argmax(logits[i]) for _ in range(200)])
    torch.cuda.synchronize()
    for w, ids in zip(want, got):
        assert all(torch.equal(w, x) for x in ids)


@pytest.mark.gpu
def test_rules_after_a_call_that_failed(monkeypatch):
    """Its words may hold anything; the next call's ids are right all the same."""
    from llm_decoder import _cabi, sampling
    real = _cabi.lib()
    logits = torch.from_numpy(np.random.default_rng(2).standard_normal((5, 700)).astype(np.float32)).cuda()
    want = sampling.adjusted_argmax(logits)
    assert torch.equal(want, logits.argmax(1).to(torch.int32))

    def answer(*_args):
        for words in sampling._rule_words.of.values():
            words.fill_(255)
        return 2
    with monkeypatch.context() as m:
        m.setattr(_cabi, "lib", lambda: Library(real, "pa_adjust_logits", answer))
        with pytest.raises(Exception):
            sampling.adjusted_argmax(logits)
    assert torch.equal(sampling.adjusted_argmax(logits), want)


def small_cache(seed):
    import llm_decoder as ld
    kv = ld.KVTileCache("f16")
    kv.init(2 * 2 * 8, 16, 64)
    kv.configure_table(2, 2, 8)
    kv.page_table_.load_host_table(np.arange(32, dtype=np.int32).reshape(2, 2, 8))
    g = torch.Generator(device="cuda").manual_seed(seed)
    kv.key_buffer_.normal_(generator=g)
    kv.value_buffer_.normal_(generator=g)
    return kv


@pytest.mark.gpu
def test_tree_attention_has_a_workspace_per_thread_and_none_per_cache(monkeypatch):
    import llm_decoder as ld
    from llm_decoder import _cabi
    real, gate, used = _cabi.lib(), threading.Barrier(2, timeout=60), []
    caches = [small_cache(i) for i in range(3)]
    trees = [ld.DraftTree([[-1, 0, 0], [-1, 0]], device="cuda") for _ in range(2)]
    q, ctx = torch.randn(5, 2, 64, device="cuda"), torch.tensor([100, 30], dtype=torch.int32, device="cuda")
    for c in caches:
        c.page_table_.device_data()

    def answer(*args):
        gate.wait()
        used.append((threading.get_ident(), args[-3]))
        return 0
    monkeypatch.setattr(_cabi, "lib", lambda: Library(real, "pa_tree_attention", answer))
    in_threads(2, lambda i: [ld.paged_tree_attention(q, c, trees[i], ctx) for c in (caches[0], caches[i + 1])])
    spaces = {}
    for thread, space in used:
        spaces.setdefault(thread, set()).add(space)
    assert len(used) == 4 and [len(s) for s in spaces.values()] == [1, 1] and len(set.union(*spaces.values())) == 2
    assert None not in set.union(*spaces.values())


@pytest.mark.gpu
def test_tree_attention_in_threads_on_one_cache():
    import llm_decoder as ld
    kv = small_cache(7)
    ctx = torch.tensor([100, 30], dtype=torch.int32, device="cuda")
    trees = [ld.DraftTree([[-1] + [0] * (3 + i), [-1, 0]], device="cuda") for i in range(4)]
    qs = [torch.randn(t.rows, 2, 64, device="cuda") for t in trees]
    want = [ld.paged_tree_attention(q, kv, t, ctx) for q, t in zip(qs, trees)]
    torch.cuda.synchronize()
    got = in_threads(4, lambda i: [ld.paged_tree_attention(qs[i], kv, trees[i], ctx) for _ in range(100)])
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(w, x) for x in outs)


@pytest.mark.gpu
def test_the_first_call_of_a_thread_is_served_as_any_other():
    """By a thread that has not called CUDA before, into memory that is there: the same bits."""
    import llm_decoder as ld
    from llm_decoder import draft_tree
    kv = small_cache(9)
    ctx = torch.tensor([100, 30], dtype=torch.int32, device="cuda")
    tree = ld.DraftTree([[-1, 0, 0, 1], [-1, 0]], device="cuda")
    q = torch.randn(tree.rows, 2, 64, device="cuda")
    want = ld.paged_tree_attention(q, kv, tree, ctx)
    outs, spaces = [torch.empty_like(want) for _ in range(8)], dict(draft_tree._workspaces.of)

    def first(i):
        draft_tree._workspaces.of.update(spaces)
        return ld.paged_tree_attention(q, kv, tree, ctx, out=outs[i])
    for i in range(8):              # one thread after the other
        in_threads(1, lambda _k, i=i: first(i))
    torch.cuda.synchronize()
    assert all(torch.equal(want, x) for x in outs)


def test_host_stage_gives_threads_regions_of_their_own(monkeypatch):
    """Two threads in the middle of a step's description: neither writes where the other's copy still reads."""
    from llm_decoder.host_stage import _PinnedStage

    class Stage(_PinnedStage):
        def __init__(self):
            monkeypatch.setattr(torch.Tensor, "pin_memory", lambda self: self)
            super().__init__()

    class View:
        """A region of the stage; its copy takes as long as the other thread needs to come here, where it may."""

        def __init__(self, view):
            self.view_ = view

        def view(self, shape):
            return self

        def copy_(self, t):
            self.view_.copy_(t)
            try:
                meet.wait(timeout=0.3)
            except threading.BrokenBarrierError:
                pass

        def to(self, device, non_blocking):
            return self.view_.clone()

    class Buffer:
        def __init__(self, t):
            self.t = t

        def __getitem__(self, key):
            return View(self.t[key])

    meet, stage = threading.Barrier(2), Stage()
    stage.buf = Buffer(stage.buf)
    got = in_threads(2, lambda i: stage.put(torch.full((100,), i, dtype=torch.int32), torch.device("cpu")))
    assert [x.tolist() for x in got] == [[0] * 100, [1] * 100]
