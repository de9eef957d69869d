"""Device-side sampling over vocabulary logits: the reference's CPU filters
(attention_cpu/softmax_lut.cpp:203-256) and its GPU sketch (attention/top_k_top_p_filter.cuh:55-111)
as three kernels of libpa_b200.so (`sample`: tensors are CUDA float32 [rows, vocab]); rules of a batch's requests (adjust_logits); and, for requests
with temperatures and truncations of their own, the distribution that is drawn from, draws from it by given numbers and drafted tokens kept or
replaced (truncated_softmax, draw_tokens, verify_drafts)."""
import ctypes

import torch

from . import _cabi


def build_exp_lut(resolution=1024, max_x=10.0, device=None):
    """build_exp_lut (softmax_lut.cpp:11-18): lut[i] = exp(-max_x + 2*max_x*i/(resolution-1)) in float32 with
    the C library's expf (what std::exp(float) calls), so the table is the reference's bit for bit."""
    import ctypes
    import ctypes.util

    import numpy as np
    libm = ctypes.CDLL(ctypes.util.find_library("m") or "libm.so.6")
    libm.expf.restype = ctypes.c_float
    libm.expf.argtypes = [ctypes.c_float]
    mx = np.float32(max_x)
    lut = np.empty(resolution, dtype=np.float32)
    for i in range(resolution):
        x = -mx + np.float32(2) * mx * np.float32(i) / np.float32(resolution - 1)
        lut[i] = libm.expf(float(np.float32(x)))
    t = torch.from_numpy(lut)
    return t.to(device) if device is not None else t


def softmax_lut(logits_i32, scale, lut, out=None):
    """fused_softmax_lut_inplace / softmax_batch_parallel (softmax_lut.cpp:60-100) over int32 logits
    [rows, n] -> f32 probabilities, bit-exact (pa_softmax_lut_i32)."""
    x = logits_i32.contiguous()
    assert x.dtype == torch.int32 and lut.dtype == torch.float32 and lut.is_cuda
    rows, n = x.shape
    p = torch.empty((rows, n), dtype=torch.float32, device=x.device) if out is None else out
    with torch.cuda.device(x.device):
        _cabi.check(_cabi.lib().pa_softmax_lut_i32(x.data_ptr(), rows, n, float(scale), lut.data_ptr(), lut.numel(),
                                                   p.data_ptr(), _cabi.stream()), "pa_softmax_lut_i32")
    return p


def softmax_temperature(logits, temperature=1.0, out=None):
    """softmax_lut_vec (softmax_lut.cpp:203-231): exp((x - max)/T) / (sum + 1e-6) per row."""
    x = logits.contiguous()
    rows, V = x.shape
    p = torch.empty_like(x) if out is None else out
    with torch.cuda.device(x.device):
        _cabi.check(_cabi.lib().pa_softmax_temperature(x.data_ptr(), rows, V, float(temperature), p.data_ptr(),
                                                       _cabi.stream()), "pa_softmax_temperature")
    return p


def apply_topk_topp_filter(probs, top_k, top_p, eos_token_id=-1, eos_thresh=0.0):
    """apply_topk_topp_filter (softmax_lut.cpp:233-256), in place on probs [rows, vocab]."""
    assert probs.is_contiguous() and probs.dtype == torch.float32
    rows, V = probs.shape
    with torch.cuda.device(probs.device):
        _cabi.check(_cabi.lib().pa_topk_topp_filter(probs.data_ptr(), rows, V, int(top_k), float(top_p),
                                                    int(eos_token_id), float(eos_thresh), _cabi.stream()),
                    "pa_topk_topp_filter")
    return probs


def sample_from_probs(probs, uniform, out=None):
    """First index whose inclusive prefix sum exceeds uniform[row] * sum(probs[row])."""
    rows, V = probs.shape
    ids = torch.empty(rows, dtype=torch.int32, device=probs.device) if out is None else out
    with torch.cuda.device(probs.device):
        _cabi.check(_cabi.lib().pa_sample_from_probs(probs.data_ptr(), rows, V, uniform.data_ptr(), ids.data_ptr(),
                                                     _cabi.stream()), "pa_sample_from_probs")
    return ids


def sample(logits, temperature=1.0, top_k=0, top_p=1.0, eos_token_id=-1, eos_thresh=0.0, generator=None):
    """logits [rows, vocab] -> sampled token ids [rows] (temperature softmax -> top-k/top-p/EOS filter ->
    inverse-CDF draw).  The uniform numbers come from a torch generator (plumbing, not math)."""
    probs = softmax_temperature(logits, temperature)
    apply_topk_topp_filter(probs, top_k, top_p, eos_token_id, eos_thresh)
    u = torch.rand(probs.shape[0], device=probs.device, generator=generator)
    return sample_from_probs(probs, u)


_LOGIT_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}      # PA_TYPE_*
_rule_words = _cabi.PerThread()         # workspaces of pa_adjust_logits


def _rules(logits, out, ids, history, history_start, repetition, presence, frequency, bias, allowed, allowed_rows, row_seq, tree):
    dev, at, kind = logits.device, logits.get_device(), _LOGIT_TYPES.get(logits.dtype)
    if logits.dim() != 2 or kind is None or not logits.is_cuda:
        raise ValueError("logits: [rows, vocab] of float32, float16 or bfloat16 on the GPU")
    (rows, V), (stride, one) = logits.shape, logits.stride()
    if V == 0 or (rows and (one != 1 or (rows > 1 and stride < V))):
        raise ValueError("logits: a vocabulary, and rows of consecutive elements that do not overlap")
    if (history is None) != (history_start is None):
        raise ValueError("history and history_start come together")

    def of(x, dtype, what, n=None):
        """The address of a vector."""
        if not isinstance(x, torch.Tensor) or x.dtype is not dtype or x.get_device() != at or x.dim() != 1 or not x.is_contiguous() or \
                (n is not None and x.numel() != n):
            raise ValueError(f"{what}: a contiguous {dtype} vector{'' if n is None else f' of {n}'} on {dev}")
        return x.data_ptr()
    i32, f32, p_seq, p_history, p_start, p_ids, p_val, p_bias, p_rows = torch.int32, torch.float32, None, None, None, None, None, None, None
    paths = (None, None, 0, None)
    if tree is not None:
        if tree.tokens is None or tree.rows != rows or tree.device != dev or row_seq is not None:
            raise ValueError("tree: one with tokens, a node for every row, on the logits' device (and then no row_seq)")
        seqs, p_seq = tree.num_seqs, tree.row_seq.data_ptr()
        paths = (tree.tokens.data_ptr(), tree.mask.data_ptr(), tree.mask.shape[1], tree.node_start.data_ptr())
    elif row_seq is not None:
        p_seq = of(row_seq, i32, "row_seq", rows)
        seqs = None             # as many as the other arguments say
    else:
        seqs = rows
    if history is not None:
        p_history = of(history, i32, "history")
        p_start = of(history_start, i32, "history_start", None if seqs is None else seqs + 1)
        seqs = history_start.numel() - 1
    arrays, values = [], []
    for x, what in ((repetition, "repetition"), (presence, "presence"), (frequency, "frequency")):
        if isinstance(x, torch.Tensor):
            arrays.append(of(x, f32, what, seqs))
            seqs = x.numel()
            values.append(0.0)
        else:
            arrays.append(None)
            values.append(float(x))
    if arrays[0] is None and not values[0] > 0:
        raise ValueError("repetition: above 0 (1 changes nothing)")
    if bias is not None:
        b_ids, b_val, b_start = bias
        p_ids, p_val = of(b_ids, i32, "bias tokens"), of(b_val, f32, "bias values", b_ids.numel())
        p_bias = of(b_start, i32, "bias starts", None if seqs is None else seqs + 1)
        seqs = b_start.numel() - 1
    masks = (0, 0)              # rows of masks, words from one to the next
    if allowed is not None:
        if allowed.dim() != 2 or allowed.dtype != torch.int32 or allowed.device != dev or allowed.shape[1] * 32 < V or \
                (allowed.numel() and allowed.stride(1) != 1) or (allowed_rows is None and allowed.shape[0] != rows):
            raise ValueError("allowed: int32 [rows, words], 32 tokens a word, the logits' vocabulary")
        if allowed_rows is not None:
            p_rows = of(allowed_rows, i32, "allowed_rows", rows)
        masks = (allowed.shape[0], allowed.stride(0) if allowed.shape[0] > 1 else allowed.shape[1])
    if rows == 0:
        return
    lib = _cabi.lib()
    with _cabi.on_device(dev):
        stream, ws, need = _cabi.stream_on(dev), None, 0
        if ids is not None:     # words that every call leaves at zero
            need = lib.pa_adjust_logits_workspace_bytes(rows)
            if _cabi.capturing(stream):         # a graph has words of its own: its replays may run beside other calls
                ws = torch.zeros(need, dtype=torch.uint8, device=dev)
            else:
                ws = _rule_words.of.get((dev.index, stream))
                if ws is None or ws.numel() < need:
                    ws = _rule_words.of[(dev.index, stream)] = torch.zeros(max(need, 1 << 14), dtype=torch.uint8, device=dev)
        # (the stride of a single row may be anything)
        status = lib.pa_adjust_logits(
            logits.data_ptr(), kind, stride if rows > 1 else V, rows, V, _cabi.ptr(out), 0 if out is None else out.stride(0) if rows > 1 else V,
            _cabi.ptr(ids), p_seq, seqs or 0, p_history, history.numel() if p_history else 0, p_start, *arrays, *values, p_ids, p_val,
            b_ids.numel() if p_ids else 0, p_bias, _cabi.ptr(allowed), *masks, p_rows, *paths, _cabi.ptr(ws), need, stream)
        if status != _cabi.PA_OK:               # what the words hold now nobody knows
            _rule_words.of.pop((dev.index, stream), None)
        _cabi.check(status, "pa_adjust_logits")


def adjust_logits(logits, history=None, history_start=None, repetition=1.0, presence=0.0, frequency=0.0, bias=None, allowed=None,
                  allowed_rows=None, row_seq=None, tree=None, out=None, ids=False):
    """What the requests of a batch ask of their logits [rows, vocab] (pa_adjust_logits), in their type; with ids=True also the greedy
    ids, (logits, ids).  For a token that stands c times in the history of the row's sequence (c > 0):
        x = x / repetition if x > 0 else x * repetition;  x -= presence;  x -= frequency * c
    then x += bias, and -inf for what is not allowed.

    history, history_start: the sequences' tokens one after the other, and where each begins [sequences + 1] (int32).
    repetition, presence, frequency: a number, or a float32 tensor per sequence.
    bias: (tokens, values, start [sequences + 1]); of two entries for a token the last counts.
    allowed: int32 [rows, words], bit v & 31 of word v >> 5 for token v; with allowed_rows, the mask of row r is allowed[allowed_rows[r]],
    and a number that there is no mask for allows everything.
    row_seq: the sequence of every row (None: row r is sequence r).  tree: the rows are the nodes of a DraftTree with tokens; the
    tokens on a node's path, its own among them, count as history.
    out: a tensor like logits (also logits itself, no other rows that overlap them)."""
    if out is None:
        out = torch.empty_like(logits, memory_format=torch.contiguous_format)
    elif out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device or (out.numel() and out.stride(1) != 1) or \
            (out.shape[0] > 1 and out.stride(0) < out.shape[1]):
        raise ValueError("out: of the logits' shape, type and device, rows of consecutive elements")
    chosen = torch.empty(logits.shape[0], dtype=torch.int32, device=logits.device) if ids else None
    _rules(logits, out, chosen, history, history_start, repetition, presence, frequency, bias, allowed, allowed_rows, row_seq, tree)
    return (out, chosen) if ids else out


def adjusted_argmax(logits, history=None, history_start=None, repetition=1.0, presence=0.0, frequency=0.0, bias=None, allowed=None,
                    allowed_rows=None, row_seq=None, tree=None):
    """The greedy ids [rows] int32 of adjust_logits' result (the lowest index of the largest), which is not written."""
    ids = torch.empty(logits.shape[0], dtype=torch.int32, device=logits.device)
    _rules(logits, None, ids, history, history_start, repetition, presence, frequency, bias, allowed, allowed_rows, row_seq, tree)
    return ids


def _matrix(logits):
    if logits.dim() != 2:
        raise ValueError("logits: [rows, vocab]")
    return logits.shape


def _draw_rules(logits, temperature, top_k, top_p, min_p, row_seq, tree):
    """(arguments of the logits, pa_draw_rules by reference, what must live until the call) of a call over logits."""
    dev, at, kind = logits.device, logits.get_device(), _LOGIT_TYPES.get(logits.dtype)
    (rows, V), (stride, one) = _matrix(logits), logits.stride()
    if kind is None or not logits.is_cuda:
        raise ValueError("logits: [rows, vocab] of float32, float16 or bfloat16 on the GPU")
    if V == 0 or (rows and ((V > 1 and one != 1) or (rows > 1 and stride < V))):
        raise ValueError("logits: a vocabulary, and rows of consecutive elements that do not overlap")
    if rows and V * logits.element_size() > _MOST_ROW_BYTES:
        raise ValueError(f"logits: rows of at most {_MOST_ROW_BYTES} bytes")

    def of(x, dtype, what, n):
        if x.dtype is not dtype or x.get_device() != at or x.dim() != 1 or not x.is_contiguous() or (n is not None and x.numel() != n):
            raise ValueError(f"{what}: a contiguous {dtype} vector{'' if n is None else f' of {n}'} on {dev}")
        return x.data_ptr()
    seqs, rules = rows, _cabi.DrawRules()
    if tree is not None:
        if tree.rows != rows or tree.device != dev or row_seq is not None:
            raise ValueError("tree: one with a node for every row, on the logits' device (and then no row_seq)")
        seqs, rules.row_seq = tree.num_seqs, tree.row_seq.data_ptr()
    elif row_seq is not None:
        rules.row_seq = of(row_seq, torch.int32, "row_seq", rows)
        seqs = None             # as many as the rules say
    for x, what, dtype in ((temperature, "temperature", torch.float32), (top_k, "top_k", torch.int32), (top_p, "top_p", torch.float32),
                           (min_p, "min_p", torch.float32)):
        if isinstance(x, torch.Tensor):
            setattr(rules, what + "s", of(x, dtype, what, seqs))
            seqs = x.numel()
        else:
            x = int(x) if dtype is torch.int32 else float(x)
            if not x >= 0 or (what == "min_p" and x > 1) or (what == "top_k" and x >= 2 ** 31):
                raise ValueError(f"{what}: not below 0{', at most 1' if what == 'min_p' else ''}")
            setattr(rules, what, x)
    rules.num_seqs = (2 ** 31 - 1) if seqs is None else seqs        # (values alone: whatever sequences the rows name)
    return (logits.data_ptr(), kind, stride if rows > 1 else V, rows, V, ctypes.byref(rules))


_MOST_ROW_BYTES = 1500000               # PA_DRAW_MOST_ROW_BYTES
_draw_spaces = _cabi.PerThread()        # workspaces of the calls below


def _draw_space(args, dev, stream, children=0):
    """(address, bytes) of a workspace for a call over these logits on a stream, and the tensor."""
    need = _cabi.lib().pa_draw_workspace_bytes(args[1], args[3], args[4], children)
    if _cabi.capturing(stream):         # a graph has a workspace of its own: its replays may run beside other calls
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
    else:
        ws = _draw_spaces.of.get((dev.index, stream))
        if ws is None or ws.numel() < need:
            ws = _draw_spaces.of[(dev.index, stream)] = torch.empty(need, dtype=torch.uint8, device=dev)
    return ws.data_ptr(), need, ws


def truncated_softmax(logits, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, row_seq=None, tree=None, out=None):
    """The distribution that the next token of every row of logits [rows, vocab] is drawn from, float32 [rows, vocab] (pa_truncated_softmax).
    With w = exp((x - max x) / temperature) a token stays if fewer than top_k are above it, if the w above it, of those that stay so far, sum up
    to less than top_p of theirs, and if its w is at least min_p; p = w / (sum of what stays).  The largest always stays, tokens of one value stay or go
    together; a row of -inf alone gives zeros.  (apply_topk_topp_filter is the reference's filter: of equal tokens the later go first, top_p counts
    before top_k, and nothing is divided again.)

    temperature, top_k, top_p, min_p: a number, or a tensor per sequence (float32; top_k int32).  temperature 0: the lowest index of the
    largest alone; top_k 0, top_p 1, min_p 0 leave nothing out.  row_seq: the sequence of every row (None: row r is sequence r); tree: the rows are the
    nodes of a DraftTree.  out: float32, rows of consecutive elements, no memory of the logits."""
    shape = _matrix(logits)
    if out is None:
        out = torch.empty(shape, dtype=torch.float32, device=logits.device)
    elif out.shape != shape or out.dtype != torch.float32 or out.device != logits.device or \
            (out.numel() and out.shape[1] > 1 and out.stride(1) != 1) or (out.shape[0] > 1 and out.stride(0) < out.shape[1]):
        raise ValueError("out: float32 of the logits' shape and device, rows of consecutive elements")
    args = _draw_rules(logits, temperature, top_k, top_p, min_p, row_seq, tree)
    if args[3]:
        with _cabi.on_device(logits.device):
            stream = _cabi.stream_on(logits.device)
            at, need, ws = _draw_space(args, logits.device, stream)
            _cabi.check(_cabi.lib().pa_truncated_softmax(*args, out.data_ptr(), out.stride(0) if args[3] > 1 else args[4], at, need, stream),
                        "pa_truncated_softmax")
    return out


def draw_tokens(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, row_seq=None, tree=None, logprobs=False):
    """Tokens drawn by the numbers `uniform` (float32 in [0, 1), [rows] or [rows, n]) from the distributions of truncated_softmax: int32 of uniform's
    shape (pa_draw_tokens).  The first token up to which the probabilities exceed the number; of n numbers a row each draws from what the ones
    before it left (n different tokens); -1 where nothing is left.  logprobs=True: (ids, log p of them, float32, -inf for -1)."""
    rows = _matrix(logits)[0]
    if uniform.dim() not in (1, 2) or uniform.shape[0] != rows or uniform.dtype is not torch.float32 or uniform.device != logits.device or \
            not uniform.is_contiguous():
        raise ValueError(f"uniform: contiguous float32 [{rows}] or [{rows}, n] on {logits.device}")
    ids = torch.empty(uniform.shape, dtype=torch.int32, device=logits.device)
    logs = torch.empty(uniform.shape, dtype=torch.float32, device=logits.device) if logprobs else None
    args = _draw_rules(logits, temperature, top_k, top_p, min_p, row_seq, tree)
    if ids.numel():
        with _cabi.on_device(logits.device):
            stream = _cabi.stream_on(logits.device)
            at, need, ws = _draw_space(args, logits.device, stream)
            _cabi.check(_cabi.lib().pa_draw_tokens(*args, uniform.data_ptr(), ids.numel() // rows, ids.data_ptr(), _cabi.ptr(logs), at, need, stream),
                        "pa_draw_tokens")
    return (ids, logs) if logprobs else ids


def verify_drafts(logits, tree, uniform, draft_probs, draft_rows=None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, distinct=False,
                  logprobs=False):
    """What a step over a DraftTree (with tokens) gives at every node, int32 [rows] (pa_verify_drafts), where the children of a node were drawn by
    chance from a draft model: the token of a child, or another one, such that the tokens along the path that tree_accept takes by these ids are distributed
    as if they had been drawn one by one from truncated_softmax(logits, ...).

    draft_probs: [n, vocab] of float32, float16 or bfloat16, rows of consecutive elements; row draft_rows[r] (int32, None: r) is what the children
    of node r were drawn from, in order, each from all of it, or with distinct=True from what the ones before it left (draw_tokens with n numbers).
    draft_rows[r] outside [0, n): children that were not drawn by chance (lookup_drafts); the id is drawn as by draw_tokens.
    uniform: float32 [rows, 2] in [0, 1): for the test of the node itself, and for the draw at it.  The rules are those of truncated_softmax,
    per sequence of the tree.  logprobs=True: (ids, log p of them)."""
    rows, V, dev = *_matrix(logits), logits.device
    if tree.tokens is None:
        raise ValueError("tree: one with tokens")
    kind = _LOGIT_TYPES.get(draft_probs.dtype)
    if kind is None or draft_probs.dim() != 2 or draft_probs.shape[1] != V or draft_probs.device != dev or \
            (draft_probs.numel() and ((V > 1 and draft_probs.stride(1) != 1) or (draft_probs.shape[0] > 1 and draft_probs.stride(0) < V))):
        raise ValueError(f"draft_probs: [n, {V}] of float32, float16 or bfloat16 on {dev}, rows of consecutive elements")
    if draft_rows is None:
        if draft_probs.shape[0] != rows:
            raise ValueError(f"draft_probs: a row for each of the {rows} nodes, or draft_rows")
    elif draft_rows.dtype is not torch.int32 or draft_rows.shape != (rows,) or draft_rows.device != dev or not draft_rows.is_contiguous():
        raise ValueError(f"draft_rows: a contiguous int32 vector of {rows} on {dev}")
    if uniform.dtype is not torch.float32 or uniform.shape != (rows, 2) or uniform.device != dev or not uniform.is_contiguous():
        raise ValueError(f"uniform: contiguous float32 [{rows}, 2] on {dev}")
    ids = torch.empty(rows, dtype=torch.int32, device=dev)
    logs = torch.empty(rows, dtype=torch.float32, device=dev) if logprobs else None
    args = _draw_rules(logits, temperature, top_k, top_p, min_p, None, tree)
    n = draft_probs.shape[0]
    if rows:
        with _cabi.on_device(dev):
            stream = _cabi.stream_on(dev)
            at, need, ws = _draw_space(args, dev, stream, tree.branches)
            _cabi.check(_cabi.lib().pa_verify_drafts(
                *args, uniform.data_ptr(), tree.tokens.data_ptr(), tree.parents.data_ptr(), tree.node_start.data_ptr(), tree.branches,
                draft_probs.data_ptr() if n else None,
                kind, draft_probs.stride(0) if n > 1 else V, n, _cabi.ptr(draft_rows), int(distinct), ids.data_ptr(), _cabi.ptr(logs),
                at, need, stream), "pa_verify_drafts")
    return (ids, logs) if logprobs else ids
