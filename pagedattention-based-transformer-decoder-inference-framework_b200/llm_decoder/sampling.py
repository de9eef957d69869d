"""Device-side sampling over vocabulary logits: the reference's CPU filters
(attention_cpu/softmax_lut.cpp:203-256) and its GPU sketch (attention/top_k_top_p_filter.cuh:55-111)
as three kernels of libpa_b200.so.  Tensors are CUDA float32 [rows, vocab]."""
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
