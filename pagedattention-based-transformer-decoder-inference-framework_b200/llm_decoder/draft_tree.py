"""Verifying trees of drafted tokens: one step of a model over several guesses of what comes next, instead of one step per token.

    tree = DraftTree(parents, tokens, device)                   # per sequence: node 0 the pending token, then guesses, parents first
    kv.append(k, v, tree.positions(ctx_lens), tree.row_seq)     # per layer: the nodes' rows behind the context ...
    out = paged_tree_attention(q, kv, tree, ctx_lens, T)        # ... and attention of every node to the context and its ancestors
    ids = sampling.adjusted_argmax(logits, tree=tree, ...)      # what the model chooses at every node
    done = tree_accept(ids, tree, TreeCaches(layers), ctx_lens) # the path that it agrees with; its rows move to their places

`done.tokens[b, :done.counts[b]]` are the tokens that the model itself would have given one by one; the last of them is the next
pending token (it has no row in the caches yet), `done.ctx_lens` the next context lengths."""
import collections
import ctypes
import itertools

import numpy as np
import torch

from . import _cabi
from .host_stage import to_device

MOST_NODES = 1024               # PA_TREE_MOST_NODES
TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.int8: 3}      # PA_TYPE_*
_PAIRS = {(torch.float32, "f16"), (torch.float32, "i8"), (torch.float32, "f32"), (torch.float16, "f16"), (torch.float16, "i8"),
          (torch.bfloat16, "bf16")}


def _on(device):
    device = torch.device(device) if device is not None else torch.device("cuda")
    return torch.device("cuda", torch.cuda.current_device()) if device.type == "cuda" and device.index is None else device


class DraftTree:
    """The drafted nodes of a batch of sequences, on the device.  parents: per sequence the parent of every node as a number within the
    sequence, -1 for node 0 and a lower node for every other (a sequence without nodes sits the step out); tokens: per
    sequence the nodes' tokens, where ids are to be adjusted or accepted.

    rows (nodes of all sequences), num_seqs, sizes, most (nodes of the largest), depth (nodes on the longest path); int32 tensors
    node_start [num_seqs + 1], row_seq, parents, depths (0 at the root), nodes (the node's number), tokens [rows] or None, and
    mask [rows, words], bit j of which says that node j is on the row's path."""

    def __init__(self, parents, tokens=None, device=None):
        sizes = [len(p) for p in parents]
        B, R, most = len(sizes), sum(sizes), max(sizes, default=0)
        if most > MOST_NODES:
            raise ValueError(f"DraftTree: at most {MOST_NODES} nodes a sequence")
        if tokens is not None and [len(t) for t in tokens] != sizes:
            raise ValueError("DraftTree: a token for every node")
        words, rows = max(1, -(-most // 32)), 4 if tokens is None else 5
        flat = np.fromiter(itertools.chain.from_iterable(parents), np.int64, R)
        host = np.zeros(B + 1 + R * (rows + words) + 1, dtype=np.int32)         # one copy; the last word stays here
        np.cumsum(sizes, out=host[1:B + 1])
        if tokens is not None:
            host[B + 1 + 4 * R:B + 1 + 5 * R] = np.fromiter(itertools.chain.from_iterable(tokens), np.int64, R)
        at = host.ctypes.data
        row = [at + 4 * (B + 1 + i * R) for i in range(rows + 1)]               # sequences, parents, depths, nodes, (tokens,) masks
        if _cabi.lib().pa_draft_trees(flat.ctypes.data, at, B, words, *row[:4], row[rows], at + 4 * (len(host) - 1)) != _cabi.PA_OK:
            raise ValueError("DraftTree: node 0 has parent -1, every other node a lower one of its sequence")
        self.rows, self.num_seqs, self.sizes, self.most, self.depth = R, B, sizes, most, int(host[-1])
        self.device = _on(device)
        dev = to_device(torch.from_numpy(host[:-1]), self.device)
        self.node_start, *parts = dev.split_with_sizes([B + 1] + [R] * rows + [R * words])
        self.row_seq, self.parents, self.depths, self.nodes = parts[:4]
        self.tokens = None if tokens is None else parts[4]
        self.mask = parts[-1].view(R, words)
        self._space = {}                # (heads, kv heads, D) -> bytes of workspace that pa_tree_attention wants for this tree

    def positions(self, ctx_lens):
        """Where the nodes' K/V rows go in the caches (`KVTileCache.append`): behind the context, in node order."""
        return ctx_lens[self.row_seq] + self.nodes


def longest_path(parents):
    """Nodes on the longest path of one sequence's tree (its parents as for DraftTree)."""
    depths = []
    for up in parents:
        depths.append(1 if up < 0 or up >= len(depths) else depths[up] + 1)
    return max(depths, default=0)


def lookup_drafts(tokens, most, depth, branches=2, longest=3):
    """A tree of guesses from the sequence itself: (parents, tokens) of at most `most` nodes in paths of at most `depth`, node 0 being the
    last of `tokens`.  Where the last `longest` tokens (then one fewer, ... then the last one) came up before, what followed is a guess, the
    latest first, up to `branches` of them; guesses that begin alike share their nodes."""
    tokens = np.asarray(tokens)
    parents, out, child, found = [-1], [int(tokens[-1])], {}, 0
    before = tokens[:-1] == tokens[-1]          # the places of the last k tokens' ends
    matches = [before]
    for k in range(1, min(longest, len(tokens) - 1)):
        before = before.copy()
        before[:k] = False
        before[k:] &= tokens[:-1 - k] == tokens[-1 - k]
        matches.append(before)
    for ends in reversed(matches):
        for end in np.flatnonzero(ends)[::-1]:
            node, new = 0, False
            for t in tokens[end + 1:end + depth].tolist():
                if (node, t) not in child:
                    if len(out) >= most:
                        break
                    child[node, t] = len(out)
                    parents.append(node)
                    out.append(t)
                    new = True
                node = child[node, t]
            found += new
            if found == branches or len(out) >= most:
                return parents, out
    return parents, out


_workspaces = _cabi.PerThread()         # of pa_tree_attention: one for the caches of all layers, whose calls on a stream come one after the other


def _vector(x, n, device, what):
    if not isinstance(x, torch.Tensor):
        x = to_device(torch.as_tensor(np.asarray(x), dtype=torch.int32), device)
    if x.dtype is not torch.int32 or x.shape != (n,) or x.device != device or not x.is_contiguous():
        raise ValueError(f"{what}: a contiguous int32 vector of {n} on {device}")
    return x


def paged_tree_attention(q, kv_cache, tree, ctx_lens, temperature=1.0, beam_ids=None, out=None):
    """Attention of the nodes of `tree` over the pages of `kv_cache` (pa_tree_attention): q [rows, heads, D] (rows may be a view of a
    wider projection); row r of sequence b sees the first ctx_lens[b] cached tokens and, of the nodes behind them, those of its mask.
    heads is a multiple of the cache's heads.  beam_ids: table row per sequence (None: b).  ctx_lens, beam_ids: int32 device tensors,
    or sequences of ints.  out: [rows, heads, D] like q, contiguous.

    Up to 1024 sequences, heads of 64 or 128, pages of 16 rows (or multiples) that are not float; what is beyond goes through the general kernel, some
    forty times as slow where contexts are long.  Partial results are kept in a workspace per host thread and stream."""
    pt, dev = kv_cache.page_table_, kv_cache.key_buffer_.device
    KVH, D = pt.num_heads_, kv_cache.head_dim_
    if q.dim() != 3 or q.shape[0] != tree.rows or q.shape[2] != D or q.shape[1] % KVH or q.shape[1] == 0:
        raise ValueError(f"paged_tree_attention: q is [{tree.rows}, a multiple of {KVH}, {D}], not {list(q.shape)}")
    if kv_cache.value_dim_ != D:
        raise ValueError("paged_tree_attention: keys and values of one width")
    if (q.dtype, kv_cache.dtype) not in _PAIRS:
        raise ValueError(f"paged_tree_attention: {q.dtype} queries on '{kv_cache.dtype}' pages")
    if q.device != dev or tree.device != dev:
        raise ValueError("paged_tree_attention: q, tree and cache on one device")
    if not temperature:
        raise ValueError("paged_tree_attention: temperature 0")
    R, H = tree.rows, q.shape[1]
    if not q.is_contiguous() and (q.stride(2) != 1 or q.stride(1) != D or (R > 1 and q.stride(0) < H * D)):
        q = q.contiguous()
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != (R, H, D) or out.dtype != q.dtype or out.device != dev or not out.is_contiguous():
        raise ValueError("paged_tree_attention: out is contiguous, of q's shape, type and device")
    ctx_lens = _vector(ctx_lens, tree.num_seqs, dev, "ctx_lens")
    if beam_ids is not None:
        beam_ids = _vector(beam_ids, tree.num_seqs, dev, "beam_ids")
    if R == 0:
        return out
    lib = _cabi.lib()
    table = pt.device_data()
    need = tree._space.get((H, KVH, D))
    with _cabi.on_device(dev):
        stream = _cabi.stream_on(dev)
        if need is None:
            need = tree._space[(H, KVH, D)] = lib.pa_tree_attention_workspace_bytes(R, tree.num_seqs, tree.most, H, KVH, D)
        if _cabi.capturing(stream):     # a graph has a workspace of its own: its replays may run beside other calls
            ws = torch.empty(need, dtype=torch.uint8, device=dev)
        else:
            ws = _workspaces.of.get((dev.index, stream))
            if need and (ws is None or ws.numel() < need):
                ws = _workspaces.of[(dev.index, stream)] = torch.empty(need, dtype=torch.uint8, device=dev)
        _cabi.check(lib.pa_tree_attention(
            q.data_ptr(), q.stride(0) if R > 1 else H * D, TYPES[q.dtype], out.data_ptr(), kv_cache.key_buffer_.data_ptr(),
            kv_cache.value_buffer_.data_ptr(), _cabi.ptr(kv_cache.k_scales_), _cabi.ptr(kv_cache.v_scales_),
            TYPES[kv_cache.key_buffer_.dtype], table.data_ptr(), pt.num_beams_, KVH, pt.num_tiles_, kv_cache.total_pages_, _cabi.ptr(beam_ids),
            ctx_lens.data_ptr(), tree.node_start.data_ptr(), tree.mask.data_ptr(), tree.mask.shape[1], R, tree.num_seqs, tree.most, H, D,
            kv_cache.tile_size_, float(temperature), _cabi.ptr(ws) if need else None, need, stream), "pa_tree_attention")
    return out


class TreeCaches:
    """The caches of a model's layers, for tree_accept: KVTileCaches of one geometry (each with a table of its own, or one shared).
    Holds their addresses: made anew after a cache's init, resize, configure_table or adopt_buffers."""

    def __init__(self, kv_caches):
        self.caches = list(kv_caches)

        def kind(k):
            pt = k.page_table_
            return (k.key_buffer_.device, k.dtype, k.single_rows_, k.head_dim_, k.value_dim_, k.tile_size_, k.total_pages_, pt.num_beams_,
                    pt.num_heads_, pt.num_tiles_)
        if len({kind(k) for k in self.caches}) > 1:
            raise ValueError("TreeCaches: caches of one device, type and geometry")
        self.tables = list({id(k.page_table_): k.page_table_ for k in self.caches}.values())
        ptrs = []
        for k in self.caches:
            ptrs += [_cabi.ptr(k.key_buffer_), _cabi.ptr(k.value_buffer_), _cabi.ptr(k.k_scales_), _cabi.ptr(k.v_scales_),
                     k.page_table_.d_table_.data_ptr()]
        self._array = (ctypes.c_void_p * max(1, len(ptrs)))(*ptrs)
        self._geometry = (0, 0, 0, 0, 0, 0, 0)
        if self.caches:
            k, pt = self.caches[0], self.caches[0].page_table_
            e = k.key_buffer_.element_size()
            self._geometry = (pt.num_beams_, pt.num_heads_, pt.num_tiles_, k.total_pages_, k.tile_size_, k.head_dim_ * e,
                              0 if k.single_rows_ else k.value_dim_ * e)


Accepted = collections.namedtuple("Accepted", "counts tokens nodes ctx_lens")


def tree_accept(ids, tree, caches, ctx_lens, beam_ids=None):
    """What the model agrees with: from node 0 on to the child whose token is the one chosen at the node (ids [rows] int32), as long
    as there is one, and the K/V rows of that path to positions ctx_lens[b] + 0, 1, 2, ... of every cache (pa_tree_accept).
    Accepted(counts [B], tokens [B, depth], nodes [B, depth], ctx_lens [B]): nodes on the path, what was chosen at them and their
    numbers (-1 behind them), the new context lengths; int32 on the device."""
    if tree.tokens is None:
        raise ValueError("tree_accept: a tree with tokens")
    if not isinstance(caches, TreeCaches):
        caches = TreeCaches(caches)
    dev, B = tree.device, tree.num_seqs
    if caches.caches and caches.caches[0].key_buffer_.device != dev:
        raise ValueError("tree_accept: tree and caches on one device")
    ids = _vector(ids, tree.rows, dev, "ids")
    ctx_lens = _vector(ctx_lens, B, dev, "ctx_lens")
    if beam_ids is not None:
        beam_ids = _vector(beam_ids, B, dev, "beam_ids")
    paths = B * tree.depth
    counts, lens, tokens, nodes = torch.empty(2 * (B + paths), dtype=torch.int32, device=dev).split_with_sizes((B, B, paths, paths))
    tokens, nodes = tokens.view(B, tree.depth), nodes.view(B, tree.depth)
    if B == 0:
        return Accepted(counts, tokens, nodes, lens)
    if tree.rows == 0:
        counts.zero_()
        lens.copy_(ctx_lens)
        return Accepted(counts, tokens, nodes, lens)
    for t in caches.tables:
        if t._pending:
            t.flush()
    with _cabi.on_device(dev):
        _cabi.check(_cabi.lib().pa_tree_accept(
            ids.data_ptr(), tree.tokens.data_ptr(), tree.parents.data_ptr(), tree.node_start.data_ptr(), B, tree.most, tree.depth,
            ctx_lens.data_ptr(), _cabi.ptr(beam_ids), *caches._geometry, len(caches.caches), caches._array, counts.data_ptr(),
            tokens.data_ptr(), nodes.data_ptr(), lens.data_ptr(), _cabi.stream_on(dev)), "pa_tree_accept")
    return Accepted(counts, tokens, nodes, lens)
