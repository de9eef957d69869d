"""What verifying drafted tokens is timed on: the three operators that a step over trees of drafted tokens is made of.

  attention   drafted nodes of every sequence attend its cached context and their own ancestors, whose K/V rows the cache holds behind
              the context (`paged_tree_attention`)
  logits      penalties for repeated tokens, per-request biases and grammar masks, over the rows of a batch or of a tree, with the
              greedy ids where they are wanted (`sampling.adjust_logits`, `sampling.adjusted_argmax`)
  accept      the walk along the tokens that the model chose, and the move of the accepted rows to their places in the caches of all
              layers (`tree_accept`)

Sizes are those of the repository's decoders (12 heads of 64, 32 heads of 128, vocabulary 50257) and of its serving benchmarks
(grouped heads of 128, some dozen sequences), from one sequence with one drafted token to long contexts and full batches."""
import math
import os
import random
import sys

import numpy as np
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "pagedattention-based-transformer-decoder-inference-framework_b200")

own = False

TILE = 16
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}


def _ld():
    if PKG not in sys.path:
        sys.path.insert(0, PKG)
    import llm_decoder
    return llm_decoder


# ------------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the smallest call: one sequence of the 12-head decoder, some hundred tokens in, eight drafted tokens; latency is all of it
        dict(name="attention_f16_single", kind="attention", pool="f16", q="f32", seqs=1, nodes=8, heads=12, kv_heads=12, dim=64, ctx=333, ragged=False),
        # a serving batch with grouped heads: 32 drafted tokens for each of 32 requests, 4K tokens of context
        dict(name="attention_bf16_batch", kind="attention", pool="bf16", q="bf16", seqs=32, nodes=32, heads=32, kv_heads=8, dim=128, ctx=4096, ragged=False),
        # one request with a long context and a wide tree: little parallelism but along the keys
        dict(name="attention_bf16_long", kind="attention", pool="bf16", q="bf16", seqs=1, nodes=64, heads=16, kv_heads=4, dim=128, ctx=131072, ragged=False),
        # int8 pages of the 32-head decoder, requests of unequal length with trees of unequal size
        dict(name="attention_i8_ragged", kind="attention", pool="i8", q="f32", seqs=48, nodes=16, heads=32, kv_heads=32, dim=128, ctx=2048, ragged=True),
        # one request's next token under penalties: the smallest call
        dict(name="logits_single", kind="logits", type="f32", seqs=1, nodes=0, vocab=50257, history=333, bias=8, masked=False, want="both"),
        # a full batch with penalties, biases and grammars, adjusted logits for a sampler
        dict(name="logits_batch", kind="logits", type="f32", seqs=256, nodes=0, vocab=128000, history=4096, bias=64, masked=True, want="logits"),
        # the nodes of a batch of trees, greedy ids only
        dict(name="logits_tree", kind="logits", type="f32", seqs=16, nodes=32, vocab=50257, history=2048, bias=0, masked=True, want="ids"),
        # 16-bit logits of an odd vocabulary, both results
        dict(name="logits_bf16_odd", kind="logits", type="bf16", seqs=100, nodes=0, vocab=100003, history=1000, bias=16, masked=True, want="both"),
        # one sequence of the 12-layer decoder
        dict(name="accept_single", kind="accept", pool="f16", seqs=1, nodes=8, layers=12, kv_heads=12, dim=64, ctx=25),
        # a serving batch: 24 requests of 32 drafted tokens, 16 layers
        dict(name="accept_batch", kind="accept", pool="f16", seqs=24, nodes=32, layers=16, kv_heads=8, dim=128, ctx=40),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "logits", "logits", "accept"])
    if kind == "attention":
        heads, kv, dim = rng.choice([(12, 12, 64), (16, 16, 64), (16, 4, 128), (32, 8, 128), (8, 1, 128), (32, 32, 128)])
        pool = rng.choice(["f16", "bf16", "bf16", "i8"])
        q = "bf16" if pool == "bf16" else rng.choice(["f32", "f16"])
        seqs, nodes = _log(rng, 1, 64), _log(rng, 1, 128)
        # no dearer than the largest listed case: 137 GFLOP, 0.5 GB of keys and values
        most = min(131072, 137e9 / (4.0 * seqs * nodes * heads * dim), 5e8 / (4.0 * seqs * kv * dim))
        return dict(kind=kind, pool=pool, q=q, seqs=seqs, nodes=nodes, heads=heads, kv_heads=kv, dim=dim,
                    ctx=_log(rng, 1, max(2, most)), ragged=rng.random() < 0.6)
    if kind == "logits":
        vocab = rng.choice([32000, 50257, _log(rng, 1000, 128000)])
        rows = _log(rng, 1, max(1, min(512, 32768000 // vocab)))
        nodes = rng.choice([0, 0, min(rows, _log(rng, 1, 64))])
        return dict(kind=kind, type=rng.choice(["f32", "f32", "bf16", "f16"]), seqs=max(1, rows // nodes) if nodes else rows, nodes=nodes,
                    vocab=vocab, history=_log(rng, 1, 4096), bias=rng.choice([0, _log(rng, 1, 200)]), masked=rng.random() < 0.6,
                    want=rng.choice(["both", "logits", "ids"]))
    kv, dim = rng.choice([(12, 64), (8, 128), (4, 128), (16, 64)])
    return dict(kind=kind, pool=rng.choice(["f16", "bf16"]), seqs=_log(rng, 1, 24), nodes=_log(rng, 2, 32), layers=rng.randint(1, 16), kv_heads=kv,
                dim=dim, ctx=rng.randint(0, 40))


# ---------------------------------------------------------------------------------------------- shapes: the case's, not the seed's
def _rand(c):
    return random.Random(" ".join("%s=%s" % (k, c[k]) for k in sorted(c) if k != "name"))


def _shape(c):
    """Per sequence: (tokens of context, parents of the drafted nodes).  Node 0 is the root; a parent comes before its children."""
    r = _rand(c)
    out = []
    for _ in range(c["seqs"]):
        ctx, n = c["ctx"], c["nodes"]
        if c.get("ragged"):
            ctx, n = r.randint(0 if r.random() < 0.1 else ctx // 8, ctx), r.randint(max(1, n // 4), n)
        out.append((ctx, [-1] + [r.randint(max(0, i - 6), i - 1) for i in range(1, n)]))
    return out


def _paths(parents):
    """Per node, the nodes from the root to it."""
    out = []
    for i, p in enumerate(parents):
        out.append((out[p] if p >= 0 else []) + [i])
    return out


def _gen(seed, *more):
    s = int(seed) & 0xFFFFFFFF
    for m in more:
        s = (s * 1000003 + m + 1) & 0x7FFFFFFFFFFF
    return torch.Generator(device="cuda").manual_seed(s)


def _i32(a):
    return torch.tensor(np.asarray(a, dtype=np.int32), device="cuda")


class _State(dict):
    __getattr__ = dict.__getitem__


def _pages(c, shape, g, rows_of):
    """A page table [seqs, kv heads, tiles] of shuffled pages, and how many there are."""
    tiles = max(1, max(-(-(ctx + n) // TILE) for ctx, n in rows_of))
    total = c["seqs"] * c["kv_heads"] * tiles
    return torch.randperm(total, device="cuda", generator=g).to(torch.int32).view(c["seqs"], c["kv_heads"], tiles), total, tiles


def _cache(s, c, k, v, ks=None, vs=None, owner=None):
    ld = _ld()
    cache = ld.KVTileCache(c["pool"])
    cache.adopt_buffers(k, v, ks, vs)
    if owner is not None:
        cache.share_pages(owner)
        return cache
    cache.configure_table(c["seqs"], c["kv_heads"], s.tiles)
    cache.page_table_.load_host_table(s.table.cpu().numpy())
    return cache


def prepare(case, seed):
    return {"attention": _prepare_attention, "logits": _prepare_logits, "accept": _prepare_accept}[case["kind"]](case, seed)


def run(state):
    return {"attention": _run_attention, "logits": _run_logits, "accept": _run_accept}[state.case["kind"]](state)


def work(case):
    return {"attention": _work_attention, "logits": _work_logits, "accept": _work_accept}[case["kind"]](case)


def exact(case, seed):
    if case["kind"] == "accept":
        return None             # moves and whole numbers: nothing is computed
    return {"attention": _exact_attention, "logits": _exact_logits}[case["kind"]](case, seed)


# -------------------------------------------------------------------------------------------------------------- attention
def _prepare_attention(c, seed):
    g = _gen(seed, 1)
    shape = _shape(c)
    sizes = [len(p) for _c, p in shape]
    s = _State(case=c, shape=shape, start=np.concatenate([[0], np.cumsum(sizes)]), temperature=math.sqrt(c["dim"]))
    s["table"], total, s["tiles"] = _pages(c, shape, g, [(ctx, len(p)) for ctx, p in shape])
    R, D = int(s.start[-1]), c["dim"]
    s["q"] = torch.randn(R, c["heads"], D, device="cuda", generator=g).to(TYPES[c["q"]])
    s["ks"] = s["vs"] = None
    if c["pool"] == "i8":
        for n in "kv":
            x = torch.randn(total, TILE, D, device="cuda", generator=g)
            s[n + "s"] = 127.0 / (x.abs().amax(-1) + 1e-6)
            s[n] = torch.round(x * s[n + "s"][..., None]).clamp(-128, 127).to(torch.int8)
    else:
        for n in "kv":
            s[n] = torch.empty(total, TILE, D, device="cuda", dtype=TYPES[c["pool"]])
            for i in range(0, total, 1 << 15):
                s[n][i:i + (1 << 15)] = torch.randn(min(1 << 15, total - i), TILE, D, device="cuda", generator=g).to(TYPES[c["pool"]])
    s["ctx"] = _i32([ctx for ctx, _p in shape])
    s["seen"] = []              # per sequence, the ancestors of every node
    for _ctx, p in shape:
        m = torch.zeros(len(p), len(p), dtype=torch.bool)
        for i, path in enumerate(_paths(p)):
            m[i, path] = True
        s.seen.append(m.cuda())
    if own:
        s["cache"] = _cache(s, c, s.k, s.v, s.ks, s.vs)
        s["tree"] = _ld().DraftTree([p for _c, p in shape], device="cuda")
    return s


def _run_attention(s):
    c = s.case
    if own:
        return _ld().paged_tree_attention(s.q, s.cache, s.tree, s.ctx, temperature=s.temperature)
    out = torch.empty_like(s.q)
    KV, D = c["kv_heads"], c["dim"]
    for b, (ctx, p) in enumerate(s.shape):
        n, r0, T = len(p), int(s.start[b]), ctx + len(p)
        pages = s.table[b, :, :-(-T // TILE)].long()
        k, v = s.k[pages].float(), s.v[pages].float()                       # [KV, tiles, TILE, D]
        if s.ks is not None:
            k, v = k / s.ks[pages][..., None], v / s.vs[pages][..., None]
        k, v = k.reshape(KV, -1, D)[:, :T], v.reshape(KV, -1, D)[:, :T]
        q = s.q[r0:r0 + n].float().view(n, KV, -1, D).permute(1, 2, 0, 3).reshape(KV, -1, D)       # rows: head of the group, node
        x = torch.matmul(q, k.transpose(1, 2)).view(KV, -1, n, T) / s.temperature
        x[..., ctx:].masked_fill_(~s.seen[b], float("-inf"))
        x = torch.exp(x - x.amax(-1, keepdim=True))
        x = x / (x.sum(-1, keepdim=True) + 1e-6)
        o = torch.matmul(x.view(KV, -1, T), v).view(KV, -1, n, D)
        out[r0:r0 + n] = o.permute(2, 0, 1, 3).reshape(n, c["heads"], D).to(out.dtype)
    return out


def _work_attention(c):
    kv = pairs = rows = 0
    for ctx, p in _shape(c):
        depth = []
        for q in p:
            depth.append(1 if q < 0 else depth[q] + 1)
        kv += ctx + len(p)
        rows += len(p)
        pairs += ctx * len(p) + sum(depth)
    row = 2 * (c["dim"] * BYTES[c["pool"]] + (4 if c["pool"] == "i8" else 0))
    return {"bytes": kv * c["kv_heads"] * row + 2 * rows * c["heads"] * c["dim"] * BYTES[c["q"]], "flops": 4 * pairs * c["heads"] * c["dim"]}


def _exact_attention(c, seed):
    """Head by head in 64 bits, by position: the row of key t of a sequence is page * TILE + t % TILE of the pool's rows."""
    s = _prepare_attention(c, seed)
    out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    G = c["heads"] // c["kv_heads"]
    krows, vrows = s.k.view(-1, c["dim"]), s.v.view(-1, c["dim"])
    for b, (ctx, p) in enumerate(s.shape):
        n, r0 = len(p), int(s.start[b])
        t = torch.arange(ctx + n, device="cuda")
        hidden = torch.zeros(n, ctx + n, dtype=torch.bool, device="cuda")
        for i, path in enumerate(_paths(p)):
            off = torch.ones(n, dtype=torch.bool)
            off[path] = False
            hidden[i, ctx:] = off.cuda()
        for g in range(c["kv_heads"]):
            at = s.table[b, g].long()[t // TILE] * TILE + t % TILE
            k, v = krows[at].double(), vrows[at].double()
            if s.ks is not None:
                k, v = k / s.ks.view(-1)[at].double()[:, None], v / s.vs.view(-1)[at].double()[:, None]
            for h in range(g * G, (g + 1) * G):
                z = s.q[r0:r0 + n, h].double() @ k.t() / float(s.temperature)
                z.masked_fill_(hidden, -math.inf)
                top = z.max(dim=1).values
                e = (z - top[:, None]).exp()
                out[r0:r0 + n, h] = (e @ v) / (e.sum(1) + 1e-6)[:, None]
    return out


# ----------------------------------------------------------------------------------------------------------------- logits
def _prepare_logits(c, seed):
    g = _gen(seed, 2)
    r = _rand(c)
    V, B = c["vocab"], c["seqs"]
    shape = _shape(dict(c, ctx=0)) if c["nodes"] else None
    sizes = [len(p) for _c, p in shape] if shape else [1] * B
    R = sum(sizes)
    s = _State(case=c, rows=R, row_seq=torch.tensor(np.repeat(np.arange(B), sizes), device="cuda"))
    s["logits"] = (torch.randn(R, V, device="cuda", generator=g) * 3).to(TYPES[c["type"]])
    lens = [r.randint(c["history"] // 2, c["history"]) for _ in range(B)]
    lens[0] = c["history"]

    def tokens(n):              # as text has them: some often, most never
        u = torch.rand(n, device="cuda", generator=g)
        return (torch.exp(u * math.log(V)) - 1).to(torch.int32).clamp_(0, V - 1)
    s["history"] = tokens(sum(lens))
    s["history_start"] = _i32(np.concatenate([[0], np.cumsum(lens)]))
    s["history_seq"] = torch.tensor(np.repeat(np.arange(B), lens), device="cuda")
    u = torch.rand(3, B, device="cuda", generator=g)
    s["repetition"], s["presence"], s["frequency"] = 1.0 + 0.5 * u[0], 0.8 * u[1], 0.3 * u[2]
    s["bias"] = None
    if c["bias"]:
        ids = torch.stack([torch.randperm(V, device="cuda", generator=g)[:c["bias"]] for _ in range(B)]).to(torch.int32)
        s["bias"] = (ids.reshape(-1), torch.randn(B * c["bias"], device="cuda", generator=g) * 2,
                     _i32(np.arange(B + 1) * c["bias"]))
    s["allowed"] = None
    if c["masked"]:             # a grammar leaves a few tokens, or most of them
        few = torch.rand(R, 1, device="cuda", generator=g) < 0.5
        words = (V + 31) // 32
        a, b, d = (torch.randint(-2 ** 31, 2 ** 31, (R, words), device="cuda", generator=g).to(torch.int32) for _ in range(3))
        s["allowed"] = torch.where(few, a & b & d, a | b | d)
    s["node_tokens"] = None
    if shape:
        s["node_tokens"] = tokens(R)
        first = np.concatenate([[0], np.cumsum(sizes)])
        s["up"] = torch.tensor(np.concatenate([[first[b] + q if q >= 0 else -1 for q in p] for b, (_c, p) in enumerate(shape)]), device="cuda")
        s["depth"] = max(len(x) for _c, p in shape for x in _paths(p))
    if own:
        s["tree"] = None
        if shape:
            host = s.node_tokens.cpu().tolist()
            s["tree"] = _ld().DraftTree([p for _c, p in shape], tokens=[host[first[b]:first[b + 1]] for b in range(B)], device="cuda")
    return s


def _run_logits(s):
    c = s.case
    if own:
        sampling = _ld().sampling
        kw = dict(history=s.history, history_start=s.history_start, repetition=s.repetition, presence=s.presence, frequency=s.frequency,
                  bias=s.bias, allowed=s.allowed, tree=s.tree)
        if c["want"] == "ids":
            return sampling.adjusted_argmax(s.logits, **kw)
        return sampling.adjust_logits(s.logits, ids=c["want"] == "both", **kw)
    V, R = c["vocab"], s.rows
    per_seq = torch.zeros(c["seqs"] * V, device="cuda").index_add_(0, s.history_seq * V + s.history, torch.ones(len(s.history), device="cuda"))
    count = per_seq.view(-1, V)[s.row_seq]
    if s.node_tokens is not None:
        at = torch.arange(R, device="cuda")
        for _ in range(s.depth):
            on = at >= 0
            count.view(-1).index_add_(0, (torch.arange(R, device="cuda") * V + s.node_tokens[at.clamp(min=0)]), on.float())
            at = torch.where(on, s.up[at.clamp(min=0)], at)
    x = s.logits.float()
    seen = count > 0
    rep = s.repetition[s.row_seq][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - torch.where(seen, s.presence[s.row_seq][:, None], 0.0)
    x = x - s.frequency[s.row_seq][:, None] * count
    if s.bias is not None:
        add = torch.zeros(c["seqs"] * V, device="cuda")
        add[torch.arange(c["seqs"], device="cuda").repeat_interleave(c["bias"]) * V + s.bias[0]] = s.bias[1]
        x = x + add.view(-1, V)[s.row_seq]
    if s.allowed is not None:
        bits = (s.allowed[:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        x = x.masked_fill(bits.view(R, -1)[:, :V] == 0, float("-inf"))
    if c["want"] == "logits":
        return x.to(s.logits.dtype)
    top = x.amax(-1, keepdim=True)
    ids = torch.where(x == top, torch.arange(V, device="cuda"), V).amin(-1).to(torch.int32)
    return ids if c["want"] == "ids" else (x.to(s.logits.dtype), ids)


def _work_logits(c):
    rows = sum(len(p) for _c, p in _shape(dict(c, ctx=0))) if c["nodes"] else c["seqs"]
    e = BYTES[c["type"]] * (1 if c["want"] == "ids" else 2)
    small = 4 * c["seqs"] * (c["history"] * 3 // 4 + 2 * c["bias"]) + 4 * rows
    return {"bytes": rows * c["vocab"] * e + (rows * ((c["vocab"] + 31) // 32) * 4 if c["masked"] else 0) + small, "flops": rows * c["vocab"]}


def _exact_logits(c, seed):
    """Row by row in 64 bits from the tokens themselves."""
    if c["want"] == "ids":
        return None
    s = _prepare_logits(c, seed)
    out = s.logits.double()
    lens = s.history_start.tolist()
    for r in range(s.rows):
        b = int(s.row_seq[r])
        past = s.history[lens[b]:lens[b + 1]].long()
        if s.node_tokens is not None:
            walk, at = [], r
            while at >= 0:
                walk.append(int(s.node_tokens[at]))
                at = int(s.up[at])
            past = torch.cat([past, torch.tensor(walk, device="cuda")])
        ids, n = torch.unique(past, return_counts=True)
        row = out[r]
        old, rep = row[ids], float(s.repetition[b])
        row[ids] = torch.where(old > 0, old / rep, old * rep) - float(s.presence[b]) - float(s.frequency[b]) * n.double()
        if s.bias is not None:
            mine = slice(b * c["bias"], (b + 1) * c["bias"])
            row[s.bias[0][mine].long()] += s.bias[1][mine].double()
        if s.allowed is not None:
            v = torch.arange(c["vocab"], device="cuda")
            row[((s.allowed[r].long()[v // 32] >> (v % 32)) & 1) == 0] = -math.inf
    return out if c["want"] == "logits" else (out, None)


# ----------------------------------------------------------------------------------------------------------------- accept
def _walks(c, shape):
    """Per sequence the accepted path: from the root down, as far as a draft is believed.  A row is moved over places that hold no row of
    the same path, so that a pass leaves what a second one finds."""
    r = _rand(dict(c, walk=1))
    out = []
    for _ctx, p in shape:
        ways = _paths(p)
        r.shuffle(ways)
        out.append(next(w for w in ways + [[0]] if all(i == d or i >= len(w) for d, i in enumerate(w))))
    return out


def _prepare_accept(c, seed):
    g = _gen(seed, 3)
    shape = _shape(c)
    sizes = [len(p) for _c, p in shape]
    R, D, start = sum(sizes), c["dim"], np.concatenate([[0], np.cumsum(sizes)])
    s = _State(case=c, shape=shape, rows=R)
    s["table"], total, s["tiles"] = _pages(c, shape, g, [(ctx, len(p)) for ctx, p in shape])
    s["k"], s["v"] = ([torch.randn(total, TILE, D, device="cuda", generator=g).to(TYPES[c["pool"]]) for _ in range(c["layers"])] for _ in range(2))
    tokens = torch.randint(0, 50257, (R,), device="cuda", generator=g).to(torch.int32)
    ids = torch.randint(50257, 60000, (R,), device="cuda", generator=g).to(torch.int32)       # what the model chose: no child has it ...
    for b, w in enumerate(_walks(c, shape)):
        for above, below in zip(w, w[1:]):
            ids[start[b] + above] = tokens[start[b] + below]                                    # ... but along the path
    s["tokens"], s["ids"], s["ctx"] = tokens, ids, _i32([ctx for ctx, _p in shape])
    n = max(sizes)
    pad = lambda rows: torch.tensor([list(x) + [-2] * (n - len(x)) for x in rows], device="cuda")  # noqa: E731
    s["parents"] = pad([p for _c, p in shape])
    s["at"] = pad([range(a, b) for a, b in zip(start, start[1:])])
    s["depth"] = max(len(x) for _c, p in shape for x in _paths(p))
    if own:
        ld = _ld()
        host = tokens.cpu().tolist()
        s["tree"] = ld.DraftTree([p for _c, p in shape], tokens=[host[a:b] for a, b in zip(start, start[1:])], device="cuda")
        caches = []
        for k, v in zip(s.k, s.v):
            caches.append(_cache(s, c, k, v, owner=caches[0] if caches else None))
        s["caches"] = ld.TreeCaches(caches)
    return s


def _run_accept(s):
    c = s.case
    if own:
        a = _ld().tree_accept(s.ids, s.tree, s.caches, s.ctx)
        return a.counts, a.tokens, a.nodes, a.ctx_lens, s.k, s.v
    B, dev = c["seqs"], "cuda"
    b = torch.arange(B, device=dev)
    node_ids, node_tokens = s.ids[s.at.clamp(min=0)], torch.where(s.at >= 0, s.tokens[s.at.clamp(min=0)], -1)
    nodes = torch.full((B, s.depth), -1, dtype=torch.int32, device=dev)
    out = torch.full((B, s.depth), -1, dtype=torch.int32, device=dev)
    counts = torch.zeros(B, dtype=torch.int32, device=dev)
    cur, on = torch.zeros(B, dtype=torch.long, device=dev), torch.ones(B, dtype=torch.bool, device=dev)
    N = s.parents.shape[1]
    for d in range(s.depth):
        chosen = node_ids[b, cur]
        nodes[:, d] = torch.where(on, cur, -1)
        out[:, d] = torch.where(on, chosen, -1)
        counts += on
        hit = (s.parents == cur[:, None]) & (node_tokens == chosen[:, None])
        nxt = torch.where(hit, torch.arange(N, device=dev), N).amin(-1)
        on = on & (nxt < N)
        cur = torch.where(on, nxt, cur)
    # the rows of the accepted nodes, layer by layer: all read before any is written
    d = torch.arange(s.depth, device=dev)
    keep = nodes >= 0
    src, dst = (s.ctx[:, None] + nodes.clamp(min=0)).long(), (s.ctx[:, None] + d).long()
    dst = torch.where(keep, dst, src)

    def rows(pos):              # [B, depth, kv heads]
        return s.table[b[:, None], :, (pos // TILE)].long() * TILE + (pos % TILE)[..., None]
    at, to = rows(src)[keep], rows(dst)[keep]
    for pool in s.k + s.v:
        flat = pool.view(-1, c["dim"])
        flat[to] = flat[at]
    return counts, out, nodes, s.ctx + counts, s.k, s.v


def _work_accept(c):
    shape = _shape(c)
    moved = sum(sum(1 for d, i in enumerate(w) if i != d) for w in _walks(c, shape))
    rows = sum(len(p) for _c, p in shape)
    row = 2 * c["layers"] * c["kv_heads"] * c["dim"] * BYTES[c["pool"]]
    return {"bytes": 2 * moved * row + 12 * rows, "flops": 4 * rows}
