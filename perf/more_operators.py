"""What sampling with drafted tokens is timed on: the operators of a step that draws its tokens by chance and keeps its pages on the GPU.

  probs       the distribution that a row's token is drawn from: temperature, the most likely k, the most likely that make up p, those
              with a share of the largest (`sampling.truncated_softmax`)
  draw        tokens drawn from it by given random numbers, one or several different ones a row, with their log probabilities
              (`sampling.draw_tokens`)
  verify      trees of tokens drawn from a draft model, kept or replaced so that what comes out is distributed as the model's own
              (`sampling.verify_drafts`)
  pages       the page table and the slots of new rows from the sequences' lengths, without the host (`DevicePages`)

Sizes are those of the repository's decoders (12 heads of 64, 32 heads, vocabulary 50257, 32000) and of its serving benchmarks (grouped heads,
some dozen sequences, vocabularies up to 128000), from one row to full batches and long contexts."""
import itertools
import math
import os
import random
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "pagedattention-based-transformer-decoder-inference-framework_b200")

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def _ld():
    if PKG not in sys.path:
        sys.path.insert(0, PKG)
    import llm_decoder
    return llm_decoder


# ------------------------------------------------------------------------------------------------------------------ cases
# rules: which of the truncations the requests ask for; "mixed": each request its own, as in a batch of strangers
def listed():
    return [
        # a batch's distributions for a caller who draws, or scores, by himself
        dict(name="probs_batch", kind="probs", type="f32", rows=64, vocab=50257, rules="p", masked=False),
        # 16-bit logits of an odd vocabulary under grammars, every request with rules of its own
        dict(name="probs_f16_odd", kind="probs", type="f16", rows=33, vocab=32001, rules="mixed", masked=True),
        # the smallest call: one request's next token; latency is all of it
        dict(name="draw_single", kind="draw", type="f32", rows=1, vocab=50257, rules="p", masked=False, count=1, logprobs=False),
        # temperature alone
        dict(name="draw_tempered", kind="draw", type="f32", rows=64, vocab=128000, rules="none", masked=False, count=1, logprobs=True),
        # a full batch of requests with rules of their own: the largest call
        dict(name="draw_batch", kind="draw", type="f32", rows=256, vocab=128000, rules="mixed", masked=False, count=1, logprobs=True),
        # four different tokens a row from 16-bit logits: what a draft model's tree is made of
        dict(name="draw_bf16_several", kind="draw", type="bf16", rows=48, vocab=100003, rules="p", masked=True, count=4, logprobs=False),
        # one sequence with a chain of seven drafted tokens
        dict(name="verify_single", kind="verify", type="f32", drafts="f32", seqs=1, nodes=8, vocab=50257, rules="p", distinct=False, most=1, logprobs=False),
        # a serving batch with chains of drafted tokens, 16-bit logits and probabilities
        dict(name="verify_chains", kind="verify", type="bf16", drafts="bf16", seqs=64, nodes=6, vocab=128000, rules="mixed", distinct=False, most=1, logprobs=True),
        # trees whose nodes have up to four different children
        dict(name="verify_trees", kind="verify", type="f32", drafts="f32", seqs=16, nodes=32, vocab=50257, rules="none", distinct=True, most=4, logprobs=False),
        # one sequence of the 12-head decoder takes room for eight rows
        dict(name="pages_single", kind="pages", seqs=1, heads=12, ctx=333, new=8, ragged=False),
        # a serving batch, long contexts of unequal length, drafted tokens
        dict(name="pages_batch", kind="pages", seqs=128, heads=8, ctx=8192, new=32, ragged=True),
        # prompts: tables for whole contexts
        dict(name="pages_prompts", kind="pages", seqs=32, heads=32, ctx=0, new=8192, ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["probs", "draw", "draw", "draw", "verify", "verify", "pages"])
    vocab = rng.choice([32000, 50257, _log(rng, 100, 128000), _log(rng, 1000, 128000)])
    rules = rng.choice(["none", "k", "p", "m", "kp", "mixed", "mixed"])
    kind_of = rng.choice(["f32", "f32", "bf16", "f16"])
    if kind == "probs":
        return dict(kind=kind, type=kind_of, rows=_log(rng, 1, max(1, min(512, 8192000 // vocab))), vocab=vocab, rules=rules, masked=rng.random() < 0.4)
    if kind == "draw":
        count = rng.choice([1, 1, 1, rng.randint(2, 8)])
        return dict(kind=kind, type=kind_of, rows=_log(rng, 1, max(1, min(1024, 32768000 // (vocab * count)))), vocab=vocab, rules=rules,
                    masked=rng.random() < 0.4, count=count, logprobs=rng.random() < 0.5)
    if kind == "verify":
        rows = _log(rng, 1, max(1, min(512, 25731584 // vocab)))
        nodes = min(rows, _log(rng, 1, 48))
        return dict(kind=kind, type=kind_of, drafts=rng.choice(["f32", "f32", "bf16", "f16"]), seqs=max(1, rows // nodes), nodes=nodes, vocab=vocab,
                    rules=rules, distinct=rng.random() < 0.5, most=rng.randint(1, 4), logprobs=rng.random() < 0.5)
    heads, seqs = rng.choice([1, 4, 8, 12, 16, 32]), _log(rng, 1, 512)
    ctx = rng.choice([0, _log(rng, 1, max(2, 8388608 // (heads * seqs)))])
    return dict(kind=kind, seqs=seqs, heads=heads, ctx=min(ctx, 131072), new=_log(rng, 1, max(1, min(16384, 4194304 // (heads * seqs)))),
                ragged=rng.random() < 0.6)


# ---------------------------------------------------------------------------------------------- shapes: the case's, not the seed's
def _rand(c):
    return random.Random(" ".join("%s=%s" % (k, c[k]) for k in sorted(c) if k != "name"))


def _trees(c):
    """Parents of every sequence's nodes: at most `most` children a node, a chain where that is one."""
    r = _rand(c)
    out = []
    for _ in range(c["seqs"]):
        parents, children = [-1], [0]
        for i in range(1, c["nodes"]):
            p = r.choice([j for j in range(max(0, i - 8), i) if children[j] < c["most"]])
            parents.append(p)
            children[p] += 1
            children.append(0)
        out.append(parents)
    return out


def _lengths(c):
    """Tokens that every sequence has, and those that it gets."""
    r = _rand(c)
    out = []
    for _ in range(c["seqs"]):
        if c["ragged"]:
            out.append((r.randint(c["ctx"] // 8, c["ctx"]), r.randint(0 if r.random() < 0.1 else max(1, c["new"] // 4), c["new"])))
        else:
            out.append((c["ctx"], c["new"]))
    return out


def _gen(seed, *more):
    s = int(seed) & 0xFFFFFFFF
    for m in more:
        s = (s * 1000003 + m + 1) & 0x7FFFFFFFFFFF
    return torch.Generator(device="cuda").manual_seed(s)


def _i32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


class _State(dict):
    __getattr__ = dict.__getitem__


def prepare(case, seed):
    return {"probs": _prepare_draw, "draw": _prepare_draw, "verify": _prepare_verify, "pages": _prepare_pages}[case["kind"]](case, seed)


def run(state):
    return {"probs": _run_probs, "draw": _run_draw, "verify": _run_verify, "pages": _run_pages}[state.case["kind"]](state)


def work(case):
    return {"probs": _work_probs, "draw": _work_draw, "verify": _work_verify, "pages": _work_pages}[case["kind"]](case)


def exact(case, seed):
    if case["kind"] == "pages":
        return None             # whole numbers: nothing is computed
    if case["rows" if "rows" in case else "seqs"] * case["vocab"] * case.get("nodes", 1) > 100_000_000:
        return None
    return {"probs": _exact_probs, "draw": _exact_draw, "verify": _exact_verify}[case["kind"]](case, seed)


# ------------------------------------------------------------------------------------------- logits, and what is asked of them
def _logits(c, g, rows):
    """As a model gives them: a bell of tokens, and in half of the rows a few that stand out."""
    V = c["vocab"]
    x = torch.randn(rows, V, device="cuda", generator=g)
    width = 1.5 + 2.0 * torch.rand(rows, 1, device="cuda", generator=g)
    x *= width
    n = min(4, V)
    top = torch.randint(0, V, (rows, n), device="cuda", generator=g)
    sure = (torch.rand(rows, 1, device="cuda", generator=g) < 0.5) * 12.0
    x.scatter_add_(1, top, sure * torch.rand(rows, n, device="cuda", generator=g))
    if c.get("masked"):         # a grammar leaves some tokens, or most of them
        keep = torch.where(torch.rand(rows, 1, device="cuda", generator=g) < 0.5, 0.05, 0.9)
        hide = torch.rand(rows, V, device="cuda", generator=g) > keep
        hide.scatter_(1, top, False)
        x.masked_fill_(hide, float("-inf"))
    return x.to(TYPES[c["type"]])


def _rules(c, g, n):
    """temperature, top_k, top_p, min_p: a number for all, or one per request."""
    u = torch.rand(4, n, device="cuda", generator=g)
    rules = c["rules"]
    if rules == "mixed":
        on = torch.rand(4, n, device="cuda", generator=g) < 0.5
        return dict(temperature=torch.where(on[0], 0.4 + 1.2 * u[0], 1.0), top_k=torch.where(on[1], 1 + (u[1] * 100).int(), 0).to(torch.int32),
                    top_p=torch.where(on[2], 0.5 + 0.49 * u[2], 1.0), min_p=torch.where(on[3], 0.1 * u[3], 0.0))
    return dict(temperature=0.5 + u[0], top_k=50 if "k" in rules else 0, top_p=0.9 if "p" in rules else 1.0, min_p=0.05 if "m" in rules else 0.0)


def _column(x, row_seq, dtype=torch.float64):
    """A rule as a column for the rows."""
    if isinstance(x, torch.Tensor):
        return x.to(dtype)[row_seq][:, None]
    return torch.full((len(row_seq), 1), x, dtype=dtype, device="cuda")


def _weights(logits, row_seq, temperature, top_k, top_p, min_p):
    """Of what is drawn from, weights in 64 bits relative to a row's largest; 0 for what the rules leave out."""
    x = logits.double()
    V = x.shape[1]
    top = x.amax(1, keepdim=True)
    w = torch.exp((x - top) / _column(temperature, row_seq))
    order = torch.sort(x, 1, descending=True).values
    if isinstance(top_k, torch.Tensor) or top_k:
        k = _column(top_k, row_seq, torch.int64)
        border = order.gather(1, (torch.where((k > 0) & (k < V), k, V) - 1))
        w = torch.where(x >= border, w, 0.0)
    if isinstance(top_p, torch.Tensor) or top_p < 1:
        p = _column(top_p, row_seq)
        v = torch.sort(w, 1, descending=True).values            # ties stay ties: equal logits have equal weights
        before = torch.cumsum(v, 1) - v
        last = ((before < p * v.sum(1, keepdim=True)).sum(1, keepdim=True) - 1).clamp(min=0)
        w = torch.where((x >= order.gather(1, last)) | (p >= 1), w, 0.0)
    return torch.where(w >= _column(min_p, row_seq), w, 0.0)


def _pick(w, target):
    """The first token up to which the weights exceed the target [rows, 1]."""
    cum = torch.cumsum(w, 1)
    V = w.shape[1]
    over = (cum > target) & (w > 0)
    return torch.where(over, torch.arange(V, device="cuda"), V - 1).amin(1)


# ------------------------------------------------------------------------------------------------------- distribution and draws
def _prepare_draw(c, seed):
    g = _gen(seed, 1)
    s = _State(case=c, row_seq=torch.arange(c["rows"], device="cuda"), logits=_logits(c, g, c["rows"]), rules=_rules(c, g, c["rows"]))
    n = c.get("count", 1)
    s["uniform"] = torch.rand((c["rows"], n) if n > 1 else (c["rows"],), device="cuda", generator=g)
    return s


def _run_probs(s):
    if own:
        return _ld().sampling.truncated_softmax(s.logits, **s.rules)
    w = _weights(s.logits, s.row_seq, **s.rules)
    return (w / w.sum(1, keepdim=True)).float()


def _run_draw(s):
    c = s.case
    if own:
        return _ld().sampling.draw_tokens(s.logits, s.uniform, logprobs=c["logprobs"], **s.rules)
    w = _weights(s.logits, s.row_seq, **s.rules)
    total = w.sum(1, keepdim=True)
    whole, at = w, torch.arange(c["rows"], device="cuda")
    u = s.uniform.double().view(c["rows"], -1)
    ids = []
    for i in range(u.shape[1]):
        if i:
            w = w.clone() if i == 1 else w
            w[at, ids[-1]] = 0.0
        left = w.sum(1, keepdim=True)
        ids.append(torch.where(left[:, 0] > 0, _pick(w, u[:, i:i + 1] * left), -1))
    ids = torch.stack(ids, 1)
    logprobs = torch.where(ids >= 0, (whole.gather(1, ids.clamp(min=0)) / total).log(), -math.inf).float()
    ids = ids.to(torch.int32)
    if s.uniform.dim() == 1:
        ids, logprobs = ids[:, 0], logprobs[:, 0]
    return (ids, logprobs) if c["logprobs"] else ids


def _work_probs(c):
    n = c["rows"] * c["vocab"]
    return {"bytes": n * (BYTES[c["type"]] + 4), "flops": 4 * n}


def _work_draw(c):
    n = c["rows"] * c["vocab"]
    return {"bytes": n * BYTES[c["type"]] + c["rows"] * c["count"] * (12 if c["logprobs"] else 8), "flops": 4 * n}


def _exact_row(x, temperature, top_k, top_p, min_p):
    """One row's distribution from the definitions: a token counts by how many, and how much, stands above it."""
    p = torch.zeros_like(x, dtype=torch.float64)
    some = torch.nonzero(x > -math.inf)[:, 0]
    values, group, size = torch.unique(x[some].double(), return_inverse=True, return_counts=True)       # ascending
    share = torch.softmax(values / temperature + size.double().log(), 0)                                 # of all tokens of a value
    many = size.flip(0).cumsum(0).flip(0) - size                                                         # tokens above a value
    keep = torch.ones_like(values, dtype=torch.bool)
    if 0 < top_k < len(x):
        keep &= many < top_k
    if top_p < 1:
        share = share * keep / (share * keep).sum()
        above = share.flip(0).cumsum(0).flip(0) - share
        keep &= above < top_p
        keep[-1] = True
    if min_p > 0:
        keep &= (values - values[-1]) / temperature >= math.log(min_p)
    each = torch.softmax(torch.where(keep, values / temperature + size.double().log(), -math.inf), 0) / size
    p[some] = each[group]
    return p


def _of(x, i):
    return x[i].item() if isinstance(x, torch.Tensor) else x


def _exact_rows(s, row_seq):
    at = row_seq.tolist()
    return [_exact_row(x, *(_of(s.rules[k], at[r]) for k in ("temperature", "top_k", "top_p", "min_p"))) for r, x in enumerate(s.logits)]


def _exact_probs(c, seed):
    s = _prepare_draw(c, seed)
    return torch.stack(_exact_rows(s, s.row_seq))


def _exact_draw(c, seed):
    """Log probabilities of the tokens that the numbers draw; the tokens are whole numbers."""
    if not c["logprobs"]:
        return None
    s = _prepare_draw(c, seed)
    out = torch.empty(s.uniform.shape, dtype=torch.float64, device="cuda")
    for r, p in enumerate(_exact_rows(s, s.row_seq)):
        gone = p.clone()
        for i, u in enumerate(s.uniform[r].double().view(-1).tolist()):
            cum = gone.cumsum(0)
            t = min(int(torch.searchsorted(cum, u * cum[-1], right=True)), len(p) - 1) if cum[-1] > 0 else -1
            out[r].view(-1)[i] = p[t].log() if t >= 0 else -math.inf
            gone[t] = 0
    return None, out


# ------------------------------------------------------------------------------------------------------------- verification
def _prepare_verify(c, seed):
    g = _gen(seed, 2)
    trees = _trees(c)
    first = [0]
    for p in trees:
        first.append(first[-1] + len(p))
    R, V = first[-1], c["vocab"]
    s = _State(case=c, rows=R, logits=_logits(c, g, R), rules=_rules(c, g, c["seqs"]))
    s["row_seq"] = torch.repeat_interleave(torch.arange(c["seqs"], device="cuda"), torch.tensor([len(p) for p in trees], device="cuda"), output_size=R)
    children = [[] for _ in range(R)]
    for b, parents in enumerate(trees):
        for i, p in enumerate(parents):
            if p >= 0:
                children[first[b] + p].append(first[b] + i)
    # a draft model that is near the model: its distributions at the nodes that have children, and the children drawn from them
    inner = [r for r in range(R) if children[r]]
    place = {r: i for i, r in enumerate(inner)}
    s["draft_rows"] = _i32([place.get(r, -1) for r in range(R)])
    at = torch.tensor(inner, dtype=torch.int64, device="cuda")
    near = s.logits[at].float() / _column(s.rules["temperature"], s.row_seq[at], torch.float32)
    near = near + 0.7 * torch.randn(len(inner), V, device="cuda", generator=g)
    q = torch.softmax(near, 1)
    s["draft_probs"] = q.to(TYPES[c["drafts"]])
    tokens = torch.randint(0, V, (R,), device="cuda", generator=g)
    if inner:
        most = max(len(x) for x in children)
        drawn = torch.multinomial(s.draft_probs.float(), most, not c["distinct"], generator=g)
        pad = torch.tensor([children[r] + [-1] * (most - len(children[r])) for r in inner], device="cuda")
        tokens[pad[pad >= 0]] = drawn[pad >= 0]
    s["tokens"] = tokens
    s["children"] = torch.tensor([x + [-1] * (c["most"] - len(x)) for x in children], device="cuda")
    s["uniform"] = torch.rand(R, 2, device="cuda", generator=g)
    if own:
        host = tokens.cpu().tolist()
        s["tree"] = _ld().DraftTree(trees, tokens=[host[a:b] for a, b in zip(first, first[1:])], device="cuda")
    return s


def _run_verify(s):
    c = s.case
    if own:
        return _ld().sampling.verify_drafts(s.logits, s.tree, s.uniform, s.draft_probs, draft_rows=s.draft_rows, distinct=c["distinct"],
                                            logprobs=c["logprobs"], **s.rules)
    R = s.rows
    w = _weights(s.logits, s.row_seq, **s.rules)
    p = w / w.sum(1, keepdim=True)
    u = s.uniform.double()
    ids = torch.full((R,), -1, dtype=torch.int64, device="cuda")
    rest = p.clone()                                        # what is drawn from where no child is kept
    inner = torch.nonzero(s.draft_rows >= 0)[:, 0]          # the nodes with children, all alike below
    if len(inner):
        q, mine, kids = s.draft_probs.double(), p[inner], s.children[inner]
        n = len(inner)
        at = torch.arange(n, device="cuda")
        a, Q = torch.zeros(2, n, 1, dtype=torch.float64, device="cuda")
        S = torch.ones(n, 1, dtype=torch.float64, device="cuda")
        kept = torch.full((n,), -1, dtype=torch.int64, device="cuda")
        left = mine
        for j in range(kids.shape[1]):
            child = kids[:, j]
            there = (child >= 0) & (kept < 0)
            token = s.tokens[child.clamp(min=0)]
            qt = q[at, token]
            yes = there & (u[child.clamp(min=0), 0] * qt * S[:, 0] < left[at, token] * (1 - Q[:, 0]))
            kept = torch.where(yes, token, kept)
            no = (there & ~yes)[:, None]
            a = torch.where(no, a + S / (1 - Q).clamp(min=1e-18), a)
            if c["distinct"]:
                Q = torch.where(no, Q + qt[:, None], Q)
            left = torch.where(no, (mine - a * q).clamp(min=0), left)
            S = torch.where(no, left.sum(1, keepdim=True), S)
        rest[inner] = torch.where(S > 0, left, mine)
        ids[inner] = kept
    drawn = _pick(rest, u[:, 1:] * rest.sum(1, keepdim=True))
    ids = torch.where(ids >= 0, ids, drawn)
    logprobs = p.gather(1, ids[:, None])[:, 0].log().float()
    ids = ids.to(torch.int32)
    return (ids, logprobs) if c["logprobs"] else ids


def _work_verify(c):
    """The logits of every node, whose sums no test can do without; a row of draft probabilities counts where its children cannot all be kept."""
    trees = _trees(c)
    R = c["seqs"] * c["nodes"]
    inner = sum(len(set(p[1:])) for p in trees)
    n = R * c["vocab"]
    return {"bytes": n * BYTES[c["type"]] + inner * c["vocab"] * BYTES[c["drafts"]] // 2 + R * (16 if c["logprobs"] else 12), "flops": 4 * n}


def _exact_verify(c, seed):
    """Node by node: every child's own test, each time against what the children before it have left."""
    if not c["logprobs"]:
        return None
    s = _prepare_verify(c, seed)
    out = torch.empty(s.rows, dtype=torch.float64, device="cuda")
    rank, kids, tokens, u = s.draft_rows.tolist(), s.children.tolist(), s.tokens.tolist(), s.uniform.double().tolist()
    for r, p in enumerate(_exact_rows(s, s.row_seq)):
        left, took, gone = p, None, []
        if rank[r] >= 0:
            q = s.draft_probs[rank[r]].double()
            for child in kids[r]:
                if child < 0:
                    continue
                t = tokens[child]
                if u[child][0] * q[t] < left[t]:
                    took = t
                    break
                less = (left - q).clamp(min=0)
                if less.sum() <= 0:
                    left = torch.zeros_like(p)
                    continue
                left = less / less.sum()
                if c["distinct"]:
                    gone.append(t)
                    q = _without(s.draft_probs[rank[r]], gone)
        if took is None:
            if left.sum() <= 0:
                left = p
            cum = left.cumsum(0)
            took = min(int(torch.searchsorted(cum, u[r][1] * cum[-1], right=True)), len(p) - 1)
        out[r] = p[took].log()
    return None, out


def _without(q, gone):
    """A draft distribution after tokens were drawn from it: what is left of it, as much as it said it had."""
    q = q.double()
    more = 1 / (1 - q[torch.tensor(gone, device="cuda")].sum()).clamp(min=1e-18)
    q = q.clone()
    q[torch.tensor(gone, device="cuda")] = 0
    return q * more


# -------------------------------------------------------------------------------------------------------------------- pages
TILE = 16


def _prepare_pages(c, seed):
    g = _gen(seed, 3)
    lens = _lengths(c)
    s = _State(case=c, rows=sum(n for _h, n in lens), tiles=max(1, max(-(-(h + n) // TILE) for h, n in lens)))
    s["lengths"], s["start"] = _i32([h for h, _n in lens]), _i32([0, *itertools.accumulate(n for _h, n in lens)])
    total = sum(-(-(h + n) // TILE) for h, n in lens) * c["heads"] + 64
    s["total"] = total
    free = torch.randperm(total, device="cuda", generator=g).to(torch.int32)
    held, before = torch.zeros(c["seqs"], dtype=torch.int32, device="cuda"), _i32([0, *itertools.accumulate(h for h, _n in lens)])
    if own:
        ld = _ld()
        table = ld.PageTable()
        table.init(c["seqs"], c["heads"], s.tiles)
        s["pages"] = ld.DevicePages(table, total, TILE, free=free)
        s.pages.take(held, before, int(before[-1]))
    else:
        s.update(free=free, count=total, held=held, table=torch.full((c["seqs"], c["heads"], s.tiles), -1, dtype=torch.int32, device="cuda"))
        _take(s, held, before, int(before[-1]))
    return s


def _entries(s, first, last):
    """Of the tiles first[b] to last[b] of every sequence, head by head within a tile: places in the table, and their number."""
    H = s.case["heads"]
    size = (last - first).clamp(min=0).long()
    n = int(size.sum())
    seq = torch.repeat_interleave(torch.arange(len(size), device="cuda"), size, output_size=n)
    tile = first.long()[seq] + torch.arange(n, device="cuda") - (size.cumsum(0) - size)[seq]
    head = torch.arange(H, device="cuda")
    return ((seq[:, None] * H + head) * s.tiles + tile[:, None]).view(-1), n * H


def _take(s, lengths, start, rows):
    """Pages for rows behind the lengths, from the end of the free list; the new rows' sequences, positions and slots."""
    size = (start[1:] - start[:-1]).long()
    last = torch.maximum(s.held, ((lengths + size + TILE - 1) // TILE).to(torch.int32))
    at, n = _entries(s, s.held, last)
    s.table.view(-1)[at] = s.free[s.count - n:s.count].flip(0)
    s["count"], s["held"] = s.count - n, last
    seq = torch.repeat_interleave(torch.arange(len(size), device="cuda"), size, output_size=rows)
    pos = (lengths[seq] + torch.arange(rows, device="cuda") - start.long()[seq])
    slots = s.table[seq, :, pos // TILE] * TILE + (pos % TILE)[:, None]
    return seq.to(torch.int32), pos.to(torch.int32), slots.to(torch.int32)


def _run_pages(s):
    """What was taken beyond the lengths goes back, as after a step whose drafts were turned down; then room for the next rows."""
    if own:
        s.pages.release(s.lengths)
        new = s.pages.take(s.lengths, s.start, s.rows)
        return new.row_seq, new.positions, new.slots, s.pages.table.device_data().view(s.case["seqs"], s.case["heads"], s.tiles)
    keep = torch.minimum(s.held, (s.lengths + TILE - 1) // TILE)
    at, n = _entries(s, keep, s.held)
    s.free[s.count:s.count + n] = s.table.view(-1)[at].flip(0)
    s.table.view(-1)[at] = -1
    s["count"], s["held"] = s.count + n, keep
    return *_take(s, s.lengths, s.start, s.rows), s.table


def _work_pages(c):
    """An entry: read and cleared, its page into the free list and out of it, the entry written; a row: its two numbers and a slot a head."""
    entries = rows = 0
    for h, n in _lengths(c):
        entries += c["heads"] * max(0, -(-(h + n) // TILE) - -(-h // TILE))
        rows += n
    return {"bytes": 20 * entries + rows * (8 + 4 * c["heads"]) + 12 * c["seqs"], "flops": 4 * entries + 4 * rows * c["heads"]}
