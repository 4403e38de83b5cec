"""Operators that check drafted tokens over a paged key/value cache, as a serving program calls them: the rotation and the
append of a step's tokens to the pages, attention of single tokens, of trees of drafted tokens and of pieces of prompts over
them, the decision which drafted tokens stand against the target's probabilities, and the move of the accepted ones' keys.

A step's tokens are nodes, packed: sequence b owns rows cu[b] .. cu[b + 1] - 1.  Node 0 of a sequence is the token that was
accepted last, the others are drafted; parents[i] is the node of the same sequence that node i continues (-1 for node 0).
Without parents node i continues node i - 1.  A layer of the cache is [2][pages][Nkv][page size][H] (keys, values), slot s of
sequence b lies in page table[b][s // page size] at s % page size, and past[b] slots are filled before the step.
"""
import functools
import math
import os
import random
import sys

import torch

own = False

BF16 = torch.bfloat16
EPS = 1e-6
MAX_POSITIONS = 16384

# query heads, key heads, head size
HEADS = {
    "llama-7b": (32, 32, 128),
    "llama-70b": (64, 8, 128),
    "qwen2-7b": (28, 4, 128),
    "gptj-6b": (16, 16, 256),
    "small": (12, 4, 64),
    "odd": (10, 2, 96),
}
LOGITS = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # a single token of one sequence goes to its page: latency alone
        {"name": "append 1 token", "op": "append", "heads": "qwen2-7b", "batch": 1, "longest": 1, "shortest": 1, "past": 700, "page": 16,
         "tree": False, "norm": False, "style": "llama", "strided": True},
        # trees of drafted tokens of a serving batch, norms of the heads, q, k and v as views of one projection's rows
        {"name": "append 24 trees", "op": "append", "heads": "llama-70b", "batch": 24, "longest": 61, "shortest": 20, "past": 2500, "page": 64,
         "tree": True, "norm": True, "style": "llama", "strided": True},
        # one sequence decoding, small pages, a key head per query head
        {"name": "decode 1 x 1900", "op": "attn", "heads": "llama-7b", "batch": 1, "longest": 1, "shortest": 1, "past": 1900, "page": 16,
         "tree": False},
        # the largest step of single tokens: a serving batch of uneven lengths, where the cache's bytes count
        {"name": "decode 48 up to 9000", "op": "attn", "heads": "llama-70b", "batch": 48, "longest": 1, "shortest": 1, "past": 9000, "page": 64,
         "tree": False},
        # a tree of drafted tokens of one sequence
        {"name": "tree 60 behind 5000", "op": "attn", "heads": "qwen2-7b", "batch": 1, "longest": 60, "shortest": 60, "past": 5000, "page": 64,
         "tree": True},
        # trees of a batch, odd sizes, pages that end inside the step's tokens
        {"name": "16 trees up to 25", "op": "attn", "heads": "llama-70b", "batch": 16, "longest": 25, "shortest": 9, "past": 4000, "page": 32,
         "tree": True},
        # the next piece of a long prompt
        {"name": "chunk 700 behind 9000", "op": "attn", "heads": "llama-70b", "batch": 1, "longest": 700, "shortest": 700, "past": 9000,
         "page": 256, "tree": False},
        # a short chain from a lookup in the prompt, greedy
        {"name": "verify 5 greedy", "op": "verify", "vocab": 32000, "batch": 1, "longest": 5, "shortest": 5, "tree": False, "drafts": False,
         "temperature": 0.0, "dtype": "bf16"},
        # chains drawn by a draft model, sampled
        {"name": "verify 24 chains drawn", "op": "verify", "vocab": 128000, "batch": 24, "longest": 7, "shortest": 4, "tree": False,
         "drafts": True, "temperature": 0.8, "dtype": "bf16"},
        # trees of likely continuations, sampled
        {"name": "verify 10 trees", "op": "verify", "vocab": 152000, "batch": 10, "longest": 60, "shortest": 25, "tree": True, "drafts": False,
         "temperature": 1.0, "dtype": "bf16"},
        # the accepted path of one sequence in a small stack
        {"name": "keep 1 in 4 layers", "op": "keep", "heads": "small", "batch": 1, "longest": 24, "shortest": 24, "past": 90, "page": 16,
         "layers": 4},
        # the same for a batch in a whole stack
        {"name": "keep 12 in 28 layers", "op": "keep", "heads": "qwen2-7b", "batch": 12, "longest": 61, "shortest": 30, "past": 200, "page": 64,
         "layers": 28},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(["append", "attn", "attn", "attn", "verify", "verify", "keep"])
    case = {"op": op}
    if op == "verify":
        case["vocab"] = rng.choice([_log_int(rng, 500, 152000), 32000, 50401, 128000])
        case["drafts"] = rng.random() < 0.4
        case["tree"] = not case["drafts"] and rng.random() < 0.7
        case["batch"] = _log_int(rng, 1, 24)
        rows = min(400, 60000000 // case["vocab"]) // case["batch"]
        case["longest"] = _log_int(rng, 1, max(1, min(64 if case["tree"] else 9, rows)))
        case["shortest"] = rng.randint(1, case["longest"])
        case["temperature"] = rng.choice([0.0, 1.0, round(rng.uniform(0.3, 1.5), 2)])
        case["dtype"] = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        return case
    case["heads"] = rng.choice(list(HEADS))
    case["page"] = rng.choice([16, 32, 64, 128, 256])
    if op == "keep":
        case["batch"], case["layers"] = _log_int(rng, 1, 12), _log_int(rng, 1, 28)
        case["longest"] = _log_int(rng, 2, 64)
        case["shortest"] = rng.randint(1, case["longest"])
        case["past"] = rng.randint(1, 200)
        return case
    if op == "append":
        case["batch"] = _log_int(rng, 1, 32)
        case["tree"] = rng.random() < 0.5
        case["longest"] = rng.choice([1, _log_int(rng, 1, 1 + (64 if case["tree"] else 1400 // case["batch"]))])
        case["past"] = rng.choice([0, rng.randint(1, 3000)])
        case["norm"], case["strided"] = rng.random() < 0.4, rng.random() < 0.5
        case["style"] = rng.choice(["llama", "llama", "gptj"])
    else:
        kind = rng.choice(["decode", "tree", "chunk"])
        case["tree"] = kind == "tree"
        case["batch"] = _log_int(rng, 1, {"decode": 48, "tree": 16, "chunk": 6}[kind])
        case["longest"] = 1 if kind == "decode" else _log_int(rng, 2, 64) if kind == "tree" else _log_int(rng, 2, 700 // case["batch"])
        keys = {"decode": 100000, "tree": 30000, "chunk": 9000}[kind] // case["batch"]
        case["past"] = rng.choice([0, _log_int(rng, 1, min(9000, keys)), _log_int(rng, 1, min(9000, keys))])
    case["shortest"] = rng.randint(1, case["longest"])
    return case


def _lengths(batch, longest, shortest):
    """`batch` lengths from `longest` to `shortest`, in no order of size but the first."""
    step = [(7 * b) % batch for b in range(batch)] if batch % 7 else list(range(batch))
    return [round(longest * (shortest / longest) ** (s / max(1, batch - 1))) for s in step]


def _pasts(case):
    past = case["past"]
    return _lengths(case["batch"], past, max(1, past // 8)) if past else [0] * case["batch"]


@functools.lru_cache(maxsize=None)
def _tree(nodes, which):
    """Parents of a tree of that many nodes, level by level: a wide first level, fewer continuations of its first nodes."""
    rng = random.Random(1000 * which + nodes)
    parents, level = [-1], [0]
    while len(parents) < nodes:
        wide = min(nodes - len(parents), max(1, round(nodes * (0.4 if len(level) == 1 and level[0] == 0 else 0.2))))
        # (earlier candidates are the likelier ones and have more children)
        chosen = sorted(level[min(int(rng.expovariate(2.0) * len(level)), len(level) - 1)] for _ in range(wide))
        level = list(range(len(parents), len(parents) + wide))
        parents += chosen
    return tuple(parents)


def _parents(case):
    """Of every sequence, as lists."""
    new = _lengths(case["batch"], case["longest"], case["shortest"])
    if case["op"] == "keep" or case["tree"]:
        return [list(_tree(n, b % 5)) for b, n in enumerate(new)]
    return [list(range(-1, n - 1)) for n in new]


def _depths(parents):
    depth = []
    for p in parents:
        depth.append(0 if p < 0 else depth[p] + 1)
    return depth


def _path(parents, which):
    """An accepted path through a later branch of the tree: node 0, then nodes that lie behind the slots they move to."""
    rng, at = random.Random(which), 0
    path = [0]
    while True:
        children = [i for i, p in enumerate(parents) if p == at]
        children = [i for i in children if i > max(_depths(parents))] if at == 0 else children
        if not children:
            return path
        at = rng.choice(children)
        path.append(at)


# ----------------------------------------------------------------------------------------------------------------------
# inputs
def _table(style, width):
    """cos / sin of every position: [2][MP][width] with the frequencies twice, or [MP][width] sin | cos for adjacent pairs."""
    freq = 10000.0 ** (-torch.arange(0, width, 2, dtype=torch.float64, device="cuda") / width)
    angle = torch.arange(MAX_POSITIONS, dtype=torch.float64, device="cuda")[:, None] * freq
    if style == "gptj":
        return torch.cat((angle.sin(), angle.cos()), 1).float()
    return torch.stack((torch.cat((angle, angle), 1).cos(), torch.cat((angle, angle), 1).sin())).float()


def _rows(g, tokens, counts, head, strided):
    """q, k and v as projections leave them: channels of different size; strided: views of one matrix's rows."""
    def make(n):
        gain = torch.exp(0.5 * torch.randn(n * head, generator=g, device="cuda"))
        return (torch.randn((tokens, n * head), generator=g, device="cuda") * gain).to(BF16)

    if strided:
        whole = make(sum(counts)).view(tokens, sum(counts), head)
        return [whole[:, sum(counts[:i]):sum(counts[:i + 1])] for i in range(len(counts))]
    return [make(n).view(tokens, n, head) for n in counts]


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _page_table(g, lengths, page):
    """Pages of sequences that hold `lengths` slots, in the order that a pool gives them out after some use: none after the
    other.  Returns (table [B][most pages], pages of the pool)."""
    need = [-(-n // page) for n in lengths]
    pool = sum(need) + 3
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(need), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pool


def _filled(g, shape):
    """Keys (with channels of different size) and values of `shape`[2:] pages."""
    layer = torch.empty(shape, dtype=BF16, device="cuda")
    gain = torch.exp(0.5 * torch.randn((shape[-3], 1, shape[-1]), generator=g, device="cuda"))
    for i in range(0, shape[-4], 256):
        n = min(256, shape[-4] - i)
        layer[..., 0, i:i + n, :, :, :] = torch.randn(shape[:-5] + (n,) + shape[-3:], generator=g, device="cuda") * gain
        layer[..., 1, i:i + n, :, :, :] = torch.randn(shape[:-5] + (n,) + shape[-3:], generator=g, device="cuda")
    return layer


def _target_logits(g, rows, vocab):
    """Logits as a model gives them: a wide bulk and a few likely tokens."""
    x = 1.5 * torch.randn((rows, vocab), generator=g, device="cuda")
    some = torch.randint(0, vocab, (rows, 24), generator=g, device="cuda")
    return x.scatter_add_(1, some, 10.0 + 2.0 * torch.randn((rows, 24), generator=g, device="cuda"))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    parents = _parents(case)
    new = [len(p) for p in parents]
    starts = [sum(new[:b]) for b in range(len(new) + 1)]
    tokens = starts[-1]
    single = max(new) == 1
    state = {"op": case["op"], "new": new, "starts": starts, "cu": None if single else _i32(starts), "parents": None}
    if not single and case.get("tree"):
        state["parents"] = _i32([p for of in parents for p in of])
    if case["op"] == "verify":
        dtype = LOGITS[case["dtype"]]
        target = _target_logits(g, tokens, case["vocab"])
        guess = target + 1.2 * torch.randn(target.shape, generator=g, device="cuda")
        state["temperature"] = case["temperature"]
        state["target"], guess = target.to(dtype), guess.to(dtype)
        state["draft"] = guess if case["drafts"] else None
        state["uniforms"] = torch.rand(tokens, generator=g, device="cuda")
        state["sample"] = torch.rand(case["batch"], generator=g, device="cuda")
        if case["drafts"] and case["temperature"] > 0:  # drawn from the draft's probabilities
            noise = -torch.log(-torch.log(torch.rand(guess.shape, generator=g, device="cuda").clamp_(1e-20, 1 - 1e-7)))
            ranked = (guess.float() / case["temperature"] + noise).argmax(1, keepdim=True)
        else:
            ranked = guess.float().topk(min(64, case["vocab"]), 1).indices
        row, rank = [], []
        for b, of in enumerate(parents):
            seen = [0] * len(of)
            for p in of:
                row.append(starts[b] + max(p, 0))
                rank.append(seen[p] if p >= 0 else 0)
                if p >= 0:
                    seen[p] += 1
        at = torch.tensor(rank, device="cuda") % ranked.shape[1]
        state["tokens"] = ranked[torch.tensor(row, device="cuda"), at].contiguous()
        return state
    nq, nkv, head = HEADS[case["heads"]]
    past = _pasts(case)
    state["past_host"], state["past"], state["page"] = past, _i32(past), case["page"]
    held = [p + n for p, n in zip(past, new)]
    # room for the tokens of the next steps, as a program hands out pages
    state["table"], pool = _page_table(g, [n + 20 for n in held], case["page"])
    shape = (2, pool, nkv, case["page"], head)
    if case["op"] == "keep":
        state["cache"] = _filled(g, (case["layers"],) + shape)
        paths = [_path(p, seed + b) for b, p in enumerate(parents)]
        state["path"] = _i32([i for p, n in zip(paths, new) for i in p + [-1] * (n - len(p))])
        state["count"] = _i32([len(p) for p in paths])
        state["cu"] = _i32(starts)
        return state
    if case["op"] == "append":
        state["rows"] = _rows(g, tokens, [nq, nkv, nkv], head, case["strided"])
        for name in ("wq", "wk"):
            state[name] = 1.0 + 0.2 * torch.randn(head, generator=g, device="cuda") if case["norm"] else None
        state["style"] = case["style"]
        state["angles"] = _table(case["style"], head if case["style"] == "llama" else 64)
        state["layer"] = torch.zeros(shape, dtype=BF16, device="cuda")
        return state
    state["q"] = (torch.randn((tokens, nq, head), generator=g, device="cuda") * 1.5).to(BF16)
    state["layer"] = _filled(g, shape)
    return state


# ----------------------------------------------------------------------------------------------------------------------
# plain forms
def _sequence_of(state):
    """(sequence, index within it) of every node."""
    new = torch.tensor(state["new"], device="cuda")
    seq = torch.repeat_interleave(torch.arange(len(state["new"]), device="cuda"), new)
    return seq, torch.arange(state["starts"][-1], device="cuda") - torch.tensor(state["starts"][:-1], device="cuda")[seq]


def _seen_nodes(parents, n):
    """[n][n]: node j is node i or one that it continues."""
    if parents is None:
        return torch.ones((n, n), dtype=torch.bool, device="cuda").tril()
    seen = torch.eye(n, device="cuda")
    seen += (parents[:, None] == torch.arange(n, device="cuda")) & (parents[:, None] >= 0)
    for _ in range((n - 1).bit_length()):  # twice as many generations each time
        seen = ((seen @ seen) > 0).float()
    return seen > 0


def _normed(x, weight):
    if weight is None:
        return x
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight


def _rotated(x, table, pos, style):
    """x [T][heads][H] turned by the table's angles at `pos`; channels past the table's width stay."""
    width = table.shape[-1]
    turn, rest = x[..., :width], x[..., width:]
    if style == "gptj":
        sin, cos = table[pos][:, None].chunk(2, -1)
        a, b = turn[..., 0::2], turn[..., 1::2]
        turn = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        cos, sin = table[0][pos][:, None], table[1][pos][:, None]
        a, b = turn.chunk(2, -1)
        turn = turn * cos + torch.cat((-b, a), -1) * sin
    return torch.cat((turn, rest), -1)


def _plain_append(state):
    q, k, v = state["rows"]
    seq, index = _sequence_of(state)
    depth = index
    if state["parents"] is not None:
        depth = torch.cat([_seen_nodes(state["parents"][a:b], b - a).sum(1) - 1 for a, b in zip(state["starts"], state["starts"][1:])])
    pos, slot = state["past"][seq] + depth, state["past"][seq] + index
    q = _rotated(_normed(q.float(), state["wq"]), state["angles"], pos, state["style"]).to(BF16)
    k = _rotated(_normed(k.float(), state["wk"]), state["angles"], pos, state["style"]).to(BF16)
    page = state["table"][seq, slot // state["page"]].long()
    state["layer"][0, page, :, slot % state["page"]] = k
    state["layer"][1, page, :, slot % state["page"]] = v
    return [q, state["layer"]]


def _plain_attn(state):
    out = []
    for b, (n, past) in enumerate(zip(state["new"], state["past_host"])):
        rows = slice(state["starts"][b], state["starts"][b + 1])
        q = state["q"][rows].float()
        pages = state["table"][b, :-(-(past + n) // state["page"])].long()
        k, v = (x[pages].transpose(0, 1).flatten(1, 2)[:, :past + n].float() for x in state["layer"])
        _, nq, head = q.shape
        nkv = k.shape[0]
        grouped = q.view(n, nkv, nq // nkv, head).permute(1, 2, 0, 3).reshape(nkv, nq // nkv * n, head)
        scores = (grouped @ k.transpose(1, 2)).view(nkv, nq // nkv, n, past + n) / math.sqrt(head)
        seen = _seen_nodes(None if state["parents"] is None else state["parents"][rows], n)
        scores[..., past:] = scores[..., past:].masked_fill(~seen, -math.inf)
        e = torch.exp(scores - scores.amax(-1, keepdim=True))
        o = (e / e.sum(-1, keepdim=True)).view(nkv, nq // nkv * n, past + n) @ v
        out.append(o.view(nkv, nq // nkv, n, head).permute(2, 0, 1, 3).reshape(n, nq, head))
    return torch.cat(out).to(BF16)


def _probabilities(logits, temperature):
    """In 64 bits: which token a random number falls on is a step function of their sums."""
    x = logits.double()
    top = x.amax(-1, keepdim=True)
    if temperature == 0:
        first = x.argmax(-1, keepdim=True)
        return torch.zeros_like(x).scatter_(-1, first, 1.0)
    e = torch.exp((x - top) / temperature)
    return e / e.sum(-1, keepdim=True)


def _plain_verify(state):
    out = {"path": [], "count": [], "next": []}
    for b, n in enumerate(state["new"]):
        rows = slice(state["starts"][b], state["starts"][b + 1])
        p = _probabilities(state["target"][rows], state["temperature"])
        token, u = state["tokens"][rows], state["uniforms"][rows].double()
        index = torch.arange(n, device="cuda")
        parent = index - 1 if state["parents"] is None else state["parents"][rows].long()
        up = parent.clamp_min(0)
        px = p[up, token]
        sibling = (parent[:, None] == parent) & (index[:, None] > index)  # [later][earlier]
        again = (sibling & (token[:, None] == token)).any(1)
        px = torch.where(again, torch.zeros_like(px), px)
        if state["draft"] is None or state["temperature"] == 0:
            q = None
            left = 1.0 - (sibling * px).sum(1)
            fine = u * left < px
        else:
            q = _probabilities(state["draft"][rows], state["temperature"])
            fine = u * q[up, token] < px
        fine &= index > 0
        # the first child of a node that stands, or n
        stands = torch.where(fine & (parent == index[:, None]), index, n)  # [node][child]
        after = torch.cat((stands.amin(1), torch.tensor([n], device="cuda")))
        path, at = [], torch.zeros((), dtype=torch.int64, device="cuda")
        end = at
        for _ in range(n):
            path.append(at)
            end = torch.where(at < n, at, end)
            at = after[at]
        path = torch.stack(path)
        rest = p[end]
        children = (parent == end) & (index > 0)
        if q is None:
            gone = torch.zeros(p.shape[1] + 1, dtype=torch.bool, device="cuda").scatter_(0, torch.where(children, token, p.shape[1]), True)
            rest = rest.masked_fill(gone[:-1], 0.0)
        else:
            residual = (rest - q[end]).clamp_min(0.0)
            rest = torch.where(children.any() & (residual.sum() > 0), residual, rest)
        rest = torch.where(rest.sum() > 0, rest, p[end])
        sums = rest.cumsum(0)
        beyond = sums > state["sample"][b].double() * sums[-1]
        out["next"].append(beyond.to(torch.int8).argmax())
        out["path"].append(torch.where(path < n, path, -1))
        out["count"].append((path < n).sum())
    return [torch.cat(out["path"]).to(torch.int32), torch.stack(out["count"]).to(torch.int32), torch.stack(out["next"])]


def _plain_keep(state):
    page = state["page"]
    moves = []
    for b, n in enumerate(state["new"]):
        path = state["path"][state["starts"][b]:state["starts"][b + 1]].long()
        to = state["past"][b] + torch.arange(n, device="cuda")
        come = torch.where(torch.arange(n, device="cuda") < state["count"][b], state["past"][b] + path, to)
        moves.append([(state["table"][b, s // page].long(), s % page) for s in (come, to)])
    (fp, fs), (tp, ts) = ([torch.cat([m[i][j] for m in moves]) for j in range(2)] for i in range(2))
    held = state["cache"][:, :, fp, :, fs]
    state["cache"][:, :, tp, :, ts] = held
    return state["cache"]


PLAIN = {"append": _plain_append, "attn": _plain_attn, "verify": _plain_verify, "keep": _plain_keep}


# ----------------------------------------------------------------------------------------------------------------------
# the framework's calls
@functools.lru_cache(maxsize=None)
def _operators():
    where = os.path.join(os.getcwd(), "tpp-pytorch-extension_amd")
    if where not in sys.path:
        sys.path.insert(0, where)
    import tpp_pytorch_extension  # noqa: F401
    from tpp_pytorch_extension._C import _tpp_attn
    return _tpp_attn


def _own_run(state):
    at = _operators()
    if state["op"] == "append":
        q, k, v = state["rows"]
        q = at.append_paged(q, k, v, state["layer"], state["table"], state["past"], state["cu"], state["parents"], state["wq"], state["wk"],
                            EPS, state["angles"], None, state["style"])
        return [q, state["layer"]]
    if state["op"] == "attn":
        return at.attn_paged(state["q"], state["layer"], state["table"], state["past"], state["cu"], state["parents"])
    if state["op"] == "verify":
        return list(at.verify_drafts(state["tokens"], state["target"], state["cu"], state["parents"], state["draft"], state["uniforms"],
                                     state["sample"], state["temperature"]))
    at.keep_paged(state["cache"], state["table"], state["past"], state["path"], state["count"], state["cu"])
    return state["cache"]


def run(state):
    if own:
        return _own_run(state)
    return PLAIN[state["op"]](state)


# ----------------------------------------------------------------------------------------------------------------------
def work(case):
    parents = _parents(case)
    new = [len(p) for p in parents]
    tokens = sum(new)
    if case["op"] == "verify":
        logits = tokens * case["vocab"] * (2 if case["drafts"] and case["temperature"] > 0 else 1)
        return {"bytes": logits * (4.0 if case["dtype"] == "fp32" else 2.0) + 24.0 * tokens, "flops": 4.0 * logits}
    nq, nkv, head = HEADS[case["heads"]]
    past = _pasts(case)
    if case["op"] == "append":
        width = head if case["style"] == "llama" else 64
        return {"bytes": 4.0 * tokens * nq * head + 8.0 * tokens * nkv * head + 4.0 * tokens * width,
                "flops": 8.0 * tokens * (nq + nkv) * head}
    if case["op"] == "keep":
        moved = sum(max(_depths(p)) for p in parents)
        return {"bytes": 8.0 * case["layers"] * moved * nkv * head, "flops": 0.0}
    keys = sum(p + n for p, n in zip(past, new))
    pairs = sum(p * n + sum(_depths(of)) + n for p, n, of in zip(past, new, parents))
    return {"bytes": 4.0 * tokens * nq * head + 4.0 * keys * nkv * head + 4.0 * keys / case["page"], "flops": 4.0 * nq * head * pairs}


# ----------------------------------------------------------------------------------------------------------------------
# the definitions, in 64 bits
def _exact_turn(x, weight, table, pos, style):
    """One pair of channels after the other, by complex numbers."""
    x = x.double()
    if weight is not None:
        x = x / ((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + EPS) ** 0.5 * weight.double()
    width = table.shape[-1]
    half = width // 2
    where = table.double()[pos] if style == "gptj" else table.double()[:, pos]
    sin, cos = (where[:, :half], where[:, half:]) if style == "gptj" else (where[1, :, :half], where[0, :, :half])
    angle = torch.complex(cos, sin)[:, None]
    pairs = x[..., :width].unflatten(-1, (half, 2)) if style == "gptj" else x[..., :width].unflatten(-1, (2, half)).transpose(-1, -2)
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * angle)
    turned = turned if style == "gptj" else turned.transpose(-1, -2)
    return torch.cat((turned.flatten(-2), x[..., width:]), -1)


def _exact_append(state, parents):
    pos = [p + d for p, of in zip(state["past_host"], parents) for d in _depths(of)]
    q, k, v = state["rows"]
    pos = torch.tensor(pos, device="cuda")
    q, k = (_exact_turn(x, w, state["angles"], pos, state["style"]) for x, w in ((q, state["wq"]), (k, state["wk"])))
    layer = torch.zeros(state["layer"].shape, dtype=torch.float64, device="cuda")
    table = state["table"].tolist()
    for b, of in enumerate(parents):
        for i in range(len(of)):
            page, at = divmod(state["past_host"][b] + i, state["page"])
            for side, x in enumerate((k, v)):
                layer[side, table[b][page], :, at] = x[state["starts"][b] + i].double()
    return [q, layer]


def _exact_attn(state, parents):
    """One head after the other."""
    out = torch.empty(state["q"].shape, dtype=torch.float64, device="cuda")
    nq, head = state["q"].shape[1:]
    table = state["table"].tolist()
    for b, of in enumerate(parents):
        past, n, first = state["past_host"][b], len(of), state["starts"][b]
        unseen = torch.ones((n, past + n), dtype=torch.bool)
        unseen[:, :past] = False
        for i in range(n):
            j = i
            while j >= 0:
                unseen[i, past + j] = False
                j = of[j]
        unseen = unseen.cuda()
        used = table[b][:-(-(past + n) // state["page"])]
        whole = state["layer"][:, used].permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :past + n].double()
        for h in range(nq):
            k, v = whole[:, h * whole.shape[1] // nq]
            s = torch.mm(state["q"][first:first + n, h].double(), k.t()) * head ** -0.5
            s[unseen] = -math.inf
            out[first:first + n, h] = torch.mm(torch.softmax(s, 1), v)
    return out


def _exact_verify(state, parents):
    """Token by token, as the rule is told."""
    paths, counts, following = [], [], []
    tokens, uniforms, samples = state["tokens"].tolist(), state["uniforms"].tolist(), state["sample"].tolist()
    greedy = state["temperature"] == 0
    for b, of in enumerate(parents):
        first = state["starts"][b]

        def spread(logits, node):
            x = logits[first + node].double()
            if greedy:
                one = torch.zeros_like(x)
                one[int(x.argmax())] = 1.0
                return one
            return torch.softmax(x / state["temperature"], 0)

        at, path = 0, [0]
        while True:
            p, down = spread(state["target"], at), None
            rest, rejected = p.clone(), False
            for child in (i for i, up in enumerate(of) if up == at):
                token = tokens[first + child]
                if state["draft"] is not None and not greedy:
                    q = spread(state["draft"], at)
                    if uniforms[first + child] * float(q[token]) < float(p[token]):
                        down = child
                        break
                    rest = torch.relu(p - q)
                else:
                    if uniforms[first + child] * float(rest.sum()) < float(rest[token]):
                        down = child
                        break
                    rest[token] = 0.0
                rejected = True
            if down is None:
                break
            at = down
            path.append(at)
        total = float(rest.sum())
        if rejected and total <= 0:
            rest, total = p, float(p.sum())
        sums = torch.cumsum(rest, 0)
        following.append(int((sums > samples[b] * total).nonzero()[0]))
        paths += path + [-1] * (len(of) - len(path))
        counts.append(len(path))
    return [_i32(paths), _i32(counts), torch.tensor(following, device="cuda")]


def _exact_keep(state, parents):
    out = state["cache"].double()
    path, count, table = state["path"].tolist(), state["count"].tolist(), state["table"].tolist()
    for b in range(len(parents)):
        for i in range(count[b]):
            a, z = (divmod(state["past_host"][b] + j, state["page"]) for j in (path[state["starts"][b] + i], i))
            out[:, :, table[b][z[0]], :, z[1]] = state["cache"][:, :, table[b][a[0]], :, a[1]].double()
    return out


def exact(case, seed):
    state = prepare(case, seed)
    return {"append": _exact_append, "attn": _exact_attn, "verify": _exact_verify, "keep": _exact_keep}[case["op"]](state, _parents(case))
