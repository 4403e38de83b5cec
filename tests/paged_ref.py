"""64-bit plain forms of the paged cache's operators and of the check of drafted tokens, for the tests (CPU)."""
import math
import random

import torch

F64 = torch.float64


def tree(nodes, seed, deep=0.3):
    """Parents of a random tree: node 0 the root, every other continues an earlier one; deep: how often the one right before."""
    rng = random.Random(seed)
    return ([-1] + [i - 1 if rng.random() < deep else rng.randrange(i) for i in range(1, nodes)])[:nodes]


def ancestors(parents):
    """[n][n]: node j is node i or one that it continues."""
    n = len(parents)
    seen = torch.zeros((n, n), dtype=torch.bool)
    for i in range(n):
        j = i
        while j >= 0:
            seen[i, j] = True
            j = parents[j] if parents[j] < j else -1
    return seen


def depths(parents):
    return [int(s) - 1 for s in ancestors(parents).sum(1)] if parents else []


def table_for(lengths, page, spare=2, seed=0):
    """(table [B][most pages] with -1 behind the pages of a sequence, pages of the pool), pages in no order."""
    need = [max(1, -(-n // page)) for n in lengths]
    order = list(range(sum(need) + spare))
    random.Random(seed).shuffle(order)
    table = torch.full((len(need), max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    return table, len(order)


def slots(layer, table, b, n):
    """Keys and values [2][Nkv][n][H] of a sequence's first n slots."""
    page = layer.shape[3]
    pages = table[b, :-(-n // page)].long()
    return layer[:, pages].permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :n]


def attend(q, k, v, seen):
    """q [n][Nq][H], k, v [Nkv][keys][H], seen [n][keys].  Returns the output and the largest error that the kernel's roundings may
    make of it: the probabilities in bf16 (half a step each, and their sum), scores and sums in fp32, the output rounded to bf16."""
    n, nq, H = q.shape
    nkv, keys = k.shape[:2]
    out, tol = torch.zeros((n, nq, H), dtype=F64), torch.zeros((n, nq, H), dtype=F64)
    some = seen.any(1)
    for h in range(nq):
        qq, kk, vv = q[:, h].to(F64), k[h * nkv // nq].to(F64), v[h * nkv // nq].to(F64)
        used = seen.any(0)
        kk, vv, sn = kk[used], vv[used], seen[:, used]
        s = (qq @ kk.t() / math.sqrt(H)).masked_fill(~sn, -math.inf)
        p = torch.softmax(s[some], 1)
        out[some, h] = p @ vv
        # fp32 scores: H products and sums
        es = (H + 4) * 2.0 ** -24 * (qq.abs() @ kk.abs().t()).amax(1, keepdim=True)[some] / math.sqrt(H)
        es = es + 2.0 ** -23 * s[some].masked_fill(~sn[some], 0.0).abs().amax(1, keepdim=True)
        rel = 2.0 * 2.0 ** -8 + 2 * es + 2.0 ** -12 + keys * 2.0 ** -23
        tol[some, h] = 2.0 ** -8 * out[some, h].abs() + rel * (p @ vv.abs()) * 1.01
    return out, tol + 2.0 ** -126


def shares(logits, temperature):
    """Probabilities of a row [V]."""
    x = torch.nan_to_num(logits.to(F64), nan=-math.inf, posinf=math.inf, neginf=-math.inf)
    top = x.max()
    if not temperature > 0 or math.isinf(temperature):
        p = torch.zeros_like(x)
        p[int((x == top).nonzero()[0])] = 1.0
        return p
    w = torch.where(x == top, torch.ones_like(x), torch.exp((x - top) / temperature))
    return w / w.sum()


def verify(tokens, parents, target, draft, uniforms, sample, temperature, near=None):
    """One sequence: (path, next token).  tokens: list, target [n][V].  near: a list that gets how close every decision was."""
    n, V = target.shape
    near = [] if near is None else near
    greedy = not temperature > 0 or math.isinf(temperature)
    at, path = 0, [0]
    while True:
        p, down = shares(target[at], temperature), None
        rest, tried = p.clone(), False
        for c in range(at + 1, n):
            if (parents[c] if parents is not None else c - 1) != at:
                continue
            x = tokens[c]
            u = 0.0 if greedy else float(uniforms[c])
            if draft is not None and not greedy:
                q = shares(draft[at], temperature)
                a, z = u * float(q[x]) if 0 <= x < V else 0.0, float(p[x]) if 0 <= x < V else 0.0
                left = torch.relu(p - q)
            else:
                a, z = u * float(rest.sum()), float(rest[x]) if 0 <= x < V else 0.0
                left = rest.clone()
                if 0 <= x < V:
                    left[x] = 0.0
            if not greedy and z > 0:
                near.append(abs(a - z) / z)
            if a < z:
                down = c
                break
            rest, tried = left, True
        if down is None:
            break
        at = down
        path.append(at)
    if tried and not float(rest.sum()) > 0:
        rest = p
    sums = torch.cumsum(rest, 0)
    border = 0.0 if greedy else float(sample) * float(sums[-1])
    if not greedy:
        near.append(float((sums - border).abs().min()) / float(sums[-1]))
    return path, int((sums > border).nonzero()[0])
