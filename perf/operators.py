"""Operators of the MXFP4 key/value cache and of packed prompts, as a serving program calls them: per-head norms of queries
and keys with the position rotation, the append of keys and values to a cache held in 4 bits, attention of single tokens and
of several new tokens over that cache, and causal attention of prompts of different lengths laid one after the other.

A cache layer is four byte tensors: the codes of the keys [B][Nkv][capacity][H/2] (two E2M1 codes a byte, the even channel in
the low half), their scales [B][Nkv][capacity][H/32] (one E8M0 byte for 32 channels), and the same of the values.  `past[b]` is
the number of keys that sequence b held before its new tokens; packed tokens of sequence b are rows cu[b] .. cu[b + 1] - 1.
"""
import functools
import math
import os
import sys

import torch

own = False

BF16 = torch.bfloat16
MAX_POSITIONS = 32768
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)

# query heads, key heads, head size
HEADS = {
    "llama-7b": (32, 32, 128),
    "llama-70b": (64, 8, 128),
    "qwen2-7b": (28, 4, 128),
    "gptj-6b": (16, 16, 256),
    "small": (12, 4, 64),
    "odd": (10, 2, 96),
}


def listed():
    return [
        # one token of one sequence between the projections and the attention of a decode step: latency alone
        {"name": "norm+rotary 1 token", "op": "rotary", "heads": "qwen2-7b", "batch": 1, "longest": 1, "shortest": 1, "past": 700,
         "norm": True, "style": "llama", "strided": False},
        # a long prompt, q and k as views of one fused projection's rows
        {"name": "norm+rotary 2048 tokens", "op": "rotary", "heads": "llama-70b", "batch": 1, "longest": 2048, "shortest": 2048,
         "past": 0, "norm": True, "style": "llama", "strided": True},
        # the new token of 16 sequences of different lengths goes to the cache
        {"name": "append 16 x 1 token", "op": "append", "heads": "llama-70b", "batch": 16, "longest": 1, "shortest": 1, "past": 2500,
         "norm": True, "style": "llama", "strided": True},
        # packed prompts of 5 requests go to the cache, no norm
        {"name": "append 5 prompts", "op": "append", "heads": "llama-7b", "batch": 5, "longest": 1000, "shortest": 77, "past": 0,
         "norm": False, "style": "llama", "strided": False},
        # one sequence decoding, the smallest step of a model with a head per key head
        {"name": "decode 1 x 2048", "op": "decode", "heads": "llama-7b", "batch": 1, "longest": 2048, "shortest": 2048, "mask": False},
        # a serving batch of uneven lengths, grouped heads
        {"name": "decode 16 uneven", "op": "decode", "heads": "llama-70b", "batch": 16, "longest": 4000, "shortest": 90, "mask": False},
        # the largest step: long contexts, where the cache is all that counts
        {"name": "decode 32 x 16000", "op": "decode", "heads": "llama-70b", "batch": 32, "longest": 16000, "shortest": 16000, "mask": False},
        # 256-wide heads, a batch padded on the left
        {"name": "decode 4 x 700 masked", "op": "decode", "heads": "gptj-6b", "batch": 4, "longest": 700, "shortest": 700, "mask": True},
        # a few new tokens each (a drafted continuation to be checked) on filled caches
        {"name": "extend 6 x 5..9 tokens", "op": "extend", "heads": "qwen2-7b", "batch": 6, "longest": 9, "shortest": 5, "past": 1500,
         "mask": False},
        # the next piece of a long prompt that is read piece by piece
        {"name": "extend 512 behind 6000", "op": "extend", "heads": "llama-70b", "batch": 1, "longest": 512, "shortest": 512,
         "past": 6000, "mask": False},
        # many short prompts
        {"name": "packed 16 short", "op": "packed", "heads": "qwen2-7b", "batch": 16, "longest": 200, "shortest": 17, "strided": True},
        # long prompts beside short ones
        {"name": "packed 4 up to 4100", "op": "packed", "heads": "llama-7b", "batch": 4, "longest": 4100, "shortest": 60, "strided": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "decode", "decode", "extend", "packed"])
    case = {"op": op, "heads": rng.choice(list(HEADS))}
    if op in ("rotary", "append"):
        case["batch"] = _log_int(rng, 1, 24)
        case["longest"] = rng.choice([1, _log_int(rng, 1, max(2, 2048 // case["batch"]))])
        case["shortest"] = rng.randint(1, case["longest"])
        case["past"] = rng.choice([0, rng.randint(1, 4000)])
        case["norm"], case["strided"] = rng.random() < 0.7, rng.random() < 0.5
        case["style"] = rng.choice(["llama", "llama", "gptj"])
        return case
    if op == "decode":
        case["batch"] = _log_int(rng, 1, 48)
        case["longest"] = _log_int(rng, 1, min(16000, 200000 // case["batch"]))
        case["shortest"] = rng.randint(1, case["longest"])
        case["mask"] = rng.random() < 0.3
        return case
    if op == "extend":
        case["batch"] = _log_int(rng, 1, 8)
        case["longest"] = _log_int(rng, 2, 512 // case["batch"])
        case["shortest"] = rng.randint(1, case["longest"])
        case["past"] = _log_int(rng, 1, 6000 // case["batch"])
        case["mask"] = rng.random() < 0.3
        return case
    case["batch"] = _log_int(rng, 1, 24)
    case["longest"] = _log_int(rng, 1, 4000 // math.isqrt(case["batch"]) // (2 if case["heads"] in ("llama-70b", "gptj-6b") else 1))
    case["shortest"] = rng.randint(1, case["longest"])
    case["strided"] = rng.random() < 0.5
    return case


def _lengths(batch, longest, shortest):
    """`batch` lengths from `longest` to `shortest`, in no order of size but the first."""
    step = [(7 * b) % batch for b in range(batch)] if batch % 7 else list(range(batch))
    return [round(longest * (shortest / longest) ** (s / max(1, batch - 1))) for s in step]


def _new_tokens(case):
    return _lengths(case["batch"], case["longest"], case["shortest"])


def _pasts(case):
    """Keys that the sequences hold already: different ones where they hold any."""
    if case["op"] == "decode":
        return [n - 1 for n in _new_tokens(case)]
    past = case.get("past", 0)
    return _lengths(case["batch"], past, max(1, past // 3)) if past else [0] * case["batch"]


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
    """q (, k, v) as projections leave them: channels of different size; strided: views of one matrix's rows."""
    def make(n):
        gain = torch.exp(0.5 * torch.randn(n * head, generator=g, device="cuda"))
        return (torch.randn((tokens, n * head), generator=g, device="cuda") * gain).to(BF16)

    if strided:
        whole = make(sum(counts)).view(tokens, sum(counts), head)
        return [whole[:, sum(counts[:i]):sum(counts[:i + 1])] for i in range(len(counts))]
    return [make(n).view(tokens, n, head) for n in counts]


def _codes_of(x):
    """E2M1 codes and E8M0 scales of x over blocks of 32 of the last dimension: 2^(floor(log2 max) - 2), nearest, ties to
    the even code, 6 at most.  Returns (code of every value, scale byte of every block, the values they stand for)."""
    blocks = x.unflatten(-1, (-1, 32))
    top = blocks.abs().amax(-1, keepdim=True)
    byte = (torch.frexp(top).exponent - 1 - 2 + 127).clamp_(0, 254)
    byte = torch.where(top < 2.0 ** -126, torch.zeros_like(byte), byte)
    scale = torch.ldexp(torch.ones_like(top), byte - 127)
    scale = torch.where(byte == 0, torch.zeros_like(scale), scale)
    a = torch.where(scale > 0, blocks.abs() / scale, torch.zeros_like(blocks))
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    value = torch.tensor(E2M1, dtype=x.dtype, device=x.device)[code.long()] * scale
    minus = (blocks < 0) & (code > 0)
    value = torch.where(minus, -value, value)
    return (code + 8 * minus.to(torch.uint8)).flatten(-2), byte.squeeze(-1).to(torch.uint8), value.flatten(-2)


def _packed_codes(code):
    return code[..., 0::2] | code[..., 1::2] << 4


def _values_of(codes, scales):
    """float32 values that codes [..][H/2] and scales [..][H/32] stand for."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float32, device=codes.device)
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    scale = torch.ldexp(torch.ones_like(scales, dtype=torch.float32), scales.int() - 127)
    return (table[code.int()].unflatten(-1, (-1, 32)) * scale[..., None]).flatten(-2)


def _filled(g, batch, nkv, capacity, head):
    """A layer whose every slot holds a key and a value."""
    gain = torch.exp(0.5 * torch.randn((nkv, 1, head), generator=g, device="cuda"))
    layer = []
    for _ in range(2):
        code, scale, _ = _codes_of(torch.randn((batch, nkv, capacity, head), generator=g, device="cuda") * gain)
        layer += [_packed_codes(code), scale]
        gain = 1.0
    return tuple(layer)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    nq, nkv, head = HEADS[case["heads"]]
    new, past = _new_tokens(case), _pasts(case)
    if case["op"] == "decode":
        new = [1] * case["batch"]
    starts = [sum(new[:b]) for b in range(len(new) + 1)]
    state = {"op": case["op"], "new": new, "past_host": past, "past": _i32(past), "starts": starts, "mask": None,
             "cu": None if max(new) == 1 and case["op"] != "packed" else _i32(starts)}
    tokens = starts[-1]
    if case["op"] in ("rotary", "append"):
        counts = [nq, nkv, nkv] if case["op"] == "append" else [nq, nkv]
        state["rows"] = _rows(g, tokens, counts, head, case["strided"])
        for name in ("wq", "wk"):
            state[name] = 1.0 + 0.2 * torch.randn(head, generator=g, device="cuda") if case["norm"] else None
        state["style"] = case["style"]
        state["table"] = _table(case["style"], head if case["style"] == "llama" else 64)
        state["pos"] = torch.tensor([p + i for p, n in zip(past, new) for i in range(n)], dtype=torch.int64, device="cuda")
        if case["op"] == "append":
            # room for the tokens still to come, as a generation loop allocates it
            capacity = max(p + n for p, n in zip(past, new)) + 128
            shape = (case["batch"], nkv, capacity)
            state["layer"] = tuple(torch.zeros(shape + (w,), dtype=torch.uint8, device="cuda")
                                   for w in (head // 2, head // 32, head // 2, head // 32))
        return state
    if case["op"] == "packed":
        state["q"], state["k"], state["v"] = _rows(g, tokens, [nq, nkv, nkv], head, case["strided"])
        return state
    longest = max(p + n for p, n in zip(past, new))
    state["q"] = (torch.randn((tokens, nq, head), generator=g, device="cuda") * 1.5).to(BF16)
    state["layer"] = _filled(g, case["batch"], nkv, longest + 64, head)
    if case["mask"]:  # padding on the left, more for the shorter ones
        state["mask"] = torch.zeros((case["batch"], (longest + 31) // 32 * 32), dtype=BF16, device="cuda")
        for b in range(case["batch"]):
            state["mask"][b, :(past[b] + 1) * b // (2 * case["batch"])] = torch.finfo(BF16).min
    return state


# ----------------------------------------------------------------------------------------------------------------------
# plain forms
def _normed(x, weight, eps):
    if weight is None:
        return x
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight.to(x.dtype)


def _rotated(x, table, pos, style):
    """x [T][heads][H] turned by the table's angles at `pos`; channels past the table's width stay."""
    width = table.shape[-1]
    turn, rest = x[..., :width], x[..., width:]
    if style == "gptj":
        sin, cos = table[pos].to(x.dtype)[:, None].chunk(2, -1)
        a, b = turn[..., 0::2], turn[..., 1::2]
        turn = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        cos, sin = table[0][pos].to(x.dtype)[:, None], table[1][pos].to(x.dtype)[:, None]
        a, b = turn.chunk(2, -1)
        turn = turn * cos + torch.cat((-b, a), -1) * sin
    return torch.cat((turn, rest), -1)


EPS = 1e-6


def _plain_rotary(state):
    return [_rotated(_normed(x.float(), w, EPS), state["table"], state["pos"], state["style"]).to(BF16)
            for x, w in zip(state["rows"], (state["wq"], state["wk"]))]


def _plain_append(state):
    q, k, v = state["rows"]
    q = _rotated(_normed(q.float(), state["wq"], EPS), state["table"], state["pos"], state["style"]).to(BF16)
    # a code is a step function of its value: 64 bits, so that no value next to a border falls on its other side
    k = _rotated(_normed(k.double(), state["wk"], EPS), state["table"], state["pos"], state["style"])
    seq = torch.repeat_interleave(torch.arange(len(state["new"]), device="cuda"), torch.tensor(state["new"], device="cuda"))
    first = torch.tensor(state["starts"][:-1], device="cuda")[seq]
    slot = state["past"][seq] + torch.arange(state["starts"][-1], device="cuda") - first
    held = []
    for i, x in ((0, k), (2, v.float())):
        code, scale, value = _codes_of(x)
        state["layer"][i][seq, :, slot] = _packed_codes(code)
        state["layer"][i + 1][seq, :, slot] = scale
        held.append(value.to(BF16))
    return [q, held, list(state["layer"])]


def _weights(scores):
    """Softmax over the last dimension; zeros where nothing is to be seen."""
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    return e / e.sum(-1, keepdim=True).clamp_min(torch.finfo(e.dtype).tiny)


def _attend(q, k, v, past, mask=None):
    """q [n][Nq][H] behind `past` keys, k, v [Nkv][past + n][H], float32; query i sees the keys up to past + i."""
    n, nq, head = q.shape
    nkv, keys = k.shape[:2]
    grouped = q.view(n, nkv, nq // nkv, head).permute(1, 2, 0, 3).reshape(nkv, nq // nkv * n, head)
    scores = (grouped @ k.transpose(1, 2)).view(nkv, nq // nkv, n, keys) / math.sqrt(head)
    if mask is not None:
        scores = scores + mask
    if n > 1:
        at = torch.arange(keys, device=q.device)
        scores = scores.masked_fill(at > past + torch.arange(n, device=q.device)[:, None], -math.inf)
    out = _weights(scores).view(nkv, nq // nkv * n, keys) @ v
    return out.view(nkv, nq // nkv, n, head).permute(2, 0, 1, 3).reshape(n, nq, head)


def _plain_decode(state):
    kc, ks, vc, vs = state["layer"]
    batch, nkv = kc.shape[:2]
    longest = max(state["past_host"]) + 1
    q = state["q"].float().unflatten(1, (nkv, -1))
    k = _values_of(kc[:, :, :longest], ks[:, :, :longest])
    scores = q @ k.transpose(2, 3) / math.sqrt(q.shape[-1])
    if state["mask"] is not None:
        scores = scores + state["mask"][:, None, None, :longest].float()
    at = torch.arange(longest, device="cuda")
    scores = scores.masked_fill(at > state["past"][:, None, None, None], -math.inf)
    return (_weights(scores) @ _values_of(vc[:, :, :longest], vs[:, :, :longest])).flatten(1, 2).to(BF16)


def _plain_extend(state):
    kc, ks, vc, vs = state["layer"]
    out = []
    for b, (n, past) in enumerate(zip(state["new"], state["past_host"])):
        rows, keys = slice(state["starts"][b], state["starts"][b + 1]), slice(0, past + n)
        mask = None if state["mask"] is None else state["mask"][b, :past + n].float()
        out.append(_attend(state["q"][rows].float(), _values_of(kc[b][:, keys], ks[b][:, keys]),
                           _values_of(vc[b][:, keys], vs[b][:, keys]), past, mask))
    return torch.cat(out).to(BF16)


def _plain_packed(state):
    out = []
    for b in range(len(state["new"])):
        q, k, v = (state[x][state["starts"][b]:state["starts"][b + 1]].float() for x in ("q", "k", "v"))
        out.append(_attend(q, k.transpose(0, 1), v.transpose(0, 1), 0))
    return torch.cat(out).to(BF16)


PLAIN = {"rotary": _plain_rotary, "append": _plain_append, "decode": _plain_decode, "extend": _plain_extend,
         "packed": _plain_packed}


# ----------------------------------------------------------------------------------------------------------------------
# the framework's calls
@functools.lru_cache(maxsize=None)
def _attention():
    where = os.path.join(os.getcwd(), "tpp-pytorch-extension_amd")
    if where not in sys.path:
        sys.path.insert(0, where)
    import tpp_pytorch_extension  # noqa: F401
    from tpp_pytorch_extension._C import _tpp_attn
    return _tpp_attn


def _own_run(state):
    at = _attention()
    op = state["op"]
    if op == "rotary":
        q, k = state["rows"]
        return list(at.qk_norm_rotary(q, k, state["wq"], state["wk"], EPS, state["table"], state["pos"], state["style"]))
    if op == "append":
        q, k, v = state["rows"]
        q, k, v = at.append_mx4(q, k, v, state["layer"], state["past"], state["cu"], state["wq"], state["wk"], EPS,
                                state["table"], state["pos"], state["style"], values=True)
        return [q, [k, v], list(state["layer"])]
    if op == "packed":
        return at.attn_packed(state["q"], state["k"], state["v"], state["cu"])
    return at.attn_mx4(state["q"], state["layer"], state["past"], state["cu"], state["mask"])


def run(state):
    if own:
        return _own_run(state)
    return PLAIN[state["op"]](state)


# ----------------------------------------------------------------------------------------------------------------------
def _seen(case):
    """(tokens, pairs of a token and a key that it sees, keys read)"""
    new, past = _new_tokens(case), _pasts(case)
    if case["op"] == "decode":
        new = [1] * case["batch"]
    return sum(new), sum(n * p + n * (n + 1) // 2 for n, p in zip(new, past)), sum(n + p for n, p in zip(new, past))


def work(case):
    nq, nkv, head = HEADS[case["heads"]]
    tokens, pairs, keys = _seen(case)
    four = 0.5 + 1 / 32
    if case["op"] in ("rotary", "append"):
        width = head if case["style"] == "llama" else 64
        rows = tokens * (nq + nkv) * head
        table = 8.0 * max(n + p for n, p in zip(_new_tokens(case), _pasts(case))) * width if tokens > case["batch"] else 8.0 * tokens * width
        if case["op"] == "rotary":
            return {"bytes": 4.0 * rows + min(table, 8.0 * tokens * width), "flops": 8.0 * rows}
        kv = tokens * nkv * head
        # q in and out, k and v in, their codes and the values that these stand for out
        return {"bytes": 4.0 * tokens * nq * head + 4.0 * kv + 2 * four * kv + 4.0 * kv + min(table, 8.0 * tokens * width),
                "flops": 8.0 * rows + 4.0 * kv}
    flops = 4.0 * nq * head * pairs
    if case["op"] == "packed":
        return {"bytes": 4.0 * tokens * (nq + nkv) * head, "flops": flops}
    return {"bytes": 4.0 * tokens * nq * head + 2 * four * keys * nkv * head, "flops": flops}


# ----------------------------------------------------------------------------------------------------------------------
# the definition, in 64 bits
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


def _exact_held(x):
    """The values of the grid {0, .5, 1, 1.5, 2, 3, 4, 6} times 2^(floor(log2 max) - 2) nearest to x, by distance."""
    blocks = x.unflatten(-1, (-1, 32))
    top = blocks.abs().amax(-1, keepdim=True)
    unit = torch.where(top >= 2.0 ** -126, 2.0 ** (torch.floor(torch.log2(top.clamp_min(1e-300))) - 2), torch.zeros_like(top))
    # log2 rounds just below a power of two up to it
    unit = torch.where(unit * 4 > top, unit / 2, unit)
    best, dist = torch.zeros_like(blocks), blocks.abs()
    for i, v in enumerate(E2M1[1:], 1):
        d = (blocks.abs() - v * unit).abs()
        nearer = (d < dist) | ((d == dist) & (i % 2 == 0) & (unit > 0))
        best, dist = torch.where(nearer, v * unit, best), torch.where(nearer, d, dist)
    return (best * blocks.sign()).flatten(-2)


def _exact_values(codes, scales):
    low, high = (codes % 16).double(), (codes // 16).double()
    code = torch.stack((low, high), -1).flatten(-2)
    size = code % 8
    # E2M1: two bits of exponent, one of mantissa
    exponent, mantissa = torch.floor(size / 2), size % 2
    value = torch.where(exponent > 0, 2.0 ** (exponent - 1) * (1 + mantissa / 2), mantissa / 2)
    return (torch.where(code >= 8, -value, value).unflatten(-1, (-1, 32)) * (2.0 ** (scales.double() - 127))[..., None]).flatten(-2)


def _exact_rows(q, k, v, past, mask):
    """One key head after the other: q [n][Nq][H], k, v [Nkv][keys][H]."""
    n, nq, head = q.shape
    nkv, keys = k.shape[:2]
    out = torch.empty((n, nq, head), dtype=torch.float64, device=q.device)
    hidden = torch.ones((n, keys), dtype=torch.bool, device=q.device).triu(past + 1)
    for h in range(nq):
        s = torch.mm(q[:, h].double(), k[h * nkv // nq].double().t()) * head ** -0.5
        if mask is not None:
            s += mask.double()
        s[hidden] = -math.inf
        out[:, h] = torch.mm(torch.softmax(s, 1), v[h * nkv // nq].double())
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] in ("rotary", "append"):
        turned = [_exact_turn(x, w, state["table"], state["pos"], state["style"]) for x, w in zip(state["rows"], (state["wq"], state["wk"]))]
        if case["op"] == "rotary":
            return turned
        return [turned[0], [_exact_held(turned[1]), _exact_held(state["rows"][2].double())], [None] * 4]
    out = []
    for b, (n, past) in enumerate(zip(state["new"], state["past_host"])):
        rows = slice(state["starts"][b], state["starts"][b + 1])
        if case["op"] == "packed":
            k, v = (state[x][rows].transpose(0, 1) for x in ("k", "v"))
        else:
            kc, ks, vc, vs = (x[b, :, :past + n] for x in state["layer"])
            k, v = _exact_values(kc, ks), _exact_values(vc, vs)
        out.append(_exact_rows(state["q"][rows], k, v, past, None if state["mask"] is None else state["mask"][b, :past + n]))
    return torch.cat(out)
