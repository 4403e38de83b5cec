"""The paged cache's operators and the check of drafted tokens against 64-bit plain forms (paged_ref)."""
import math

import pytest
import torch

import mx4_ref as M
import paged_ref as R

pytestmark = pytest.mark.gpu


def _at():
    import tpp_pytorch_extension  # noqa: F401
    from tpp_pytorch_extension._C import _tpp_attn
    return _tpp_attn


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _starts(lengths):
    return [sum(lengths[:i]) for i in range(len(lengths) + 1)]


def _within(got, want, tol):
    bad = ~((got.double().cpu() - want).abs() <= tol)
    assert not bool(bad.any()), (f"{int(bad.sum())} of {bad.numel()} beyond their bound, worst "
                                 f"{float(((got.double().cpu() - want).abs() / tol).max()):.3g} times it, first {bad.nonzero()[:3].tolist()}")


def _up(t):
    return None if t is None else t.cuda()


# -- append -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("H,width,style,norm", [(64, 64, "llama", True), (96, 96, "llama", False), (128, 128, "llama", True), (128, 64, "llama", False),
                                                (192, 48, "llama", True), (256, 64, "gptj", True), (96, 96, "gptj", False), (128, 0, None, True)])
@pytest.mark.parametrize("new,past,page,trees", [([1, 1, 1], [0, 15, 30], 16, False), ([5, 0, 17, 1], [3, 9, 0, 20], 16, True),
                                                 ([5, 0, 17, 1], [3, 9, -1, 31], 32, False)])
def test_append(H, width, style, norm, new, past, page, trees):
    at = _at()
    B, Nq, Nkv = len(new), 6, 3
    cu = _starts(new)
    ragged = max(new) > 1
    T = cu[-1] + (2 if ragged else 0)  # two rows behind the last sequence
    parents = [R.tree(n, n) for n in new] if trees else [list(range(-1, n - 1)) for n in new]
    q, k, v = (M.randn((T, Nq + 2 * Nkv + 1, H), 1.5, 10 + H)[:, a:z].cuda() for a, z in ((0, Nq), (Nq, Nq + Nkv), (Nq + Nkv, Nq + 2 * Nkv)))
    wq, wk = (M.randn(H, 1.0, 3).float(), M.randn(H, 1.0, 4).float()) if norm else (None, None)
    table = None if style is None else M.llama_table(40, width) if style == "llama" else M.gptj_table(40, width)
    pages, pool = R.table_for([max(p, 0) + n for p, n in zip(past, new)], page)
    pages[0, -1] = -1 if new[0] == 5 and pages.shape[1] > 1 else pages[0, -1]
    layer = torch.full((2, pool, Nkv, page, H), 7.0, dtype=torch.bfloat16, device="cuda")
    flat = [x for p in parents for x in p] + [0] * (T - cu[-1])
    out = at.append_paged(q, k, v, layer, pages.cuda(), _i32(past), _i32(cu) if ragged else None, _i32(flat) if trees else None, _up(wq), _up(wk),
                          1e-5, _up(table), None, style)
    pos = [p + d for p, of in zip(past, parents) for d in R.depths(of)]
    n = cu[-1]
    want, size = M.turn(q.cpu()[:n], wq, 1e-5, table, pos, style)
    # one bf16 rounding; fp32 inside: 12 sums, a root, a quotient, two products and the rotation, 16 roundings in all
    _within(out[:n], want, 2.0 ** -8 * want.abs() + 2.0 ** -20 * size + 2.0 ** -133)
    kw, ks = M.turn(k.cpu()[:n], wk, 1e-5, table, pos, style)
    left = torch.ones(layer.shape, dtype=torch.bool)
    held = layer.cpu()
    for b in range(B):
        for i in range(new[b]):
            s = past[b] + i
            if past[b] < 0 or s // page >= pages.shape[1] or int(pages[b, s // page]) < 0:
                continue
            row = (int(pages[b, s // page]), slice(None), s % page)
            _within(held[0][row], kw[cu[b] + i], 2.0 ** -8 * kw[cu[b] + i].abs() + 2.0 ** -20 * ks[cu[b] + i] + 2.0 ** -133)
            assert torch.equal(held[1][row], v.cpu()[cu[b] + i])
            left[0][row] = left[1][row] = False
    assert bool((held[left] == 7.0).all())
    # given positions, bf16 norm weights, no queries: the same keys
    again = torch.full_like(layer, 7.0)
    given = torch.tensor(pos + [0] * (T - n), device="cuda")
    assert at.append_paged(None, k, v, again, pages.cuda(), _i32(past), _i32(cu) if ragged else None, None, None,
                           None if wk is None else wk.to(torch.bfloat16).cuda(), 1e-5, _up(table), given, style) is None
    assert torch.equal(again, layer)


def test_append_of_bad_tables_and_pasts():
    """Entries that are no pages, slots past the table and past near the ends of int32 lead nowhere."""
    at = _at()
    k, v = M.randn((6, 2, 64), 1.0, 1).cuda(), M.randn((6, 2, 64), 1.0, 2).cuda()
    layer = torch.zeros((2, 3, 2, 16, 64), dtype=torch.bfloat16, device="cuda")
    table = _i32([[0, 1], [99, -5], [2 ** 31 - 1, -2 ** 31], [1, 2], [0, 2], [0, 1]])
    at.append_paged(None, k, v, layer, table, _i32([32, 3, 17, 2 ** 31 - 1, -2 ** 31, -1]))
    assert not bool(layer.any())
    at.append_paged(None, k, v, layer, table, _i32([31, 32, 3, 2 ** 30, -7, -1]))
    assert torch.equal(layer[1, 1, :, 15], v[0])
    layer[:, 1, :, 15] = 0
    assert not bool(layer.any())


# -- attention --------------------------------------------------------------------------------------------------------
def _layer(pool, Nkv, page, H, seed):
    return M.randn((2, pool, Nkv, page, H), 1.0, seed)


def _check_attention(new, past, page, Nq, Nkv, H, parents, seed=0, spare_rows=0):
    """parents: of every sequence, or None: chains without parents."""
    at = _at()
    cu = _starts(new)
    single = max(new) == 1 and not spare_rows
    T = cu[-1] + spare_rows
    pages, pool = R.table_for([max(p, 0) + n for p, n in zip(past, new)], page, seed=seed)
    layer = _layer(pool, Nkv, page, H, 100 + seed)
    q = M.randn((T, Nq + 1, H), 1.5, 200 + seed)[:, :Nq]
    flat = None if parents is None else _i32([x for p in parents for x in p] + [-1] * spare_rows)
    out = at.attn_paged(q.cuda(), layer.cuda(), pages.cuda(), _i32(past), None if single else _i32(cu), flat)
    for b, n in enumerate(new):
        if n == 0:
            continue
        rows = slice(cu[b], cu[b + 1])
        if past[b] < 0:
            assert not bool(out[rows].any())
            continue
        k, v = R.slots(layer, pages, b, past[b] + n)
        seen = torch.ones((n, past[b] + n), dtype=torch.bool)
        seen[:, past[b]:] = R.ancestors(parents[b] if parents is not None else list(range(-1, n - 1)))
        _within(out[rows], *R.attend(q[rows], k, v, seen))
    return out


@pytest.mark.parametrize("H,Nq,Nkv", [(64, 12, 4), (96, 10, 2), (128, 8, 8), (128, 16, 2), (192, 3, 1), (256, 4, 2), (128, 20, 1), (64, 17, 1)])
@pytest.mark.parametrize("page", [16, 64])
def test_attention_of_single_tokens(H, Nq, Nkv, page):
    _check_attention([1] * 9, [0, 1, 15, 16, 31, 33, 127, 130, 700], page, Nq, Nkv, H, None, seed=H + page)


@pytest.mark.parametrize("H,Nq,Nkv", [(64, 12, 4), (96, 10, 2), (128, 8, 8), (128, 16, 2), (192, 3, 1), (256, 4, 2)])
@pytest.mark.parametrize("page", [16, 32, 256])
@pytest.mark.parametrize("form", ["", "1", "2", "3", "4", "5", "6"])
def test_attention_of_trees(H, Nq, Nkv, page, form, monkeypatch):
    if form:  # (one of the kernel's forms instead of the one that the sizes give)
        monkeypatch.setenv("TPPX_PAGED_FORM", form)
    new, past = [9, 1, 0, 30, 70, 17], [40, 0, 3, 129, 63, 300]
    _check_attention(new, past, page, Nq, Nkv, H, [R.tree(n, n + page) if n else [] for n in new], seed=H + page, spare_rows=3)


@pytest.mark.parametrize("H,Nq,Nkv", [(64, 12, 4), (96, 10, 2), (128, 8, 8), (128, 16, 2), (192, 3, 1), (256, 4, 2)])
@pytest.mark.parametrize("new,past", [([70, 1, 200], [0, 500, 33]), ([130], [1000]), ([3, 2, 2], [15, -1, 0])])
@pytest.mark.parametrize("chunk", ["", "64"])
def test_attention_of_pieces_of_prompts(H, Nq, Nkv, new, past, chunk, monkeypatch):
    if chunk:  # (parts of 64 keys)
        monkeypatch.setenv("TPPX_PAGED_LEAST", chunk)
    _check_attention(new, past, 32, Nq, Nkv, H, None, seed=H + len(new), spare_rows=2)


@pytest.mark.parametrize("B", [65, 150, 400])
@pytest.mark.parametrize("form", ["", "1", "2", "3", "4", "5", "6"])
@pytest.mark.parametrize("kind", ["single", "chains", "trees"])
def test_attention_of_many_sequences(B, form, kind, monkeypatch):
    """More sequences than a wave has lanes, some long enough to be split, some empty, some that take no part."""
    if form:
        monkeypatch.setenv("TPPX_PAGED_FORM", form)
    monkeypatch.setenv("TPPX_PAGED_LEAST", "64")
    monkeypatch.setenv("TPPX_PAGED_ITEMS", "6000")
    new = [1] * B if kind == "single" else [(0, 3, 1, 8, 21)[i * 7 % 5] for i in range(B)]
    past = [(0, 5, 130, -1, 33)[i * 3 % 5] for i in range(B)]
    past[1], past[63], past[64], past[B - 1] = 900, 2100, 1200, 700
    trees = [R.tree(n, i) if n else [] for i, n in enumerate(new)] if kind == "trees" else None
    _check_attention(new, past, 16, 4, 2, 64, trees, seed=B)


@pytest.mark.parametrize("form", ["1", "2", "3", "4", "5", "6"])
@pytest.mark.parametrize("items", ["4", "10", "24", "100"])
@pytest.mark.parametrize("kind", ["one", "fresh", "trees", "single"])
def test_attention_in_rounds(form, items, kind, monkeypatch):
    """Launches with more blocks than run at once, `items` of them here: whole rounds, and parts of what is left."""
    monkeypatch.setenv("TPPX_PAGED_FORM", form)
    monkeypatch.setenv("TPPX_PAGED_ITEMS", items)
    monkeypatch.setenv("TPPX_PAGED_LEAST", "64")
    new, past = {"one": ([150], [1000]), "fresh": ([600, 90, 0, 33], [0, 0, 0, 500]), "trees": ([70, 3, 64, 30], [900, 1500, 0, 333]),
                 "single": ([1] * 12, [0, 2000, 30, 700, -1, 64, 1500, 1200, 5, 5, 800, 100])}[kind]
    _check_attention(new, past, 16, 8, 2, 128, [R.tree(n, n) if n else [] for n in new] if kind == "trees" else None, seed=len(items))


def test_attention_of_a_deep_tree_and_of_one_that_is_a_chain():
    n = 300
    _check_attention([n], [20], 16, 4, 2, 128, [R.tree(n, 5, deep=0.97)])
    chain = _check_attention([n], [20], 16, 4, 2, 128, [list(range(-1, n - 1))])
    assert torch.equal(chain, _check_attention([n], [20], 16, 4, 2, 128, None))


def test_attention_of_bad_parents():
    """What is no earlier node is none: such a node sees the slots before the step's and its own."""
    at = _at()
    H, page, past = 64, 16, 20
    layer = _layer(4, 1, page, H, 3).cuda()
    table = _i32([[2, 0, 1]])
    q = M.randn((5, 2, H), 1.0, 4).cuda()
    got = at.attn_paged(q, layer, table, _i32([past]), _i32([0, 5]), _i32([7, 1, -9, 2 ** 31 - 1, 3]))
    want = at.attn_paged(q, layer, table, _i32([past]), _i32([0, 5]), _i32([-1, -1, -1, -1, 3]))
    assert torch.equal(got, want)


def test_attention_past_the_table():
    """More keys than the table has slots for: those it has."""
    at = _at()
    H, page = 128, 16
    layer = _layer(3, 2, page, H, 5)
    table = torch.tensor([[2, 0], [1, 0], [0, 1]], dtype=torch.int32)
    q = M.randn((3, 4, H), 1.0, 6)
    out = at.attn_paged(q.cuda(), layer.cuda(), table.cuda(), _i32([40, 2 ** 31 - 1, 31]))
    for b in range(3):
        k, v = R.slots(layer, table, b, 32)
        _within(out[b:b + 1], *R.attend(q[b:b + 1], k, v, torch.ones((1, 32), dtype=torch.bool)))


@pytest.mark.parametrize("H,Nq,Nkv", [(64, 4, 2), (96, 4, 2), (128, 16, 2), (256, 4, 2)])
@pytest.mark.parametrize("new", [4, 40])
@pytest.mark.parametrize("form", ["1", "2", "3", "4", "5", "6"])
def test_what_a_node_does_not_see_may_be_anything(H, Nq, Nkv, new, form, monkeypatch):
    """Infinities and NaN in the keys and values of nodes that another does not continue, and behind the last one, stay there."""
    at = _at()
    monkeypatch.setenv("TPPX_PAGED_FORM", form)
    page, past = 16, 37
    parents = [-1, 0, 0, 1] + [R.tree(new, 9)[i] for i in range(4, new)]
    parents = [p if p != 2 else 0 for p in parents]  # nobody continues node 2
    table, pool = R.table_for([past + new + 20], page)
    layer = _layer(pool, Nkv, page, H, 7)
    q = M.randn((new, Nq, H), 1.0, 8)
    clean = at.attn_paged(q.cuda(), layer.cuda(), table.cuda(), _i32([past]), _i32([0, new]), _i32(parents))

    def put(slot, head, channel, key, value):
        page_id = int(table[0, slot // page])
        layer[0, page_id, head, slot % page, channel] = key
        layer[1, page_id, head, slot % page, channel] = value

    put(past + 2, 0, 3, math.nan, math.inf)
    put(past + 2, Nkv - 1, H - 1, math.inf, math.nan)
    for s in range(past + new, past + new + 20):
        put(s, 0, 0, math.nan, math.nan)
        put(s, 1, 5, -math.inf, math.inf)
    out = at.attn_paged(q.cuda(), layer.cuda(), table.cuda(), _i32([past]), _i32([0, new]), _i32(parents))
    others = [i for i in range(new) if i != 2]
    assert torch.equal(out[others], clean[others])
    assert bool(torch.isnan(out[2, 0]).all())  # (a key that is NaN)
    for h in range(Nq - Nq // Nkv, Nq):  # (an infinite one: a score of infinity, or of -infinity, whose value counts for nothing but is NaN)
        got = torch.isnan(out[2, h])
        assert bool(got.all()) if float(q[2, h, H - 1]) > 0 else bool(got[H - 1]) and not bool(got[:H - 1].any())
    # values alone: they reach the node itself, in their channel
    layer[0] = _layer(pool, Nkv, page, H, 7)[0]
    layer[1, int(table[0, (past + 2) // page]), Nkv - 1, (past + 2) % page, H - 1] = -math.inf
    out = at.attn_paged(q.cuda(), layer.cuda(), table.cuda(), _i32([past]), _i32([0, new]), _i32(parents))
    assert torch.equal(out[others], clean[others])
    assert float(out[2, 0, 3]) == math.inf and float(out[2, -1, H - 1]) == -math.inf
    same = torch.ones((Nq, H), dtype=torch.bool)
    same[:Nq // Nkv, 3] = same[-(Nq // Nkv):, H - 1] = False
    assert torch.equal(out[2].cpu()[same], clean[2].cpu()[same])
    # a value in front of the step reaches every node
    layer[1, int(table[0, 0]), 1, 5, 9] = math.nan
    out = at.attn_paged(q.cuda(), layer.cuda(), table.cuda(), _i32([past]), _i32([0, new]), _i32(parents))
    assert bool(torch.isnan(out[:, Nq // Nkv:2 * (Nq // Nkv), 9]).all())
    assert not bool(torch.isnan(out[others][:, :, 10]).any())


def test_attention_beyond_4_gib():
    """Pages whose offsets in the layer pass 2^32 bytes, and 2^32 elements for the values."""
    at = _at()
    H, Nkv, page, past = 128, 8, 256, 300
    pool = 17000  # 8.9 GB a side
    layer = torch.zeros((2, pool, Nkv, page, H), dtype=torch.bfloat16, device="cuda")
    small = _layer(4, Nkv, page, H, 11)
    ids = [16999, 8193, 4097, 3]
    layer[:, ids] = small.cuda()
    q = M.randn((3, 16, H), 1.0, 12).cuda()
    k, v = M.randn((3, Nkv, H), 1.0, 13).cuda(), M.randn((3, Nkv, H), 1.0, 14).cuda()
    high, low = _i32([ids[:2], ids[1:3], ids[2:]]), _i32([[0, 1], [1, 2], [2, 3]])
    small = small.cuda()
    p = _i32([past, past + 100, past + 150])
    for table, where in ((high, layer), (low, small)):
        at.append_paged(None, k, v, where, table, p)
    assert torch.equal(layer[:, ids], small)
    assert torch.equal(at.attn_paged(q, layer, high, p), at.attn_paged(q, small, low, p))
    path, count = _i32([0, 2, 3, -1] * 3), _i32([3, 3, 3])
    for table, where in ((high, layer), (low, small)):
        at.keep_paged(where, table, p, path, count, _i32([0, 4, 8, 12]))
    assert torch.equal(layer[:, ids], small)


# -- verification -----------------------------------------------------------------------------------------------------
def _verify_case(new, V, dtype, seed, trees, drafts, temps):
    """Logits with likely tokens, candidates among them; returns the arguments on the CPU."""
    g = torch.Generator().manual_seed(seed)
    T = sum(new)
    target = torch.randn((T, V), generator=g) * 2
    target.scatter_add_(1, torch.randint(0, V, (T, 4), generator=g), torch.full((T, 4), 5.0))
    draft = target + torch.randn((T, V), generator=g) * 0.7
    target, draft = target.to(dtype), draft.to(dtype)
    parents, tokens, at = [], [], 0
    for b, n in enumerate(new):
        of = R.tree(n, seed + b) if trees and n else list(range(-1, n - 1))
        rank = {}
        for i, p in enumerate(of):
            if p < 0:
                tokens.append(0)
                continue
            t = temps[b] if temps[b] > 0 else 1.0
            if drafts:
                tokens.append(int(torch.multinomial(torch.softmax(draft[at + p].float() / t, 0), 1, generator=g)))
            else:
                r = rank[p] = rank.get(p, -1) + 1
                tokens.append(int(draft[at + p].float().topk(min(V, r + 1)).indices[-1]))
        parents.append(of)
        at += n
    return tokens, parents, target, draft if drafts else None, torch.rand(T, generator=g), torch.rand(len(new), generator=g)


def _check_verify(new, V, dtype, seed, trees=False, drafts=False, temps=None, as_tensor=False, given=None):
    at = _at()
    temps = [1.0] * len(new) if temps is None else temps
    tokens, parents, target, draft, uniforms, sample = given or _verify_case(new, V, dtype, seed, trees, drafts, temps)
    cu = _starts(new)
    single = max(new) == 1
    path, count, following = at.verify_drafts(
        torch.tensor(tokens, device="cuda"), target.cuda(), None if single else _i32(cu), _i32([p for of in parents for p in of]) if trees else None,
        _up(draft), uniforms.cuda(), sample.cuda(), torch.tensor(temps, device="cuda") if as_tensor else temps[0])
    stood = 0
    for b, n in enumerate(new):
        rows = slice(cu[b], cu[b + 1])
        if n == 0:
            assert int(count[b]) == 0 and int(following[b]) == 0
            continue
        near = []
        want, then = R.verify(tokens[rows], parents[b] if trees else None, target[rows], None if draft is None else draft[rows],
                              uniforms[rows], sample[b], temps[b], near)
        assert not near or min(near) > 1e-10, "a draw next to a border: another seed"
        assert path[rows].tolist() == want + [-1] * (n - len(want)), b
        assert int(count[b]) == len(want) and int(following[b]) == then, b
        stood += len(want) - 1
    return stood


@pytest.mark.parametrize("V,dtype", [(1, torch.float32), (7, torch.bfloat16), (1000, torch.float16), (4099, torch.bfloat16), (32000, torch.bfloat16),
                                     (50401, torch.float32), (9000, torch.float32), (128000, torch.float16)])
@pytest.mark.parametrize("kind", ["single", "chain", "drawn", "tree", "small tree"])
def test_verify(V, dtype, kind):
    new = {"single": [1, 1, 1, 1], "chain": [5, 0, 1, 9], "drawn": [6, 1, 0, 3, 8], "tree": [20, 1, 0, 66, 7], "small tree": [0, 12, 1, 9, 8]}[kind]
    args = dict(trees="tree" in kind, drafts=kind == "drawn")
    _check_verify(new, V, dtype, V + len(new), temps=[0.8] * len(new), **args)
    _check_verify(new, V, dtype, V + 1, temps=[0.0, 1.0, 0.7, 1.3, 0.05][:len(new)], as_tensor=True, **args)
    _check_verify(new, V, dtype, V + 2, temps=[0.0] * len(new), **args)


def test_verify_of_bounds_that_do_not_ascend():
    """Sequences that share rows, end before they begin or lie outside: every call ends, and the ones after it are right."""
    at = _at()
    V = 4099
    tokens, parents, target, _, u, s = _verify_case([12, 8], V, torch.bfloat16, 3, True, False, [1.0, 1.0])
    args = [torch.tensor(tokens, device="cuda"), target.cuda(), _i32([0, 12, 20]), _i32([p for of in parents for p in of]), None, u.cuda(), s.cuda()]
    want = at.verify_drafts(*args)
    for cu in ([0, 20, 0], [20, 5, 12], [-7, 30, 9], [12, 0, 20], [0, 2 ** 31 - 1, -2 ** 31], [9, 9, 9], [0, 0, 20], [3, 15, 18]):
        path, count, following = at.verify_drafts(args[0], args[1], _i32(cu), *args[3:])
        assert 0 <= int(count.min()) and int(count.max()) <= 20 and 0 <= int(following.min()) and int(following.max()) < V
        for got, w in zip(at.verify_drafts(*args), want):
            assert torch.equal(got, w)


def test_verify_long_chain_and_wide_tree():
    _check_verify([300], 700, torch.bfloat16, 3, drafts=True)
    tokens, parents, target, _, u, s = _verify_case([200], 500, torch.float32, 4, True, False, [1.0])
    parents = [[-1] + [0] * 199]
    tokens = [0] + [int(x) for x in torch.randperm(500, generator=torch.Generator().manual_seed(1))[:199]]
    _check_verify([200], 500, torch.float32, 4, trees=True, given=(tokens, parents, target, None, u * 0 + 0.999, s))
    # more children than the kernel keeps in LDS, none of which stands; then a tree of as many nodes
    g = torch.Generator().manual_seed(8)
    target = torch.randn((400, 3000), generator=g)
    tokens = [0] + [int(x) for x in torch.randperm(3000, generator=g)[:399]]
    for s in (0.0, 0.4, 0.9999):
        _check_verify([400], 3000, torch.float32, 4, trees=True,
                      given=(tokens, [[-1] + [0] * 399], target, None, torch.full((400,), 0.999), torch.tensor([s])))
    _check_verify([400, 3, 270], 900, torch.bfloat16, 9, trees=True)


def test_verify_of_infinities_and_nan():
    g = torch.Generator().manual_seed(5)
    V = 600
    target = torch.randn((12, V), generator=g)
    draft = target + torch.randn((12, V), generator=g)
    target[0, 5:] = -math.inf
    target[1, 100] = math.nan
    target[2, [40, 300, 599]] = math.inf
    target[3] = -math.inf
    target[4] = math.nan
    draft[5, 10:] = -math.inf
    draft[6] = -math.inf
    draft[7, 3] = math.inf
    target[8, 0], target[9, V - 1] = math.nan, math.inf
    tokens = [0, 2, 100, 300, 17, 0, 5, 11, 3, 0, 599, 1]
    for temp in (1.0, 0.0):
        for with_draft in (True, False):
            for new in ([12], [1] * 12, [3, 4, 5]):
                chains = [list(range(-1, n - 1)) for n in new]
                s = torch.rand(len(new), generator=g)
                _check_verify(new, V, torch.float32, 0, drafts=with_draft, temps=[temp] * len(new),
                              given=(tokens, chains, target, draft if with_draft else None, torch.rand(12, generator=g), s))


def test_verify_at_its_borders():
    """Tokens outside of the vocabulary, the same candidate twice, numbers of zero and next to one, a draft that equals the target."""
    g = torch.Generator().manual_seed(6)
    V = 40
    target = torch.randn((6, V), generator=g)
    below = 1.0 - 2.0 ** -24
    star = [[-1, 0, 0, 0, 0, 0]]
    for tokens in ([0, -1, V, 2 ** 40, 3, 4], [0, 7, 7, 7, 8, 8]):
        for u in (0.0, 0.5, below):
            for s in (0.0, 0.3, below):
                _check_verify([6], V, torch.float32, 0, trees=True, given=(tokens, star, target, None, torch.full((6,), u), torch.tensor([s])))
    chain = [list(range(-1, 5))]
    tokens = [0, 1, 2, 3, 4, 5]
    assert _check_verify([6], V, torch.float32, 0, drafts=True, given=(tokens, chain, target, target.clone(), torch.full((6,), below), torch.tensor([0.5]))) == 5
    # candidates that are the whole vocabulary: one of them stands
    wide = torch.randn((41, V), generator=g)
    assert _check_verify([41], V, torch.float32, 0, trees=True,
                         given=([0] + list(range(V)), [[-1] + [0] * V], wide, None, torch.full((41,), 0.5), torch.tensor([0.5]))) == 1


@pytest.mark.parametrize("kind", ["drawn", "tree"])
def test_verified_tokens_are_distributed_as_the_target(kind):
    """The token behind node 0, drafted or not, over many sequences with numbers of their own."""
    at = _at()
    B, V = 200000, 8
    g = torch.Generator(device="cuda").manual_seed(7)
    p, q = torch.randn(V, generator=g, device="cuda"), torch.randn(V, generator=g, device="cuda")
    n = 2 if kind == "drawn" else 3
    target = p.expand(n * B, V).contiguous()
    if kind == "drawn":
        draft = q.expand(n * B, V).contiguous()
        drawn = torch.multinomial(torch.softmax(q, 0), B, replacement=True, generator=g)
        tokens, parents = torch.stack((drawn * 0, drawn), 1).view(-1), None
    else:
        draft, tokens = None, torch.tensor([0, 2, 5], device="cuda").repeat(B)
        parents = _i32([-1, 0, 0]).repeat(B)
    cu = torch.arange(0, n * B + 1, n, dtype=torch.int32, device="cuda")
    path, count, following = at.verify_drafts(tokens, target, cu, parents, draft, torch.rand(n * B, generator=g, device="cuda"),
                                              torch.rand(B, generator=g, device="cuda"))
    second = path.view(B, n)[:, 1].long().clamp_min(0)
    out = torch.where(count > 1, tokens.view(B, n).gather(1, second[:, None])[:, 0], following)
    share = torch.softmax(p.double(), 0)
    seen = torch.bincount(out, minlength=V).double()
    # six standard deviations of a count; 8 counts, so by chance once in 10^7 runs of numbers that differ
    assert bool(((seen - B * share).abs() < 6 * (B * share * (1 - share)).sqrt()).all()), (seen / B, share)


# -- keeping an accepted path -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("H,Nkv,page,layers", [(64, 4, 16, 3), (96, 1, 32, 2), (128, 8, 64, 5), (192, 2, 16, 1), (256, 3, 256, 2)])
def test_keep(H, Nkv, page, layers):
    at = _at()
    new, past = [9, 0, 40, 1, 12, 6], [14, 3, 60, 0, -1, 31]
    paths = [[0, 1, 4, 8], [], [0, 7, 8, 9, 20, 21, 22, 23, 24, 30, 39], [0], [0, 3], [0, 1, 2, 3, 4, 5]]
    cu = _starts(new)
    table, pool = R.table_for([max(p, 0) + n for p, n in zip(past, new)], page)
    cache = torch.stack([_layer(pool, Nkv, page, H, 20 + i) for i in range(layers)])
    path = [x for p, n in zip(paths, new) for x in p + [-1] * (n - len(p))]
    got = cache.cuda()
    at.keep_paged(got, table.cuda(), _i32(past), _i32(path), _i32([len(p) for p in paths]), _i32(cu))
    want = cache.clone()
    for b, p in enumerate(paths):
        if past[b] < 0:
            continue
        for i, node in enumerate(p):
            a, z = (divmod(past[b] + s, page) for s in (node, i))
            want[:, :, int(table[b, z[0]]), :, z[1]] = cache[:, :, int(table[b, a[0]]), :, a[1]]
    assert torch.equal(got.cpu(), want)
    one = cache[0].cuda()
    at.keep_paged(one, table.cuda(), _i32(past), _i32(path), _i32([len(p) for p in paths]), _i32(cu))
    assert torch.equal(one.cpu(), want[0])


def test_keep_of_bad_paths():
    """Numbers that are no nodes, counts beyond them, slots without a page: nothing outside of the sequence's pages changes."""
    at = _at()
    cache = _layer(4, 2, 16, 64, 30).cuda()
    table = _i32([[0, -1], [1, 77]])
    before = cache.clone()
    at.keep_paged(cache, table, _i32([14, 10]), _i32([5, 2 ** 31 - 1, -2 ** 31, 3, 9, -1]), _i32([100, 3]), _i32([0, 3, 6]))
    assert torch.equal(cache[:, 2:], before[:, 2:])
    at.keep_paged(cache, table, _i32([2 ** 31 - 1, -2 ** 31]), _i32([0, 2, 1, 0, 2, 1]), _i32([3, 3]), _i32([0, 3, 6]))
    assert torch.equal(cache[:, 2:], before[:, 2:])
    now = cache.clone()
    for cu in ([6, 3, 0], [2 ** 31 - 1, -2 ** 31, 3], [-2 ** 31, -1, -2 ** 31], [7, 2 ** 31 - 1, 7]):
        at.keep_paged(cache, table, _i32([2, 2]), _i32([0, 2, 3, 0, 2, 3]), _i32([3, 3]), _i32(cu))
    assert torch.equal(cache[:, 2:], now[:, 2:])


# -- together ---------------------------------------------------------------------------------------------------------
def _step(at, x, layers, table, past, cu, parents, head, emb, out=None):
    """A step of a small stack without MLPs: q, k, v are slices of the hidden state; then logits, check and keep."""
    h = x
    for layer in layers:
        q, k, v = h[:, :4], h[:, 4:6], h[:, 6:8]
        q = at.append_paged(q, k, v, layer, table, past, cu, parents, None, None, 1e-6, emb)
        o = at.attn_paged(q, layer, table, past, cu, parents)
        h = torch.cat((o, h[:, 4:]), 1) * 0.5 + x * 0.5
    return (h.flatten(1).float() @ head).to(torch.bfloat16)


def test_steps_in_a_replayed_graph():
    """append, attention, check and keep of a step, captured once and replayed on other nodes, lengths and tables, against eager calls."""
    at = _at()
    B, n, H, page, layers, V = 3, 7, 64, 16, 3, 300
    T = B * n
    cu = torch.arange(0, T + 1, n, dtype=torch.int32, device="cuda")
    emb = M.llama_table(200, H).cuda()
    head = (M.randn((8 * H, V), 0.3, 40)).float().cuda()
    table, pool = R.table_for([120] * B, page)
    start = torch.stack([_layer(pool, 2, page, H, 50 + i) for i in range(layers)]).cuda()

    def inputs(i):
        g = torch.Generator(device="cuda").manual_seed(60 + i)
        parents = _i32([p for b in range(B) for p in R.tree(n, 10 * i + b)])
        return {"x": M.randn((T, 8, H), 1.0, 70 + i).cuda(), "past": _i32([5 * i, 40 - i, 70]), "parents": parents, "table": table.roll(i, 1).cuda().contiguous(),
                "tokens": torch.randint(0, V, (T,), generator=g, device="cuda"), "u": torch.rand(T, generator=g, device="cuda"),
                "s": torch.rand(B, generator=g, device="cuda")}

    def step(cache, a):
        logits = _step(at, a["x"], list(cache), a["table"], a["past"], cu, a["parents"], head, emb)
        path, count, following = at.verify_drafts(a["tokens"], logits, cu, a["parents"], None, a["u"], a["s"], 0.9)
        at.keep_paged(cache, a["table"], a["past"], path, count, cu)
        return logits, path, count, following

    cache, fixed = start.clone(), inputs(0)
    step(cache, fixed)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(cache, fixed)
    for i in (1, 2, 3, 1):
        a = inputs(i)
        for name, t in a.items():
            fixed[name].copy_(t)
        cache.copy_(start)
        graph.replay()
        again = start.clone()
        want = step(again, a)  # (eager work between the replays)
        torch.cuda.synchronize()
        for got, w in zip(outs, want):
            assert torch.equal(got, w)
        assert torch.equal(cache, again)


def test_drawn_chains_in_a_replayed_graph():
    at = _at()
    new, V = [6, 1, 0, 3, 8], 30000

    def inputs(i):
        tokens, _, target, draft, u, s = _verify_case(new, V, torch.bfloat16, 80 + i, False, True, [1.0] * 5)
        return [t.cuda() for t in (torch.tensor(tokens), target, draft, u, s, torch.tensor([1.0, 0.7, 1.0, 0.0, 1.2]))]

    def check(a):
        return at.verify_drafts(a[0], a[1], cu, None, a[2], a[3], a[4], a[5])

    cu, fixed = _i32(_starts(new)), inputs(0)
    check(fixed)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = check(fixed)
    for i in (1, 2, 3, 1, 4):
        a = inputs(i)
        for to, t in zip(fixed, a):
            to.copy_(t)
        graph.replay()
        want = check(a)
        torch.cuda.synchronize()
        assert all(torch.equal(got, w) for got, w in zip(outs, want))


def test_two_graphs_replayed_at_once():
    """Steps of drafted tokens keep what they leave for their later launches apart: replays of two graphs need no order."""
    at = _at()
    jobs, want, graphs, outs = [], [], [], []
    for i in range(2):
        new, past = [20, 9], [2000 + 300 * i, 900]
        table, pool = R.table_for([p + n for p, n in zip(past, new)], 32, seed=i)
        parents = _i32([x for n in new for x in R.tree(n, n + i)])
        tokens, _, target, _, u, s = _verify_case(new, 4000, torch.bfloat16, i, True, False, [1.0, 1.0])
        jobs.append([t.cuda() for t in (M.randn((29, 16, 128), 1.0, i), _layer(pool, 2, 32, 128, 90 + i), table, _i32(past), _i32([0, 20, 29]), parents,
                                        torch.tensor(tokens), target, u, s)])

    def work(j):
        q, layer, table, past, cu, parents, tokens, target, u, s = j
        return (at.attn_paged(q, layer, table, past, cu, parents), *at.verify_drafts(tokens, target, cu, parents, None, u, s))

    for j in jobs:
        want.append(work(j))
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(work(j))
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, z) for a, z in zip(outs[i], want[i]))
            for t in outs[i]:
                t.zero_()
        torch.cuda.synchronize()


def test_two_streams_at_once():
    at = _at()
    H, page = 128, 32
    jobs = []
    for i in range(2):
        new, past = [20, 9], [700 + i, 300]
        table, pool = R.table_for([p + n for p, n in zip(past, new)], page, seed=i)
        parents = _i32([x for n in new for x in R.tree(n, n + i)])
        tokens, _, target, _, u, s = _verify_case(new, 4000, torch.bfloat16, i, True, False, [1.0, 1.0])
        jobs.append((M.randn((29, 16, H), 1.0, i).cuda(), _layer(pool, 2, page, H, 90 + i).cuda(), table.cuda(), _i32(past), _i32([0, 20, 29]), parents,
                     torch.tensor(tokens, device="cuda"), target.cuda(), u.cuda(), s.cuda()))

    def work(j):
        q, layer, table, past, cu, parents, tokens, target, u, s = j
        return (at.attn_paged(q, layer, table, past, cu, parents), *at.verify_drafts(tokens, target, cu, parents, None, u, s))

    want = [work(j) for j in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, j in enumerate(jobs):
            with torch.cuda.stream(streams[i]):
                got[i].append(work(j))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, z) for a, z in zip(r, want[i]))
