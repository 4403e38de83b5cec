"""The MXFP4 key/value cache and packed prompts: per-head norms with the rotation, the append, attention of single, several
and many tokens over the cache, causal attention of packed prompts, against 64-bit plain forms (mx4_ref)."""
import math

import pytest
import torch

import mx4_ref as R

pytestmark = pytest.mark.gpu


def _at():
    import tpp_pytorch_extension  # noqa: F401
    from tpp_pytorch_extension._C import _tpp_attn
    return _tpp_attn


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _starts(lengths):
    return [sum(lengths[:i]) for i in range(len(lengths) + 1)]


def _table(style, positions, H, width):
    return None if style is None else R.llama_table(positions, width) if style == "llama" else R.gptj_table(positions, width)


def _within(got, want, tol):
    bad = ~((got.double().cpu() - want).abs() <= tol)
    assert not bool(bad.any()), (f"{int(bad.sum())} of {bad.numel()} beyond their bound, worst "
                                 f"{float(((got.double().cpu() - want).abs() / tol).max()):.3g} times it, first {bad.nonzero()[:3].tolist()}")


def _prompt_form(queries, monkeypatch):
    """Empty: the form that the sizes give; "64", "128": the prompt kernels in the form of small or of large launches."""
    if queries:
        monkeypatch.setenv("TPPX_MX4_PROMPT_QUERIES", queries)


# -- norm and rotation ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("H,width,style", [(64, 64, "llama"), (96, 96, "llama"), (128, 128, "llama"), (128, 64, "llama"), (192, 48, "llama"),
                                           (256, 256, "llama"), (256, 64, "gptj"), (96, 96, "gptj"), (128, 128, None)])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("T,Nq,Nkv,strided", [(1, 4, 4, False), (5, 7, 1, True)])
def test_norm_and_rotation(H, width, style, norm, T, Nq, Nkv, strided):
    at = _at()
    whole = R.randn((T, Nq + Nkv + 1, H), 2.0, H + T).cuda()
    q, k = whole[:, :Nq], whole[:, Nq:Nq + Nkv]
    if not strided:
        q, k = q.contiguous(), k.contiguous()
    wq, wk = (R.randn(H, 1.0, 3), R.randn(H, 1.0, 4)) if norm else (None, None)
    table = _table(style, 50, H, width)
    pos = torch.tensor([(13 * t + 49) % 53 for t in range(T)])  # some past the table
    up = lambda t: None if t is None else t.cuda()  # noqa: E731
    qo, ko = at.qk_norm_rotary(q, k, up(wq), up(wk), 1e-5, up(table), pos.cuda(), style or "llama")
    qo2, _ = at.qk_norm_rotary(q, k, None if wq is None else wq.float().cuda(), None if wk is None else wk.float().cuda(), 1e-5, up(table), pos.cuda(), style)
    assert torch.equal(qo, qo2)
    for x, w, got in ((q, wq, qo), (k, wk, ko)):
        want, size = R.turn(x.cpu(), w, 1e-5, table, pos, style)
        # one bf16 rounding; fp32 inside: 12 sums, a root, a quotient, two products and the rotation, 16 roundings in all
        _within(got, want, 2.0 ** -8 * want.abs() + 2.0 ** -20 * size + 2.0 ** -133)


# -- append -----------------------------------------------------------------------------------------------------------
def _empty_layer(B, Nkv, cap, H, fill=0):
    at = _at()
    return at.Mx4Layer(*(torch.full((B, Nkv, cap, w), fill, dtype=torch.uint8, device="cuda") for w in (H // 2, H // 32, H // 2, H // 32)))


@pytest.mark.parametrize("H,style,norm", [(64, "llama", True), (96, "llama", False), (128, "llama", True), (192, None, True), (256, "gptj", False)])
@pytest.mark.parametrize("new,past", [([1, 1, 1], [0, 4, 30]), ([5, 0, 17, 1], [3, 9, 0, 20])])
def test_append(H, style, norm, new, past):
    at = _at()
    B, Nq, Nkv, cap = len(new), 6, 3, 31
    cu = _starts(new)
    T = cu[-1] + 2  # two rows behind the last sequence
    if max(new) == 1:
        T = cu[-1]
    q, k, v = (R.randn((T, n, H), 1.5, 10 + H + n).cuda() for n in (Nq, Nkv, Nkv))
    k[0, 0, :32] = 0.0  # a block of zeros
    k[-1, 1, 0] = 2.0 ** -130
    v[0, 0, :32] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0] * 4)  # ties
    v[0, 1, :32] = torch.tensor([-0.25, -0.1, 0.0, -0.75, -2.5, -3.5, -5.0, -7.9] * 4)
    v[0, 2, :32] = 2.0 ** -126
    wq, wk = (R.randn(H, 1.0, 3).float().cuda(), R.randn(H, 1.0, 4).float().cuda()) if norm else (None, None)
    table = _table(style, 64, H, 64)
    layer = _empty_layer(B, Nkv, cap, H, 0xAB)
    pos = [p + i for n, p in zip(new, past) for i in range(n)]
    ragged = max(new) > 1
    qo, ko, vo = at.append_mx4(q, k, v, layer, _i32(past), _i32(cu) if ragged else None, wq, wk, 1e-5,
                               None if table is None else table.cuda(), None, style, values=True)
    n = cu[-1]
    want, size = R.turn(q.cpu()[:n], None if wq is None else wq.cpu(), 1e-5, table, pos, style)
    _within(qo[:n], want, 2.0 ** -8 * want.abs() + 2.0 ** -20 * size + 2.0 ** -133)
    kw, _ = R.turn(k.cpu()[:n], None if wk is None else wk.cpu(), 1e-5, table, pos, style)
    untouched = [torch.ones(t.shape, dtype=torch.bool) for t in layer]
    for i, x, held in ((0, kw, ko), (2, v.cpu()[:n].double(), vo)):
        codes, scales = R.encode(x)
        assert torch.equal(held[:n].cpu().double(), R.decode(codes, scales).to(torch.bfloat16).double())
        for b in range(B):
            for j in range(new[b]):
                slot = past[b] + j
                if slot >= cap:
                    continue
                assert torch.equal(layer[i][b, :, slot].cpu(), codes[cu[b] + j])
                assert torch.equal(layer[i + 1][b, :, slot].cpu(), scales[cu[b] + j])
                untouched[i][b, :, slot] = untouched[i + 1][b, :, slot] = False
    for t, same in zip(layer, untouched):
        assert bool((t.cpu()[same] == 0xAB).all())


def test_append_of_infinities_and_of_a_full_cache():
    at = _at()
    H, Nkv = 128, 2
    k, v = R.randn((3, Nkv, H), 1.0, 1).cuda(), R.randn((3, Nkv, H), 1.0, 2).cuda()
    k[0, 0, 3], v[0, 1, 127], v[1, 0, 40], v[1, 1, 5] = math.inf, math.nan, -math.inf, 3.0e38
    layer = _empty_layer(3, Nkv, 4, H, 7)
    _, ko, vo = at.append_mx4(None, k, v, layer, _i32([0, 1, 4]), values=True)
    for held, x, scales in ((ko, k, layer.k_scales), (vo, v, layer.v_scales)):
        c, s = R.encode(x.cpu().double())
        want = R.decode(c, s)
        assert torch.equal(torch.isnan(held.cpu()), torch.isnan(want))
        assert torch.equal(held.cpu().double().nan_to_num(), want.to(torch.bfloat16).double().nan_to_num())
        assert torch.equal(scales[0, :, 0].cpu(), s[0]) and torch.equal(scales[1, :, 1].cpu(), s[1])
        assert bool((scales[2] == 7).all())  # no room: dropped


# -- attention over the cache -------------------------------------------------------------------------------------------
def _filled(B, Nkv, cap, H, seed):
    """A layer of normal keys and values, and the layer's values in 64 bits."""
    at = _at()
    kc, ks = R.encode(R.randn((B, Nkv, cap, H), 1.0, seed))
    vc, vs = R.encode(R.randn((B, Nkv, cap, H), 1.0, seed + 1))
    return at.Mx4Layer(kc.cuda(), ks.cuda(), vc.cuda(), vs.cuda()), R.decode(kc, ks), R.decode(vc, vs)


def _junk_behind(layer, lengths):
    """What lies behind the keys is anything: NaN scales, any codes."""
    for t in layer:
        for b, n in enumerate(lengths):
            t[b, :, n:] = 255


@pytest.mark.parametrize("H", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("Nq,Nkv,past,cap", [(4, 4, [0], 1), (4, 2, [0, 62, 63, 64], 67), (28, 4, [300, 5], 333), (36, 2, [130, 257], 259),
                                             (3, 1, [-1, 1000, 7], 1001)])
def test_single_tokens(H, Nq, Nkv, past, cap):
    at = _at()
    B = len(past)
    layer, k, v = _filled(B, Nkv, cap, H, H + cap)
    _junk_behind(layer, [p + 1 for p in past])
    q = R.randn((B, Nq, H), 1.5, 5)
    got = at.attn_mx4(q.cuda(), layer, _i32(past))
    for b in range(B):
        n = past[b] + 1
        want, tol = R.attend(q[b:b + 1], k[b, :, :n], v[b, :, :n], past[b])
        _within(got[b:b + 1], want, tol)


@pytest.mark.parametrize("H", [64, 96, 128, 256])
@pytest.mark.parametrize("Nq,Nkv,new,past", [(4, 4, [2, 1, 0, 3], [0, 70, 5, 1]), (14, 2, [9, 5], [120, 64]), (8, 1, [3], [700]), (2, 2, [70, 33], [0, 90]),
                                             (4, 2, [130, 1, 65], [0, 3, 64])])
@pytest.mark.parametrize("queries", ["", "64"])
def test_several_tokens(H, Nq, Nkv, new, past, queries, monkeypatch):
    at = _at()
    _prompt_form(queries, monkeypatch)
    B, cu = len(new), _starts(new)
    cap = max(p + n for p, n in zip(past, new)) + 3
    layer, k, v = _filled(B, Nkv, cap, H, H + cap)
    _junk_behind(layer, [p + n for p, n in zip(past, new)])
    q = R.randn((cu[-1], Nq + 1, H), 1.5, 5).cuda()[:, 1:]  # rows further apart than their heads
    got = at.attn_mx4(q, layer, _i32(past), _i32(cu))
    for b in range(B):
        n = past[b] + new[b]
        if new[b]:
            want, tol = R.attend(q[cu[b]:cu[b + 1]].cpu(), k[b, :, :n], v[b, :, :n], past[b])
            _within(got[cu[b]:cu[b + 1]], want, tol)


def _masks(kind, B, keys):
    low = torch.finfo(torch.bfloat16).min
    m = torch.zeros((B, keys), dtype=torch.bfloat16)
    if kind == "padding":
        for b in range(B):
            m[b, :keys * (b + 1) // (B + 1)] = low
    elif kind == "lowest everywhere":
        m[:] = low
    elif kind == "nothing":
        m[:] = -math.inf
    elif kind == "some":
        m[:, ::3] = -math.inf
        m[:, 1::7] = -2.5
    elif kind == "short":
        m = m[:, :5].contiguous()
        m[:, :2] = -math.inf
    return m


@pytest.mark.parametrize("kind", ["padding", "lowest everywhere", "nothing", "some", "short"])
@pytest.mark.parametrize("H,Nq,Nkv,new,past", [(128, 8, 2, None, [100, 3]), (64, 4, 4, None, [64, 300]), (128, 6, 3, [4, 2], [90, 0]),
                                               (128, 2, 1, [140, 70], [10, 0]), (256, 2, 2, [130], [5])])
@pytest.mark.parametrize("queries", ["", "128", "64"])
def test_masks(kind, H, Nq, Nkv, new, past, queries, monkeypatch):
    at = _at()
    _prompt_form(queries, monkeypatch)
    B = len(past)
    lens = new or [1] * B
    cu = _starts(lens)
    total = [p + n for p, n in zip(past, lens)]
    layer, k, v = _filled(B, Nkv, max(total) + 1, H, 77)
    mask = _masks(kind, B, max(total) - (kind == "some"))
    if kind == "some":  # a key that is not looked at may hold anything
        layer.k_scales[:, :, 0] = 255
        layer.v_scales[:, :, 0] = 255
        k[:, :, 0], v[:, :, 0] = math.nan, math.nan
    q = R.randn((cu[-1], Nq, H), 1.5, 6)
    got = at.attn_mx4(q.cuda(), layer, _i32(past), _i32(cu) if new else None, mask.cuda())
    for b in range(B):
        want, tol = R.attend(q[cu[b]:cu[b + 1]], k[b, :, :total[b]], v[b, :, :total[b]], past[b], mask[b])
        _within(got[cu[b]:cu[b + 1]], want, tol)
        if kind == "nothing" and mask.shape[1] >= total[b]:
            assert not bool(got[cu[b]:cu[b + 1]].any())


@pytest.mark.parametrize("new,past", [([1], [80]), ([3], [80]), ([140], [0])])
@pytest.mark.parametrize("queries", ["", "128", "64"])
def test_a_block_of_nan_reaches_the_tokens_that_see_it_alone(new, past, queries, monkeypatch):
    at = _at()
    _prompt_form(queries, monkeypatch)
    H, Nq, Nkv = 128, 4, 2
    n = past[0] + new[0]
    layer, k, v = _filled(1, Nkv, n, H, 9)
    q = R.randn((new[0], Nq, H), 1.0, 3)
    clean = at.attn_mx4(q.cuda(), layer, _i32(past), _i32([0, new[0]])).clone()
    hit = n - 1  # the last token's own value, second block of the first head
    layer.v_scales[0, 0, hit, 1] = 255
    layer.v_codes[0, 0, hit, 16:32] = 0
    got = at.attn_mx4(q.cuda(), layer, _i32(past), _i32([0, new[0]]))
    assert torch.equal(got[:-1], clean[:-1])
    bad = torch.zeros((Nq, H), dtype=torch.bool)
    bad[:Nq // Nkv, 32:64] = True
    assert torch.equal(torch.isnan(got[-1].cpu()), bad)
    assert torch.equal(got[-1].cpu()[~bad], clean[-1].cpu()[~bad])


def test_many_sequences_and_one_without_tokens():
    at = _at()
    H, Nq, Nkv = 64, 2, 1
    new = [(3 * b) % 5 for b in range(150)]
    past = [(7 * b) % 90 for b in range(150)]
    cu = _starts(new)
    layer, k, v = _filled(150, Nkv, 95, H, 21)
    q = R.randn((cu[-1], Nq, H), 1.0, 22)
    got = at.attn_mx4(q.cuda(), layer, _i32(past), _i32(cu))
    kp, vp = R.randn((cu[-1], Nkv, H), 1.0, 23), R.randn((cu[-1], Nkv, H), 1.0, 24)
    packed = at.attn_packed(q.cuda(), kp.cuda(), vp.cuda(), _i32(cu))
    for b in range(150):
        rows = slice(cu[b], cu[b + 1])
        if new[b]:
            n = past[b] + new[b]
            _within(got[rows], *R.attend(q[rows], k[b, :, :n], v[b, :, :n], past[b]))
            _within(packed[rows], *R.attend(q[rows], kp[rows].transpose(0, 1).double(), vp[rows].transpose(0, 1).double(), 0))


# -- packed prompts -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("H", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("Nq,Nkv,new,strided", [(2, 2, [1], False), (4, 1, [63, 65, 1], True), (6, 2, [0, 130, 17], True), (2, 1, [200], False)])
def test_packed_prompts(H, Nq, Nkv, new, strided):
    at = _at()
    cu = _starts(new)
    T = cu[-1] + 3
    whole = R.randn((T, Nq + 2 * Nkv, H), 1.3, H + T)
    whole[cu[-1]:] = math.nan  # rows behind the last sequence
    up = whole.cuda()
    q, k, v = up[:, :Nq], up[:, Nq:Nq + Nkv], up[:, Nq + Nkv:]
    if not strided:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    got = at.attn_packed(q, k, v, _i32(cu))
    q, k, v = whole[:, :Nq], whole[:, Nq:Nq + Nkv].transpose(0, 1).double(), whole[:, Nq + Nkv:].transpose(0, 1).double()
    for b in range(len(new)):
        rows = slice(cu[b], cu[b + 1])
        if new[b]:
            _within(got[rows], *R.attend(q[rows], k[:, rows], v[:, rows], 0))


@pytest.mark.parametrize("kind", ["padding", "nothing", "some"])
def test_packed_prompts_with_masks(kind):
    at = _at()
    H, Nq, Nkv, new = 128, 4, 2, [90, 33]
    cu = _starts(new)
    q, k, v = (R.randn((cu[-1], n, H), 1.0, 40 + i) for i, n in enumerate((Nq, Nkv, Nkv)))
    mask = _masks(kind, 2, 90)
    if kind == "some":
        k[0], v[0], k[90], v[93] = math.nan, math.inf, math.nan, math.nan
    got = at.attn_packed(q.cuda(), k.cuda(), v.cuda(), _i32(cu), mask.cuda())
    for b in range(2):
        rows = slice(cu[b], cu[b + 1])
        _within(got[rows], *R.attend(q[rows], k[rows].transpose(0, 1).double(), v[rows].transpose(0, 1).double(), 0, mask[b]))


def test_values_that_are_not_finite_reach_later_tokens_alone():
    at = _at()
    H, Nq, Nkv, n = 128, 2, 1, 150
    q, k, v = (R.randn((n, m, H), 1.0, 50 + i) for i, m in enumerate((Nq, Nkv, Nkv)))
    clean = at.attn_packed(q.cuda(), k.cuda(), v.cuda(), _i32([0, n])).cpu()
    v[70, 0, 5], v[100, 0, 9], v[101, 0, 9], v[101, 0, 77] = math.nan, math.inf, -math.inf, -math.inf
    got = at.attn_packed(q.cuda(), k.cuda(), v.cuda(), _i32([0, n])).cpu()
    want = clean.clone()
    want[70:, :, 5] = math.nan
    want[100:, :, 9] = math.inf
    want[101:, :, 9] = math.nan
    want[101:, :, 77] = -math.inf
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(), want.nan_to_num())


# -- together, and around them -----------------------------------------------------------------------------------------
def test_prompt_then_decode_from_a_graph_on_its_own_stream():
    """Packed prompts go to the cache, their attention over the values it holds equals attention over the cache, then single
    tokens are appended and attended from a captured graph, replayed with eager work between the replays."""
    at = _at()
    H, Nq, Nkv, new, cap = 128, 8, 2, [70, 5, 33], 90
    B, cu = 3, _starts(new)
    table, w = R.llama_table(100, H).cuda(), (1 + 0.1 * torch.randn(H)).cuda()
    q, k, v = (R.randn((cu[-1], m, H), 1.0, 60 + i).cuda() for i, m in enumerate((Nq, Nkv, Nkv)))
    layer = _empty_layer(B, Nkv, cap, H)
    past = _i32([0, 0, 0])
    qo, ko, vo = at.append_mx4(q, k, v, layer, past, _i32(cu), w, w, 1e-6, table, values=True)
    a = at.attn_packed(qo, ko, vo, _i32(cu))
    for b in range(B):
        rows = slice(cu[b], cu[b + 1])
        want, tol = R.attend(qo[rows].cpu(), ko[rows].cpu().transpose(0, 1).double(), vo[rows].cpu().transpose(0, 1).double(), 0)
        _within(a[rows], want, tol)
        _within(at.attn_mx4(qo, layer, past, _i32(cu))[rows], want, tol)
    past.copy_(_i32(new))
    steps = [[R.randn((B, m, H), 1.0, 70 + 3 * s + i).cuda() for i, m in enumerate((Nq, Nkv, Nkv))] for s in range(4)]

    def step(x, layer, past):
        qs, _, _ = at.append_mx4(*x, layer, past, None, w, w, 1e-6, table)
        return at.attn_mx4(qs, layer, past)

    eager_layer, eager_past, eager = at.Mx4Layer(*(t.clone() for t in layer)), past.clone(), []
    for x in steps:
        eager.append(step(x, eager_layer, eager_past).clone())
        eager_past.add_(1)
    x = [t.clone() for t in steps[0]]
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, at.Mx4Layer(*(t.clone() for t in layer)), past)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = step(x, layer, past)
        past.add_(1)
    for s in range(4):
        for t, u in zip(x, steps[s]):
            t.copy_(u)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[s])
        step([t.clone() for t in steps[s]], at.Mx4Layer(*(t.clone() for t in layer)), past.clone())
    for t, u in zip(layer, eager_layer):
        assert torch.equal(t, u)


def test_split_over_workgroups_and_unsplit_agree():
    at = _at()
    from tpp_pytorch_extension import _lib
    H, Nq, Nkv, cap, past = 128, 8, 2, 3000, [2990, 700]
    layer, k, v = _filled(2, Nkv, cap, H, 31)
    q = R.randn((2, Nq, H), 1.0, 32)
    got = at.attn_mx4(q.cuda(), layer, _i32(past))
    again = at.attn_mx4(q.cuda(), layer, _i32(past))
    assert torch.equal(got, again)
    one = torch.empty_like(got)
    qc, pc = q.cuda(), _i32(past)
    _lib.check(_lib.lib().tppx_attn_mx4(qc.data_ptr(), *(t.data_ptr() for t in layer), pc.data_ptr(), None, None, 0, one.data_ptr(), 2, 2, Nq, Nkv, H,
                                        cap, Nq * H, None, 0, None, 0, _lib.stream_of(qc)))
    for b in range(2):
        n = past[b] + 1
        want, tol = R.attend(q[b:b + 1], k[b, :, :n], v[b, :, :n], past[b])
        _within(got[b:b + 1], want, tol)
        _within(one[b:b + 1], want, tol)


def test_bounds_on_the_device_that_do_not_fit_stay_inside():
    """cu_seqlens and past that point outside are clamped: rows they do not name are left as they were."""
    at = _at()
    from tpp_pytorch_extension import _lib
    H, Nq, Nkv, T = 128, 4, 2, 10
    q, k, v = (R.randn((T, m, H), 1.0, 80 + i).cuda() for i, m in enumerate((Nq, Nkv, Nkv)))
    out = torch.full((T, Nq, H), 3.0, dtype=torch.bfloat16, device="cuda")
    cu = _i32([4, 2, 6])  # descending, then rows 2 .. 5
    _lib.check(_lib.lib().tppx_attn_packed(q.data_ptr(), k.data_ptr(), v.data_ptr(), cu.data_ptr(), None, 0, out.data_ptr(), T, 2, Nq, Nkv, H, Nq * H,
                                           Nkv * H, Nkv * H, _lib.stream_of(q)))
    assert bool((out[:2] == 3.0).all()) and bool((out[6:] == 3.0).all())
    _within(out[2:6], *R.attend(q[2:6].cpu(), k[2:6].cpu().transpose(0, 1).double(), v[2:6].cpu().transpose(0, 1).double(), 0))
    layer = _empty_layer(2, Nkv, 5, H, 9)
    at.append_mx4(q, k, v, layer, _i32([-3, 1 << 30]), _i32([0, 4, 99]))
    assert bool((layer.k_codes[1] == 9).all()) and bool((layer.k_codes[0, :, 1:] == 9).all())
    c, _ = R.encode(k[3].cpu())
    assert torch.equal(layer.k_codes[0, :, 0].cpu(), c)
    at.attn_mx4(q, layer, _i32([-3, 1 << 30]), _i32([0, 4, 99]))
    torch.cuda.synchronize()


def test_offsets_beyond_32_bits(monkeypatch):
    """Slots whose codes lie more than 4 GiB into a layer: the append, single tokens, several, and the prompt kernel over the cache."""
    at = _at()
    H, far = 256, 1 << 25  # 128 bytes of codes a slot
    layer = _empty_layer(1, 1, far + 300, H)
    layer.v_codes.fill_(0x22)  # 1.0
    layer.v_scales.fill_(127)
    k = torch.ones((130, 1, H), dtype=torch.bfloat16, device="cuda")
    cu = _i32([0, 130])
    at.append_mx4(None, k, 2 * k, layer, _i32([far]), cu, style=None)
    assert bool((layer.v_codes[0, 0, far:far + 130] == layer.v_codes[0, 0, far, 0]).all()) and bool((layer.k_scales[0, 0, far:far + 130] == 125).all())
    assert not bool(layer.k_scales[0, 0, :far].any()) and bool((layer.v_codes[0, 0, far + 130:] == 0x22).all())
    # scores: 0 before slot `far`, sqrt(H) = 16 from it on
    q = torch.ones((130, 1, H), dtype=torch.bfloat16, device="cuda")

    def want(n):
        return (far + 2 * n * math.exp(16)) / (far + n * math.exp(16))

    one = at.attn_mx4(q[:1], layer, _i32([far + 129]))
    some = at.attn_mx4(q, layer, _i32([far]), cu)
    _prompt_form("64", monkeypatch)
    many = at.attn_mx4(q, layer, _i32([far]), cu)
    # (the sums of 2^25 equal terms are exact in fp32, 32 or more at a time; what rounds is the output, the probabilities and exp)
    for n, got in ((130, one[0]), (1, some[0]), (130, some[129]), (1, many[0]), (130, many[129])):
        assert bool(((got.double() - want(n)).abs() <= (2.0 ** -8 + 2.0 ** -8 + 2.0 ** -12) * want(n)).all()), (n, got[0, 0].item(), want(n))


def test_two_streams_at_once():
    """Split attention on two streams at the same time: each has its own partial results and counters."""
    at = _at()
    H, Nq, Nkv, cap = 128, 8, 2, 4000
    layer, _, _ = _filled(2, Nkv, cap, H, 41)
    qs = [R.randn((2, Nq, H), 1.0, 42 + i).cuda() for i in range(2)]
    past = [_i32([3990, 2700]), _i32([900, 3999])]
    alone = [at.attn_mx4(q, layer, p) for q, p in zip(qs, past)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i].append(at.attn_mx4(qs[i], layer, past[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, alone[i]) for o in outs[i])


# -- the forms that larger calls take ------------------------------------------------------------------------------------
@pytest.mark.parametrize("H", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("queries", ["128", "64"])
def test_prompt_forms(H, queries, monkeypatch):
    """Both forms of a prompt's workgroup at sizes that the rule would give the other one: packed rows and the cache, tiles that end
    in a sequence, blocks that end in a tile, a mask."""
    monkeypatch.setenv("TPPX_MX4_PROMPT_QUERIES", queries)
    at = _at()
    Nq, Nkv, new, past = 4, 2, [150, 1, 129, 200], [0, 70, 33, 1]
    cu = _starts(new)
    layer, k, v = _filled(4, Nkv, 210, H, H)
    _junk_behind(layer, [p + n for p, n in zip(past, new)])
    q, kp, vp = R.randn((cu[-1], Nq, H), 1.3, 1), R.randn((cu[-1], Nkv, H), 1.0, 2), R.randn((cu[-1], Nkv, H), 1.0, 3)
    got = at.attn_mx4(q.cuda(), layer, _i32(past), _i32(cu))
    packed = at.attn_packed(q.cuda(), kp.cuda(), vp.cuda(), _i32(cu))
    for b in range(4):
        rows, n = slice(cu[b], cu[b + 1]), past[b] + new[b]
        _within(got[rows], *R.attend_rows(q[rows], k[b, :, :n], v[b, :, :n], past[b]))
        _within(packed[rows], *R.attend_rows(q[rows], kp[rows].transpose(0, 1).double(), vp[rows].transpose(0, 1).double(), 0))
    zeros = torch.zeros((4, 210), dtype=torch.bfloat16, device="cuda")
    assert torch.equal(at.attn_mx4(q.cuda(), layer, _i32(past), _i32(cu), zeros)[cu[1]:cu[2]].isnan(), torch.zeros((1, Nq, H), dtype=torch.bool, device="cuda"))
    for b, rows in ((0, slice(0, 150)), (3, slice(cu[3], cu[4]))):
        _within(at.attn_packed(q.cuda(), kp.cuda(), vp.cuda(), _i32(cu), zeros)[rows],
                *R.attend_rows(q[rows], kp[rows].transpose(0, 1).double(), vp[rows].transpose(0, 1).double(), 0))
    kp[cu[3] + 130], vp[cu[3] + 131] = math.nan, math.inf  # seen by later tokens alone
    hit = at.attn_packed(q.cuda(), kp.cuda(), vp.cuda(), _i32(cu))
    assert torch.equal(hit[:cu[3] + 130], packed[:cu[3] + 130]) and bool(hit[cu[3] + 130:].isnan().all())


@pytest.mark.parametrize("H", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("queries", ["128", "64"])
def test_prompt_forms_with_values_that_are_not_finite(H, queries, monkeypatch):
    """Infinite and NaN keys and values behind a mask of -inf, of a neighbouring sequence and of later tokens, in both forms."""
    monkeypatch.setenv("TPPX_MX4_PROMPT_QUERIES", queries)
    at = _at()
    Nq, Nkv, new = 2, 1, [133, 70]
    cu = _starts(new)
    q, k, v = (R.randn((cu[-1] + 3, n, H), 1.0, 60 + i) for i, n in enumerate((Nq, Nkv, Nkv)))
    mask = torch.zeros((2, 133), dtype=torch.bfloat16)
    mask[0, 3:7] = mask[0, 66] = -math.inf
    k[3:7], v[5:7], v[66] = math.nan, math.inf, math.nan
    v[132], k[cu[1] + 69], v[cu[2]:] = -math.inf, math.nan, math.nan  # seen by the last token alone, by the last of the other one, by none
    got = at.attn_packed(q.cuda(), k.cuda(), v.cuda(), _i32(cu), mask.cuda()).cpu()
    assert bool((got[132] == -math.inf).all()) and bool(got[cu[2] - 1].isnan().all())
    for b in range(2):
        rows = slice(cu[b], cu[b + 1] - 1)
        _within(got[rows], *R.attend(q[rows], k[rows].transpose(0, 1).double(), v[rows].transpose(0, 1).double(), 0, mask[b]))


@pytest.mark.parametrize("H", [64, 96, 128])
def test_prompts_of_many_heads(H):
    """More than 400 workgroups of 128 queries: the form of large launches, by its own rule."""
    at = _at()
    Nq, new, past = 104, [131, 130], [0, 40]
    cu = _starts(new)
    layer, k, v = _filled(2, Nq, 172, H, H)
    q, kp, vp = (R.randn((cu[-1], Nq, H), 1.2, i) for i in range(3))
    got = at.attn_mx4(q.cuda(), layer, _i32(past), _i32(cu))
    packed = at.attn_packed(q.cuda(), kp.cuda(), vp.cuda(), _i32(cu))
    for b in range(2):
        rows, n = slice(cu[b], cu[b + 1]), past[b] + new[b]
        _within(got[rows], *R.attend_rows(q[rows], k[b, :, :n], v[b, :, :n], past[b]))
        _within(packed[rows], *R.attend_rows(q[rows], kp[rows].transpose(0, 1).double(), vp[rows].transpose(0, 1).double(), 0))


@pytest.mark.parametrize("H,Nq,Nkv", [(128, 72, 8), (192, 26, 13), (256, 26, 26)])
def test_many_short_prompts(H, Nq, Nkv):
    """The form of large launches of short prompts, by its own rule: a mask, keys and values that are not finite where they are not
    seen, prompts of one token and of none."""
    at = _at()
    new = [70, 1, 33, 0, 32, 97, 64, 65]
    cu = _starts(new)
    q, k, v = (R.randn((cu[-1], n, H), 1.1, 90 + i) for i, n in enumerate((Nq, Nkv, Nkv)))
    got = at.attn_packed(q.cuda(), k.cuda(), v.cuda(), _i32(cu))
    for b in range(len(new)):
        rows = slice(cu[b], cu[b + 1])
        if new[b]:
            _within(got[rows], *R.attend_rows(q[rows], k[rows].transpose(0, 1).double(), v[rows].transpose(0, 1).double(), 0))
    v[cu[5] + 40, 0], k[cu[5] + 96, Nkv - 1] = math.inf, math.nan  # seen from there on, by the last token alone
    hit = at.attn_packed(q.cuda(), k.cuda(), v.cuda(), _i32(cu))
    first = Nq // Nkv
    assert torch.equal(hit[cu[5]:cu[5] + 40], got[cu[5]:cu[5] + 40]) and bool((hit[cu[5] + 40:cu[5] + 96, :first] == math.inf).all())
    assert torch.equal(hit[cu[5] + 40:cu[5] + 96, first:], got[cu[5] + 40:cu[5] + 96, first:]) and bool(hit[cu[5] + 96, -first:].isnan().all())
    assert torch.equal(hit[:cu[5]], got[:cu[5]]) and torch.equal(hit[cu[6]:], got[cu[6]:])
    mask = _masks("some", 8, 97)
    k[cu[5] + 96] = 0.0
    v[cu[5] + 40] = 0.0
    k[cu[5] + 3], v[cu[5] + 6] = math.nan, math.nan  # behind -inf
    got = at.attn_packed(q.cuda(), k.cuda(), v.cuda(), _i32(cu), mask.cuda())
    rows = slice(cu[5], cu[6])
    _within(got[rows, ::13], *R.attend(q[rows, ::13], k[rows].transpose(0, 1).double()[torch.arange(0, Nq, 13) * Nkv // Nq],
                                       v[rows].transpose(0, 1).double()[torch.arange(0, Nq, 13) * Nkv // Nq], 0, mask[5]))


@pytest.mark.parametrize("H", [64, 128, 192])
@pytest.mark.parametrize("splits", ["1", "3", "32"])
def test_splits(H, splits, monkeypatch):
    """Every number of splits, also where sequences are too short for theirs."""
    monkeypatch.setenv("TPPX_MX4_SPLITS", splits)
    at = _at()
    Nq, Nkv, past = 6, 2, [1500, 0, 255, 256, 700]
    layer, k, v = _filled(5, Nkv, 1600, H, H)
    _junk_behind(layer, [p + 1 for p in past])
    q = R.randn((5, Nq, H), 1.2, 1)
    for _ in range(2):
        got = at.attn_mx4(q.cuda(), layer, _i32(past))
        for b in range(5):
            _within(got[b:b + 1], *R.attend_rows(q[b:b + 1], k[b, :, :past[b] + 1], v[b, :, :past[b] + 1], past[b]))


@pytest.mark.parametrize("H,style,width", [(128, "llama", 128), (96, "llama", 96), (192, "gptj", 64)])
@pytest.mark.parametrize("wgs", ["1", "100000"])
def test_append_by_few_and_by_many_workgroups(H, style, width, wgs, monkeypatch):
    """Some hundred tokens of sequences that begin and end inside a workgroup's tokens, one head or all of them to a workgroup."""
    monkeypatch.setenv("TPPX_MX4_ROWS_WGS", wgs)
    at = _at()
    new, past, Nq, Nkv = [100, 0, 3, 1, 70], [5, 1, 0, 9, 31], 3, 2
    cu = _starts(new)
    q, k, v = (R.randn((cu[-1], n, H), 1.5, i) for i, n in enumerate((Nq, Nkv, Nkv)))
    w = R.randn(H, 0.2, 9).float() + 1
    table = _table(style, 128, H, width)
    layer = _empty_layer(5, Nkv, 120, H)
    qo, ko, vo = at.append_mx4(q.cuda(), k.cuda(), v.cuda(), layer, _i32(past), _i32(cu), w.cuda(), w.cuda(), 1e-6, table.cuda(), None, style, values=True)
    pos = [p + i for n, p in zip(new, past) for i in range(n)]
    want, size = R.turn(q, w, 1e-6, table, pos, style)
    _within(qo, want, 2.0 ** -8 * want.abs() + 2.0 ** -20 * size + 2.0 ** -133)
    kw, _ = R.turn(k, w, 1e-6, table, pos, style)
    for i, x, held in ((0, kw, ko), (2, v.double(), vo)):
        codes, scales = R.encode(x)
        assert torch.equal(held.cpu().double(), R.decode(codes, scales).to(torch.bfloat16).double())
        for b in range(5):
            at_slots = slice(past[b], past[b] + new[b])
            assert torch.equal(layer[i][b, :, at_slots].cpu(), codes[cu[b]:cu[b + 1]].transpose(0, 1))
            assert torch.equal(layer[i + 1][b, :, at_slots].cpu(), scales[cu[b]:cu[b + 1]].transpose(0, 1))
