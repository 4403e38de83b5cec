"""The MXFP4 cache and its operators at the edges of what their documentation allows: lengths at the ends of their type, sequences of
different lengths in a second turn, positions and masks in every shape that the blocks take, refused calls that change nothing."""
import math

import pytest
import torch

import mx4_ref as R

pytestmark = pytest.mark.gpu


def _at():
    import tpp_pytorch_extension  # noqa: F401
    from tpp_pytorch_extension._C import _tpp_attn
    return _tpp_attn


def _llm():
    import tpp_pytorch_extension  # noqa: F401
    from tpp_pytorch_extension.llm import fused_llama_infer as F
    return F


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _starts(lengths):
    return [sum(lengths[:i]) for i in range(len(lengths) + 1)]


def _within(got, want, tol):
    bad = ~((got.double().cpu() - want).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), bad.numel(), float(((got.double().cpu() - want).abs() / tol).max()))


def _filled(B, Nkv, cap, H, seed):
    """A layer of normal keys and values, and the layer's values in 64 bits."""
    kc, ks = R.encode(R.randn((B, Nkv, cap, H), 1.0, seed))
    vc, vs = R.encode(R.randn((B, Nkv, cap, H), 1.0, seed + 1))
    return _at().Mx4Layer(kc.cuda(), ks.cuda(), vc.cuda(), vs.cuda()), R.decode(kc, ks), R.decode(vc, vs)


def _prompt_form(queries, monkeypatch):
    """Empty: the form that the sizes give (here the split kernel); "64": the prompt kernel."""
    if queries:
        monkeypatch.setenv("TPPX_MX4_PROMPT_QUERIES", queries)


def _decoder(**kw):
    F = _llm()
    return F, F.LlamaDecoder(hidden=512, inter=1024, n_layers=2, n_heads=4, n_kv_heads=2, vocab=512, max_positions=256, seed=3, **kw)


@pytest.mark.parametrize("H", [64, 128, 256])
@pytest.mark.parametrize("queries", ["", "64"])
def test_past_at_the_end_of_its_type(H, queries, monkeypatch):
    """past at the end of int32: an append finds no slot, attention sees the whole cache, in both kernels."""
    at = _at()
    _prompt_form(queries, monkeypatch)
    Nq, Nkv, new, cap = 4, 2, [70, 130, 2], 40
    past = [2 ** 31 - 1, 2 ** 31 - 100, 2 ** 31 - 2]
    cu = _starts(new)
    layer, k, v = _filled(3, Nkv, cap, H, H)
    before = [t.clone() for t in layer]
    q, kn, vn = (R.randn((cu[-1], n, H), 1.2, i) for i, n in enumerate((Nq, Nkv, Nkv)))
    qo, _, _ = at.append_mx4(q.cuda(), kn.cuda(), vn.cuda(), layer, _i32(past), _i32(cu), emb_pos=R.llama_table(64, H).cuda())
    assert all(torch.equal(a, b) for a, b in zip(layer, before)) and torch.equal(qo.cpu(), q)  # (positions outside the table)
    got = at.attn_mx4(q.cuda(), layer, _i32(past), _i32(cu))
    one = at.attn_mx4(q[:3].cuda(), layer, _i32(past))
    for b in range(3):
        rows = slice(cu[b], cu[b + 1])
        _within(got[rows], *R.attend_rows(q[rows], k[b], v[b], cap))
        _within(one[b:b + 1], *R.attend_rows(q[b:b + 1], k[b], v[b], cap))


@pytest.mark.parametrize("H", [64, 128, 256])
@pytest.mark.parametrize("queries", ["", "64"])
@pytest.mark.parametrize("masked", [False, True])
def test_tokens_before_the_first_slot(H, queries, masked, monkeypatch):
    """A negative past: token i sees the keys 0 .. past + i, those before the first slot none, in both kernels and appended alike; a block of
    NaN in a seen key reaches the tokens that see it."""
    at = _at()
    _prompt_form(queries, monkeypatch)
    Nq, Nkv, new, past, cap = 4, 2, [70, 230, 9, 5], [-3, -200, -9, -2 ** 31], 68
    cu = _starts(new)
    layer, k, v = _filled(4, Nkv, cap, H, H + 5)
    q = R.randn((cu[-1], Nq, H), 1.2, 3)
    mask = torch.zeros((4, 70), dtype=torch.bfloat16)
    if masked:
        mask[:, 1] = -math.inf
    args = (q.cuda(), layer, _i32(past), _i32(cu), mask.cuda() if masked else None)
    got = at.attn_mx4(*args)
    for b in range(4):
        rows = slice(cu[b], cu[b + 1])
        n = max(past[b] + new[b], 0)
        _within(got[rows], *R.attend(q[rows], k[b, :, :n], v[b, :, :n], past[b], mask[b] if masked else None))
        assert not bool(got[cu[b]:cu[b] - past[b]].any())
    layer.v_scales[1, 0, 10, 0] = 255
    hit = at.attn_mx4(*args)
    bad = torch.zeros(got.shape, dtype=torch.bool)
    bad[cu[1] + 210:cu[2], :Nq // Nkv, :32] = True
    assert torch.equal(hit.isnan().cpu(), bad) and torch.equal(hit.cpu()[~bad], got.cpu()[~bad])


def test_a_second_turn_behind_sequences_of_different_lengths():
    """prefill on a cache whose sequences differ: each sequence's tokens are rotated at its own positions."""
    F, dec = _decoder(kv_dtype="mxfp4")
    g = torch.Generator().manual_seed(11)
    first = [torch.randint(0, 512, (n,), generator=g).cuda() for n in (40, 7)]
    turn = torch.randint(0, 512, (2, 5), generator=g).cuda()
    caches = [F.Mx4Cache(80) for _ in range(2)]
    for c in caches:
        dec.prefill_packed(first, c)
    dec.prefill(turn, caches[0])
    h = dec.embed.index_select(0, turn.reshape(-1)).view(2, 5, 512)
    pos = torch.stack([torch.arange(n, n + 5) for n in (40, 7)]).cuda()
    for layer in dec.layers:
        h = layer.forward([h, None, pos], caches[1])[0]
    caches[1].advance(5)
    assert caches[0].seq_len_dev.tolist() == caches[1].seq_len_dev.tolist() == [45, 12]
    for i in range(2):
        for a, b in zip(caches[0].layers[i], caches[1].layers[i]):
            assert torch.equal(a, b)
    # and as the sequences alone: the first layer's keys differ by what a step of bf16 (2^-7) moves, one code in 2^-7 / (1/4) at most,
    # each by half of its value at most: rel-L2 sqrt(2^-5 / 4) < 0.09
    for b in range(2):
        c = F.Mx4Cache(80)
        dec.prefill(first[b].view(1, -1), c)
        dec.prefill(turn[b:b + 1], c)
        n = first[b].numel()
        want, got = c.get(0)[0][0, :, n:n + 5].double(), caches[0].get(0)[0][b, :, n:n + 5].double()
        assert float((got - want).norm() / want.norm()) < 0.09


def _tiny(family):
    T = pytest.importorskip("transformers")
    F = _llm()
    torch.manual_seed(43)
    if family in ("llama", "qwen2"):
        cls, model = (T.LlamaConfig, T.LlamaForCausalLM) if family == "llama" else (T.Qwen2Config, T.Qwen2ForCausalLM)
        kw = dict(head_dim=128) if family == "llama" else {}
        cfg = cls(hidden_size=512, intermediate_size=1024, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, vocab_size=1024,
                  max_position_embeddings=256, attn_implementation="eager", **kw)
        if family == "llama":
            return F.OptimizeModelForLlama(model(cfg).eval(), torch.bfloat16, "cuda", "mxfp4").eval()
        from tpp_pytorch_extension.llm import fused_qwen2_infer as Q
        return Q.OptimizeModelForQwen2(model(cfg).eval(), torch.bfloat16, "cuda", "mxfp4").eval()
    if family == "gptj":
        from tpp_pytorch_extension.llm import fused_gptj_infer as G
        return G.OptimizeModelForGPTJ(T.GPTJForCausalLM(T.GPTJConfig(n_embd=512, n_head=2, n_layer=2, n_positions=256, rotary_dim=64, vocab_size=1600,
                                                                     bos_token_id=1, eos_token_id=2)).eval(), torch.bfloat16, "cuda", "mxfp4").eval()
    from tpp_pytorch_extension.llm import fused_opt_infer as O
    cfg = T.OPTConfig(hidden_size=512, ffn_dim=1024, num_hidden_layers=2, num_attention_heads=4, vocab_size=1600, max_position_embeddings=256,
                      word_embed_proj_dim=512, attn_implementation="eager")
    return O.OptimizeModelForOPT(T.OPTForCausalLM(cfg).eval(), torch.bfloat16, "cuda", "mxfp4").eval()


@pytest.mark.parametrize("family", ["llama", "qwen2", "gptj", "opt"])
def test_front_ends_count_the_positions_of_every_sequence(family):
    """Packed prompts through a front-end's forward, then a turn of both sequences, without position_ids: what explicit ones give."""
    from tpp_pytorch_extension.llm.llm_common import TppCache
    opt = _tiny(family)
    core = next(m for m in opt.modules() if getattr(m, "_tpp_core_model", False))
    g = torch.Generator().manual_seed(12)
    packed, turn = (torch.randint(3, 1000, s, generator=g).cuda() for s in ((1, 13), (2, 3)))
    outs, keys = [], []
    for explicit in (False, True):
        cache = TppCache(capacity=64, kv_dtype="mxfp4")
        where = [torch.cat([torch.arange(9), torch.arange(4)]).unsqueeze(0).cuda(), torch.stack([torch.arange(9, 12), torch.arange(4, 7)]).cuda()]
        with torch.no_grad():
            if family != "opt":  # (whose forward makes a padding mask, which packed prompts do not take)
                cache.get_cpp().prompts([9, 4])
                a = core(input_ids=packed, past_key_values=cache, position_ids=where[0] if explicit else None).last_hidden_state
            else:
                core(input_ids=turn.repeat(1, 3), past_key_values=cache)
                cache.get_cpp()._short = [0, 5]
                cache.get_cpp().seq_len_dev.sub_(_i32([0, 5]))
                a = None
            b = core(input_ids=turn, past_key_values=cache, position_ids=where[1] if explicit else None).last_hidden_state
        outs.append((a, b))
        keys.append([t.clone() for layer in cache.get_cpp().layers.values() for t in layer])
        assert cache.get_cpp().seq_len_dev.tolist() == [12, 7]
    for x, y in zip(outs[0], outs[1]):
        assert x is y or torch.equal(x, y)
    assert all(torch.equal(x, y) for x, y in zip(*keys))


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("kv", ["mxfp4", "bfloat16"])
def test_one_position_for_all_sequences(norm, kv):
    """Single tokens of several sequences with position_ids [1][1], as the blocks take them."""
    F = _llm()
    B, Nq, Nkv, H = 3, 4, 2, 128
    table = R.llama_table(64, H).cuda()
    w = (1 + 0.1 * R.randn(H, 1.0, 5).float()).cuda()
    q, k, v = (R.randn((B, 1, n * H), 1.0, i).cuda() for i, n in enumerate((Nq, Nkv, Nkv)))
    outs = []
    for pos in (torch.tensor([[9]]).cuda(), torch.tensor([[9]] * B).cuda(), torch.tensor([[9]]).cuda().expand(B, 1)):
        cache = F.kv_cache(32, kv)
        outs.append(F.rotate_append_attend(q.clone(), k.clone(), v, None, pos.contiguous() if kv == "bfloat16" else pos, cache, 0, B, 1, Nq, Nkv, H, table,
                                           "llama", (w, w, 1e-6) if norm else None))
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[2], outs[1])


@pytest.mark.parametrize("family", ["llama", "qwen2", "gptj", "opt"])
def test_front_ends_without_a_mask(family, monkeypatch):
    """Greedy loops of two sequences without an attention mask (one row of positions for both) on the MXFP4 cache, eager and replayed."""
    monkeypatch.setenv("TPPX_KV_DTYPE", "mxfp4")
    F = _llm()
    opt = _tiny(family)
    ids = torch.randint(3, 1000, (2, 21), generator=torch.Generator().manual_seed(8)).cuda()
    out = F.generate_greedy(opt, ids, 8)
    assert out.shape == (2, 29) and torch.equal(F.generate_greedy(opt, ids, 8, torch.ones_like(ids)), out)
    assert torch.equal(F.generate_greedy_graph(opt, ids, 8), out)


def test_one_token_with_any_stride():
    """The row stride of a single token is not looked at."""
    at = _at()
    H, Nq, Nkv = 128, 4, 2
    x = [R.randn((1, n, H), 1.0, n).cuda() for n in (Nq, Nkv, Nkv + 1)]
    x[2] = x[2][:, :Nkv].contiguous()
    odd = []
    for t, stride in zip(x, (7, 8, 0)):
        o = torch.empty_strided(t.shape, (stride, H, 1), dtype=t.dtype, device="cuda")
        odd.append(o.copy_(t))
    a, b = at.qk_norm_rotary(*x[:2]), at.qk_norm_rotary(*odd[:2])
    assert all(torch.equal(s, t) for s, t in zip(a, b))
    outs = []
    for q, k, v in (x, odd):
        layer = at.Mx4Layer(*(torch.zeros((1, Nkv, 4, n), dtype=torch.uint8, device="cuda") for n in (64, 4, 64, 4)))
        r, kr, vr = at.append_mx4(q, k, v, layer, _i32([0]), style=None, values=True)
        outs.append([r, kr, vr, *layer, at.attn_mx4(q, layer, _i32([0])), at.attn_packed(q, k, v, _i32([0, 1]))])
    assert all(torch.equal(s, t) for s, t in zip(*outs))


def test_a_context_of_no_tokens():
    """new_cache with a context of no tokens, on both caches."""
    for kv in ("bfloat16", "mxfp4"):
        F, dec = _decoder(kv_dtype=kv)
        cache = dec.new_cache(2, 0, 40)
        assert cache.get_seq_length() == 0 and set(cache.seq_len_dev.tolist()) == {0}
        out = dec.greedy_decode(torch.tensor([3, 5]).cuda(), cache, 4)
        again = dec.greedy_decode(torch.tensor([3, 5]).cuda(), dec.new_cache(2, 0, 40), 4, use_graph=False)
        assert torch.equal(out, again) and cache.get_seq_length() == 4


def test_several_tokens_first_asked_for_inside_a_capture():
    """A pass of several tokens that is captured first and run eagerly before the first replay, then replayed."""
    F = _llm()
    B, S, Nq, Nkv, H = 2, 3, 4, 2, 128
    q, k, v = (R.randn((B, S, n * H), 1.0, i).cuda() for i, n in enumerate((Nq, Nkv, Nkv)))

    def fresh():
        c = F.Mx4Cache(32)
        zeros = torch.zeros((B, Nkv, 5, H), dtype=torch.bfloat16, device="cuda")
        return c.fill_(0, zeros, zeros + 1)

    pos = torch.zeros((1, S), dtype=torch.int64, device="cuda")

    def run(cache, q):
        return F.rotate_append_attend(q, k, v, None, pos, cache, 0, B, S, Nq, Nkv, H, None, None)

    want = run(fresh(), q)  # (and the workspace exists)
    cache = fresh()
    x = q.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(cache, x)
    other = torch.cuda.Stream()
    with torch.cuda.stream(other):
        assert torch.equal(run(cache, q), want)
    torch.cuda.synchronize()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        junk = [torch.full((B + 1,), 77, dtype=torch.int32, device="cuda") for _ in range(20)]
        del junk


def test_a_refused_mask_leaves_the_cache_as_it_was():
    F = _llm()
    B, Nkv, Rr, H = 2, 2, 2, 64
    cache = F.kv_cache(16, "mxfp4")
    q, k, v = (R.randn((B, Nkv, 3, n, H), 1.0, n).cuda() for n in (Rr, 1, 3))
    k, v = k[:, :, :, 0].contiguous(), v[:, :, :, 1].contiguous()
    F.attn(q, k, v, None, cache, 0)
    before = [t.clone() for t in cache.layers[0]]
    for mask in (torch.zeros(1, 6), torch.zeros(B, 1, 3, 6), torch.zeros(B, 6).cuda().expand(3, B, 6)):
        with pytest.raises(F.TppxError):
            F.attn(q, k, v, mask.to(torch.bfloat16).cuda(), cache, 0)
        assert cache.get_seq_length() == 3 and cache.seq_len_dev.tolist() == [3, 3] and cache.get_capacity() == 16
        assert all(torch.equal(a, b) for a, b in zip(cache.layers[0], before))


@pytest.mark.parametrize("S", [1, 4])
def test_masks_of_the_blocks_in_four_dimensions(S):
    """The additive mask [B][1][1][keys] through a decoder block: what [B][keys] gives, on both caches."""
    for kv in ("bfloat16", "mxfp4"):
        F, dec = _decoder(kv_dtype=kv)
        mask = torch.zeros((2, 32), dtype=torch.bfloat16, device="cuda")
        mask[1, :6] = torch.finfo(torch.bfloat16).min
        h = R.randn((2, S, 512), 1.0, 4).cuda()
        outs = []
        for m in (mask, mask.view(2, 1, 1, 32)):
            cache = dec.new_cache(2, 20, 40)
            outs.append(dec.layers[0].forward([h, m, cache.positions(2, "cuda") + torch.arange(S, device="cuda")], cache)[0])
        assert torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("H,style,width", [(128, "llama", 128), (96, "llama", 64), (256, "gptj", 64)])
def test_norms_of_heads_that_hold_an_infinity(H, style, width):
    """Their mean square is infinite: the finite channels become zeros and the infinite ones NaN, for queries and for the codes of keys."""
    at = _at()
    T, Nq, Nkv = 4, 2, 2
    table = (R.llama_table if style == "llama" else R.gptj_table)(16, width)
    w = R.randn(H, 0.2, 9).float() + 1
    q, k, v = (R.randn((T, n, H), 1.0, i) for i, n in enumerate((Nq, Nkv, Nkv)))
    q[0, 0, 5], k[0, 1, 3], k[1, 0, H - 1], k[2, 1, 7] = math.inf, math.inf, -math.inf, math.nan
    layer = at.Mx4Layer(*(torch.zeros((1, Nkv, 8, n), dtype=torch.uint8, device="cuda") for n in (H // 2, H // 32, H // 2, H // 32)))
    qo, ko, _ = at.append_mx4(q.cuda(), k.cuda(), v.cuda(), layer, _i32([1]), _i32([0, T]), w.cuda(), w.cuda(), 1e-6, table.cuda(), None, style, values=True)
    pos = range(1, 1 + T)
    want, size = R.turn(q, w, 1e-6, table, pos, style)
    assert torch.equal(qo.isnan().cpu(), want.isnan())
    _within(qo.nan_to_num(), want.nan_to_num(), (2.0 ** -8 * want.abs() + 2.0 ** -20 * size.abs()).nan_to_num() + 2.0 ** -133)
    codes, scales = R.encode(R.turn(k, w, 1e-6, table, pos, style)[0])
    assert torch.equal(layer.k_scales[0, :, 1:1 + T].cpu(), scales.transpose(0, 1))
    held = R.decode(codes, scales)
    assert torch.equal(ko.isnan().cpu(), held.isnan()) and torch.equal(ko.nan_to_num().cpu().double(), held.nan_to_num().to(torch.bfloat16).double())
