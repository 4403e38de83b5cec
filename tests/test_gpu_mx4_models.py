"""The MXFP4 cache under the decoder blocks, the decoder, the attention entry point and the front-ends; norms of the heads in a
block; packed prompts of different lengths."""
import pytest
import torch

import mx4_ref as R

pytestmark = pytest.mark.gpu


def _llm():
    import tpp_pytorch_extension  # noqa: F401
    from tpp_pytorch_extension.llm import fused_llama_infer as F
    return F


def _within(got, want, tol):
    bad = ~((got.double().cpu() - want).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), bad.numel(), float(((got.double().cpu() - want).abs() / tol).max()))


def _rel(a, b):
    a, b = a.double(), b.double()
    return float((a - b).norm() / b.norm())


@pytest.mark.parametrize("style,width", [("llama", 128), ("gptj", 64), (None, 0)])
@pytest.mark.parametrize("norm", [False, True])
def test_rotate_append_attend_over_an_mx4_cache(style, width, norm):
    """A prompt, single tokens and a few tokens, with a padding mask, each over what the cache holds then."""
    F = _llm()
    B, Nq, Nkv, H, cap = 2, 4, 2, 128, 96
    table = None if style is None else R.llama_table(64, width) if style == "llama" else R.gptj_table(64, width)
    wq, wk = (R.randn(H, 0.2, 1).float() + 1, R.randn(H, 0.2, 2).float() + 1) if norm else (None, None)
    qk_norm = (wq.cuda(), wk.cuda(), 1e-6) if norm else None
    cache = F.Mx4Cache(cap)
    held_k, held_v = torch.zeros((B, Nkv, 0, H), dtype=torch.float64), torch.zeros((B, Nkv, 0, H), dtype=torch.float64)
    keep = torch.ones((B, 60))
    keep[1, :5] = 0
    at = 0
    for i, S in enumerate((13, 1, 1, 4, 1)):
        q, k, v = (R.randn((B, S, n * H), 1.0, 10 * i + n) for n in (Nq, Nkv, Nkv + 10))
        v = v[..., :Nkv * H].contiguous()
        pos = torch.arange(at, at + S).unsqueeze(0)
        if S == 1:
            pos = pos.expand(B, 1).contiguous()
        mask = cache.align_and_invert_mask(keep[:, :at + S].to(torch.bfloat16), torch.finfo(torch.bfloat16).min)
        ctx = F.rotate_append_attend(q.cuda(), k.cuda(), v.cuda(), mask.cuda(), pos.cuda(), cache, 0, B, S, Nq, Nkv, H,
                                     None if table is None else table.cuda(), style, qk_norm)
        flat = pos.expand(B, S).reshape(-1)
        qr, _ = R.turn(q.view(B * S, Nq, H), wq, 1e-6, table, flat, style)
        kr, _ = R.turn(k.view(B * S, Nkv, H), wk, 1e-6, table, flat, style)
        kr, vr = (R.decode(*R.encode(t)).view(B, S, Nkv, H).transpose(1, 2) for t in (kr, v.view(B * S, Nkv, H).double()))
        held_k, held_v = torch.cat((held_k, kr), 2), torch.cat((held_v, vr), 2)
        for b in range(B):
            rows = qr.view(B, S, Nq, H)[b].to(torch.bfloat16)
            want, tol = R.attend(rows, held_k[b], held_v[b], at, mask[b])
            # the queries were rounded to bf16 there and here, from fp32 and from 64 bits: where the two fall on different sides
            # a query is a step of 2^-7 off, and a score by that of its products
            shift = 2.0 ** -7 * float((held_k[b].abs().amax((0, 1)) @ rows.abs().amax((0, 1)).double())) / H ** 0.5 / 64
            _within(ctx.view(B, S, Nq, H)[b], want, tol + 2 * shift * held_v[b].abs().max())
        cache.advance(S)
        at += S
    k, v = cache.get(0)
    assert torch.equal(k.cpu().double(), held_k.to(torch.bfloat16).double()) and torch.equal(v.cpu().double(), held_v.to(torch.bfloat16).double())


def test_head_norms_of_a_block_on_the_bf16_cache():
    """The norms in front of the rotation, then the bf16 cache: what rotate_append_attend gives for rows normed and rotated before."""
    F = _llm()
    from tpp_pytorch_extension._C import _tpp_attn as at
    B, S, Nq, Nkv, H = 2, 9, 4, 2, 128
    table, w = R.llama_table(64, H).cuda(), (1 + 0.1 * torch.randn(H)).cuda()
    q, k, v = (R.randn((B, S, n * H), 1.0, n).cuda() for n in (Nq, Nkv, 7))
    v = v[..., :Nkv * H].contiguous()
    pos = torch.arange(S).unsqueeze(0).cuda()
    a, b = F.TppCache(32), F.TppCache(32)
    one = F.rotate_append_attend(q.clone(), k.clone(), v, None, pos, a, 0, B, S, Nq, Nkv, H, table, "llama", (w, w, 1e-6))
    qr, kr = at.qk_norm_rotary(q.view(-1, Nq, H), k.view(-1, Nkv, H), w, w, 1e-6, table, pos.expand(B, S).reshape(-1))
    two = F.rotate_append_attend(qr.view(q.shape), kr.view(k.shape), v, None, pos, b, 0, B, S, Nq, Nkv, H, table, None)
    assert torch.equal(one, two) and all(torch.equal(x, y) for x, y in zip(a.layers[0], b.layers[0]))


def _decoder(**kw):
    F = _llm()
    return F, F.LlamaDecoder(hidden=512, inter=1024, n_layers=2, n_heads=4, n_kv_heads=2, vocab=512, max_positions=256, seed=3, **kw)


@pytest.mark.parametrize("qk_norm", [False, True])
def test_packed_prompts_through_the_layers(qk_norm):
    """Hidden states of prompts packed one after the other equal those of each prompt alone: apart from the order of fp32 sums (row
    counts pick the GEMM kernels), which moves some 10^-3 of the bf16 values by a step and a few codes with them: rel-L2 1e-2
    over two layers, as the bf16 roundings of two layers allow."""
    F, dec = _decoder(kv_dtype="mxfp4", qk_norm=qk_norm)
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, 512, (n,), generator=g).cuda() for n in (40, 1, 17, 90)]

    def run(ps, cache):
        bounds = cache.prompts([p.numel() for p in ps])
        pos = torch.cat([torch.arange(p.numel()) for p in ps]).unsqueeze(0).cuda()
        h = dec.embed.index_select(0, torch.cat(ps)).unsqueeze(0)
        for layer in dec.layers:
            h = layer.forward([h, None, pos], cache)[0]
        cache.advance()
        return [h[0, bounds[i]:bounds[i + 1]] for i in range(len(ps))]

    cache = F.Mx4Cache(128)
    together = run(prompts, cache)
    assert cache.seq_len_dev.tolist() == [40, 1, 17, 90] and cache.get_seq_length() == 90
    for p, h in zip(prompts, together):
        assert _rel(h, run([p], F.Mx4Cache(128))[0]) <= 1e-2
    # a second packed pass behind the first: the shorter ones catch up
    more = [torch.randint(0, 512, (n,), generator=g).cuda() for n in (3, 100, 1, 2)]
    cache.prompts([p.numel() for p in more])
    cache._packed = None
    first = dec.prefill_packed(more, cache)
    assert first.shape == (4,) and cache.seq_len_dev.tolist() == [43, 101, 18, 92] and cache.get_seq_length() == 101
    with pytest.raises(F.TppxError):
        cache.prompts([1, 28, 1, 1])
    assert cache.prompts([85, 27, 110, 36]).tolist() == [0, 85, 112, 222, 258]


def test_generate_packed_equals_its_graph_and_refuses_others():
    F, dec = _decoder(kv_dtype="mxfp4", qk_norm=True)
    g = torch.Generator().manual_seed(6)
    prompts = [torch.randint(0, 512, (n,), generator=g).cuda() for n in (30, 7, 64)]
    eager = dec.generate_packed(prompts, 12, use_graph=False)
    assert eager.shape == (3, 12)
    assert torch.equal(dec.generate_packed(prompts, 12), eager)
    same = torch.stack([prompts[0], prompts[0]])
    assert torch.equal(dec.generate(same, 10), dec.generate(same, 10, use_graph=False))
    assert dec.time_decode_steps(prompts[0][:2], dec.new_cache(2, 50, 100), 5) > 0
    with pytest.raises(F.TppxError):
        dec.prefill_packed(prompts, F.TppCache(128))
    with pytest.raises(F.TppxError):
        dec.prefill_packed([prompts[0], prompts[0][:0]], F.Mx4Cache(128))
    with pytest.raises(F.TppxError):
        F.kv_cache(8, "int3")


def test_attention_entry_point_and_cache_methods():
    """_tpp_attn.attn, update, get, crop, reorder and growth of an Mx4Cache."""
    F = _llm()
    from tpp_pytorch_extension._C import _tpp_attn as at
    B, Nkv, Rr, H = 2, 2, 3, 64
    cache = at.kv_cache(8, "mxfp4")
    ks, vs = [], []
    for i, S in enumerate((6, 1, 5)):
        q, k, v = (R.randn((B, Nkv, S, n, H), 1.0, 20 * i + n) for n in (Rr, 1, 2))
        k, v = k[:, :, :, 0], v[:, :, :, 1].contiguous()
        out = at.attn(q.cuda(), k.cuda(), v.cuda(), None, cache, 0)
        ks.append(R.decode(*R.encode(k)))
        vs.append(R.decode(*R.encode(v)))
        past = sum(t.shape[2] for t in ks) - S
        for b in range(B):
            rows = q[b].permute(1, 0, 2, 3).reshape(S, Nkv * Rr, H)
            want, tol = R.attend(rows, torch.cat(ks, 2)[b], torch.cat(vs, 2)[b], past)
            _within(out[b].permute(1, 0, 2, 3).reshape(S, Nkv * Rr, H), want, tol)
    assert cache.get_seq_length() == 12 and cache.get_capacity() >= 12  # it grew
    k, v = cache.get(0)
    assert torch.equal(k.cpu().double(), torch.cat(ks, 2)) and torch.equal(v.cpu().double(), torch.cat(vs, 2))
    cache.reorder_cache(torch.tensor([1, 1]))
    assert torch.equal(cache.get(0)[0][0], k[1]) and torch.equal(cache.get(0)[1][1], v[1])
    cache.crop(7)
    assert cache.get_seq_length() == 7 and cache.seq_len_dev.tolist() == [7, 7]
    nk, _ = cache.update(R.randn((B, Nkv, 2, H), 1.0, 90).cuda(), R.randn((B, Nkv, 2, H), 1.0, 91).cuda(), 0)
    assert nk.shape[2] == 9 and torch.equal(nk[:, :, :7], k[1:].expand(2, -1, -1, -1)[:, :, :7])
    mask = torch.zeros((B, 9), dtype=torch.bfloat16)
    mask[1, 2:5] = float("-inf")
    q, k, v = R.randn((B, Nkv, 1, Rr, H), 1.0, 92), R.randn((B, Nkv, 1, H), 1.0, 93), R.randn((B, Nkv, 1, H), 1.0, 94)
    outs = []
    for m in (mask, mask.view(B, 1, 1, 9)):  # the same mask in two shapes
        outs.append(at.attn(q.cuda(), k.cuda(), v.cuda(), m.cuda(), cache, 0))
        cache.crop(9)
    assert torch.equal(outs[0], outs[1])
    with pytest.raises(F.TppxError):
        at.attn(R.randn((B, Nkv, 1, 1, 80), 1.0, 1).cuda(), R.randn((B, Nkv, 1, 80), 1.0, 1).cuda(), R.randn((B, Nkv, 1, 80), 1.0, 1).cuda(), None,
                at.kv_cache(8, "mxfp4"), 0)


@pytest.mark.parametrize("family", ["llama", "gptj"])
def test_front_ends_on_an_mx4_cache(family, monkeypatch):
    """TPPX_KV_DTYPE=mxfp4: greedy loops of the optimized transformers models with left padding, eager and from a graph, give the same
    tokens, and each token maximises the logits of a pass over the finished sequence (3 % of the largest logit, as for the bf16
    cache: both passes see the same codes); beam search moves the codes."""
    T = pytest.importorskip("transformers")
    monkeypatch.setenv("TPPX_KV_DTYPE", "mxfp4")
    F = _llm()
    torch.manual_seed(41)
    if family == "llama":
        cfg = T.LlamaConfig(hidden_size=512, intermediate_size=1024, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, vocab_size=1024,
                            max_position_embeddings=256, head_dim=128, attn_implementation="eager")
        opt = F.OptimizeModelForLlama(T.LlamaForCausalLM(cfg).eval(), torch.bfloat16, "cuda", "mxfp4").eval()
    else:
        from tpp_pytorch_extension.llm import fused_gptj_infer as G
        opt = G.OptimizeModelForGPTJ(T.GPTJForCausalLM(T.GPTJConfig(n_embd=512, n_head=2, n_layer=2, n_positions=256, rotary_dim=64, vocab_size=1600,
                                                                    bos_token_id=1, eos_token_id=2)).eval(), torch.bfloat16, "cuda", "mxfp4").eval()
    ids = torch.randint(3, 1000, (2, 21), generator=torch.Generator().manual_seed(8)).cuda()
    am = torch.ones_like(ids)
    am[1, :6] = 0
    out = F.generate_greedy(opt, ids, 20, attention_mask=am)
    assert torch.equal(F.generate_greedy_graph(opt, ids, 20, attention_mask=am), out)
    with torch.no_grad():
        past = opt(input_ids=ids, attention_mask=am, use_cache=True).past_key_values
        assert past.get_cpp().kv_dtype == "mxfp4"
        whole = torch.cat([am, am.new_ones((2, 20))], 1)
        pos = (whole.cumsum(-1) - 1).clamp(min=0)
        pos = pos.masked_fill(whole == 0, 1)
        logits = opt(input_ids=out[:, :-1], attention_mask=whole[:, :-1], position_ids=pos[:, :-1]).logits.float()
    for t in range(20, 40):
        lt = logits[:, t]
        gap = lt.max(-1).values - lt.gather(1, out[:, t + 1:t + 2])[:, 0]
        assert bool((gap <= 0.03 * lt.abs().max(-1).values).all()), (t, gap.tolist())
    beams = opt.generate(input_ids=ids, attention_mask=am, max_new_tokens=5, num_beams=2, do_sample=False, pad_token_id=0)
    assert beams.shape[0] == 2
