"""The cache in pages under the decoder blocks and the decoder, and generation with drafted tokens."""
import pytest
import torch

import mx4_ref as M
import paged_ref as R

pytestmark = pytest.mark.gpu


def _llm():
    import tpp_pytorch_extension  # noqa: F401
    from tpp_pytorch_extension.llm import fused_llama_infer as F
    return F


@pytest.mark.parametrize("style,width", [("llama", 128), ("gptj", 64), (None, 0)])
@pytest.mark.parametrize("norm", [False, True])
def test_rotate_append_attend_over_pages(style, width, norm):
    """A prompt, single tokens, a few tokens, and trees of nodes of which a path is kept, each over what the cache holds then."""
    F = _llm()
    B, Nq, Nkv, H, page = 2, 4, 2, 128, 16
    table = None if style is None else M.llama_table(64, width) if style == "llama" else M.gptj_table(64, width)
    wq, wk = (M.randn(H, 0.2, 1).float() + 1, M.randn(H, 0.2, 2).float() + 1) if norm else (None, None)
    qk_norm = (wq.cuda(), wk.cuda(), 1e-6) if norm else None
    cache = F.PagedCache(60, 2, page=page)
    held = [[torch.zeros((Nkv, 0, H), dtype=torch.float64)] * 2 for _ in range(B)]
    trees = [R.tree(6, 1), R.tree(9, 2)]
    paths = [[0, 1, 3], [0]]
    for i, S in enumerate((13, 1, "trees", 1, 4)):
        nodes = [6, 9] if S == "trees" else [S] * B
        T = sum(nodes)
        q, k, v = (M.randn((T, n, H), 1.0, 10 * i + j) for j, n in enumerate((Nq, Nkv, Nkv)))
        parents = trees if S == "trees" else [list(range(-1, S - 1))] * B
        at = [h[0].shape[1] for h in held]
        pos = torch.tensor([a + d for a, p in zip(at, parents) for d in R.depths(p)])
        shape = (1, T) if S == "trees" else (B, S)
        if S == "trees":
            cache.nodes(nodes, trees)
            assert torch.equal(cache.next_positions(T, "cuda").cpu()[0], pos)
        got = F.rotate_append_attend(*(t.view(*shape, -1).cuda() for t in (q, k, v)), None, pos.view(shape).cuda(), cache, 1, *shape, Nq, Nkv, H,
                                     None if table is None else table.cuda(), style, qk_norm).view(T, Nq, H)
        qr, _ = M.turn(q, wq, 1e-6, table, pos, style)
        kr, _ = M.turn(k, wk, 1e-6, table, pos, style)
        qr, kr = qr.to(torch.bfloat16), kr.to(torch.bfloat16)
        first = 0
        for b, n in enumerate(nodes):
            rows = slice(first, first + n)
            kk, vv = (torch.cat((h, x[rows].double().transpose(0, 1)), 1) for h, x in zip(held[b], (kr, v)))
            seen = torch.ones((n, at[b] + n), dtype=torch.bool)
            seen[:, at[b]:] = R.ancestors(parents[b])
            want, tol = R.attend(qr[rows], kk, vv, seen)
            # queries and keys are rounded to bf16 there and here, from 64 bits and from fp32: where the two fall on different sides one of
            # them is a step of 2^-7 off, and a score by that of its products; one in some 2^8 is
            shift = 2 * 2.0 ** -7 * float((kk.abs().amax((0, 1)) @ qr[rows].double().abs().amax((0, 1)))) / H ** 0.5 / 64
            assert bool(((got[rows].double().cpu() - want).abs() <= tol + shift * vv.abs().amax()).all())
            keep = list(range(n)) if S != "trees" else paths[b]
            held[b] = [torch.cat((h, x[rows].double().transpose(0, 1)[:, keep]), 1) for h, x in zip(held[b], (kr, v))]
            first += n
        if S == "trees":
            path = torch.tensor([x for p, n in zip(paths, nodes) for x in p + [-1] * (n - len(p))], dtype=torch.int32, device="cuda")
            assert cache.keep(path, torch.tensor([3, 1], dtype=torch.int32, device="cuda")) == [3, 1]
        else:
            cache.advance(S)
        assert cache.lengths == cache.seq_len_dev.tolist() == [h[0].shape[1] for h in held]
    for side, got in enumerate(cache.get(1)):
        for b in range(B):
            n = cache.lengths[b]
            d = (got[b, :, :n].double().cpu() - held[b][side]).abs()
            assert bool((d <= 2.0 ** -7 * held[b][side].abs() + 1e-30).all()) and float((d > 0).double().mean()) < 0.02


def _decoder(**kw):
    F = _llm()
    return F, F.LlamaDecoder(hidden=256, inter=512, n_layers=2, n_heads=4, n_kv_heads=2, vocab=1024, max_positions=256, seed=3, kv_dtype="paged", **kw)


def _logits(dec, F, text):
    """Of every position of a text, by one pass over an empty cache."""
    cache = F.PagedCache(256, dec.n_layers)
    cache.nodes([len(text)])
    h = dec.embed.index_select(0, torch.tensor(text, device="cuda")).unsqueeze(0)
    for layer in dec.layers:
        h = layer.forward([h, None, cache.next_positions(len(text), "cuda")], cache)[0]
    from tpp_pytorch_extension import _ops
    return _ops.fc_plain(F.rms_norm(h[0].contiguous(), dec.norm_w, dec.eps), dec.lm_head, None).float()


def _is_greedy(dec, F, prompt, new):
    """Every new token has the largest logit, but for roundings: of this pass and of the one that chose it, in some 8 places each that are
    rounded to bf16 (stream, norms, projections, attention, MLP, of two layers; the logits), 2^-8 of the value at most: 16 of those."""
    logits = _logits(dec, F, prompt + new[:-1])[len(prompt) - 1:]
    chosen = logits.gather(1, torch.tensor(new, device="cuda")[:, None])[:, 0]
    return bool((chosen >= logits.amax(1) - 16 * 2.0 ** -8 * logits.abs().amax(1)).all())


def _prompts(lengths, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 1024, (n,), generator=g).cuda() for n in lengths]


def test_generation_over_pages():
    F, dec = _decoder(qk_norm=True)
    prompts = _prompts([17, 3, 40])
    out = dec.generate_packed(prompts, 12)
    assert torch.equal(out, dec.generate_packed(prompts, 12, use_graph=False))  # (the same kernels, replayed)
    for p, o in zip(prompts, out):
        assert _is_greedy(dec, F, p.tolist(), o.tolist())
    even = torch.stack(_prompts([20, 20], 1))
    out = dec.generate(even, 9)
    assert torch.equal(out, dec.generate(even, 9, use_graph=False))
    for p, o in zip(even, out):
        assert _is_greedy(dec, F, p.tolist(), o.tolist())
    one = dec.generate(even[:1], 9)  # (a single counter: the greedy launch moves it)
    assert _is_greedy(dec, F, even[0].tolist(), one[0].tolist())


def test_generation_with_drafts_is_greedy():
    F, dec = _decoder()
    prompts = _prompts([17, 3, 40], 2)
    n_new = 20
    known = [p.tolist() + o.tolist() for p, o in zip(prompts, dec.generate_packed(prompts, n_new + 8))]

    def right(text):
        """The continuation that is known, as one branch of a tree."""
        for k in known:
            if k[:len(text)] == text:
                true = k[len(text):len(text) + 4]
                return [5, 6] + true, [-1, 0] + [-1] + list(range(2, 1 + len(true)))
        return [], []

    for propose in (right, None, lambda t: ([9, 8, 7], [-1, -1, 1]), lambda t: ([], [])):
        out, passes = dec.generate_drafted(prompts, n_new, propose)
        for p, o in zip(prompts, out):
            assert o.numel() == n_new and _is_greedy(dec, F, p.tolist(), o.tolist())
        assert passes <= n_new if propose is not right else passes < n_new


def test_generation_with_drafts_samples():
    F, dec = _decoder()
    prompts = _prompts([5, 30], 3)
    runs = []
    for seed in (1, 1, 2):
        g = torch.Generator(device="cuda").manual_seed(seed)
        runs.append(dec.generate_drafted(prompts, 15, lambda t: ([t[-1], 3, 4], [-1, -1, 0]), temperature=0.9, generator=g)[0])
    assert all(o.numel() == 15 and int(o.min()) >= 0 and int(o.max()) < 1024 for r in runs for o in r)
    assert all(torch.equal(a, b) for a, b in zip(runs[0], runs[1]))
    assert not all(torch.equal(a, b) for a, b in zip(runs[0], runs[2]))


def test_pages_go_back_to_the_pool():
    """A sequence that is done makes room for another one, whose results do not depend on what the pages held."""
    F, dec = _decoder()
    a, b, c = (p.tolist() for p in _prompts([40, 70, 60], 4))
    cache = F.PagedCache(128, dec.n_layers, page=16, pages=9)

    def read(texts):
        cache.nodes([len(t) for t in texts])
        flat = torch.tensor([x for t in texts for x in t], device="cuda")
        h = dec.embed.index_select(0, flat).unsqueeze(0)
        for layer in dec.layers:
            h = layer.forward([h, None, cache.next_positions(flat.numel(), "cuda")], cache)[0]
        cache.advance()
        return h[0]

    first = read([a, b])
    with pytest.raises(Exception, match="free"):
        cache.nodes([60, 0])
    cache.release(1)
    assert cache.lengths == cache.seq_len_dev.tolist() == [40, 0] and len(cache._free) == 6
    again = read([[], c])
    cache.release(1)
    cache.storage.fill_(float("nan"))  # (what a page held before)
    cache.release(0)
    assert torch.equal(read([[], c]), again)
    cache.release(1)
    assert torch.equal(read([a, b]), first)


def test_a_decoder_without_pages_refuses_drafts():
    F = _llm()
    dec = F.LlamaDecoder(hidden=256, inter=512, n_layers=1, n_heads=2, n_kv_heads=2, vocab=512, max_positions=64, seed=1)
    for call in (lambda: dec.generate_drafted(_prompts([3]), 4), lambda: dec.generate_packed(_prompts([3]), 4)):
        with pytest.raises(F.TppxError):
            call()


def test_drafted_tokens_outside_of_the_vocabulary():
    F, dec = _decoder()
    for bad in (-1, 1 << 20):
        with pytest.raises(F.TppxError, match="vocabulary"):
            dec.generate_drafted(_prompts([5], 6), 4, lambda t: ([3, bad], [-1, 0]))
    assert dec.generate_drafted(_prompts([5], 6), 4)[0][0].numel() == 4
