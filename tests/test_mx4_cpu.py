"""What the operators of the MXFP4 cache and of packed prompts refuse, before anything is launched, and their 64-bit plain
forms against known values."""
import math

import pytest
import torch

import mx4_ref as R


def _mods():
    import tpp_pytorch_extension  # noqa: F401
    from tpp_pytorch_extension import _lib
    from tpp_pytorch_extension._C import _tpp_attn
    return _lib, _lib.lib(), _tpp_attn


A = 1 << 20  # a fake, aligned "device pointer": refused before it is touched


def test_c_refusals():
    _lib, L, _ = _mods()

    def rotary(q=A, k=A, gq=A, gk=A, gdt=0, emb=A, pos=A, qo=A, ko=A, T=3, Nq=4, Nkv=2, H=128, q_ld=512, k_ld=256, MP=10, HR=128):
        return L.tppx_qk_norm_rotary(q, k, gq, gk, gdt, 1e-6, emb, 0, pos, qo, ko, T, Nq, Nkv, H, q_ld, k_ld, MP, HR, None)

    assert rotary(q=None) == rotary(k=None) == rotary(qo=None) == rotary(ko=None) == rotary(pos=None) == _lib.EINVAL
    assert rotary(q=A + 8) == rotary(gk=A + 4) == rotary(emb=A + 4) == rotary(gdt=2) == _lib.EINVAL
    assert rotary(H=80) == rotary(H=32) == rotary(H=512) == _lib.EUNSUPPORTED
    assert rotary(HR=24) == rotary(HR=144) == rotary(MP=0) == rotary(q_ld=504) == rotary(k_ld=260) == rotary(T=-1) == rotary(Nkv=0) == _lib.ESHAPE
    assert rotary(T=0) == _lib.OK

    def append(q=A, k=A, v=A, kc=A, ks=A, vc=A, vs=A, past=A, cu=A, qo=A, ko=A, vo=A, T=3, B=2, Nkv=2, H=128, Smax=9, v_ld=256):
        return L.tppx_append_mx4(q, k, v, None, None, 0, 1e-6, None, 0, None, kc, ks, vc, vs, past, cu, qo, ko, vo, T, B, 4, Nkv, H, Smax,
                                 512, 256, v_ld, 0, 0, None)

    for name in ("k", "v", "kc", "ks", "vc", "vs", "past", "qo"):
        assert append(**{name: None}) == _lib.EINVAL
    assert append(kc=A + 8) == append(vo=A + 2) == _lib.EINVAL
    assert append(H=48) == _lib.EUNSUPPORTED
    assert append(cu=None) == append(Smax=0) == append(B=0) == append(v_ld=128) == append(Nkv=-1) == _lib.ESHAPE
    assert append(T=0) == append(T=0, q=None, qo=None) == _lib.OK

    def attn(q=A, kc=A, vs=A, past=A, cu=A, mask=None, mask_ld=0, out=A, T=3, B=2, Nq=4, Nkv=2, H=128, Smax=9, q_ld=512, ws=None, wb=0, ct=None, cb=0):
        return L.tppx_attn_mx4(q, kc, A, A, vs, past, cu, mask, mask_ld, out, T, B, Nq, Nkv, H, Smax, q_ld, ws, wb, ct, cb, None)

    for name in ("q", "kc", "vs", "past", "out"):
        assert attn(**{name: None}) == _lib.EINVAL
    assert attn(q=A + 4) == attn(vs=A + 2) == attn(mask=A) == attn(wb=64) == attn(cb=64) == attn(ct=A + 1, cb=64) == _lib.EINVAL
    assert attn(H=160) == _lib.EUNSUPPORTED
    assert attn(Nq=5) == attn(Smax=1 << 30) == attn(cu=None) == attn(q_ld=500) == attn(B=0) == attn(T=-1) == _lib.ESHAPE
    assert attn(T=0) == _lib.OK

    def packed(q=A, k=A, v=A, cu=A, out=A, T=3, B=2, Nq=4, Nkv=2, H=128, k_ld=256, v_ld=256):
        return L.tppx_attn_packed(q, k, v, cu, None, 0, out, T, B, Nq, Nkv, H, 512, k_ld, v_ld, None)

    for name in ("q", "k", "v", "cu", "out"):
        assert packed(**{name: None}) == _lib.EINVAL
    assert packed(k=A + 8) == _lib.EINVAL and packed(H=100) == _lib.EUNSUPPORTED
    assert packed(Nq=3) == packed(k_ld=250) == packed(v_ld=100) == packed(T=1 << 31) == _lib.ESHAPE
    assert packed(T=0) == _lib.OK


def test_python_refuses_tensors_off_the_gpu():
    _lib, _, at = _mods()
    q, k = torch.zeros((3, 4, 128), dtype=torch.bfloat16), torch.zeros((3, 2, 128), dtype=torch.bfloat16)
    i = torch.zeros(3, dtype=torch.int32)
    layer = at.Mx4Layer(*(torch.zeros((3, 2, 8, w), dtype=torch.uint8) for w in (64, 4, 64, 4)))
    for call in (lambda: at.qk_norm_rotary(q, k), lambda: at.append_mx4(q, k, k, layer, i), lambda: at.attn_mx4(q, layer, i),
                 lambda: at.attn_packed(q, k, k, i)):
        with pytest.raises(_lib.TppxError) as e:
            call()
        assert e.value.code == _lib.EINVAL


def test_plain_forms():
    grid = torch.tensor([0.0, 0.25, 0.26, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9, -0.25, -0.75, -3.49, 4.0, 6.0, -6.0] * 2)
    codes, scales = R.encode(grid)
    assert scales.tolist() == [127]
    want = torch.tensor([0.0, 0.0, 0.5, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0, 0.0, -1.0, -3.0, 4.0, 6.0, -6.0] * 2).double()
    assert torch.equal(R.decode(codes, scales), want)
    _, s = R.encode(torch.tensor([[2.0 ** -125] * 32, [2.0 ** -124] * 32, [3.0e38] * 32, [math.inf] * 32]))
    assert s[:, 0].tolist() == [0, 1, 252, 255]
    # a rotation keeps the length of its pairs; equal keys give the mean of the values
    x = R.randn((2, 1, 64), 1.0, 1)
    for style, table in (("llama", R.llama_table(9, 32)), ("gptj", R.gptj_table(9, 32))):
        y, _ = R.turn(x, None, 0.0, table, torch.tensor([3, 8]), style)
        assert torch.allclose(y.norm(dim=-1), x.double().norm(dim=-1), rtol=1e-6)
        assert torch.equal(y[..., 32:], x[..., 32:].double())
    v = torch.randn((1, 5, 64), dtype=torch.float64)
    out, _ = R.attend(x, torch.zeros((1, 5, 64), dtype=torch.float64), v, 3)
    assert torch.allclose(out[:, 0], torch.stack((v[0, :4].mean(0), v[0].mean(0))))


def test_lengths_of_sequences_follow_a_reorder():
    """Host and device agree on every sequence's length after packed prompts, a beam reorder and a crop; appends of one length are
    refused while the lengths differ and taken once they do not."""
    from tpp_pytorch_extension.llm import fused_llama_infer as F
    cache = F.Mx4Cache(40)
    cache.prompts([9, 3, 5], "cpu")
    cache.advance()
    cache.reorder_cache(torch.tensor([1, 1, 2]))
    assert cache.seq_len_dev.tolist() == [3, 3, 5] and cache.get_seq_length() == 5
    with pytest.raises(F.TppxError):
        cache.update(torch.zeros(3, 1, 1, 64), torch.zeros(3, 1, 1, 64), 0)
    with pytest.raises(F.TppxError):
        cache.prompts([1, 1, 36], "cpu")
    cache.prompts([37, 0, 1], "cpu")
    cache.advance()
    assert cache.seq_len_dev.tolist() == [40, 3, 6] and cache.get_seq_length() == 40
    cache.crop(4)
    assert cache.seq_len_dev.tolist() == [4, 3, 4] and cache.get_seq_length() == 4
    cache.reorder_cache(torch.tensor([1, 1, 1]))
    assert cache.seq_len_dev.tolist() == [3, 3, 3] and cache.get_seq_length() == 3 and not any(cache._short)


def test_generate_packed_refuses_no_prompts():
    from tpp_pytorch_extension.llm import fused_llama_infer as F
    with pytest.raises(F.TppxError):
        F.LlamaDecoder.generate_packed(None, [], 3)


def test_positions_of_the_next_tokens():
    """One row for sequences of one length, a row each otherwise; a cache that was not used yet begins at 0."""
    from tpp_pytorch_extension.llm import fused_llama_infer as F
    for cache in (F.TppCache(40), F.Mx4Cache(40)):
        assert cache.positions(2, "cpu").tolist() == [[0], [0]]
        assert cache.next_positions(3, "cpu").tolist() == [[0, 1, 2]]
    cache = F.Mx4Cache(40)
    cache.prompts([9, 3], "cpu")
    cache.advance()
    assert cache.positions(2, "cpu").tolist() == [[9], [3]]
    assert cache.next_positions(3, "cpu").tolist() == [[9, 10, 11], [3, 4, 5]]
    cache.crop(3)
    assert cache.next_positions(2, "cpu").tolist() == [[3, 4]]
    with pytest.raises(F.TppxError):
        cache.positions(3, "cpu")


def test_positions_of_packed_tokens():
    from tpp_pytorch_extension.llm import fused_llama_infer as F
    cache = F.Mx4Cache(40)
    cache.prompts([3, 0, 2], "cpu")
    assert cache.next_positions(5, "cpu").tolist() == [[0, 1, 2, 0, 1]]
    cache.advance()
    cache.prompts([1, 2, 1], "cpu")
    assert cache.next_positions(4, "cpu").tolist() == [[3, 0, 1, 2]]


def test_positions_of_every_token():
    from tpp_pytorch_extension.llm.fused_llama_infer import _token_positions
    one, row = torch.tensor([[7]]), torch.tensor([[3, 4]])
    for pos, T, S, want in ((one, 3, 1, [7, 7, 7]), (one.expand(3, 1), 3, 1, [7, 7, 7]), (row, 4, 2, [3, 4, 3, 4]), (row, 2, 2, [3, 4]),
                            (torch.tensor([[1, 2], [5, 6]]), 4, 2, [1, 2, 5, 6])):
        got = _token_positions(pos, T, S)
        assert got.is_contiguous() and got.stride() == (1,) and got.tolist() == want


def test_bounds_of_sequences_of_one_length():
    from tpp_pytorch_extension.llm import fused_llama_infer as F
    cache = F.Mx4Cache(8)
    for B, S in ((3, 0), (1, 1), (2, 5)):
        b = cache._bounds_of(B, S, "cpu")
        assert b.dtype == torch.int32 and b.tolist() == [S * i for i in range(B + 1)]


def test_few_bounds_are_kept():
    """The last ones that were asked for: a prompt of every length leaves no tensor each."""
    from tpp_pytorch_extension.llm import fused_llama_infer as F
    cache = F.Mx4Cache(8)
    first = cache._bounds_of(2, 1, "cpu")
    for S in range(2, 40):
        cache._bounds_of(2, S, "cpu")
        assert cache._bounds_of(2, 1, "cpu") is first
    assert len(cache._bounds) <= cache.KEPT_BOUNDS and cache._bounds_of(2, 39, "cpu").tolist() == [0, 39, 78]


def test_an_announced_pass_over_packed_prompts():
    """Other passes, appends and reorders are refused until it ends or is dropped; a crop and new contents drop it."""
    from tpp_pytorch_extension.llm import fused_llama_infer as F
    cache = F.Mx4Cache(40)
    pos = torch.zeros((1, 3), dtype=torch.int64)

    def announce(lengths):
        cache.prompts(lengths, "cpu")

    def refused(call):
        with pytest.raises(F.TppxError):
            call()
        assert cache._packed is not None

    announce([4, 2])
    refused(lambda: F.check_layer_inputs("block", torch.zeros((2, 3, 8)), pos, cache))  # as many tokens, another shape
    refused(lambda: F.check_layer_inputs("block", torch.zeros((2, 1, 8)), pos[:, :1], cache))
    refused(lambda: cache.rotate_append_attend(None, None, None, None, None, 0, 2, 3, 2, 1, 64, None, None))
    refused(lambda: cache.rotate_append_attend(None, None, None, None, None, 0, 2, 6, 2, 1, 64, None, None))
    refused(lambda: cache.advance(1))
    refused(lambda: cache.advance(100))
    refused(lambda: cache.reorder_cache(torch.tensor([0, 0])))
    refused(lambda: cache.update(torch.zeros(2, 1, 1, 64), torch.zeros(2, 1, 1, 64), 0))
    assert cache.room_for(6) and cache.seq_len_dev.tolist() == [0, 0] and cache.get_seq_length() == 0
    cache.advance(6)
    assert cache.seq_len_dev.tolist() == [4, 2] and cache._packed is None
    announce([1, 36])
    cache.cancel_prompts()
    assert cache.seq_len_dev.tolist() == [4, 2] and cache.room_for(36) and not cache.room_for(37)
    cache.advance()
    cache.advance(2)
    assert cache.seq_len_dev.tolist() == [7, 5]
    announce([1, 1])
    cache.crop(6)
    assert cache._packed is None and cache.seq_len_dev.tolist() == [6, 5]
    cache.reorder_cache(torch.tensor([1, 1]))
    cache.advance(1)
    assert cache.seq_len_dev.tolist() == [6, 6]


def test_generate_packed_refuses_a_decoder_on_the_bf16_cache():
    from types import SimpleNamespace
    from tpp_pytorch_extension.llm import fused_llama_infer as F
    with pytest.raises(F.TppxError) as e:
        F.LlamaDecoder.generate_packed(SimpleNamespace(kv_dtype="bfloat16"), [torch.tensor([1, 2])], 3)
    assert e.value.code == F._lib.EINVAL and "kv_dtype" in str(e.value)
