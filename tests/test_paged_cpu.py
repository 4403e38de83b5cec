"""What the paged cache's operators and the check of drafted tokens refuse, before anything is launched, and their plain forms
against known values."""
import pytest
import torch

import paged_ref as R


def _mods():
    import tpp_pytorch_extension  # noqa: F401
    from tpp_pytorch_extension import _lib
    from tpp_pytorch_extension._C import _tpp_attn
    return _lib, _lib.lib(), _tpp_attn


A = 1 << 20  # a fake, aligned "device pointer": refused before it is touched


def test_c_refusals():
    _lib, L, _ = _mods()

    def append(q=A, k=A, v=A, gq=A, gdt=0, emb=A, pos=A, layer=A, table=A, past=A, cu=A, parents=A, out=A, T=3, B=2, Nq=4, Nkv=2, H=128, P=5, page=16,
               ld=3, q_ld=512, k_ld=256, v_ld=256, MP=10, HR=128):
        return L.tppx_append_paged(q, k, v, gq, None, gdt, 1e-6, emb, 0, pos, layer, table, past, cu, parents, out, T, B, Nq, Nkv, H, P, page, ld,
                                   q_ld, k_ld, v_ld, MP, HR, None)

    for name in ("k", "v", "layer", "table", "past", "out"):
        assert append(**{name: None}) == _lib.EINVAL
    assert append(k=A + 8) == append(layer=A + 8) == append(emb=A + 4) == append(table=A + 2) == append(cu=A + 1) == append(parents=A + 2) == _lib.EINVAL
    assert append(pos=A + 4) == append(gdt=2) == _lib.EINVAL
    assert append(H=80) == append(page=24) == append(page=8) == append(page=0) == append(page=1 << 17) == _lib.EUNSUPPORTED
    assert append(cu=None) == append(T=-1) == append(B=0) == append(Nkv=0) == append(Nq=0) == append(P=0) == append(ld=0) == append(ld=1 << 27) == _lib.ESHAPE
    assert append(HR=24) == append(HR=144) == append(MP=0) == append(q_ld=504) == append(k_ld=260) == append(v_ld=128) == _lib.ESHAPE
    assert append(T=0) == append(T=0, q=None, out=None) == _lib.OK

    def attn(q=A, layer=A, table=A, past=A, cu=A, parents=None, out=A, T=3, B=2, Nq=4, Nkv=2, H=128, P=5, page=16, ld=3, q_ld=512, ws=None, wb=0,
             ct=None, cb=0):
        return L.tppx_attn_paged(q, layer, table, past, cu, parents, out, T, B, Nq, Nkv, H, P, page, ld, q_ld, ws, wb, ct, cb, None)

    for name in ("q", "layer", "table", "past", "out"):
        assert attn(**{name: None}) == _lib.EINVAL
    assert attn(q=A + 4) == attn(layer=A + 2) == attn(out=A + 8) == attn(parents=A + 1) == attn(wb=64) == attn(cb=64) == attn(ct=A + 1, cb=64) == _lib.EINVAL
    assert attn(H=160) == attn(page=48) == _lib.EUNSUPPORTED
    assert attn(Nq=5) == attn(cu=None) == attn(q_ld=500) == attn(B=0) == attn(T=-1) == attn(T=1 << 30) == attn(P=1 << 31) == _lib.ESHAPE
    assert attn(T=0) == _lib.OK

    def verify(tok=A, target=A, draft=None, dt=1, cu=A, parents=None, u=A, s=A, temps=None, t=1.0, path=A, count=A, nxt=A, T=3, B=2, V=100, t_ld=100,
               d_ld=100, ws=A, wb=1 << 30, ct=None, cb=0):
        return L.tppx_verify_drafts(tok, target, draft, dt, cu, parents, u, s, temps, t, path, count, nxt, T, B, V, t_ld, d_ld, ws, wb, ct, cb, None)

    for name in ("tok", "target", "path", "count", "nxt", "u", "s"):
        assert verify(**{name: None}) == _lib.EINVAL
    assert verify(dt=3) == verify(tok=A + 4) == verify(target=A + 1) == verify(u=A + 2) == verify(cu=A + 2) == verify(nxt=A + 4) == _lib.EINVAL
    assert verify(t=-1.0) == verify(t=float("nan")) == verify(t=float("inf")) == verify(temps=A, u=None) == verify(ws=None) == verify(cb=64) == verify(ct=A + 2, cb=64) == _lib.EINVAL
    assert verify(draft=A, parents=A) == _lib.EUNSUPPORTED
    assert verify(V=0) == verify(B=0) == verify(T=-1) == verify(cu=None) == verify(t_ld=99) == verify(draft=A, d_ld=99) == _lib.ESHAPE

    def keep(cache=A, table=A, past=A, path=A, count=A, cu=A, layers=2, T=3, B=2, Nkv=2, H=128, P=5, page=16, ld=3):
        return L.tppx_keep_paged(cache, table, past, path, count, cu, layers, T, B, Nkv, H, P, page, ld, None)

    for name in ("cache", "table", "past", "path", "count"):
        assert keep(**{name: None}) == _lib.EINVAL
    assert keep(cache=A + 8) == keep(path=A + 2) == keep(count=A + 1) == _lib.EINVAL
    assert keep(H=100) == keep(page=17) == _lib.EUNSUPPORTED
    assert keep(layers=0) == keep(cu=None) == keep(Nkv=1 << 16, layers=1 << 16) == keep(B=1 << 24) == _lib.ESHAPE
    assert keep(T=0) == _lib.OK


def test_python_refuses_tensors_off_the_gpu():
    _lib, _, at = _mods()
    q, k = torch.zeros((3, 4, 128), dtype=torch.bfloat16), torch.zeros((3, 2, 128), dtype=torch.bfloat16)
    i = torch.zeros(3, dtype=torch.int32)
    layer, table = torch.zeros((2, 4, 2, 16, 128), dtype=torch.bfloat16), torch.zeros((3, 2), dtype=torch.int32)
    for call in (lambda: at.append_paged(q, k, k, layer, table, i), lambda: at.attn_paged(q, layer, table, i),
                 lambda: at.verify_drafts(i.long(), torch.zeros((3, 9)), temperature=0.0), lambda: at.keep_paged(layer, table, i, i, i)):
        with pytest.raises(_lib.TppxError) as e:
            call()
        assert e.value.code == _lib.EINVAL


def test_plain_forms():
    assert R.ancestors([-1, 0, 0, 1, 9, -5]).tolist() == [[1, 0, 0, 0, 0, 0], [1, 1, 0, 0, 0, 0], [1, 0, 1, 0, 0, 0], [1, 1, 0, 1, 0, 0],
                                                          [0, 0, 0, 0, 1, 0], [0, 0, 0, 0, 0, 1]]
    assert R.depths([-1, 0, 0, 1]) == [0, 1, 1, 2]
    half = torch.tensor([[0.5, 0.25, 0.25], [0.2, 0.8, 0.0]], dtype=torch.float64).log()
    one = [0, 2]
    assert R.verify(one, None, half, None, [0.0, 0.2], 0.7, 1.0) == ([0, 1], 1)   # stands: then 0.7 of (0.2, 0.8)
    assert R.verify(one, None, half, None, [0.0, 0.3], 0.6, 1.0) == ([0], 0)      # not: 0.6 of what is left, (0.5, 0.25)
    assert R.verify(one, None, half, None, [0.0, 0.3], 0.7, 1.0) == ([0], 1)
    drawn = torch.tensor([[0.1, 0.1, 0.8], [0.3, 0.3, 0.4]], dtype=torch.float64).log()
    assert R.verify(one, None, half, drawn, [0.0, 0.3], 0.5, 1.0) == ([0, 1], 1)  # 0.3 * 0.8 < 0.25
    assert R.verify(one, None, half, drawn, [0.0, 0.4], 0.7, 1.0) == ([0], 0)     # left: (0.4, 0.15, 0)
    assert R.verify(one, None, half, drawn, [0.0, 0.4], 0.8, 1.0) == ([0], 1)
    assert R.verify(one, None, half, drawn, [0.0, 0.4], 0.8, 0.0) == ([0], 0)
    assert R.verify([0, 0], None, half, None, None, None, 0.0) == ([0, 1], 1)
    assert R.verify([0, 1, 2], [-1, 0, 0], half[[0, 1, 1]], None, [0.0, 0.3, 0.3], 0.1, 1.0) == ([0, 2], 0)  # 0.3 * 0.75 < 0.25


def test_lookup_drafts():
    from tpp_pytorch_extension.llm.paged_cache import lookup_drafts
    assert lookup_drafts([1, 2, 3, 4, 1, 2, 3]) == ([4, 1, 2, 3], [-1, 0, 1, 2])
    assert lookup_drafts([7, 1, 2, 9, 8, 7, 5, 1, 2], most=2) == ([9, 8], [-1, 0])
    assert lookup_drafts([1]) == lookup_drafts([5, 6, 7]) == lookup_drafts([]) == ([], [])


def test_pages_of_a_cache():
    """What a PagedCache keeps on the host: pages taken and given back, lengths, announced passes, refusals that change nothing."""
    _lib, _, at = _mods()
    cache = at.PagedCache(100, 2, page=16, pages=10)
    assert cache.get_capacity() == 112 and cache.get_seq_length() == 0 and cache.room_for(112) and not cache.room_for(113)
    bounds = cache.nodes([20, 0, 33], device="cpu")
    assert bounds.tolist() == [0, 20, 20, 53] and cache.next_positions(53, "cpu")[0].tolist() == list(range(20)) + list(range(33))
    assert (cache.table >= 0).sum(1).tolist() == [2, 0, 3] and len(set(cache.table[cache.table >= 0].tolist())) == 5
    assert cache.room_for(53)

    def refuses(call, code=_lib.ESHAPE):
        before = (list(cache.lengths), cache.table.clone(), len(cache._free))
        with pytest.raises(_lib.TppxError) as e:
            call()
        assert e.value.code == code
        assert cache.lengths == before[0] and torch.equal(cache.table, before[1]) and len(cache._free) == before[2]

    refuses(lambda: cache.room_for(7), _lib.EINVAL)
    refuses(lambda: cache.nodes([1, 1, 1], device="cpu"), _lib.EINVAL)
    refuses(lambda: cache.release(0), _lib.EINVAL)
    refuses(lambda: cache.advance(9), _lib.EINVAL)
    cache.advance(53)
    assert cache.lengths == cache.seq_len_dev.tolist() == [20, 0, 33] and cache.get_seq_length() == 33
    refuses(lambda: cache.nodes([3, 3], device="cpu"))
    refuses(lambda: cache.nodes([0, 0, 80], device="cpu"))      # past the capacity
    refuses(lambda: cache.nodes([60, 60, 0], device="cpu"))     # past the pool
    refuses(lambda: cache.nodes([1, -1, 0], device="cpu"))
    refuses(lambda: cache.nodes([1, 2, 0], [[-1], [-1], []], device="cpu"))
    refuses(lambda: cache.reorder_cache(torch.tensor([0, 1, 2])), _lib.EUNSUPPORTED)
    refuses(lambda: cache.keep(None, None), _lib.EINVAL)
    cache.nodes([4, 1, 3], [[-1, 0, 0, 2], [-1], [-1, 0, 0]], device="cpu")
    assert cache.next_positions(8, "cpu")[0].tolist() == [20, 21, 21, 22, 0, 33, 34, 34]
    refuses(lambda: cache.advance(), _lib.EINVAL)               # (a tree: which of its nodes?)
    path = torch.tensor([0, 2, 3, -1, 0, 0, 1, -1], dtype=torch.int32)
    assert cache.keep(path, torch.tensor([3, 1, 2], dtype=torch.int32)) == [3, 1, 2]  # (no layer has been written: nothing to move)
    assert cache.lengths == cache.seq_len_dev.tolist() == [23, 1, 35]
    cache.nodes([30, 0, 0], device="cpu")
    cache.cancel_nodes()
    assert cache.lengths == [23, 1, 35]
    cache.release(2)
    assert cache.lengths == cache.seq_len_dev.tolist() == [23, 1, 0] and (cache.table >= 0).sum(1).tolist() == [4, 1, 0]
    cache.crop(10)
    assert cache.lengths == cache.seq_len_dev.tolist() == [10, 1, 0] and (cache.table >= 0).sum(1).tolist() == [1, 1, 0] and len(cache._free) == 8
    cache.reserve(16)
    assert (cache.table >= 0).sum(1).tolist() == [2, 2, 1]
    with pytest.raises(_lib.TppxError):
        at.PagedCache(0, 2)
    with pytest.raises(_lib.TppxError):
        at.PagedCache(10, 0)
