"""Keys and values held in MXFP4, for sequences of different lengths, and attention of packed prompts.

The reference keeps its cache in bf16 or fp32 and one length for the whole batch (`TppCache` / `LayerCache`,
src/csrc/llm/attn.h:164-404); the operators here stand beside its `attn` (src/csrc/llm/attn.cpp:957-1043) and its rotary
embeddings (src/csrc/llm/fused_llm_infer.cpp:150-253).

Packed tokens are rows `[T][heads][H]`: sequence b owns rows `cu_seqlens[b] .. cu_seqlens[b + 1] - 1` (int32 `[B + 1]` on the
device), or one row each where `cu_seqlens` is None.  `past[b]` (int32 `[B]`, device) is the number of keys that a sequence
held before these tokens (negative: the first of them have no slot and see nothing).  Rows of a batch behind the last sequence
take no part: the cache is left as it was, and the results hold whatever `torch.empty` gave there.

A layer of the cache is `Mx4Layer(k_codes, k_scales, v_codes, v_scales)`, uint8 `[B][Nkv][capacity][H/2]` (two E2M1 codes a
byte, the even channel in the low half) and `[B][Nkv][capacity][H/32]` (E8M0).  Head sizes 64, 96, 128, 192 and 256.
"""
from collections import namedtuple

import torch

from .. import _lib
from .._lib import TppxError

Mx4Layer = namedtuple("Mx4Layer", "k_codes k_scales v_codes v_scales")

HEAD_SIZES = (64, 96, 128, 192, 256)

# (An eager call of a few tokens is host time: attributes are read once, and new tensors are asked for by their sizes one by one,
# 0.35 us less than by a tuple.)
BF16, F32, U8, I32, I64 = torch.bfloat16, torch.float32, torch.uint8, torch.int32, torch.int64


def _run(dev, fn, *args):
    """A call of the library on device number `dev` and its current stream (the last argument)."""
    if dev == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    if rc != _lib.OK:
        _lib.check(rc)


def _rows(t, name, dev=None):
    """Packed rows of heads: bf16 [T][heads][H] on the GPU (`dev`: on that one), heads of a row side by side; other strides are
    copied.  Returns (tensor, device number, T, heads, H, elements from row to row, address)."""
    if t.dtype is not BF16 or t.dim() != 3 or not t.is_cuda:
        raise TppxError(_lib.EINVAL, f"{name} must be a bfloat16 tensor [tokens][heads][head size] on the GPU, got "
                                     f"{tuple(t.shape)} {t.dtype} on {t.device}")
    at = t.get_device()
    if dev is not None and at != dev:
        raise TppxError(_lib.EINVAL, f"{name} is on {t.device}, not on cuda:{dev}")
    T, n, h = t.shape
    a, b, c = t.stride()
    ptr = t.data_ptr()
    if T == 1:
        a = n * h  # (of a single row the stride may be anything)
    if c != 1 or (b != h and n != 1) or a % 8 or a < n * h or ptr & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        a, ptr = n * h, t.data_ptr()
    return t, at, T, n, h, a, ptr


def _index(t, name, n, dev, dtype=I32):
    if t.dtype is not dtype or t.dim() != 1 or t.numel() != n or t.get_device() != dev or not t.is_contiguous():
        raise TppxError(_lib.EINVAL, f"{name} must be a contiguous {dtype} tensor [{n}] on cuda:{dev}, got "
                                     f"{tuple(t.shape)} {t.dtype} on {t.device}")
    return t.data_ptr()


def _norm_weight(w, name, H, dev, code):
    """(address, dtype number) of a per-head norm's weights; code: the dtype number of the other one, or None."""
    at = w.data_ptr()
    if w.dim() != 1 or w.numel() != H or w.get_device() != dev or not w.is_contiguous() or at & 15:
        raise TppxError(_lib.EINVAL, f"{name} must be a contiguous, 16-byte aligned tensor [{H}] on cuda:{dev}, got "
                                     f"{tuple(w.shape)} on {w.device}")
    kind = _lib.DT_F32 if w.dtype is F32 else _lib.DT_BF16 if w.dtype is BF16 else None
    if kind is None or (code is not None and kind != code):
        raise TppxError(_lib.EINVAL, f"{name}: norm weights are both float32 or both bfloat16, got {w.dtype}")
    return at, kind


def _norm_weights(q_weight, k_weight, H, dev):
    """(address, address, dtype number) of the per-head norms' weights; None: no norm."""
    gq = gk = code = None
    if q_weight is not None:
        gq, code = _norm_weight(q_weight, "q_weight", H, dev, None)
    if k_weight is not None:
        gk, code = _norm_weight(k_weight, "k_weight", H, dev, code)
    return gq, gk, _lib.DT_F32 if code is None else code


def _rotation(emb_pos, style, H, dev):
    """(address, gptj, positions, width) of a rotary table: float32 [2][MP][HR] cos / sin ("llama"; a row's first HR/2 entries serve
    both halves) or [MP][HR] sin | cos ("gptj")."""
    llama = style == "llama"
    if not llama and style not in ("gptj", None):
        raise TppxError(_lib.EINVAL, f"rotation style {style!r} (\"llama\", \"gptj\" or None)")
    if emb_pos is None or style is None:
        return None, 0, 0, 0
    shape = emb_pos.shape
    at = emb_pos.data_ptr()
    if (emb_pos.dtype is not F32 or emb_pos.get_device() != dev or not emb_pos.is_contiguous() or len(shape) != (3 if llama else 2)
            or (llama and shape[0] != 2) or at & 15):
        raise TppxError(_lib.EINVAL, f"emb_pos must be a contiguous float32 table {'[2][positions][width]' if llama else '[positions][width]'} "
                                     f"on cuda:{dev}, got {tuple(shape)} {emb_pos.dtype} on {emb_pos.device}")
    MP, HR = shape[-2:]
    if HR > H or HR % 16 or HR == 0 or MP == 0:
        raise TppxError(_lib.ESHAPE, f"rotary width {HR} must be a multiple of 16 and at most the head size {H}")
    return at, 0 if llama else 1, MP, HR


def qk_norm_rotary(q, k, q_weight=None, k_weight=None, eps=1e-6, emb_pos=None, pos=None, style="llama"):
    """RMSNorm of every head of q [T][Nq][H] and k [T][Nkv][H] with weights [H] (None: no norm), then the rotation by
    `emb_pos` at the positions `pos` (int64 [T]), in one pass; fp32 inside, rounded once.  Returns new (q, k).  The rotation alone, in
    place, is `apply_rotary_pos_emb_llama` / `_gptj`."""
    q, dev, T, Nq, H, q_ld, q_at = _rows(q, "q")
    k, _, Tk, Nkv, Hk, k_ld, k_at = _rows(k, "k", dev)
    if Tk != T or Hk != H:
        raise TppxError(_lib.ESHAPE, f"qk_norm_rotary: q {tuple(q.shape)} and k {tuple(k.shape)}")
    gq, gk, gdt = _norm_weights(q_weight, k_weight, H, dev)
    table, gptj, MP, HR = _rotation(emb_pos, style, H, dev)
    if table is not None and pos is None:
        raise TppxError(_lib.EINVAL, "qk_norm_rotary: a rotation needs the positions")
    at = _index(pos, "pos", T, dev, I64) if pos is not None else None
    qo = q.new_empty(T, Nq, H)
    ko = q.new_empty(T, Nkv, H)
    if T == 0:
        return qo, ko
    _run(dev, _lib.lib().tppx_qk_norm_rotary, q_at, k_at, gq, gk, gdt, eps, table, gptj, at, qo.data_ptr(), ko.data_ptr(),
         T, Nq, Nkv, H, q_ld, k_ld, MP, HR)
    return qo, ko


def _layer(layer, B, Nkv, H, dev):
    """Addresses and capacity of a cache layer, checked."""
    kc, ks, vc, vs = layer
    codes, scales = kc.shape, ks.shape
    cap = codes[2] if len(codes) == 4 else 0
    if (cap == 0 or codes != (B, Nkv, cap, H // 2) or vc.shape != codes or scales != (B, Nkv, cap, H // 32) or vs.shape != scales
            or kc.dtype is not U8 or vc.dtype is not U8 or ks.dtype is not U8 or vs.dtype is not U8
            or not (kc.is_contiguous() and vc.is_contiguous() and ks.is_contiguous() and vs.is_contiguous())
            or kc.get_device() != dev or vc.get_device() != dev or ks.get_device() != dev or vs.get_device() != dev):
        raise TppxError(_lib.ESHAPE, f"cache layer: contiguous uint8 tensors [{B}][{Nkv}][capacity][{H // 2}] (codes) and [{H // 32}] (scales) of "
                                     f"keys and values on cuda:{dev} are wanted, got {[(tuple(t.shape), t.dtype, t.device) for t in layer]}")
    return kc.data_ptr(), ks.data_ptr(), vc.data_ptr(), vs.data_ptr(), cap


def _sequences(T, past, cu_seqlens, dev):
    """(B, address of past, address of cu_seqlens)"""
    B = past.numel() if past.dim() == 1 else 0
    if B == 0:
        raise TppxError(_lib.ESHAPE, f"past must be int32 [sequences], got {tuple(past.shape)}")
    at = _index(past, "past", B, dev)
    if cu_seqlens is None:
        if T != B:
            raise TppxError(_lib.ESHAPE, f"{T} tokens of {B} sequences need cu_seqlens")
        return B, at, None
    return B, at, _index(cu_seqlens, "cu_seqlens", B + 1, dev)


def append_mx4(q, k, v, layer, past, cu_seqlens=None, q_weight=None, k_weight=None, eps=1e-6, emb_pos=None, pos=None, style="llama",
               values=False):
    """`qk_norm_rotary` of packed tokens with the append: the keys and the values v [T][Nkv][H] go to `layer` in MXFP4, at slots
    past[b], past[b] + 1, ... of their sequence (what does not fit its capacity is dropped); `past` itself stays.  pos None:
    the slots are the positions.  q may be None.  Returns (q, k, v): the queries, and with `values` the keys and values as the
    cache holds them, in bf16 (None otherwise): attention over those (`attn_packed`) is attention over the cache."""
    k, dev, T, Nkv, H, k_ld, k_at = _rows(k, "k")
    v, _, Tv, Nv, Hv, v_ld, v_at = _rows(v, "v", dev)
    if Tv != T or Nv != Nkv or Hv != H:
        raise TppxError(_lib.ESHAPE, f"append_mx4: k {tuple(k.shape)} and v {tuple(v.shape)}")
    Nq = q_ld = 0
    q_at = qo = qo_at = ko = ko_at = vo = vo_at = None
    if q is not None:
        q, _, Tq, Nq, Hq, q_ld, q_at = _rows(q, "q", dev)
        if Tq != T or Hq != H:
            raise TppxError(_lib.ESHAPE, f"append_mx4: q {tuple(q.shape)} and k {tuple(k.shape)}")
    B, past_at, cu_at = _sequences(T, past, cu_seqlens, dev)
    kc, ks, vc, vs, cap = _layer(layer, B, Nkv, H, dev)
    gq, gk, gdt = _norm_weights(q_weight, k_weight, H, dev)
    table, gptj, MP, HR = _rotation(emb_pos, style, H, dev)
    at = _index(pos, "pos", T, dev, I64) if pos is not None else None
    if q is not None:
        qo = k.new_empty(T, Nq, H)
        qo_at = qo.data_ptr()
    if values:
        ko, vo = k.new_empty(T, Nkv, H), k.new_empty(T, Nkv, H)
        ko_at, vo_at = ko.data_ptr(), vo.data_ptr()
    if T == 0:
        return qo, ko, vo
    _run(dev, _lib.lib().tppx_append_mx4, q_at, k_at, v_at, gq, gk, gdt, eps, table, gptj, at, kc, ks, vc, vs, past_at, cu_at,
         qo_at, ko_at, vo_at, T, B, Nq, Nkv, H, cap, q_ld, k_ld, v_ld, MP, HR)
    return qo, ko, vo


def check_mask(mask, B, dev):
    """(address, keys) of an additive mask, or (None, 0)."""
    if mask is None or mask.numel() == 0:
        return None, 0
    if mask.dim() != 2 or mask.shape[0] != B or mask.dtype is not BF16 or not mask.is_contiguous() or mask.get_device() != dev:
        raise TppxError(_lib.EINVAL, f"mask must be a contiguous bfloat16 tensor [{B}][keys] on cuda:{dev}, got "
                                     f"{tuple(mask.shape)} {mask.dtype} on {mask.device}")
    return mask.data_ptr(), mask.shape[1]


def attn_mx4(q, layer, past, cu_seqlens=None, mask=None):
    """Attention of packed tokens q [T][Nq][H] over a layer of the MXFP4 cache, after their own keys were appended: token i of
    sequence b sees the keys 0 .. past[b] + i.  mask: additive, bf16 [B][keys] (0 past its end; keys under -inf are not looked
    at).  A token that sees nothing gets zeros.  Returns [T][Nq][H]."""
    q, dev, T, Nq, H, q_ld, q_at = _rows(q, "q")
    B, past_at, cu_at = _sequences(T, past, cu_seqlens, dev)
    Nkv = layer[0].shape[1] if layer[0].dim() == 4 else 0
    kc, ks, vc, vs, cap = _layer(layer, B, Nkv, H, dev)
    m_at, m_ld = check_mask(mask, B, dev)
    out = q.new_empty(T, Nq, H)
    if T == 0:
        return out
    _run(dev, _lib.lib().tppx_attn_mx4, q_at, kc, ks, vc, vs, past_at, cu_at, m_at, m_ld, out.data_ptr(), T, B, Nq, Nkv, H, cap, q_ld,
         *_lib.with_counters(_lib.workspace(q)))
    return out


def attn_packed(q, k, v, cu_seqlens, mask=None):
    """Causal attention of packed prompts q [T][Nq][H] over their own k, v [T][Nkv][H] (bf16, query heads in groups of
    Nq / Nkv): token i of a sequence sees its tokens 0 .. i.  mask: additive, bf16 [B][tokens of a sequence].  Returns [T][Nq][H]."""
    q, dev, T, Nq, H, q_ld, q_at = _rows(q, "q")
    k, _, Tk, Nkv, Hk, k_ld, k_at = _rows(k, "k", dev)
    v, _, Tv, Nv, Hv, v_ld, v_at = _rows(v, "v", dev)
    if Tk != T or Tv != T or Hk != H or Hv != H or Nv != Nkv or Nkv == 0 or Nq % Nkv:
        raise TppxError(_lib.ESHAPE, f"attn_packed: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    B = cu_seqlens.numel() - 1 if cu_seqlens.dim() == 1 else 0
    if B < 1:
        raise TppxError(_lib.ESHAPE, f"cu_seqlens must be int32 [sequences + 1], got {tuple(cu_seqlens.shape)}")
    cu_at = _index(cu_seqlens, "cu_seqlens", B + 1, dev)
    m_at, m_ld = check_mask(mask, B, dev)
    out = q.new_empty(T, Nq, H)
    if T == 0:
        return out
    _run(dev, _lib.lib().tppx_attn_packed, q_at, k_at, v_at, cu_at, m_at, m_ld, out.data_ptr(), T, B, Nq, Nkv, H, q_ld, k_ld, v_ld)
    return out


def read_mx4(codes, scales):
    """What codes [..][H/2] and their scales [..][H/32] of a cache layer stand for, bf16 [..][H]."""
    _lib.require_gpu(codes, "cache codes")
    shape = codes.shape[:-1] + (codes.shape[-1] * 2,)
    codes, scales = codes.contiguous(), scales.to(codes.device).contiguous()
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or scales.shape != codes.shape[:-1] + (codes.shape[-1] // 16,):
        raise TppxError(_lib.ESHAPE, f"read_mx4: codes {tuple(codes.shape)} {codes.dtype} with scales {tuple(scales.shape)} {scales.dtype}")
    out = torch.empty(shape, dtype=torch.float32, device=codes.device)
    if out.numel():
        _run(codes.get_device(), _lib.lib().tppx_dequantize_per_block, codes.data_ptr(), scales.data_ptr(), _lib.Q_MXFP4, scales.numel(), 16, 1, 2, out.data_ptr())
    return out.to(torch.bfloat16)
