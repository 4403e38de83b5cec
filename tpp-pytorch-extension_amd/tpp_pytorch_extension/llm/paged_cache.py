"""Keys and values in pages, and passes that check drafted tokens over them.

The reference keeps one block of keys per batch (`TppCache` / `LayerCache`, src/csrc/llm/attn.h:164-404) and decodes one token a
step; the operators here stand beside its `attn` (src/csrc/llm/attn.cpp:957-1043), its rotary embeddings
(src/csrc/llm/fused_llm_infer.cpp:150-253) and the argmax of its generation loop.

A layer of the cache is bf16 `[2][pages][Nkv][page][H]`, keys then values; slot s of sequence b lies in page `table[b][s // page]`
(int32 `[B][pages of a sequence]`, device) at `s % page`.  Entries outside of 0 .. pages - 1 are no pages.  Head sizes 64, 96, 128, 192
and 256, pages of a power of two of slots from 16 to 65536.

The tokens of a step are nodes, packed: sequence b owns rows `cu_seqlens[b] .. cu_seqlens[b + 1] - 1` (int32 `[B + 1]`, device), or one
row each where `cu_seqlens` is None, and held `past[b]` keys before them (int32 `[B]`, device; negative: the sequence takes no
part).  Node i has slot past[b] + i.  Node 0 is the token accepted last, the others are drafted: `parents` (int32 `[T]`, device) is
the number within its sequence of the node that a node continues, smaller than its own (anything else: none).  Without parents every
node continues the one before it: drafted chains, pieces of prompts, single tokens.  Rows behind the last sequence take no part:
the cache is left as it was, and the results hold whatever `torch.empty` gave there.

A step: `append_paged` and `attn_paged` in every layer, `verify_drafts` on the logits, `keep_paged` once for all layers, and `past`
moves on by the counts.
"""
import torch

from .. import _lib
from .._lib import TppxError
from .mx4_cache import BF16, F32, HEAD_SIZES, I32, I64, _index, _norm_weights, _rotation, _rows, _run, _sequences  # noqa: F401

LOGITS = {torch.float32: _lib.DT_F32, torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16}


def _pages(layer, table, Nkv, H, B, dev, dims=5):
    """(address, pages, slots of a page, address of the table, pages of a sequence) of a cache layer, checked; Nkv, H None: its own."""
    shape = layer.shape
    if (len(shape) != dims or shape[-5] != 2 or (Nkv is not None and (shape[-3] != Nkv or shape[-1] != H)) or layer.dtype is not BF16
            or layer.get_device() != dev or not layer.is_contiguous()):
        raise TppxError(_lib.ESHAPE, f"a cache layer is a contiguous bfloat16 tensor [2][pages][{Nkv or 'Nkv'}][page][{H or 'H'}] on cuda:{dev}"
                                     f"{', a cache one of them per layer' if dims == 6 else ''}, got {tuple(shape)} {layer.dtype} on {layer.device}")
    if table.dtype is not I32 or table.dim() != 2 or table.shape[0] != B or table.get_device() != dev or not table.is_contiguous():
        raise TppxError(_lib.EINVAL, f"table must be a contiguous int32 tensor [{B}][pages of a sequence] on cuda:{dev}, got "
                                     f"{tuple(table.shape)} {table.dtype} on {table.device}")
    return layer.data_ptr(), shape[-4], shape[-2], table.data_ptr(), table.shape[1]


def append_paged(q, k, v, layer, table, past, cu_seqlens=None, parents=None, q_weight=None, k_weight=None, eps=1e-6, emb_pos=None,
                 pos=None, style="llama"):
    """RMSNorm of every head of q [T][Nq][H] and k [T][Nkv][H] with weights [H] (None: no norm) and the rotation by `emb_pos` at
    `pos` (int64 [T]; None: past plus the number of nodes that a node continues); keys and values v [T][Nkv][H] go to their slots of
    `layer` (a slot without a page is dropped); `past` itself stays.  fp32 inside, rounded once.  q may be None.  Returns the
    queries [T][Nq][H]."""
    k, dev, T, Nkv, H, k_ld, k_at = _rows(k, "k")
    v, _, Tv, Nv, Hv, v_ld, v_at = _rows(v, "v", dev)
    if Tv != T or Nv != Nkv or Hv != H:
        raise TppxError(_lib.ESHAPE, f"append_paged: k {tuple(k.shape)} and v {tuple(v.shape)}")
    Nq = q_ld = 0
    q_at = out = out_at = None
    if q is not None:
        q, _, Tq, Nq, Hq, q_ld, q_at = _rows(q, "q", dev)
        if Tq != T or Hq != H:
            raise TppxError(_lib.ESHAPE, f"append_paged: q {tuple(q.shape)} and k {tuple(k.shape)}")
        out = k.new_empty(T, Nq, H)
        out_at = out.data_ptr()
    B, past_at, cu_at = _sequences(T, past, cu_seqlens, dev)
    at, pages, page, table_at, table_ld = _pages(layer, table, Nkv, H, B, dev)
    gq, gk, gdt = _norm_weights(q_weight, k_weight, H, dev)
    angles, gptj, MP, HR = _rotation(emb_pos, style, H, dev)
    up = _index(parents, "parents", T, dev) if parents is not None else None
    pos_at = _index(pos, "pos", T, dev, I64) if pos is not None else None
    _run(dev, _lib.lib().tppx_append_paged, q_at, k_at, v_at, gq, gk, gdt, eps, angles, gptj, pos_at, at, table_at, past_at, cu_at, up, out_at,
         T, B, Nq, Nkv, H, pages, page, table_ld, q_ld, k_ld, v_ld, MP, HR)
    return out


def attn_paged(q, layer, table, past, cu_seqlens=None, parents=None):
    """Attention of nodes q [T][Nq][H] over a layer of the cache, after their own keys were appended: a node sees the slots before the
    step's, its own and those of the nodes that it continues.  One that sees nothing gets zeros.  Returns [T][Nq][H]."""
    q, dev, T, Nq, H, q_ld, q_at = _rows(q, "q")
    B, past_at, cu_at = _sequences(T, past, cu_seqlens, dev)
    Nkv = layer.shape[2] if layer.dim() == 5 else 0
    at, pages, page, table_at, table_ld = _pages(layer, table, Nkv, H, B, dev)
    up = _index(parents, "parents", T, dev) if parents is not None else None
    out = q.new_empty(T, Nq, H)
    # Single tokens merge their parts in the launch itself, by counters that only the shared workspace has.  Two parts of 128 columns for
    # every workgroup that can run, 66 KB each, do not fit in there.
    ws = _lib.workspace(q, own=cu_at is not None) if T * Nq * H < 1 << 20 or cu_at is None else torch.empty(72 << 20, dtype=torch.uint8, device=q.device)
    _run(dev, _lib.lib().tppx_attn_paged, q_at, at, table_at, past_at, cu_at, up, out.data_ptr(), T, B, Nq, Nkv, H, pages, page, table_ld, q_ld,
         *(_lib.with_counters(ws) if cu_at is None else (ws.data_ptr(), ws.numel(), None, 0)))
    return out


def _logits(t, name, T, V, dtype, dev):
    """(tensor, address, elements from row to row) of logits [T][V]; other strides than those of rows are copied."""
    if t.dim() != 2 or t.shape[0] != T or (V is not None and t.shape[1] != V) or t.get_device() != dev or t.dtype is not dtype:
        raise TppxError(_lib.EINVAL, f"{name} must be logits [{T}][{V or 'vocabulary'}] of {dtype} on cuda:{dev}, got "
                                     f"{tuple(t.shape)} {t.dtype} on {t.device}")
    a, b = t.stride()
    if (b != 1 and t.shape[1] != 1) or (a < t.shape[1] and T != 1):
        t = t.contiguous()
        a = t.shape[1]
    return t, t.data_ptr(), max(a, t.shape[1])


def verify_drafts(tokens, target, cu_seqlens=None, parents=None, draft=None, uniforms=None, sample=None, temperature=1.0):
    """Which drafted nodes stand against the target's probabilities, and the token behind them.

    tokens: int64 [T], the nodes'; target: logits [T][V] (float32, bfloat16, float16), row i what the target says behind node i; draft:
    for chains (no parents), the logits that the node behind each was drawn from, of the same type, or None for candidates that were
    chosen, not drawn.  p = softmax(target / temperature); temperature: a number, or float32 [B] on the device; 0: the first
    maximal logit alone.  From node 0 on a node's children are tried in order: candidate x stands where uniforms * M < p(x), M
    being 1 less the p of the siblings before it; drawn x where uniforms * q(x) < p(x), q = softmax(draft / temperature).  Where none
    stands the next token is drawn by sample from what is left: p without the children, max(p - q, 0), p itself behind a leaf
    (the first token whose cumulative sum exceeds sample times all).  uniforms: float32 [T], sample: float32 [B], in [0, 1); not needed at
    a temperature 0 that is a number.  fp64 inside.  A NaN logit counts as -inf, infinite ones share their row, a token outside of the
    vocabulary never stands.

    Returns (path int32 [T]: of every sequence the numbers of the nodes that stand, node 0 first, then -1; count int32 [B]: how many;
    next int64 [B]).  A sequence without nodes has count 0 and next 0."""
    _lib.require_gpu(target, "target")
    dev, T, V = target.get_device(), *(target.shape if target.dim() == 2 else (0, 0))
    code = LOGITS.get(target.dtype)
    if code is None or V == 0:
        raise TppxError(_lib.EINVAL, f"verify_drafts: target must be logits [tokens][vocabulary] in float32, bfloat16 or float16, got {tuple(target.shape)} {target.dtype}")
    target, t_at, t_ld = _logits(target, "target", T, V, target.dtype, dev)
    d_at, d_ld = None, 0
    if draft is not None:
        if parents is not None:
            raise TppxError(_lib.EUNSUPPORTED, "verify_drafts: draft logits are taken for chains, without parents")
        draft, d_at, d_ld = _logits(draft, "draft", T, V, target.dtype, dev)
    B = cu_seqlens.numel() - 1 if cu_seqlens is not None and cu_seqlens.dim() == 1 else T
    if B < 1:
        raise TppxError(_lib.ESHAPE, "verify_drafts: no sequences")
    cu = _index(cu_seqlens, "cu_seqlens", B + 1, dev) if cu_seqlens is not None else None
    tok = _index(tokens, "tokens", T, dev, I64)
    up = _index(parents, "parents", T, dev) if parents is not None else None
    temps, number = None, 0.0
    if isinstance(temperature, torch.Tensor):
        temps = _index(temperature, "temperature", B, dev, F32)
    else:
        number = float(temperature)
    u_at = s_at = None
    if temps is not None or number != 0.0:
        if uniforms is None or sample is None:
            raise TppxError(_lib.EINVAL, "verify_drafts: sampling needs uniforms and sample")
    if uniforms is not None:
        u_at = _index(uniforms, "uniforms", T, dev, F32)
    if sample is not None:
        s_at = _index(sample, "sample", B, dev, F32)
    path = tokens.new_empty(T, dtype=I32)
    count = tokens.new_empty(B, dtype=I32)
    following = tokens.new_empty(B)
    need = _lib.lib().tppx_verify_drafts_bytes(T, B, V, draft is not None)
    if need > _lib.WORKSPACE_BYTES:
        ws = torch.empty(need, dtype=torch.uint8, device=tokens.device)
        scratch = ws.data_ptr(), need, None, 0
    else:
        ws = _lib.workspace(target, own=True)
        # (a capture's own scratch has no counters, which replays of two graphs would share)
        scratch = (ws.data_ptr(), _lib.WORKSPACE_BYTES, None, 0) if torch._C._cuda_isCurrentStreamCapturing() else _lib.with_counters(ws)
    _run(dev, _lib.lib().tppx_verify_drafts, tok, t_at, d_at, code, cu, up, u_at, s_at, temps, number, path.data_ptr(), count.data_ptr(),
         following.data_ptr(), T, B, V, t_ld, d_ld, *scratch)
    return path, count, following


def keep_paged(cache, table, past, path, count, cu_seqlens=None):
    """Moves the keys and values of accepted paths to the slots from past on, in place, in all layers of `cache`
    (`[layers][2][pages][Nkv][page][H]`, or a single layer): for i < count[b] node path[cu[b] + i] goes to slot past[b] + i.  `path` and
    `count` as `verify_drafts` returns them (ascending nodes); `past` itself stays."""
    _lib.require_gpu(cache, "cache")
    dev, T = cache.get_device(), path.numel()
    whole = cache if cache.dim() != 5 else cache.unsqueeze(0)
    B, past_at, cu_at = _sequences(T, past, cu_seqlens, dev)
    at, pages, page, table_at, table_ld = _pages(whole, table, None, None, B, dev, 6)
    _run(dev, _lib.lib().tppx_keep_paged, at, table_at, past_at, _index(path, "path", T, dev), _index(count, "count", B, dev), cu_at,
         whole.shape[0], T, B, whole.shape[3], whole.shape[5], pages, page, table_ld)


def lookup_drafts(tokens, most=8, longest=3):
    """Drafts from the text itself: what followed the last earlier occurrence of its last `longest` (or fewer) tokens, at most `most`
    of them, as a chain (tokens, parents)."""
    for n in range(min(longest, len(tokens) - 1), 0, -1):
        tail = tokens[-n:]
        for at in range(len(tokens) - n - 1, -1, -1):
            if tokens[at:at + n] == tail:
                found = tokens[at + n:at + n + most]
                return found, list(range(-1, len(found) - 1))
    return [], []
