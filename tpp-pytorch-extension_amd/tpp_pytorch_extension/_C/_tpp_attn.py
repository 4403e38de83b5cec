"""Reference: REGISTER_SUBMODULE(_tpp_attn, m) (src/csrc/llm/attn.cpp:1955-1969): the KV cache class and the
attention entry point over it.  Beside them, without a counterpart there: the operators of an MXFP4 cache for sequences of
different lengths and of packed prompts, and those of a cache in pages and of drafted tokens checked over it."""
from ..llm.fused_llama_infer import Mx4Cache, PagedCache, TppCache, attn, kv_cache  # noqa: F401
from ..llm.mx4_cache import Mx4Layer, append_mx4, attn_mx4, attn_packed, qk_norm_rotary, read_mx4  # noqa: F401
from ..llm.paged_cache import append_paged, attn_paged, keep_paged, verify_drafts  # noqa: F401
