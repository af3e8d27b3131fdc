"""Python call surface: the reference's ``decoding_attn_fwd``
(decoding_attn/decoding_attn_interface.py:24-53) plus the two named entry points ``dmha_fwd`` /
``dmla_fwd`` with an explicit softmax scale.  Everything goes through the torch extension
``decoding_attn_cuda`` (csrc/torch_binding.cpp), i.e. the C++ binding over the C ABI.
"""
import os
import sys

import torch

_PKG = os.path.dirname(os.path.abspath(__file__))
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)
try:
    import decoding_attn_cuda  # noqa: E402  (built in-tree by decoding_attention_b200.build)
except ImportError as e:  # no fallback: fail loudly
    raise ImportError("the decoding_attn_cuda extension is not built: run "
                      "`python -m decoding_attention_b200.build`") from e


def maybe_contiguous(x):
    return x.contiguous() if x is not None and x.stride(-1) != 1 else x


def decoding_attn_fwd(q, k, v, cu_seq_k, max_seq_k, dim_v, is_alibi, *, softmax_scale=None):
    """Same arguments and result as the reference's ``decoding_attn_fwd``.

    q [total_q, head_q, dim]; k [total_k, head_k, dim] (MLA: the latent KV cache); v [total_k, head_k,
    dim_v] or None for MLA; cu_seq_k int32 [batch + 1]; returns o [total_q, head_q, dim_v].
    ``softmax_scale`` (keyword-only, an extension) defaults to the reference's 1/sqrt(dim).
    """
    q, k, v = [maybe_contiguous(x) for x in (q, k, v)]
    if softmax_scale is None:
        return decoding_attn_cuda.fwd(q, k, v, None, cu_seq_k, max_seq_k, dim_v, is_alibi)
    if v is None:
        return decoding_attn_cuda.dmla_fwd(q, k, cu_seq_k, max_seq_k, dim_v, is_alibi, softmax_scale)
    return decoding_attn_cuda.dmha_fwd(q, k, v, cu_seq_k, max_seq_k, is_alibi, softmax_scale)


def dmha_fwd(q, k, v, cu_seq_k, max_seq_k, is_alibi=False, softmax_scale=None, out=None, return_lse=False,
             k_scale=1.0, v_scale=1.0):
    """MHA / GQA / MQA decode attention; ``return_lse`` adds the fp32 natural-log LSE [batch, head_q].
    ``k`` / ``v`` may be an FP8 cache (torch.float8_e4m3fn) standing for ``k * k_scale`` / ``v * v_scale``."""
    q, k, v = [maybe_contiguous(x) for x in (q, k, v)]
    return decoding_attn_cuda.dmha_fwd(q, k, v, cu_seq_k, max_seq_k, is_alibi, softmax_scale, out, return_lse,
                                       k_scale, v_scale)


def dmla_fwd(q, kv, cu_seq_k, max_seq_k, dim_v=512, softmax_scale=None, out=None, return_lse=False, is_alibi=False):
    """MLA decode attention over the latent KV cache ``kv`` [total_k, 1, 576]; V = kv[..., :dim_v]."""
    q, kv = [maybe_contiguous(x) for x in (q, kv)]
    return decoding_attn_cuda.dmla_fwd(q, kv, cu_seq_k, max_seq_k, dim_v, is_alibi, softmax_scale, out, return_lse)


def paged_fwd(q, k_cache, v_cache, seq_lens, block_table, max_seq_k=None, dim_v=None, is_alibi=False, softmax_scale=None,
              out=None, return_lse=False):
    """Decode attention over a paged KV cache (the layout serving engines keep).

    q [batch, head_q, dim]; k_cache [num_pages, page_size, head_k, dim]; v_cache the same with dim_v, or
    None for the latent-KV (MLA) shape; seq_lens int32 [batch]; block_table int32 [batch, blocks]: key j
    of sequence b is row ``j % page_size`` of page ``block_table[b, j // page_size]``.  page_size must be a
    power of two >= 16.  The reference has no paged entry point; its Python benchmark builds such
    layouts for the libraries it compares against (benchmarks/python/benchmark_decoding_attn.py:182-190).
    """
    cu_seq_k = torch.zeros(seq_lens.numel() + 1, dtype=torch.int32, device=seq_lens.device)
    cu_seq_k[1:] = torch.cumsum(seq_lens, 0)
    if max_seq_k is None:
        max_seq_k = block_table.shape[1] * k_cache.shape[1]
    if dim_v is None:
        dim_v = v_cache.shape[-1] if v_cache is not None else 512
    return decoding_attn_cuda.paged_fwd(q, k_cache, v_cache, cu_seq_k, block_table, max_seq_k, dim_v, is_alibi,
                                        softmax_scale, out, return_lse)


def merge_partials(part_o, part_lse, out_dtype):
    """LSE merge of partial results over disjoint key ranges: part_o fp32 [parts, ..., dim_v]."""
    return decoding_attn_cuda.merge_partials(part_o.contiguous(), part_lse.contiguous(), out_dtype)


def kv_cache_write(k, v, k_cache, v_cache, k_scale, v_scale, slots=None):
    """Quantise the rows of new tokens into a cache of 8- or 4-bit codes, one fp32 scale per (token, KV head).

    k, v [tokens, head_k, dim], fp16 or bf16.  k_cache, v_cache: torch.float8_e4m3fn, torch.int8, or torch.uint8 for
    int4 (two codes a byte, the even element in the low nibble, last dimension dim / 2); packed [rows, head_k, dim] or
    paged [num_pages, page_size, head_k, dim]; dim 64, 96, 128 or 256.  k_scale, v_scale: float32 of that shape without
    the last dimension.  ``slots`` (int64 [tokens]) names each token's cache row, ``page * page_size + offset`` in a
    paged cache; a token whose slot is negative (padding) or past the cache is skipped, and two tokens of a call must
    not name the same row.  Without ``slots`` token i goes to row i.  Written in place.

    With a = max |x| of a row and Q = 448, 127 or 7: scale = a / Q, code = x * (Q / a) to the nearest, ties to even.
    A row whose a is below 2^-100 becomes zeros, a row with an infinity or a NaN reads back as NaN.
    k and v may be expanded over their tokens, like the inputs of the calls below (they are copied first); an ``out`` may not.
    The reference does not quantise its cache (README.md:154-156).
    """
    decoding_attn_cuda.kv_cache_write(k, v, k_cache, v_cache, k_scale, v_scale, slots)


def kv_cache_read(k_cache, v_cache, k_scale, v_scale, slots=None, dtype=torch.bfloat16, out=None):
    """The rows ``slots`` (int64 [tokens]; None: all of them, in order) of such a cache as (k, v) [tokens, head_k, dim].

    ``dtype``: torch.float16, torch.bfloat16 or torch.float32; values are code * scale in fp32, rounded to it.  A slot that
    is negative or past the cache gives a row of zeros.  ``out``: an optional pair of tensors to write to.
    """
    return decoding_attn_cuda.kv_cache_read(k_cache, v_cache, k_scale, v_scale, slots, dtype, out)


def quantized_fwd(q, k_cache, v_cache, k_scale, v_scale, cu_seq_k, is_alibi=False, softmax_scale=None, out=None,
                  return_lse=False, block_table=None):
    """Decode attention over a cache that ``kv_cache_write`` filled (any group size; dim 64, 96, 128 or 256).

    q [batch, head_q, dim]; cu_seq_k int32 [batch + 1], cumulative lengths.  A packed cache holds key j of sequence b in
    row ``cu_seq_k[b] + j``; a paged one (4-D, page_size a power of two) in row ``j % page_size`` of page
    ``block_table[b, j // page_size]`` (int32).  Keys whose row or page lies outside the cache are masked.  No length hint
    is needed: the work is divided on the device.  (Which kernel takes 8-bit codes goes by how much the cache or a row of the
    table holds a sequence: of a table that is much wider than the batch's sequences pass the columns in use.)  ``return_lse`` adds the fp32 natural-log LSE [batch, head_q].
    """
    return decoding_attn_cuda.quantized_fwd(q, k_cache, v_cache, k_scale, v_scale, cu_seq_k, is_alibi, softmax_scale, out,
                                            return_lse, block_table)


def shared_prefix_fwd(q, k_prefix, v_prefix, k, v, cu_seq_k, is_alibi=False, softmax_scale=None, out=None, return_lse=False,
                      k_scale=None, v_scale=None, block_table=None, prefix_table=None, prefix_len=None):
    """Decode attention of a batch whose sequences share their first keys, which are read once for all of them.

    Sequence b attends to the prefix and then to its own keys ``cu_seq_k[b] .. cu_seq_k[b + 1]`` (int32 [batch + 1]; a
    sequence may have none).  q [batch, head_q, dim], dim 64, 96 or 128, at most 128 query heads per KV head.

    The prefix is k_prefix, v_prefix [prefix_len, head_k, dim] in q's dtype (``prefix_len`` may name fewer rows), or pages
    ``prefix_table`` (int32 [blocks]) with ``prefix_len`` keys of a pool [num_pages, page_size, head_k, dim]: k_prefix and
    v_prefix, or k and v themselves where those are None.  page_size: a power of two >= 16.
    The own keys k, v are packed [total_k, head_k, dim] or paged with a ``block_table`` [batch, blocks], in q's dtype, or as
    codes with ``k_scale``, ``v_scale`` as ``kv_cache_write`` leaves them.  ALiBi counts positions through the prefix.
    ``return_lse`` adds the fp32 natural-log LSE [batch, head_q] over prefix and own keys.
    """
    return decoding_attn_cuda.shared_prefix_fwd(q, k_prefix, v_prefix, k, v, cu_seq_k, is_alibi, softmax_scale, out, return_lse,
                                                k_scale, v_scale, block_table, prefix_table, prefix_len)
