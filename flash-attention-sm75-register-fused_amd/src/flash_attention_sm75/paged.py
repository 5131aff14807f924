"""Paged key/value cache: writing new tokens, reading them back, attention over it.

No reference counterpart (the reference has neither a cache nor a decode path).

A cache is a pool of pages that the sequences of a serving batch share:

* ``k_cache``, ``v_cache``: [pages, H_kv, page_size, D], float16 or bfloat16, or
  float8_e4m3fn with ``k_scale``, ``v_scale``: [pages, H_kv, page_size]
  float8_e8m0fnu, one power of two for each row (a row stands for codes * scale).
  page_size is a power of two, 16 or more, D 64 or 128.  Any strides with head_dim
  contiguous and the others multiples of 16 bytes, e.g. a [pages, page_size, H_kv, D]
  buffer viewed as above.
* ``block_table``: [B, max_pages] int32; entry i of a row is the page that holds that
  sequence's positions [i * page_size, (i + 1) * page_size).  An entry outside
  [0, pages), such as -1, names no page: its positions are not written, read as
  zeros, and hidden from every query (a window's early pages that were given back).
* ``seq_lens``: [B] int32, tokens of each sequence, the new ones included.
* ``cu_seqlens``: [B + 1] int32, rising from 0: rows cu_seqlens[b] ..
  cu_seqlens[b + 1] - 1 of the new tokens' tensors are sequence b's last tokens.  None: each
  sequence has one new token, row b.

The index tensors stay on the device and are not looked at by the host, so a call
captured in a graph takes what they hold at each replay.

The calls record no gradient: inputs that require one are refused while autograd
records, and so are inputs with a forward-mode tangent.  What a call writes to counts as
changed in place (tensor versions).
"""
import math

import torch

import flash_attn_sm75_cuda as _C


def _no_backward(name):
    return RuntimeError(f"{name} has no backward pass: call it under torch.no_grad() "
                        "or on detached tensors")


def paged_cache_write(K, V, k_cache, v_cache, block_table, seq_lens, cu_seqlens=None,
                      k_scale=None, v_scale=None):
    """Writes new tokens' K and V into their pages.

    Args:
        K, V: [tokens, H_kv, D] float16 or bfloat16 (the cache's dtype, unless that is 8
            bits), views read in place where head_dim is contiguous and the other strides are
            multiples of 8.
        k_cache, v_cache, block_table, seq_lens, cu_seqlens, k_scale, v_scale: see the
            module.

    An 8-bit row takes the smallest power of two s for its scale (2^-126 to 2^7, from bfloat16 to
    2^119) with which no finite value of it exceeds 448 s in magnitude (larger ones are
    stored as 448 s), and x / s rounded to nearest even as its codes; infinities
    and NaN are stored as NaN.  Read in the dtype they were written from, such rows
    are exact 16-bit numbers.

    Rows behind cu_seqlens[B], and positions that have no page, are left out.
    Sequences of one call that share a page must not write the same positions
    of it (which of their values stays is not defined), and K and V must not be views of
    the rows that are written.
    """
    if torch.is_grad_enabled() and (K.requires_grad or V.requires_grad or k_cache.requires_grad
                                    or v_cache.requires_grad):
        raise _no_backward("paged_cache_write")
    _C.paged_cache_write(K, V, k_cache, v_cache, block_table, seq_lens, cu_seqlens, k_scale, v_scale)


def paged_cache_read(k_cache, v_cache, block_table, seq_lens, max_len=None, k_scale=None,
                     v_scale=None, dtype=None):
    """The sequences' K and V out of their pages.

    Args:
        max_len: positions to read (default: all that block_table has room for);
            B * H_kv * max_len is up to 2^27.
        dtype: float16 or bfloat16, for an 8-bit cache; a 16-bit one is read in its own.

    Returns:
        (K, V), each [B, H_kv, max_len, D]: what :func:`flash_attention_forward_ex`
        takes, zeros past a sequence's end and where it has no page.
    """
    if torch.is_grad_enabled() and (k_cache.requires_grad or v_cache.requires_grad):
        raise _no_backward("paged_cache_read")
    if max_len is None:
        max_len = block_table.size(1) * k_cache.size(2) if block_table.dim() == 2 and k_cache.dim() == 4 else 0
    return _C.paged_cache_read(k_cache, v_cache, block_table, seq_lens, int(max_len), k_scale, v_scale,
                               dtype)


def flash_attention_paged(Q, k_cache, v_cache, block_table, seq_lens, cu_seqlens=None,
                          max_query_len=None, causal="bottom_right", scale=None, k_scale=None,
                          v_scale=None, return_lse=False, out=None):
    """Attention of new tokens (a prompt's chunk, or one generated token) over the
    paged cache, which holds their own K and V already (:func:`paged_cache_write`).

    Args:
        Q: [tokens, H_q, D] float16 or bfloat16 (the cache's dtype, unless that is 8 bits);
            H_kv divides H_q.
        k_cache, v_cache, block_table, seq_lens, cu_seqlens, k_scale, v_scale: see the
            module.
        max_query_len: the most new tokens any sequence has, if the caller knows
            (default: not known).  It picks the kernel; a wrong value costs time only.
        causal: "bottom_right" (new token i of n sees keys 0 .. seq_len - n + i) or False
            (all of the sequence's keys).
        scale: softmax scale (default 1/sqrt(D)).
        return_lse: also return the fp32 natural-log row LSE, [H_q, tokens].
        out: a tensor like Q to write to, 16-byte aligned, head_dim contiguous and the other
            strides multiples of 8; it may be a view of the buffer Q is a view of (its rows
            beside Q's, or its heads between them) but must share no element with Q or the
            cache.  Its rows behind cu_seqlens[B] are left as they are (of a new tensor
            they are not defined, nor are the LSE's).

    Returns:
        O [tokens, H_q, D] in Q's dtype, or (O, LSE).  A query that sees no key gets
        a zero row and LSE -inf.  Deterministic: the same call gives the same bits.
        What lies in hidden pages and past a sequence's end reaches no query; a new token's
        V row that is not finite can reach its sequence's earlier tokens of the same call
        (0 times NaN, as in a plain product).
    """
    if torch.is_grad_enabled() and (Q.requires_grad or k_cache.requires_grad or v_cache.requires_grad
                                    or (out is not None and out.requires_grad)):
        raise _no_backward("flash_attention_paged")
    if causal is False:
        code = 0
    elif causal == "bottom_right":
        code = 2
    else:
        raise ValueError(f"causal must be 'bottom_right' or False, got {causal!r}")
    if scale is None:
        scale = 1.0 / math.sqrt(Q.size(-1))
    if max_query_len is None:
        max_query_len = 0
    elif max_query_len < 0:
        raise ValueError(f"max_query_len must be non-negative, got {max_query_len}")
    o, lse = _C.flash_attention_paged(Q, k_cache, v_cache, block_table, seq_lens, cu_seqlens,
                                      int(max_query_len), code, float(scale), k_scale, v_scale,
                                      bool(return_lse), out)
    return (o, lse) if return_lse else o
