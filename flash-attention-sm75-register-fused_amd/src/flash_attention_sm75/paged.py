"""Paged key/value cache: writing new tokens, reading them back, attention over it, prefixes
that sequences share, the weight that attention gave each row, and eviction by it.

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


def _causal_code(causal):
    if causal is False:
        return 0
    if causal == "bottom_right":
        return 2
    raise ValueError(f"causal must be 'bottom_right' or False, got {causal!r}")


def _hint(value, name):
    if value is None:
        return 0
    if value < 0:
        raise ValueError(f"{name} must be non-negative, got {value}")
    return int(value)


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
    code = _causal_code(causal)
    if scale is None:
        scale = 1.0 / math.sqrt(Q.size(-1))
    o, lse = _C.flash_attention_paged(Q, k_cache, v_cache, block_table, seq_lens, cu_seqlens,
                                      _hint(max_query_len, "max_query_len"), code, float(scale), k_scale, v_scale,
                                      bool(return_lse), out)
    return (o, lse) if return_lse else o


def flash_attention_paged_prefix(Q, k_cache, v_cache, prefix_table, prefix_lens, block_table, seq_lens,
                                 cu_seqlens=None, cu_prefix=None, max_query_len=None,
                                 max_prefix_queries=None, causal="bottom_right", scale=None, k_scale=None,
                                 v_scale=None, return_lse=False, out=None):
    """Attention of new tokens whose sequences share prefixes (an instruction, a document): a
    prefix's rows are read once for all of its sequences (or, where few rows and short tables make
    that faster, by each in one launch).

    What :func:`flash_attention_paged` gives where each sequence's table lists its prefix's pages
    first, with these differences: block_table and seq_lens are of a sequence's own tokens
    (new ones included) and do not count its prefix, whose length need not fill its last page.

    Args:
        prefix_table: [G, max_prefix_pages] int32, the pages of each prefix, as block_table.
        prefix_lens: [G] int32, tokens of each prefix.
        cu_prefix: [G + 1] int32, rising: sequences cu_prefix[g] .. cu_prefix[g + 1] - 1 have
            prefix g, those before cu_prefix[0] and from cu_prefix[G] on none.  (Where it falls, which
            prefix a sequence gets is not said.)  None: there is one prefix, and every sequence has it.
        max_prefix_queries: the most new tokens behind one prefix, if the caller knows: a hint
            as max_query_len.
        causal: by which a new token sees its sequence's own keys; it sees all of its prefix.

        The others, and what is returned, are those of :func:`flash_attention_paged`; LSE is
        over the prefix and the own keys.
    """
    if torch.is_grad_enabled() and (Q.requires_grad or k_cache.requires_grad or v_cache.requires_grad
                                    or (out is not None and out.requires_grad)):
        raise _no_backward("flash_attention_paged_prefix")
    code = _causal_code(causal)
    if scale is None:
        scale = 1.0 / math.sqrt(Q.size(-1))
    o, lse = _C.flash_attention_paged_prefix(
        Q, k_cache, v_cache, prefix_table, prefix_lens, block_table, seq_lens, cu_seqlens, cu_prefix,
        _hint(max_query_len, "max_query_len"), _hint(max_prefix_queries, "max_prefix_queries"), code,
        float(scale), k_scale, v_scale, bool(return_lse), out)
    return (o, lse) if return_lse else o


def paged_attention_weights(Q, LSE, k_cache, block_table, seq_lens, cu_seqlens=None, max_len=None,
                            max_query_len=None, causal="bottom_right", scale=None, k_scale=None, add_to=None):
    """The weight that attention gave each cached row: its probabilities, summed over the new
    tokens and the query heads that share its KV head.

    Args:
        Q, k_cache, block_table, seq_lens, cu_seqlens, max_query_len, causal, scale, k_scale: the
            attention call's.
        LSE: the log-sum-exp it returned, [H_q, tokens] float32; a row of -inf adds nothing, whatever its query.
        max_len: positions to weigh (default: all that block_table has room for).
        add_to: [B, H_kv, max_len] float32, positions contiguous: the weights are added to
            those of the positions that hold a row, the others are left as they are.  Its rows
            must not overlap, nor share memory with the other tensors.

    Returns:
        weights [B, H_kv, max_len] float32 (add_to where that is given): entry j is position j's;
        0 past a sequence's end and where it has no page.  Deterministic: the same call gives the
        same bits.

    The rows of a shared prefix get theirs from a call over its table (prefix_table, prefix_lens, and for
    cu_seqlens the bounds of its sequences' tokens) with causal=False and the LSE of
    :func:`flash_attention_paged_prefix`.  A key that is not finite gives its own weight only;
    a query that is NaN (of a row whose LSE is not -inf) or an LSE that is gives every row it sees NaN.
    """
    if torch.is_grad_enabled() and (Q.requires_grad or LSE.requires_grad or k_cache.requires_grad
                                    or (add_to is not None and add_to.requires_grad)):
        raise _no_backward("paged_attention_weights")
    code = _causal_code(causal)
    if scale is None:
        scale = 1.0 / math.sqrt(Q.size(-1))
    if max_len is None:
        max_len = block_table.size(1) * k_cache.size(2) if block_table.dim() == 2 and k_cache.dim() == 4 else 0
    elif add_to is not None:
        raise ValueError("max_len goes without add_to, whose size says it")
    return _C.paged_attention_weights(Q, LSE, k_cache, block_table, seq_lens, cu_seqlens, int(max_len),
                                      _hint(max_query_len, "max_query_len"), code, float(scale), k_scale, add_to)


def paged_cache_evict(k_cache, v_cache, block_table, seq_lens, weights, to_table, keep, recent=0,
                      k_scale=None, v_scale=None):
    """Cuts each sequence to ``keep`` rows, for each KV head those that attention gave most
    weight: they are copied, in order, to other pages.

    Args:
        weights: [B, H_kv, max_len] float32, max_len at least what block_table has room for: of each
            position (:func:`paged_attention_weights`).
        to_table: [B, max_to_pages] int32, the pages that the rows go to, with room for keep rows (or for
            as many as block_table has room for).  None of them may be one of block_table's that hold
            rows, and none may be listed twice; rows whose place has no page are dropped.
        keep: rows that stay (all, where a sequence holds no more).
        recent: those of the sequence's last ``recent`` positions (at most keep) stay whatever their weights.

    Of the other rows the heaviest stay; of equal ones those at the lowest positions; NaN
    counts as less than any number.  Positions without a page hold no row, so what is kept
    closes up over them.  block_table's rows and seq_lens are left as they are, and its pages may be shared
    between sequences; the caller goes on with to_table and what is returned:

    Returns:
        (seq_lens, weights): [B] int32, rows that stayed; [B, H_kv, max_to_pages * page_size] float32, their
        weights, 0 behind them.
    """
    if torch.is_grad_enabled() and (k_cache.requires_grad or v_cache.requires_grad or weights.requires_grad):
        raise _no_backward("paged_cache_evict")
    return _C.paged_cache_evict(k_cache, v_cache, block_table, seq_lens, weights, to_table, int(keep), int(recent),
                                k_scale, v_scale)
