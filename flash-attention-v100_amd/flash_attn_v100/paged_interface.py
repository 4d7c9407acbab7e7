"""Serving from a cache of keys and values that lies in pages: attention of new tokens over it, its writing and its reading.
No counterpart in the reference, whose attention is over queries, keys and values of the same length.

The cache is two tensors ``k_cache`` and ``v_cache`` of shape (pages, page_size, kv_heads, head_size), page_size a multiple of
16, head_size 64 or 128, in fp16 or bf16 as q, k and v are, or in torch.float8_e4m3fn with scales ``k_scale`` and ``v_scale`` of
shape (pages, page_size, kv_heads) in torch.float8_e8m0fnu.  Strides are free as long as rows of head_size elements are
contiguous and begin on 16-byte boundaries, slots less than 2 ** 24 and heads less than 2 ** 30 elements apart; pages that hold head by head (a transpose(1, 2) of such a tensor) are read up to a
tenth faster.

``page_table`` (batch, columns), int32: position p of sequence b is slot p % page_size of page
page_table[b, p // page_size].  ``cache_seqlens`` (batch), int32: how many keys a sequence has, those of its new tokens among
them; new token i of n is at position cache_seqlens[b] - n + i.  Both stay on the GPU and are read there, so a captured graph
takes what they hold at its replay.  What is not valid in them never leads out of the tensors: positions behind the table's
columns, or on a page that the cache does not have, are left out when written, and give NaN when read or attended to.  Scales
other than those that kv_cache_write makes are 2 ** -126 or more, and no NaN.

New tokens come as (batch, seqlen, heads, head_size), all sequences with as many, or packed as (tokens, heads, head_size) with
``cu_seqlens`` (batch + 1), int32: sequence b has tokens cu_seqlens[b] .. cu_seqlens[b + 1] - 1.

The three calls have no gradients and refuse tensors that ask for them, those that they write to among them.
"""
import torch  # noqa: F401  (before the kernels, so that they bind to the HIP runtime it has loaded)

try:
    import flash_attn_v100_paged_cuda as paged_cuda
except ImportError as exc:  # fail loudly: there is no fallback path
    raise ImportError(
        "flash_attn_v100 needs its compiled extension flash_attn_v100_paged_cuda "
        "(run `python setup.py build_ext --inplace` in flash-attention-v100_amd/): %s" % exc
    ) from exc

_attention, _write, _read = paged_cuda.attention, paged_cuda.write, paged_cuda.read


def flash_attn_paged_func(q, k_cache, v_cache, page_table, cache_seqlens, softmax_scale=None, causal=False, *, cu_seqlens=None,
                          max_seqlen=None, k_scale=None, v_scale=None, out=None):
    """Attention of new tokens over the cache, which already holds their own keys and values (kv_cache_write).

    q has a multiple of the cache's heads: query head h attends to head h // (heads // kv_heads).  causal: a token sees keys up to
    its own position, otherwise all of its sequence.  Rows that see no key are zero.  Keys that a token does not see do not matter to
    it, whatever they and their values hold.  softmax_scale: head_size ** -0.5 if None.
    max_seqlen: no sequence has more new tokens (with cu_seqlens).  Not needed for the result, but without it all tokens could be one
    sequence's: 64 single tokens over about 4096 keys each, 32 heads of 128, then take 179 us instead of 163, 16 over 2000 35 instead of
    27, out of 8 bits 31 instead of 21, with a workspace of 65 MiB instead of 8; a batch with chunks takes as long either way.
    out: dense tensor of q's shape on a 16-byte boundary to write to, which shares no memory with the others; rows of tokens that belong to no sequence stay as they are there, and are zero
    in a tensor made here.  Returns it."""
    return _attention(q, k_cache, v_cache, page_table, cache_seqlens, softmax_scale, causal, cu_seqlens, max_seqlen,
                      k_scale, v_scale, out)


def kv_cache_write(k, v, k_cache, v_cache, page_table, cache_seqlens, *, cu_seqlens=None, k_scale=None, v_scale=None):
    """Writes the new tokens' keys and values to their places in the cache.  Tokens at negative positions (a sequence with more
    new tokens than keys) are left out.  Into a float8_e4m3fn cache a row goes with a scale of its own: the least power of two,
    2 ** -126 or more, for which none of its numbers is over 448 scales, after clipping to the largest value of the inputs' type
    with four significant bits (fp16 61440, bf16 1.875 * 2 ** 127; infinities too, NaN stays).  Values are rounded to nearest, and
    what comes back are values of the inputs' type.  A place that several tokens have, where a page is twice in the table, holds
    one of them or parts of several."""
    _write(k, v, k_cache, v_cache, page_table, cache_seqlens, cu_seqlens, k_scale, v_scale)


def kv_cache_read(k_cache, v_cache, page_table, cache_seqlens, max_seqlen, *, k_scale=None, v_scale=None, dtype=None):
    """The cache's keys and values as two dense tensors (batch, max_seqlen, kv_heads, head_size), with zeros behind a
    sequence's length.  dtype: of a float8_e4m3fn cache's values, torch.float16 if None."""
    return _read(k_cache, v_cache, page_table, cache_seqlens, max_seqlen, k_scale, v_scale, dtype)
