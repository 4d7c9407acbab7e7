"""Attention over a paged cache, its writing and its reading, restated in 64 bits on the CPU.  TEST INFRASTRUCTURE ONLY.

There is nothing of the kind in the reference, so the functions are pinned by the definitions alone (tests/test_paged.py
checks them against closed forms and against each other): plain loops over sequences and heads, no tiles, no online softmax.
Tensors may live anywhere; all arithmetic is on the CPU.
"""
import torch

E4M3_MAX = 448.0
#: a type's largest value of four significant bits: what rounds to it stays finite in the type
LARGEST_KEPT = {torch.float16: 61440.0, torch.bfloat16: 1.875 * 2.0 ** 127}


def to_e4m3(x):
    """Rows (.., d) of fp16 or bf16 as (values float64, exponents int): a row is values * 2 ** exponent."""
    most = LARGEST_KEPT[x.dtype]
    x = x.detach().cpu().double().clamp(-most, most)  # clamp keeps NaN
    amax = torch.nan_to_num(x, nan=0.0).abs().amax(-1)
    m, e = torch.frexp(amax / E4M3_MAX)  # amax / 448 = m 2^e, m in [1/2, 1)
    e = torch.where(amax == 0, torch.tensor(-126), torch.where(m == 0.5, e - 1, e)).clamp(min=-126).to(torch.int64)
    y = x * torch.pow(2.0, -e.double()).unsqueeze(-1)
    at = torch.frexp(y.abs().clamp(min=2.0 ** -6))[1] - 1  # 2^at <= |y| < 2^(at + 1); below 2^-6 the steps stay 2^-9
    step = torch.pow(2.0, (at - 3).double())
    return torch.round(y / step) * step, e  # torch.round: ties to even


def places(page_table, page_size, b, positions):
    ids = page_table[b].cpu().long()[torch.div(positions, page_size, rounding_mode="floor")]
    return ids, positions % page_size


def held(cache, scale, page_table, b, count):
    """The first `count` rows of sequence b, (count, kv heads, d) in 64 bits."""
    ids, slots = places(page_table, cache.shape[1], b, torch.arange(count))
    where = (ids.to(cache.device), slots.to(cache.device))
    x = cache[where].cpu().double()
    return x if scale is None else x * scale[where].cpu().double().unsqueeze(-1)


def attention(q, k, v, scale, causal):
    """One sequence's new tokens q (n, heads, d) over its keys and values (L, kv heads, d), in 64 bits: the result, and what
    errors are multiplied with: sum_j p_j |v_j| over the visible keys (n, heads, d), and the largest sum of the magnitudes of
    a score's products (n, heads, 1)."""
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    n, heads, d = q.shape
    keys = k.shape[0]
    out, weight, size = (torch.zeros(n, heads, w, dtype=torch.float64) for w in (d, d, 1))
    if n == 0 or keys == 0:
        return out, weight, size
    seen = torch.arange(keys)[None] <= (keys - n + torch.arange(n)[:, None] if causal else torch.full((n, 1), keys))
    some = seen.any(1)
    for h in range(heads):
        kh, vh = k[:, h // (heads // k.shape[1])], v[:, h // (heads // k.shape[1])]
        s = (q[some, h] @ kh.t() * scale).masked_fill(~seen[some], -torch.inf)
        p = torch.softmax(s, -1)
        out[some, h], weight[some, h] = p @ vh, p @ vh.abs()
        size[some, h, 0] = (q[some, h].abs() @ kh.abs().t()).amax(-1) * abs(scale)
    return out, weight, size


def sequences(cu_seqlens, batch, tokens):
    """(first, end) of each sequence's tokens, of `tokens` a sequence where there is no cu_seqlens."""
    if cu_seqlens is None:
        return [(b * tokens, (b + 1) * tokens) for b in range(batch)]
    c = cu_seqlens.tolist()
    return list(zip(c[:-1], c[1:]))


def paged_attention(q, k_cache, v_cache, page_table, cache_seqlens, scale=None, causal=False, cu_seqlens=None, k_scale=None,
                    v_scale=None):
    """attention of a batch: its three results, the first two of q's shape."""
    flat = q.reshape(-1, *q.shape[-2:])
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    results = [torch.zeros(*flat.shape[:2], w, dtype=torch.float64) for w in (flat.shape[2], flat.shape[2], 1)]
    lengths = cache_seqlens.tolist()
    for b, (first, end) in enumerate(sequences(cu_seqlens, len(lengths), q.shape[-3])):
        k, v = (held(c, s, page_table, b, max(lengths[b], 0)) for c, s in ((k_cache, k_scale), (v_cache, v_scale)))
        for r, x in zip(results, attention(flat[first:end], k, v, scale, causal)):
            r[first:end] = x
    return [r.reshape(*q.shape[:-1], -1) for r in results]


def attention_tolerance(dtype, d, out, weight, size, keys, v_max):
    """How far the kernels' result may be from `out`, value by value, by arithmetic:

    - a score is a sum of d products in 32 bits, off by at most (d + 2) 2^-24 of the sum of their magnitudes; as an exponent of 2
      it is multiplied, the maximum subtracted, and exponentiated: 3 2^-24 of its size and 2^-22.  Probabilities are off
      relatively by that, and so is their sum: twice;
    - probabilities are rounded to the type: eps / 2, and in fp16, where they are small, half a subnormal step, 2^-25, for each
      key against a sum of at least 1;
    - sums over keys in 32 bits: 2^-24 for each key, for each of up to keys / 32 rescalings, and for joining parts;
    - the result is rounded to the type."""
    u = torch.finfo(dtype).eps / 2
    in_score = (d + 2) * 2.0 ** -24 * size + 3 * 2.0 ** -24 * 1.4427 * size + 2.0 ** -22
    relative = 2 * in_score + u + 2 * (1.1 * keys + 64) * 2.0 ** -24
    subnormal = keys * v_max * 2.0 ** -25 if dtype == torch.float16 else 0.0
    return relative * weight + u * out.abs() + subnormal + 2.0 ** -25
