"""Attention over a paged cache, its writing and its reading, on the GPU against the oracle in 64 bits."""
import pytest
import torch

import paged
from oracle import paged_oracle as po

pytestmark = pytest.mark.gpu

TYPES = (torch.float16, torch.bfloat16)


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.fail("this test needs a GPU")
    import flash_attn_v100
    return flash_attn_v100


def check_attention(ops, batch, causal, scale=None, **more):
    want, tolerance = batch.expected(causal, scale)
    got = ops.flash_attn_paged_func(batch.q, *batch.args(), scale, causal, cu_seqlens=batch.cu_seqlens, **batch.scales(), **more)
    assert got.dtype == batch.dtype and got.shape == batch.q.shape and got.is_contiguous()
    off = (got.cpu().double() - want).abs()
    assert torch.isfinite(got).all(), "%d values are not finite" % int((~torch.isfinite(got)).sum())
    worst = float((off / tolerance).max())
    assert worst <= 1, worst
    return got


# lengths about the borders of pages, units of 32 keys and tiles of 64, with empty sequences
@pytest.mark.parametrize("cache", paged.CACHES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", (64, 128))
@pytest.mark.parametrize("group", (1, 4, 16))
def test_single_tokens(ops, dim, dtype, cache, group):
    lengths = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 0, 127, 128, 129, 200, 255, 256, 257, 300]
    batch = paged.Batch(lengths, 1, 2, group, dim, 16, dtype, cache, seed=group)
    check_attention(ops, batch, True)
    check_attention(ops, batch, False)


@pytest.mark.parametrize("cache", paged.CACHES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", (64, 128))
@pytest.mark.parametrize("causal", (False, True))
@pytest.mark.parametrize("new,group,page", [(2, 1, 16), (5, 3, 48), (17, 2, 16), (33, 1, 32), (64, 4, 64), (129, 1, 16), (150, 5, 128)])
def test_chunks(ops, dim, dtype, cache, causal, new, group, page):
    """Also of sequences that have fewer keys than new tokens: the first rows see nothing under a causal mask."""
    batch = paged.Batch([new, new + 1, 40, 333, 1, 0, new + 63], new, 2, group, dim, page, dtype, cache, seed=new)
    check_attention(ops, batch, causal)


@pytest.mark.parametrize("cache", paged.CACHES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", (64, 128))
@pytest.mark.parametrize("group", (1, 5, 8))
def test_packed_batches(ops, dim, dtype, cache, group):
    """Single tokens, chunks and sequences without new tokens in one call; rows behind the last sequence are zero, or left as they
    are where the caller gives the output."""
    lengths, new = [70, 1, 300, 260, 0, 1000, 129, 50], [1, 1, 40, 0, 0, 130, 129, 2]
    batch = paged.Batch(lengths, new, 3, group, dim, 16, dtype, cache, packed=True, seed=group, tail=3)
    for causal in (True, False):
        got = check_attention(ops, batch, causal, max_seqlen=130)
        assert not got[-3:].any()
    assert torch.equal(got, check_attention(ops, batch, False))
    out = torch.full_like(batch.q, 7.0)
    same = ops.flash_attn_paged_func(batch.q, *batch.args(), cu_seqlens=batch.cu_seqlens, out=out, **batch.scales())
    assert same.data_ptr() == out.data_ptr()
    assert torch.equal(out[:-3], got[:-3]) and (out[-3:] == 7).all()


@pytest.mark.parametrize("cache", paged.CACHES)
@pytest.mark.parametrize("dim", (64, 128))
@pytest.mark.parametrize("new,group", [(1, 8), (1, 1), (3, 8), (70, 4)])
def test_long_sequences_in_parts(ops, dim, cache, new, group):
    batch = paged.Batch([5000, 4097, 1, 9000], new, 2, group, dim, 64, torch.float16, cache, seed=dim)
    check_attention(ops, batch, True)


@pytest.mark.parametrize("new", (1, 20))
def test_tokens_in_front_of_the_first_sequence(ops, new):
    """Rows that belong to none, as those behind the last one.  max_seqlen: the kernel goes by the tokens in all otherwise, and its
    roundings with it."""
    how = {"max_seqlen": max(new, 3)}
    batch = paged.Batch([70, 300, 90], [new, 2, 3], 1, 4, 64, packed=True)
    want = ops.flash_attn_paged_func(batch.q, *batch.args(), None, True, cu_seqlens=batch.cu_seqlens, **how)
    q = torch.cat([torch.full_like(batch.q[:3], float("nan")), batch.q, torch.full_like(batch.q[:2], float("nan"))])
    spoilt = torch.full_like(q, 7.0)  # most likely what the next call gets
    del spoilt
    got = ops.flash_attn_paged_func(q, *batch.args(), None, True, cu_seqlens=batch.cu_seqlens + 3, **how)
    assert torch.equal(got[3:-2], want) and not got[:3].any() and not got[-2:].any()
    out = torch.full_like(q, 7.0)
    ops.flash_attn_paged_func(q, *batch.args(), None, True, cu_seqlens=batch.cu_seqlens + 3, **how, out=out)
    assert torch.equal(out[3:-2], want) and (out[:3] == 7).all() and (out[-2:] == 7).all()


@pytest.mark.parametrize("dim", (64, 128))
@pytest.mark.parametrize("new", (9, 50))
@pytest.mark.parametrize("value", (float("nan"), float("inf"), -float("inf")))
def test_keys_of_later_tokens_do_not_matter(ops, dim, new, value):
    batch = paged.Batch([new, 333, 64 + new], new, 2, 2, dim, 16, torch.bfloat16)
    want = ops.flash_attn_paged_func(batch.q, *batch.args(), None, True)
    for b, m in enumerate(batch.lengths):
        ids, slots = po.places(batch.page_table.cpu(), 16, b, torch.arange(m - 3, m))
        batch.k_cache[ids.cuda(), slots.cuda()] = value
    got = ops.flash_attn_paged_func(batch.q, *batch.args(), None, True)
    assert torch.equal(got[:, :-3], want[:, :-3])


@pytest.mark.parametrize("cache", paged.CACHES)
@pytest.mark.parametrize("dim", (64, 128))
@pytest.mark.parametrize("lengths,new,group,kv_heads", [
    ([150000], 1, 3, 1), ([70000, 40, 90000], 1, 2, 1), ([33000, 35000], 2, 1, 2), ([3000] * 66, 1, 1, 1), ([200000], 33, 1, 1),
    ([40000, 45000, 60], 40, 4, 2), ([41000], 200, 2, 1), ([9000] * 18, 35, 1, 1)])
def test_parts_of_all_work_groups(ops, dim, cache, lengths, new, group, kv_heads):
    """So many keys that each work group has some: parts up to the last place."""
    batch = paged.Batch(lengths, new, kv_heads, group, dim, 64, torch.float16, cache, seed=dim)
    check_attention(ops, batch, True, 0.5)  # few keys have most of the weight
    if new < 40:
        batch = paged.Batch(lengths + [5, 64], [new] * len(lengths) + [1, 0], kv_heads, group, dim, 64, torch.bfloat16, cache, packed=True, seed=dim)
        check_attention(ops, batch, False, 0.5)


@pytest.mark.parametrize("count", (65, 130, 4200))
def test_many_sequences(ops, count):
    """More than a wave looks at together."""
    g = torch.Generator().manual_seed(count)
    lengths = torch.randint(0, 90, (count,), generator=g).tolist()
    batch = paged.Batch(lengths, 1, 1, 2, 64, 16, torch.bfloat16, seed=count)
    check_attention(ops, batch, True)
    new = torch.randint(0, 3, (count,), generator=g).tolist()
    batch = paged.Batch(lengths, new, 1, 2, 64, 16, torch.bfloat16, packed=True, seed=count, tail=2)
    check_attention(ops, batch, True)


@pytest.mark.parametrize("cache", paged.CACHES)
@pytest.mark.parametrize("layout", ("heads", "beside"))
@pytest.mark.parametrize("dim", (64, 128))
@pytest.mark.parametrize("new", (1, 50))
def test_strides(ops, dim, cache, layout, new):
    batch = paged.Batch([130, 77, 600], new, 3, 2, dim, 32, torch.float16, cache, seed=5, layout=layout)
    assert not batch.k_cache.is_contiguous()
    packed = torch.randn(3, new, 3, batch.heads, dim, device="cuda").half()
    batch.q = packed[:, :, 1]
    check_attention(ops, batch, True)
    batch.q = packed[:, :, 1].transpose(1, 2).contiguous().transpose(1, 2)
    check_attention(ops, batch, True)
    odd = torch.randn(3, new, batch.heads, dim + 1, device="cuda").half()
    batch.q = odd[..., 1:]  # rows on no 16-byte boundary
    check_attention(ops, batch, True)
    batch.page_table = torch.cat([batch.page_table] * 2, 1)[:, :batch.page_table.shape[1]]  # another row stride
    check_attention(ops, batch, True)


@pytest.mark.parametrize("cache", paged.CACHES)
@pytest.mark.parametrize("new", (1, 3))
@pytest.mark.parametrize("group", (33, 71, 160))
def test_many_query_heads_to_a_key_head(ops, group, new, cache):
    """Single tokens in blocks of many rows, and tokens that go over two of them."""
    batch = paged.Batch([1, 77, 300, 0, 64], new, 1, group, 64, 16, torch.bfloat16, cache, seed=group)
    check_attention(ops, batch, True)
    batch = paged.Batch([5, 77, 300], [new, 0, 1], 2, group, 128, 16, torch.float16, cache, packed=True, seed=group)
    check_attention(ops, batch, True)


@pytest.mark.parametrize("hint", (None, 1, 3, 40, 1 << 40))
@pytest.mark.parametrize("cache", paged.CACHES)
def test_the_hint_does_not_matter(ops, cache, hint):
    batch = paged.Batch([70, 40, 500, 9], [1, 40, 17, 3], 2, 4, 128, 16, torch.float16, cache, packed=True)
    check_attention(ops, batch, True, max_seqlen=hint)


@pytest.mark.parametrize("cache", paged.CACHES)
@pytest.mark.parametrize("new", (1, 40))
def test_keys_and_values_laid_out_differently(ops, cache, new):
    """Each cache and scale with strides of its own, rows of the page table apart, q the same for all sequences."""
    kinds = {name: paged.Batch([100, 65, 333], new, 2, 4, 128, 16, torch.bfloat16, cache, seed=2, layout=name) for name in ("pages", "heads", "beside")}
    for a, b, c, d in (("pages", "heads", "beside", "heads"), ("beside", "pages", "heads", "pages")):
        batch = kinds["pages"]
        batch.k_cache, batch.v_cache, batch.k_scale, batch.v_scale = kinds[a].k_cache, kinds[b].v_cache, kinds[c].k_scale, kinds[d].v_scale
        width = batch.page_table.shape[1]
        batch.page_table = torch.cat([batch.page_table, batch.page_table.flip(0) ^ 1], 1)[:, :width]
        batch.q = batch.q[:1].expand_as(batch.q)
        check_attention(ops, batch, True)


@pytest.mark.parametrize("scale", (0.0, -0.2, 0.9))
@pytest.mark.parametrize("new", (1, 40))
def test_scales(ops, scale, new):
    check_attention(ops, paged.Batch([700, 64, 41], new, 2, 2, 128, 16, torch.float16, seed=3), True, scale)


@pytest.mark.parametrize("new", (1, 40))
def test_growing_maximum(ops, new):
    """Scores that grow along the sequence, and ones of the type's size."""
    batch = paged.Batch([900, 300], new, 1, 4, 64, 16, torch.float16, seed=9)
    for b, m in enumerate(batch.lengths):
        ids, slots = po.places(batch.page_table.cpu(), 16, b, torch.arange(m))
        batch.k_cache[ids.cuda(), slots.cuda()] *= (torch.arange(m, device="cuda") / 100).half()[:, None, None]
    check_attention(ops, batch, True)


@pytest.mark.parametrize("dim,cache", [(64, "same"), (128, "e4m3")])
@pytest.mark.parametrize("new", (1, 60))
def test_bad_pages_and_lengths(ops, dim, cache, new):
    """Nothing is read outside of the cache: sequences that would are NaN, the others as ever."""
    batch = paged.Batch([100, 200, 300, 90, 400], new, 2, 2, dim, 16, torch.float16, cache, seed=1)
    pages = batch.k_cache.shape[0]
    want, tolerance = batch.expected(True)
    table, lengths = batch.page_table.clone(), batch.cache_seqlens.clone()
    table[1, 3] = pages
    table[2, 0] = -1
    lengths[4] = batch.page_table.shape[1] * 16 + 1  # behind the table's columns
    lengths[3] = -5
    got = ops.flash_attn_paged_func(batch.q, batch.k_cache, batch.v_cache, table, lengths, None, True, **batch.scales()).cpu().double()
    assert ((got[0] - want[0]).abs() <= tolerance[0]).all()
    assert got[1].isnan().all() and got[2].isnan().all() and got[4].isnan().all()  # all rows see the pages
    assert not got[3].any()
    k, v = ops.kv_cache_read(batch.k_cache, batch.v_cache, table, lengths, 310, **batch.scales())
    k0, v0 = ops.kv_cache_read(*batch.args(), 310, **batch.scales())
    for x, y in ((k, k0), (v, v0)):
        bad = torch.zeros_like(x, dtype=torch.bool)
        bad[1, 48:64] = bad[2, :16] = True
        assert x[bad].isnan().all()
        keep = ~bad
        keep[3] = keep[4] = False
        assert torch.equal(x[keep], y[keep]) and not x[3].any()
    before = [t.clone().view(torch.uint8) for t in (batch.k_cache, batch.v_cache)]
    ops.kv_cache_write(batch.k, batch.v, batch.k_cache, batch.v_cache, torch.full_like(table, pages), lengths, **batch.scales())
    ops.kv_cache_write(batch.k, batch.v, batch.k_cache, batch.v_cache, torch.full_like(table, -1), lengths, **batch.scales())
    ops.kv_cache_write(batch.k, batch.v, batch.k_cache, batch.v_cache, table, torch.zeros_like(lengths), **batch.scales())
    ops.kv_cache_write(batch.k, batch.v, batch.k_cache, batch.v_cache, table, lengths + 2 ** 30, **batch.scales())
    for x, y in zip(before, (batch.k_cache, batch.v_cache)):
        assert torch.equal(x, y.view(torch.uint8))


@pytest.mark.parametrize("ends", ([0, 5, 3, 9, 9], [-4, 2, 4, 100, 7], [7, 7, 7, 7, 7], [9, 6, 4, 2, 0]))
@pytest.mark.parametrize("times", (1, 150))
def test_token_ranges_that_make_no_sense(ops, ends, times):
    """They are not checked, but nothing is read or written outside of the tensors."""
    batch = paged.Batch([40, 50, 60, 1300] * times, [2, 3, 2, 2] * times, 1, 2, 64, 16, torch.float16, packed=True)
    cu = torch.tensor(ends[:4] * times + ends[4:], dtype=torch.int32, device="cuda") * times
    room = torch.full((3, *batch.q.shape), 3.0, device="cuda", dtype=torch.float16)
    ops.flash_attn_paged_func(batch.q, *batch.args(), None, True, cu_seqlens=cu, out=room[1])
    assert (room[0] == 3).all() and (room[2] == 3).all()
    ops.kv_cache_write(batch.k, batch.v, *batch.args(), cu_seqlens=cu)
    torch.cuda.synchronize()


@pytest.mark.parametrize("cache", paged.CACHES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", (64, 128))
@pytest.mark.parametrize("kv_heads", (1, 3, 8))
@pytest.mark.parametrize("layout", ("pages", "heads", "beside"))
def test_write_and_read(ops, dim, dtype, cache, kv_heads, layout):
    lengths, new = [70, 1, 300, 260, 0, 129, 50, 2], [1, 1, 40, 0, 0, 129, 2, 5]
    batch = paged.Batch(lengths, new, kv_heads, 1, dim, 32, dtype, cache, packed=True, seed=kv_heads, layout=layout, tail=2)
    batch.k[::3] *= 100
    batch.k[1::3] *= 1e-4
    want = {}
    for name in "kv":
        data, scale = getattr(batch, name + "_cache").cpu().double(), getattr(batch, name + "_scale")
        scale = None if scale is None else scale.cpu().view(torch.uint8).clone()
        x = getattr(batch, name).cpu()
        for b, (first, end) in enumerate(po.sequences(batch.cu_seqlens, len(lengths), 0)):
            at = lengths[b] - (end - first) + torch.arange(end - first)
            ids, slots = po.places(batch.page_table, 32, b, at[at >= 0])
            rows = x[first:end][at >= 0]
            if scale is not None:
                rows, e = po.to_e4m3(rows)
                scale[ids, slots] = (e + 127).to(torch.uint8)
            data[ids, slots] = rows.double()
        want[name] = data, scale
    ops.kv_cache_write(batch.k, batch.v, *batch.args(), cu_seqlens=batch.cu_seqlens, **batch.scales())
    for name in "kv":
        data, scale = want[name]
        assert torch.equal(torch.nan_to_num(getattr(batch, name + "_cache").cpu().double(), nan=-1e9), torch.nan_to_num(data, nan=-1e9))
        if scale is not None:
            assert torch.equal(getattr(batch, name + "_scale").cpu().view(torch.uint8), scale)
    for longest in (1, 33, 300, 400):
        got = ops.kv_cache_read(*batch.args(), longest, dtype=dtype, **batch.scales())
        for name, x in zip("kv", got):
            assert x.shape == (len(lengths), longest, kv_heads, dim) and x.dtype == dtype and x.is_contiguous()
            for b, m in enumerate(lengths):
                rows = po.held(getattr(batch, name + "_cache"), getattr(batch, name + "_scale"), batch.page_table, b, min(m, longest))
                assert torch.equal(x[b, :m].cpu().double(), rows)  # exactly: the values are some of the type
                assert not x[b, m:].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_values_at_the_ends_of_the_type(ops, dtype):
    """Infinities, NaN, the largest and smallest numbers, zeros: clipped, kept, with exact scales."""
    batch = paged.Batch([16, 16], 16, 1, 1, 64, 16, dtype, "e4m3", seed=2)
    top, tiny = torch.finfo(dtype).max, torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    rows = batch.k.view(-1, 64)
    rows[0] = 0
    rows[1] = top
    rows[2, :3] = torch.tensor([float("inf"), -float("inf"), 1.0])
    rows[3, 5] = float("nan")
    rows[4] = float("nan")
    rows[5] = tiny
    rows[6] = tiny * torch.arange(64, device="cuda")
    rows[7] = torch.linspace(-448, 448, 64, device="cuda").to(dtype)
    rows[8] = 449
    rows[9] = 2.0 ** -6
    rows[10, 0] = top / 2
    rows[11] = -0.0
    rows[12] = po.LARGEST_KEPT[dtype]
    rows[13] = torch.arange(64, device="cuda").to(dtype) * 2.0 ** -9
    batch.v.copy_(batch.k.flip(0))
    ops.kv_cache_write(batch.k, batch.v, *batch.args(), **batch.scales())
    for name in "kv":
        values, e = po.to_e4m3(getattr(batch, name).cpu())
        k, v = ops.kv_cache_read(*batch.args(), 16, dtype=dtype, **batch.scales())
        got = (k if name == "k" else v).cpu().double()
        want = values * torch.pow(2.0, e.double()).unsqueeze(-1)
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
        assert (got.isnan() | got.isfinite()).all()
        fine = getattr(batch, name).cpu().double().clamp(-po.LARGEST_KEPT[dtype], po.LARGEST_KEPT[dtype])
        # half a step of 3 bits, or of the row's smallest steps
        room = torch.maximum(2.0 ** -4 * fine.abs(), 2.0 ** -10 * torch.pow(2.0, e.double()).unsqueeze(-1))
        assert (((got - fine).abs() <= room) | got.isnan()).all()


@pytest.mark.parametrize("cache", paged.CACHES)
def test_offsets_past_32_bits(ops, cache):
    """Pages that lie more than 4 GiB behind the cache's first byte."""
    page, kv_heads, dim = 64, 8, 128
    one = paged.Batch([500, 130], 3, kv_heads, 2, dim, page, torch.float16, cache, seed=4)
    pages = (1 << 32) // (page * kv_heads * dim * one.k_cache.element_size()) + 40
    used = one.k_cache.shape[0]
    for name in ("k_cache", "v_cache", "k_scale", "v_scale"):
        small = getattr(one, name)
        if small is not None:
            large = torch.empty((pages, *small.shape[1:]), dtype=small.dtype, device="cuda")
            large[-used:].view(torch.uint8).copy_(small.view(torch.uint8))
            setattr(one, name, large)
    one.page_table += torch.where(one.page_table >= 0, pages - used, 0).int()
    check_attention(ops, one, True)
    ops.kv_cache_write(one.k, one.v, *one.args(), **one.scales())
    check_attention(ops, one, True)
    k, _ = ops.kv_cache_read(*one.args(), 500, **one.scales())
    if cache == "same":
        assert torch.equal(k[0, 497:500], one.k[0])


@pytest.mark.parametrize("new", (1, 70))
def test_half_a_billion_keys(ops, new):
    """The same page over and over, then five keys that outweigh all before them: scores of 40, where 2^29 others have 1.1 at most
    (0.5 * 64 * 0.03 rounded, + 16 times a step), so together 2^29 e^-38.9 / 5 < 2e-9 of the weight.  Probabilities of the five are
    1 of a sum of 5; the result rounds to 2^-11 of itself."""
    page, dim, last = 1 << 20, 64, 5
    g = torch.Generator().manual_seed(6)
    k = (torch.rand(2 * page, dim, generator=g) * 0.06 - 0.03).half()
    v = torch.randn(2 * page, dim, generator=g).half()
    k[page:page + last] = 2.5
    table = torch.zeros(1, 513, dtype=torch.int32, device="cuda")
    table[0, 512] = 1
    lengths = torch.tensor([512 * page + last], dtype=torch.int32, device="cuda")
    caches = [x.view(2, page, 1, dim).cuda() for x in (k, v)]
    got = ops.flash_attn_paged_func(torch.full((1, new, 1, dim), 2.0).half().cuda(), *caches, table, lengths).cpu().double()
    want = v[page:page + last].double().mean(0)
    assert ((got - want).abs() <= want.abs() * 2.0 ** -11 + 2.0 ** -20 * 4).all()


@pytest.mark.parametrize("cache", paged.CACHES)
def test_a_conversation(ops, cache):
    """Prompts in chunks, then single tokens, as a server does it: written, attended to, and against flash_attn_func over the
    whole of it."""
    dim, heads, page = 64, 4, 16
    g = torch.Generator(device="cuda").manual_seed(0)
    total, steps = [150, 97], [(60, 40), (70, 50), (1, 1), (1, 1), (18, 5)]
    q, k, v = ([torch.randn(m, heads, dim, generator=g, device="cuda").half() for m in total] for _ in range(3))
    pages = 40
    kind = torch.float16 if cache == "same" else torch.float8_e4m3fn
    k_cache, v_cache = (torch.empty(pages, page, heads, dim, device="cuda", dtype=kind) for _ in range(2))
    scales = {"k_scale": None, "v_scale": None}
    if cache == "e4m3":
        scales = {n: torch.empty(pages, page, heads, device="cuda", dtype=torch.float8_e8m0fnu) for n in scales}
    table = torch.randperm(pages, generator=g, device="cuda").int().view(2, -1)
    done, outs = [0, 0], [[], []]
    for step in steps:
        cu = torch.tensor([0, step[0], sum(step)], dtype=torch.int32, device="cuda")
        pick = lambda x: torch.cat([x[b][done[b]:done[b] + step[b]] for b in range(2)])
        lengths = torch.tensor([d + s for d, s in zip(done, step)], dtype=torch.int32, device="cuda")
        ops.kv_cache_write(pick(k), pick(v), k_cache, v_cache, table, lengths, cu_seqlens=cu, **scales)
        out = ops.flash_attn_paged_func(pick(q), k_cache, v_cache, table, lengths, None, True, cu_seqlens=cu, max_seqlen=max(step), **scales)
        for b in range(2):
            outs[b].append(out[cu[b]:cu[b + 1]])
            done[b] += step[b]
    held_k, held_v = ops.kv_cache_read(k_cache, v_cache, table, lengths, max(total), **scales)
    for b in range(2):
        kb, vb = held_k[b:b + 1, :total[b]].contiguous(), held_v[b:b + 1, :total[b]].contiguous()
        if cache == "same":
            assert torch.equal(kb[0], k[b]) and torch.equal(vb[0], v[b])
        got = torch.cat(outs[b])
        want, weight, size = po.attention(q[b], kb[0], vb[0], dim ** -0.5, True)
        tolerance = po.attention_tolerance(torch.float16, dim, want, weight, size, total[b], float(vb.abs().max()))
        assert ((got.cpu().double() - want).abs() <= tolerance).all()
        whole = ops.flash_attn_func(q[b][None], kb, vb, None, True)[0]
        assert ((got.double() - whole.double()).abs().cpu() <= 2 * tolerance).all()


def test_side_streams(ops):
    """Two streams at a time, each with a workspace of its own."""
    batches = [paged.Batch([3000, 2000], 1, 2, 4, 128, 16, torch.float16, seed=s) for s in (1, 2)]
    alone = [ops.flash_attn_paged_func(b.q, *b.args()) for b in batches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in batches]
    outs = [[], []]
    for _ in range(5):
        for b, s, o in zip(batches, streams, outs):
            with torch.cuda.stream(s):
                o.append(ops.flash_attn_paged_func(b.q, *b.args()))
    torch.cuda.synchronize()
    for want, got in zip(alone, outs):
        assert all(torch.equal(want, x) for x in got)


@pytest.mark.parametrize("cache", paged.CACHES)
def test_capture_and_replay(ops, cache):
    """A captured step of writing and attention follows the lengths, pages and values that are there at each replay; two graphs
    replayed in turn do not disturb each other."""
    batch = paged.Batch([700, 900, 40], 1, 2, 4, 64, 16, torch.bfloat16, cache, seed=6)
    chunk = paged.Batch([700, 900, 140], [60, 1, 90], 2, 4, 64, 16, torch.bfloat16, cache, packed=True, seed=7)

    def step(b):
        ops.kv_cache_write(b.k, b.v, *b.args(), cu_seqlens=b.cu_seqlens, **b.scales())
        return ops.flash_attn_paged_func(b.q, *b.args(), None, True, cu_seqlens=b.cu_seqlens, **b.scales())

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for b in (batch, chunk):
            step(b)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for b in (batch, chunk):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(b))
        graphs.append(graph)
    for n in range(4):
        for b, graph, out in zip((batch, chunk), graphs, outs):
            for x in (b.q, b.k, b.v):
                x.normal_()
            b.cache_seqlens -= 13 * n
            out.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            replayed = out.clone()
            assert torch.equal(replayed, step(b))
            b.lengths = b.cache_seqlens.tolist()
            want, tolerance = b.expected(True)
            assert ((replayed.cpu().double() - want).abs() <= tolerance).all()


def test_repeatable(ops):
    for batch in (paged.Batch([5000, 100, 7000], 1, 2, 8, 128, 16, torch.bfloat16, "e4m3"), paged.Batch([5000, 300], 200, 2, 4, 128, 16)):
        first = ops.flash_attn_paged_func(batch.q, *batch.args(), None, True, **batch.scales())
        for _ in range(3):
            assert torch.equal(first, ops.flash_attn_paged_func(batch.q, *batch.args(), None, True, **batch.scales()))


def test_gradients_are_refused(ops):
    batch = paged.Batch([40], 1)
    q = batch.q.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradients"):
        ops.flash_attn_paged_func(q, *batch.args())
    with torch.no_grad():
        assert torch.equal(ops.flash_attn_paged_func(q, *batch.args()), ops.flash_attn_paged_func(batch.q, *batch.args()))
    with pytest.raises(RuntimeError, match="no gradients"):
        ops.kv_cache_write(batch.k.clone().requires_grad_(), batch.v, *batch.args())


def test_outputs_that_overlap_inputs_are_refused(ops):
    batch = paged.Batch([40], 1, 2, 2)
    with pytest.raises(RuntimeError, match="memory"):
        ops.flash_attn_paged_func(batch.q, *batch.args(), out=batch.q)


def test_caches_that_overlap_are_refused(ops):
    batch = paged.Batch([40], 1, 2, 1)
    _, v_cache, *rest = batch.args()
    with pytest.raises(RuntimeError, match="memory"):
        ops.kv_cache_write(batch.k, batch.v, v_cache, v_cache, *rest)
    row = v_cache[:1, :1]  # of a token, as k of one
    with pytest.raises(RuntimeError, match="memory"):
        ops.kv_cache_write(row, batch.v, *batch.args())
    batch = paged.Batch([40], 1, 2, 1, cache="e4m3")
    with pytest.raises(RuntimeError, match="memory"):
        ops.kv_cache_write(batch.k, batch.v, *batch.args(), k_scale=batch.v_scale, v_scale=batch.v_scale)


def test_written_tensors_count_as_changed(ops):
    """A graph that saved one of them must not use it afterwards."""
    batch = paged.Batch([40], 1, cache="e4m3")
    tensors = [batch.k_cache, batch.v_cache, batch.k_scale, batch.v_scale]
    before = [x._version for x in tensors]
    ops.kv_cache_write(batch.k, batch.v, *batch.args(), **batch.scales())
    assert all(x._version > n for x, n in zip(tensors, before))
    out = torch.empty_like(batch.q)
    leaf = torch.ones_like(out, requires_grad=True)
    product = (leaf * out).sum()
    ops.flash_attn_paged_func(batch.q, *batch.args(), out=out, **batch.scales())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.backward()
    with torch.inference_mode():  # tensors without a version
        ops.flash_attn_paged_func(batch.q, *batch.args(), out=torch.empty_like(batch.q), **batch.scales())


def off_boundary(x):
    """The same values, contiguous, one element behind a 16-byte boundary."""
    room = torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)
    y = room[1:].view(x.shape)
    y.copy_(x)
    assert y.is_contiguous() and y.data_ptr() % 16 == x.element_size()
    return y


@pytest.mark.parametrize("packed", (False, True))
@pytest.mark.parametrize("new", (1, 40))
def test_contiguous_tokens_off_16_byte_boundaries(ops, new, packed):
    batch = paged.Batch([130, 77, 600], [new] * 3 if packed else new, 2, 2, 64, 16, torch.float16, packed=packed, seed=11)
    other = paged.Batch([130, 77, 600], [new] * 3 if packed else new, 2, 2, 64, 16, torch.float16, packed=packed, seed=11)
    ops.kv_cache_write(batch.k, batch.v, *batch.args(), cu_seqlens=batch.cu_seqlens)
    ops.kv_cache_write(off_boundary(batch.k), off_boundary(batch.v), *other.args(), cu_seqlens=batch.cu_seqlens)
    for name in ("k_cache", "v_cache"):
        assert torch.equal(getattr(batch, name).view(torch.int16), getattr(other, name).view(torch.int16))
    batch.q = off_boundary(batch.q)
    check_attention(ops, batch, True)


def any_stride(x, dim):
    """The same values, with a stride of a dimension of size 1 that no other one has a multiple of."""
    strides = list(x.stride())
    strides[dim] = 1
    y = x.as_strided(x.shape, strides)
    assert x.shape[dim] == 1 and torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))
    return y


@pytest.mark.parametrize("cache", paged.CACHES)
@pytest.mark.parametrize("new", (1, 40))
def test_strides_of_dimensions_of_size_1(ops, new, cache):
    """They say nothing: one head, one page, one sequence, one token."""
    batch = paged.Batch([130], new, 1, 1, 64, 160, torch.float16, cache, seed=12)
    ids = batch.page_table[0, :1].long()
    for name in ("k_cache", "v_cache", "k_scale", "v_scale"):
        x = getattr(batch, name)
        if x is not None:
            x = x.view(torch.uint8)[ids].view(x.dtype)
            setattr(batch, name, any_stride(any_stride(x, 2), 0))
    batch.page_table[0, 0] = 0
    for dim in (0, 2) + ((1,) if new == 1 else ()):
        batch.q, batch.k, batch.v = (any_stride(x, dim) for x in (batch.q, batch.k, batch.v))
    check_attention(ops, batch, True)
    ops.kv_cache_write(batch.k, batch.v, *batch.args(), **batch.scales())
    check_attention(ops, batch, True)
    k, _ = ops.kv_cache_read(*batch.args(), 130, **batch.scales())
    if cache == "same":
        assert torch.equal(k[0, -new:], batch.k[0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", (64, 128))
@pytest.mark.parametrize("less", (12, 20, 26))
@pytest.mark.parametrize("new,group", [(1, 4), (5, 5), (20, 4)])
def test_values_of_very_different_scales(ops, new, group, less, dim, dtype):
    """Out of 8 bits, rows of values up to 57344 in one half of the features beside rows 2^-less as large in the other half, which
    are not to be lost.  Beside what every call is off by, blocks of few rows round p_j 2^e_j to fp16 with steps of 2^-24, where the largest
    is 2^14, before it is multiplied with the value's 8 bits y_j: half a step is 2^-39 of the largest.  Blocks of many rows round p_j the
    same where the largest is 1 or more: 2^-25, times the value."""
    batch = paged.Batch([300, 40, 3000], new, 2, group, dim, 16, dtype, "e4m3", seed=less)
    g = torch.Generator().manual_seed(less)
    shape = batch.v_cache.shape
    rows = (torch.rand(shape, generator=g) * 0.75 + 0.25) * 57344
    small = (torch.rand(shape[:3], generator=g) < 0.5)[..., None]
    first = torch.arange(dim) < dim // 2
    rows = torch.where(small, rows * 2.0 ** -less, rows).masked_fill(small == first, 0.0).to(dtype)
    y, e = po.to_e4m3(rows)
    batch.v_cache.copy_(y.float().to(torch.float8_e4m3fn))
    batch.v_scale.view(torch.uint8).copy_((e + 127).to(torch.uint8))
    results = po.paged_attention(batch.q, *batch.args(), None, True, **batch.scales())
    want = results[0]
    tolerance = po.attention_tolerance(dtype, dim, *results, 3000, 0.0)
    if dtype == torch.float16:
        for b, m in enumerate(batch.lengths):
            k = po.held(batch.k_cache, batch.k_scale, batch.page_table, b, m)
            ids, slots = po.places(batch.page_table, 16, b, torch.arange(m))
            for h in range(batch.heads):
                s = batch.q[b, :, h].cpu().double() @ k[:, h // group].t() * dim ** -0.5
                p = torch.softmax(s.masked_fill(torch.arange(m) > m - new + torch.arange(new)[:, None], -torch.inf), -1)
                ys, es = y[ids, slots, h // group], e[ids, slots, h // group]
                if new * group <= 32:
                    tolerance[b, :, h] += 2.0 ** -39 * (p * torch.pow(2.0, es.double())).amax(-1, keepdim=True) * ys.abs().sum(0)
                else:
                    tolerance[b, :, h] += 2.0 ** -25 * p.amax(-1, keepdim=True) * (ys * torch.pow(2.0, es.double())[:, None]).abs().sum(0)
    got = ops.flash_attn_paged_func(batch.q, *batch.args(), None, True, **batch.scales()).cpu().double()
    assert ((got - want).abs() <= tolerance).all(), float(((got - want).abs() / tolerance).max())


@pytest.mark.parametrize("cache", paged.CACHES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", (64, 128))
@pytest.mark.parametrize("new,group", [(1, 4), (3, 2), (7, 4), (9, 9), (50, 1), (200, 2)])
def test_values_of_later_tokens_do_not_matter(ops, new, group, dim, dtype, cache):
    """Infinite and NaN values of the last three keys: rows that see them have them, with all other features bit by bit as without; the
    others do not change at all."""
    batch = paged.Batch([5, 31, 32, 33, 64, 65, 130, 333, 4100], new, 2, group, dim, 16, dtype, cache, seed=new)
    for causal in (True, False):
        want = ops.flash_attn_paged_func(batch.q, *batch.args(), None, causal, **batch.scales())
        assert torch.isfinite(want).all()
        clean = batch.v_cache.clone()
        for back, first, end, value in ((3, 0, 16, "inf"), (2, 8, 24, "-inf"), (1, 20, 32, "nan")):
            for b, m in enumerate(batch.lengths):
                ids, slots = po.places(batch.page_table, 16, b, torch.tensor([m - back]))
                row = batch.v_cache[int(ids), int(slots)]
                if cache == "same":
                    row[:, first:end] = float(value)
                else:  # no infinities
                    row.view(torch.uint8)[:, first:end] = 0x7f if back > 1 else 0xff
                sees = torch.arange(new, device="cuda") + m - new >= m - back if causal else torch.ones(new, dtype=torch.bool, device="cuda")
                want[b, sees, :, first:end] += float(value if cache == "same" else "nan")
        got = ops.flash_attn_paged_func(batch.q, *batch.args(), None, causal, **batch.scales())
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.masked_fill(got.isnan(), 0), want.masked_fill(want.isnan(), 0))
        batch.v_cache.copy_(clean)


@pytest.mark.parametrize("dim", (64, 128))
@pytest.mark.parametrize("new,group", [(1, 4), (40, 2)])
def test_values_of_later_tokens_in_packed_batches(ops, new, group, dim):
    """Single tokens and chunks, split over work groups: tokens before the spoilt one as without it."""
    batch = paged.Batch([9000, 700, 300], [new, 1, 65], 2, group, dim, 32, torch.bfloat16, packed=True, seed=dim)
    want = ops.flash_attn_paged_func(batch.q, *batch.args(), None, True, cu_seqlens=batch.cu_seqlens)
    ends = batch.cu_seqlens.tolist()[1:]
    for b, m in enumerate(batch.lengths):
        ids, slots = po.places(batch.page_table, 32, b, torch.tensor([m - 1]))
        batch.v_cache[int(ids), int(slots)] = float("inf")
        want[ends[b] - 1] = float("inf")
    got = ops.flash_attn_paged_func(batch.q, *batch.args(), None, True, cu_seqlens=batch.cu_seqlens)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", (64, 128))
@pytest.mark.parametrize("new,group,packed", [(1, 4, False), (6, 4, False), (40, 2, False), (20, 3, True)])
def test_scores_of_minus_infinity(ops, new, group, packed, dim, dtype):
    """Keys with such scores have no weight beside others; a softmax over none but those is NaN, also where parts of it are joined, while a
    row that sees no key is zero."""
    lengths = [40, 300, 9000, 40, 300, 9000, 9000, max(new // 2, 1), 0]
    batch = paged.Batch(lengths, [new] * len(lengths) if packed else new, 2, group, dim, 16, dtype, packed=packed, seed=new)
    batch.q.abs_()
    none = (0, 1, 2)  # sequences without any other scores
    for b, m in enumerate(lengths):
        at = torch.arange(m) if b in none else torch.arange(0, m, 2) if b < 6 else torch.arange(m // 2) if b == 6 else torch.arange(0)
        ids, slots = po.places(batch.page_table, 16, b, at)
        batch.k_cache[ids.cuda(), slots.cuda(), :, 3] = -float("inf")
    got = ops.flash_attn_paged_func(batch.q, *batch.args(), None, False, cu_seqlens=batch.cu_seqlens).cpu().double()
    got = got.view(len(lengths), new, batch.heads, dim)
    causal = ops.flash_attn_paged_func(batch.q, *batch.args(), None, True, cu_seqlens=batch.cu_seqlens).cpu().double()
    causal = causal.view(len(lengths), new, batch.heads, dim)
    for b, m in enumerate(lengths):
        q = batch.q.view(len(lengths), new, batch.heads, dim)[b]
        k, v = (po.held(c, None, batch.page_table, b, m) for c in (batch.k_cache, batch.v_cache))
        if b in none:
            assert got[b].isnan().all()
            first = max(new - m, 0)
            assert causal[b, first:].isnan().all() and not causal[b, :first].any()
            continue
        want, weight, _ = po.attention(q, k, v, dim ** -0.5, False)
        size = po.attention(q, k.masked_fill(k.isinf(), 0), v, dim ** -0.5, False)[2]
        v_max = float(v.abs().max()) if m else 0.0
        assert ((got[b] - want).abs() <= po.attention_tolerance(dtype, dim, want, weight, size, max(m, 1), v_max)).all()
