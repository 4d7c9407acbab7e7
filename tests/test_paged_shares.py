"""Attention over a paged cache with every tile of keys in evidence: keys are zero, so that all have the same weight, and values are zero
but for one in each tile of 64, in a feature that goes by the tile and the head.  What is expected is a closed form, sums are exact in
32 bits, and a tile that is lost or counted twice shows."""
import ctypes

import pytest
import torch

import abi
import paged
from oracle import paged_oracle as po
from test_paged_host import BatchOf, Cache, Strides, lib  # noqa: F401

pytestmark = pytest.mark.gpu

TILE = 64


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.fail("this test needs a GPU")
    import flash_attn_v100
    return flash_attn_v100


class Marked(paged.Batch):
    def __init__(self, lengths, new, **more):
        super().__init__(lengths, new, **more)
        eight = self.cache == "e4m3"
        for b, m in enumerate(lengths):
            ids, slots = (x.cuda() for x in po.places(self.page_table.cpu(), self.page, b, torch.arange(m)))
            for cache in (self.k_cache, self.v_cache):
                (cache.view(torch.uint8) if eight else cache)[ids, slots] = 0
            tile, at, power = self.markers(m)
            for h in range(self.k_cache.shape[2]):
                where = ids[at], slots[at], h, self.feature(tile, h).cuda()
                if eight:
                    self.v_cache.view(torch.uint8)[where] = 0x38  # 1
                    self.v_scale.view(torch.uint8)[where[:3]] = (127 + power).to(torch.uint8).cuda()
                else:
                    self.v_cache[where] = torch.pow(2.0, power.double()).to(self.dtype).cuda()

    def markers(self, keys):
        """(tile, its marked key, that value's power of two)"""
        tile = torch.arange(-(-keys // TILE))
        return tile, torch.minimum(TILE * tile + 7 * tile % TILE, torch.tensor(keys - 1)), 8 + tile % 3

    def feature(self, tile, kv_head):
        return (tile + 5 * kv_head) % self.dim

    def check(self, got, causal):
        """got is what is expected but for roundings: of the result half a step, of 1 / sum and of scales by powers of two 2^-22 each."""
        rounding = torch.finfo(self.dtype).eps / 2
        rounding += 2.0 ** -20
        for b, (first, end) in enumerate(po.sequences(self.cu_seqlens, len(self.lengths), self.q.shape[-3])):
            rows = got.view(-1, *got.shape[-2:])[first:end].cpu().double()
            m, n = self.lengths[b], end - first
            tile, at, power = self.markers(m)
            value = torch.pow(2.0, power.double())
            for i in sorted({0, 1, n // 2, n - 2, n - 1} & set(range(n))):
                sees = max(m - n + i + 1, 0) if causal else m
                for h in range(self.heads):
                    f = self.feature(tile, h // (self.heads // self.k_cache.shape[2]))
                    seen = at < sees
                    total = torch.zeros(self.dim, dtype=torch.float64).index_add(0, f[seen], value[seen])
                    want = total / max(sees, 1)
                    off = (rows[i, h] - want).abs()
                    assert (off <= rounding * want).all(), (b, i, h, int(off.argmax()), float((off / want.clamp(min=1e-9)).max()))
                    # each tile is a larger share of its feature than two roundings, less what it is of all keys
                    share = value[seen] / total[f[seen]] - TILE / max(sees, TILE)
                    assert len(share) < 3 or share.min() > 2 * rounding


@pytest.mark.parametrize("cache", paged.CACHES)
@pytest.mark.parametrize("dim", (64, 128))
@pytest.mark.parametrize("lengths,new,group,kv_heads", [
    ([150000], 1, 3, 1), ([70000, 40, 90000], 1, 2, 1), ([33000, 35000], 2, 1, 2), ([3000] * 66, 1, 1, 1), ([200000], 33, 1, 1),
    ([40000, 45000, 60], 40, 4, 2), ([41000], 200, 2, 1), ([9000] * 18, 35, 1, 1), ([2000, 1900], 1500, 2, 1), ([5000, 1, 64, 700], 17, 1, 3)])
def test_every_tile_counts_once(ops, lengths, new, group, kv_heads, dim, cache):
    batch = Marked(lengths, new, kv_heads=kv_heads, group=group, dim=dim, page=64, cache=cache, seed=dim)
    for causal in (True, False):
        batch.check(ops.flash_attn_paged_func(batch.q, *batch.args(), None, causal, **batch.scales()), causal)


@pytest.mark.parametrize("cache", paged.CACHES)
@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
def test_every_tile_counts_once_in_packed_batches(ops, dtype, cache):
    batch = Marked([9000, 12000, 300, 7000, 1, 2500], [300, 1, 300, 1, 1, 5], kv_heads=2, group=2, dim=128, page=48, dtype=dtype, cache=cache,
                   packed=True, seed=3)
    for causal in (True, False):
        batch.check(ops.flash_attn_paged_func(batch.q, *batch.args(), None, causal, cu_seqlens=batch.cu_seqlens, **batch.scales()), causal)


def way_taken(lib, b, causal):
    """(result, how a batch is shared out), by the table of parts that a call leaves in its workspace: a whole item has one part; parts of
    different items lie in different stretches or, where stretches do not end with items, some in the same."""
    kinds = {torch.float16: 0, torch.bfloat16: 1}
    strides = lambda x: Strides(*x.stride()[:3]) if x is not None else Strides(0, 0, 0)
    pointer = lambda x: None if x is None else x.data_ptr()
    caches = b.k_cache, b.v_cache, b.k_scale, b.v_scale
    c = Cache(*map(pointer, caches), *map(strides, caches), *b.k_cache.shape, 2 if b.cache == "e4m3" else kinds[b.dtype], kinds[b.dtype])
    tokens = b.q.shape[-3]
    t = BatchOf(b.page_table.data_ptr(), b.page_table.stride(0), b.page_table.shape[1], b.cache_seqlens.data_ptr(), pointer(b.cu_seqlens),
                len(b.lengths), tokens)
    size = lib.paged_mha_forward_workspace_bytes(c, t, b.heads, 0)
    workspace = torch.empty(size, dtype=torch.uint8, device="cuda")
    out = torch.empty_like(b.q)
    q_strides = abi.Strides(b.q.stride(0) if b.cu_seqlens is None else 0, *b.q.stride()[-3:-1])
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.paged_mha_forward(c, t, b.q.data_ptr(), ctypes.byref(q_strides), out.data_ptr(), b.heads, 0, b.dim ** -0.5, causal, 0,
                                 workspace.data_ptr(), size, stream) == 0
    rows = out.numel() // b.dim
    groups = 512
    place_rows = (size - 8 * rows) // (2 * groups * (b.dim * 4 + 8))
    table = workspace[2 * groups * place_rows * (b.dim * 4 + 8):].view(torch.int32).view(rows, 2).cpu()
    spans = sorted({(int(x) // (2 * place_rows), int(n)) for x, n in table[table[:, 1] > 1]})
    if not spans:
        return out, "whole"
    return out, "parts" if all(x + n <= y for (x, n), (y, _) in zip(spans, spans[1:])) else "stretches"


@pytest.mark.parametrize("cache", paged.CACHES)
@pytest.mark.parametrize("way,lengths,new,group,kv_heads", [
    ("parts", [4000, 3500, 4096, 3000], 1, 4, 2), ("parts", [8192], 200, 4, 1),
    ("stretches", [3000 + 40 * i for i in range(40)], 1, 4, 4), ("stretches", [900 + 100 * i for i in range(70)], 1, 2, 1),
    ("whole", [1024] * 4, 1024, 4, 2), ("parts", [500] * 20, 20, 1, 8), ("whole", [500] * 64, 20, 1, 8)])
def test_ways_of_sharing_out(lib, cache, way, lengths, new, group, kv_heads):  # noqa: F811
    """Each of the three, as the kernels choose them by their model of time."""
    batch = Marked(lengths, new, kv_heads=kv_heads, group=group, dim=128, page=64, cache=cache, seed=8)
    out, taken = way_taken(lib, batch, True)
    batch.check(out, True)
    assert taken == way
