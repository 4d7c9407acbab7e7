"""Batches over a paged cache, for the tests: made on the CPU from a seed, moved to a device where one is named."""
import torch

from oracle import paged_oracle as po

CACHES = ("same", "e4m3")


class Batch:
    """Sequences of given lengths with their pages scattered over a cache that has more of them; everything that belongs to no
    sequence (other pages, slots behind the last key) holds NaN."""

    def __init__(self, lengths, new, kv_heads=2, group=2, dim=64, page=16, dtype=torch.float16, cache="same", packed=False, seed=0,
                 device="cuda", extra_columns=1, layout="pages", tail=0):
        g = torch.Generator().manual_seed(seed)
        self.lengths, self.dtype, self.dim, self.page, self.cache = lengths, dtype, dim, page, cache
        counts = list(new) if packed else [new] * len(lengths)
        self.counts = counts
        normal = lambda *s: torch.randn(s, generator=g).to(dtype)
        used = [-(-max(m, 0) // page) for m in lengths]
        pages = sum(used) + 2
        order = torch.randperm(pages, generator=g).int()
        table = torch.full((len(lengths), max(max(used), 1) + extra_columns), -1, dtype=torch.int32)
        at = 0
        for b, m in enumerate(used):
            table[b, :m] = order[at:at + m]
            at += m
        self.heads = kv_heads * group
        lead = (sum(counts) + tail,) if packed else (len(lengths), new)
        self.q = normal(*lead, self.heads, dim).to(device)
        self.k, self.v = (normal(*lead, kv_heads, dim).to(device) for _ in range(2))
        self.page_table = table.to(device)
        self.cache_seqlens = torch.tensor(lengths, dtype=torch.int32, device=device)
        self.cu_seqlens = None
        if packed:
            self.cu_seqlens = torch.tensor([0] + counts, dtype=torch.int32).cumsum(0).int().to(device)
        self.rows = {}
        for name in "kv":
            rows = normal(pages, page, kv_heads, dim)
            live = torch.zeros(pages, page, dtype=torch.bool)
            for b, m in enumerate(lengths):
                ids, slots = po.places(table, page, b, torch.arange(max(m, 0)))
                live[ids, slots] = True
            if cache == "e4m3":
                values, e = po.to_e4m3(rows)
                data = values.float().to(torch.float8_e4m3fn)
                scale = (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)
                data.view(torch.uint8)[~live] = 0x7f
                scale.view(torch.uint8)[~live] = 0xff
                scale = self._placed(scale, layout, device)
            else:
                data, scale = rows, None
                data[~live] = float("nan")
            setattr(self, name + "_cache", self._placed(data, layout, device))
            setattr(self, name + "_scale", scale)

    @staticmethod
    def _placed(x, layout, device):
        """The same values with other strides: pages of heads of slots, or beside something else in a larger tensor."""
        if layout == "heads":
            return x.transpose(1, 2).contiguous().to(device).transpose(1, 2)
        if layout == "beside":
            both = torch.stack([x.view(torch.uint8) ^ 0x55, x.view(torch.uint8)], 1).to(device)
            return both.view(x.dtype)[:, 1]
        return x.to(device)

    def scales(self):
        return {"k_scale": self.k_scale, "v_scale": self.v_scale}

    def args(self):
        return self.k_cache, self.v_cache, self.page_table, self.cache_seqlens

    def expected(self, causal, scale=None):
        """(result, tolerance) of flash_attn_paged_func, by the oracle."""
        results = po.paged_attention(self.q, *self.args(), scale, causal, self.cu_seqlens, **self.scales())
        keys = max(max(self.lengths), 1)
        v_max = max([float(po.held(self.v_cache, self.v_scale, self.page_table, b, m).abs().max()) for b, m in enumerate(self.lengths) if m > 0],
                    default=0.0)
        return results[0], po.attention_tolerance(self.dtype, self.dim, *results, keys, v_max)
