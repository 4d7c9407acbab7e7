"""CPU tests of the paged cache's host side: what the library exports, refusals of the C interface and of the Python calls, and
how work is shared out.  No kernel runs."""
import ctypes
import inspect
import os
import re
import subprocess

import pytest
import torch

import abi
import paged
from oracle import paged_oracle as po

HEADER = os.path.join(abi.ROOT, "include", "paged_mha.h")
LIB = os.path.join(os.path.dirname(abi.LIB_PATH), "libpaged_mha.so")
CSRC = os.path.join(abi.ROOT, "flash-attention-v100_amd", "csrc")
ERR_BAD_TYPE, ERR_BAD_PAGE_SIZE, ERR_BAD_GROUP, ERR_WORKSPACE = -11, -12, -13, -14

vp, i32, i64, sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_size_t


class Strides(ctypes.Structure):
    _fields_ = [("page", i64), ("slot", i64), ("head", i64)]


class Cache(ctypes.Structure):
    _fields_ = [("key", vp), ("value", vp), ("key_scale", vp), ("value_scale", vp), ("key_strides", Strides),
                ("value_strides", Strides), ("key_scale_strides", Strides), ("value_scale_strides", Strides), ("pages", i32),
                ("page_size", i32), ("kv_head", i32), ("d", i32), ("cache_type", i32), ("type", i32)]


class BatchOf(ctypes.Structure):
    _fields_ = [("page_table", vp), ("table_stride", i64), ("table_width", i32), ("cache_seqlens", vp), ("cu_seqlens", vp),
                ("batch", i32), ("tokens", i32)]


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(LIB)
    cache, batch, strides = ctypes.POINTER(Cache), ctypes.POINTER(BatchOf), ctypes.POINTER(abi.Strides)
    lib.paged_mha_write.argtypes = [cache, batch, vp, strides, vp, strides, vp]
    lib.paged_mha_read.argtypes = [cache, batch, i32, vp, vp, vp]
    lib.paged_mha_forward_workspace_bytes.argtypes = [cache, batch, i32, i32]
    lib.paged_mha_forward_workspace_bytes.restype = sz
    lib.paged_mha_forward.argtypes = [cache, batch, vp, strides, vp, i32, i32, ctypes.c_float, i32, i32, vp, sz, vp]
    lib.paged_mha_error_string.argtypes = [i32]
    lib.paged_mha_error_string.restype = ctypes.c_char_p
    return lib


def test_exports_every_declared_symbol(lib):
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(paged_mha_\w+)\s*\(", text)))
    assert names == ["paged_mha_error_string", "paged_mha_forward", "paged_mha_forward_workspace_bytes", "paged_mha_read",
                     "paged_mha_write"]
    for name in names:
        assert hasattr(lib, name), name


def test_error_strings(lib):
    codes = [0, *range(-1, -9, -1), *range(-11, -15, -1)]
    texts = {lib.paged_mha_error_string(c) for c in codes}
    assert len(texts) == len(codes) and b"unknown error" not in texts
    assert lib.paged_mha_error_string(-99) == b"unknown error"


P = 0x10000  # a pointer that no refused call follows


def problem(**changes):
    """A valid problem, but for the changes."""
    d, heads, page = 128, 4, 16
    dense = lambda: Strides(page * heads * d, heads * d, d)
    c = Cache(P, P, None, None, dense(), dense(), Strides(page * heads, heads, 1), Strides(page * heads, heads, 1), 10, page, heads, d, 0, 0)
    b = BatchOf(P, 8, 8, P, None, 3, 5)
    call = {"q": P, "q_st": abi.Strides(5 * 8 * d, 8 * d, d), "o": P, "head": 8, "max_new": 0, "scale": 1.0, "ws": P, "bytes": 1 << 40}
    for name, value in changes.items():
        where = next((x for x in (c, b) if hasattr(x, name)), None)
        if where is None:
            assert name in call
            call[name] = value
        else:
            setattr(where, name, value)
    return c, b, call


CHANGES = [
    ({"key": None}, abi.ERR_NULL_POINTER), ({"page_table": None}, abi.ERR_NULL_POINTER), ({"cache_seqlens": None}, abi.ERR_NULL_POINTER),
    ({"type": 2}, ERR_BAD_TYPE), ({"cache_type": 1}, ERR_BAD_TYPE), ({"cache_type": 3}, ERR_BAD_TYPE),
    ({"cache_type": 2}, abi.ERR_NULL_POINTER), ({"key_scale": P}, ERR_BAD_TYPE), ({"d": 96}, abi.ERR_BAD_HEAD_DIM),
    ({"pages": 0}, abi.ERR_BAD_SHAPE), ({"kv_head": 0}, abi.ERR_BAD_SHAPE), ({"batch": 0}, abi.ERR_BAD_SHAPE),
    ({"tokens": 0}, abi.ERR_BAD_SHAPE), ({"table_width": 0}, abi.ERR_BAD_SHAPE), ({"table_stride": -1}, abi.ERR_BAD_SHAPE),
    ({"page_size": 8}, ERR_BAD_PAGE_SIZE), ({"page_size": 0}, ERR_BAD_PAGE_SIZE), ({"page_size": 17}, ERR_BAD_PAGE_SIZE),
    ({"table_width": 1 << 26}, abi.ERR_TOO_LARGE), ({"batch": 1 << 21}, abi.ERR_TOO_LARGE),
    ({"key_strides": Strides(-128, 128, 128)}, abi.ERR_BAD_STRIDE), ({"key_strides": Strides(1, 128, 128)}, abi.ERR_BAD_STRIDE),
    ({"value_strides": Strides(0, 1 << 24, 128)}, abi.ERR_BAD_STRIDE), ({"value_strides": Strides(0, 128, 4)}, abi.ERR_BAD_STRIDE),
    ({"key": P + 8}, abi.ERR_MISALIGNED), ({"value": P + 2}, abi.ERR_MISALIGNED),
]


@pytest.mark.parametrize("changes,code", CHANGES)
def test_refusals_of_every_call(lib, changes, code):
    c, b, call = problem(**changes)
    st = ctypes.byref(call["q_st"])
    assert lib.paged_mha_write(c, b, P, st, P, st, None) == code
    assert lib.paged_mha_read(c, b, 100, P, P, None) == code
    assert lib.paged_mha_forward(c, b, P, st, P, 8, 0, 1.0, 1, 0, P, 1 << 40, None) == code
    assert lib.paged_mha_forward_workspace_bytes(c, b, 8, 0) == 0


@pytest.mark.parametrize("changes,code", [
    ({"q": None}, abi.ERR_NULL_POINTER), ({"o": None}, abi.ERR_NULL_POINTER), ({"head": 6}, ERR_BAD_GROUP), ({"head": 0}, abi.ERR_BAD_SHAPE),
    ({"max_new": -1}, abi.ERR_BAD_SHAPE), ({"scale": float("inf")}, abi.ERR_BAD_SCALE), ({"scale": float("nan")}, abi.ERR_BAD_SCALE),
    ({"q_st": abi.Strides(0, 4, 128)}, abi.ERR_BAD_STRIDE), ({"q_st": abi.Strides(0, -8, 128)}, abi.ERR_BAD_STRIDE),
    ({"q": P + 2}, abi.ERR_MISALIGNED), ({"o": P + 8}, abi.ERR_MISALIGNED), ({"tokens": 1 << 26}, abi.ERR_TOO_LARGE),
    ({"ws": None, "table_width": 1000}, abi.ERR_NULL_POINTER), ({"bytes": 100, "table_width": 1000}, ERR_WORKSPACE),
    ({"ws": P + 4, "table_width": 1000}, abi.ERR_MISALIGNED)])
def test_refusals_of_attention(lib, changes, code):
    c, b, call = problem(**changes)
    assert lib.paged_mha_forward(c, b, call["q"], ctypes.byref(call["q_st"]), call["o"], call["head"], call["max_new"], call["scale"], 1, 0,
                                 call["ws"], call["bytes"], None) == code


def test_refusals_of_write_and_read(lib):
    c, b, call = problem()
    st, bad = ctypes.byref(call["q_st"]), ctypes.byref(abi.Strides(0, 4, 128))
    assert lib.paged_mha_write(c, b, None, st, P, st, None) == abi.ERR_NULL_POINTER
    assert lib.paged_mha_write(c, b, P, st, P, None, None) == abi.ERR_NULL_POINTER
    assert lib.paged_mha_write(c, b, P, bad, P, st, None) == abi.ERR_BAD_STRIDE
    assert lib.paged_mha_write(c, b, P, st, P + 8, st, None) == abi.ERR_MISALIGNED
    assert lib.paged_mha_read(c, b, 0, P, P, None) == abi.ERR_BAD_SHAPE
    assert lib.paged_mha_read(c, b, 1 << 29, P, P, None) == abi.ERR_TOO_LARGE
    assert lib.paged_mha_read(c, b, 100, P, None, None) == abi.ERR_NULL_POINTER
    assert lib.paged_mha_read(c, b, 100, P, P + 2, None) == abi.ERR_MISALIGNED


def test_launches_too_large_for_a_grid(lib):
    """Of 256 threads a work group, 2^32 work items in all at most."""
    c, b, call = problem(tokens=1 << 27, batch=1)
    st = ctypes.byref(call["q_st"])
    assert lib.paged_mha_write(c, b, P, st, P, st, None) == abi.ERR_TOO_LARGE
    c, b, call = problem(batch=1 << 20)
    assert lib.paged_mha_read(c, b, 2000, P, P, None) == abi.ERR_TOO_LARGE
    for heads, width in ((64, 8), (512, 1000)):  # a work group for each item; rows that may have parts
        c, b, call = problem(batch=1 << 20, tokens=1, kv_head=heads, table_width=width)
        assert lib.paged_mha_forward_workspace_bytes(c, b, heads, 0) == 0
        assert lib.paged_mha_forward(c, b, P, st, P, heads, 0, 1.0, 1, 0, P, 1 << 40, None) == abi.ERR_TOO_LARGE


def test_sizes_whose_product_wraps(lib):
    for tokens, batch, heads in ((1 << 30, 1 << 18, 1 << 16), (1 << 30, 1 << 20, 1 << 14), ((1 << 31) - 1, 1 << 20, 1 << 16)):
        c, b, call = problem(tokens=tokens, batch=batch, kv_head=heads)
        st = ctypes.byref(call["q_st"])
        assert lib.paged_mha_forward_workspace_bytes(c, b, heads, 0) == 0
        assert lib.paged_mha_forward(c, b, P, st, P, heads, 0, 1.0, 1, 0, P, 1 << 40, None) == abi.ERR_TOO_LARGE
        assert lib.paged_mha_write(c, b, P, st, P, st, None) == abi.ERR_TOO_LARGE


def test_python_signatures():
    import flash_attn_v100 as f
    assert str(inspect.signature(f.flash_attn_paged_func)) == (
        "(q, k_cache, v_cache, page_table, cache_seqlens, softmax_scale=None, causal=False, *, cu_seqlens=None, max_seqlen=None, "
        "k_scale=None, v_scale=None, out=None)")
    assert str(inspect.signature(f.kv_cache_write)) == (
        "(k, v, k_cache, v_cache, page_table, cache_seqlens, *, cu_seqlens=None, k_scale=None, v_scale=None)")
    assert str(inspect.signature(f.kv_cache_read)) == (
        "(k_cache, v_cache, page_table, cache_seqlens, max_seqlen, *, k_scale=None, v_scale=None, dtype=None)")


def call(b, **more):
    """flash_attn_paged_func on a batch's tensors, but for the changes."""
    import flash_attn_v100 as f
    a = {"q": b.q, "k_cache": b.k_cache, "v_cache": b.v_cache, "page_table": b.page_table, "cache_seqlens": b.cache_seqlens,
         "cu_seqlens": b.cu_seqlens, **b.scales(), **more}
    return f.flash_attn_paged_func(**a)


@pytest.mark.parametrize("cache", paged.CACHES)
@pytest.mark.parametrize("change,text", [
    (lambda b: {}, "must be on the GPU"),
    (lambda b: {"q": b.q.float()}, "fp16 or bf16"),
    (lambda b: {"q": b.q[0]}, "4 dimensions"),
    (lambda b: {"q": b.q[:1]}, "batch size of cache_seqlens"),
    (lambda b: {"q": b.q[..., :32]}, "head size of the cache"),
    (lambda b: {"q": b.q[:, :, :3]}, "multiple of the cache's heads"),
    (lambda b: {"q": b.q[:, :0]}, "seqlen must be positive"),
    (lambda b: {"q": b.q[:, :, :0]}, "must have heads"),
    (lambda b: {"k_cache": b.k_cache[0]}, "cache must have 4 dimensions"),
    (lambda b: {"v_cache": b.v_cache[1:]}, "same shape"),
    (lambda b: {"v_cache": b.v_cache.to(torch.float32)}, "same dtype"),
    (lambda b: {"k_cache": b.k_cache.float(), "v_cache": b.v_cache.float(), "k_scale": None, "v_scale": None}, "dtype of the inputs"),
    (lambda b: {"k_cache": b.k_cache[..., ::2], "v_cache": b.v_cache[..., ::2]}, "contiguous last dimension"),
    (lambda b: {"k_cache": b.k_cache[..., :32], "v_cache": b.v_cache[..., :32]}, "head dimension 64 or 128"),
    (lambda b: {"k_cache": b.k_cache[:0], "v_cache": b.v_cache[:0]}, "must not be empty"),
    (lambda b: {"page_table": b.page_table.long()}, "page_table must be int32"),
    (lambda b: {"page_table": b.page_table[0]}, "page_table must have 2 dimensions"),
    (lambda b: {"page_table": b.page_table[:1]}, "a row for each sequence"),
    (lambda b: {"page_table": b.page_table[:, :0]}, "must have columns"),
    (lambda b: {"page_table": b.page_table[:, ::2]}, "contiguous last dimension"),
    (lambda b: {"cache_seqlens": b.cache_seqlens.long()}, "cache_seqlens must be int32"),
    (lambda b: {"cache_seqlens": b.cache_seqlens[:0], "page_table": b.page_table[:0], "q": b.q[:0]}, "batch size must be"),
    (lambda b: {"cu_seqlens": torch.tensor([0, 1, 2], dtype=torch.int32)}, "one element more"),
    (lambda b: {"cu_seqlens": torch.tensor([0, 1, 2, 3], dtype=torch.int32)}, "3 dimensions"),
    (lambda b: {"max_seqlen": 0}, "max_seqlen must be positive"),
    (lambda b: {"out": b.q.float()}, "Output must have the same dtype"),
    (lambda b: {"out": b.q[:, 1:].clone()}, "shape of q"),
    (lambda b: {"out": torch.empty_like(b.q).transpose(1, 2).contiguous().transpose(1, 2)}, "must be contiguous"),
    (lambda b: {"k_scale": torch.ones(1)} if b.k_scale is None else {"k_scale": None}, "float8_e4m3fn cache"),
    (lambda b: {"softmax_scale": "x"}, "incompatible function arguments"),
])
def test_refusals_in_python(cache, change, text):
    b = paged.Batch([40, 50, 60], 2, 2, 2, 64, 16, torch.float16, cache, device="cpu")
    with pytest.raises((RuntimeError, TypeError), match=text):
        call(b, **change(b))


@pytest.mark.parametrize("change,text", [
    (lambda b: {"k_scale": b.k_scale.float()}, "float8_e8m0fnu"),
    (lambda b: {"v_scale": b.v_scale[1:]}, "must have shape"),
])
def test_refusals_of_scales(change, text):
    b = paged.Batch([40, 50, 60], 2, 2, 2, 64, 16, torch.float16, "e4m3", device="cpu")
    with pytest.raises(RuntimeError, match=text):
        call(b, **change(b))


def test_refusals_of_cache_calls_in_python():
    import flash_attn_v100 as f
    b = paged.Batch([40, 50], 2, 2, 1, 64, 16, torch.float16, device="cpu")
    with pytest.raises(RuntimeError, match="must be on the GPU"):
        f.kv_cache_write(b.k, b.v, *b.args())
    with pytest.raises(RuntimeError, match="same shape"):
        f.kv_cache_write(b.k, b.v[:, :1], *b.args())
    with pytest.raises(RuntimeError, match="heads of the cache"):
        f.kv_cache_write(b.k[:, :, :1], b.v[:, :, :1], *b.args())
    with pytest.raises(RuntimeError, match="same dtype"):
        f.kv_cache_write(b.k, b.v.bfloat16(), *b.args())
    with pytest.raises(RuntimeError, match="more than one element of the written-to tensor"):
        f.kv_cache_write(b.k, b.v, b.k_cache[:1].expand(5, -1, -1, -1), b.v_cache[:1].expand(5, -1, -1, -1), b.page_table, b.cache_seqlens)
    with pytest.raises(RuntimeError, match="must be on the GPU"):
        f.kv_cache_read(*b.args(), 10)
    with pytest.raises(RuntimeError, match="max_seqlen must be positive"):
        f.kv_cache_read(*b.args(), 0)
    with pytest.raises(RuntimeError, match="dtype of the inputs"):
        f.kv_cache_read(*b.args(), 10, dtype=torch.bfloat16)


def test_written_and_read_tensors_that_ask_for_gradients_are_refused():
    """The output among them: it would go on with the graph of what it held before.  Without gradients the next check is reached."""
    import flash_attn_v100 as f
    b = paged.Batch([40, 50, 60], 2, 2, 2, 64, 16, torch.float16, "e4m3", device="cpu")
    leaf = torch.empty_like(b.q, requires_grad=True)
    scale = b.k_scale.clone().requires_grad_()
    for change in ({"out": leaf}, {"out": leaf * 1}, {"k_scale": scale}, {"v_scale": scale}):
        with pytest.raises(RuntimeError, match="no gradients"):
            call(b, **change)
        with torch.no_grad(), pytest.raises(RuntimeError, match="must be on the GPU"):
            call(b, **change)
    with pytest.raises(RuntimeError, match="no gradients"):
        f.kv_cache_write(b.k, b.v, *b.args(), k_scale=scale, v_scale=b.v_scale)
    with pytest.raises(RuntimeError, match="no gradients"):
        f.kv_cache_read(*b.args(), 10, k_scale=b.k_scale, v_scale=scale)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(torch.empty_like(b.q), torch.ones_like(b.q))
        with pytest.raises(RuntimeError, match="no gradients"):
            call(b, out=dual)


def sharing(x, y):
    """Tensors like both, that share their first bytes."""
    room = torch.zeros(max(x.numel() * x.element_size(), y.numel() * y.element_size()) + 16, dtype=torch.uint8)
    return [room[:t.numel() * t.element_size()].view(t.dtype).view(t.shape) for t in (x, y)]


@pytest.mark.parametrize("packed", (False, True))
def test_written_tensors_that_share_memory_with_others_are_refused(packed):
    """Each pair of a tensor that is written and one that is read, or is written too."""
    import flash_attn_v100 as f
    b = paged.Batch([40, 50, 60], [2] * 3 if packed else 2, 2, 2, 64, 16, torch.float16, "e4m3", device="cpu", packed=packed)
    tensors = {"out": torch.empty_like(b.q), "q": b.q, "k": b.k, "v": b.v, "k_cache": b.k_cache, "v_cache": b.v_cache,
               "page_table": b.page_table, "cache_seqlens": b.cache_seqlens, **b.scales()}
    if packed:
        tensors["cu_seqlens"] = b.cu_seqlens
    attention = set(inspect.signature(f.flash_attn_paged_func).parameters) & set(tensors)
    write = set(inspect.signature(f.kv_cache_write).parameters) & set(tensors)
    for function, names, outputs in ((f.flash_attn_paged_func, attention, ["out"]),
                                     (f.kv_cache_write, write, ["k_cache", "v_cache", "k_scale", "v_scale"])):
        for output in outputs:
            for other in names - {output}:
                shared = dict(zip((output, other), sharing(tensors[output], tensors[other])))
                with pytest.raises(RuntimeError, match="memory"):
                    function(**{name: shared.get(name, tensors[name]) for name in names})
        with pytest.raises(RuntimeError, match="must be on the GPU"):
            function(**{name: tensors[name] for name in names})


def test_oracle_rounds_as_torch_does():
    """The oracle's 8-bit values against torch's conversion of x / 2^e, which is exact, and its scales against their definition."""
    g = torch.Generator().manual_seed(0)
    for dtype in (torch.float16, torch.bfloat16):
        x = (torch.randn(500, 64, generator=g) * torch.logspace(-6, 4, 500)[:, None]).to(dtype)
        values, e = po.to_e4m3(x)
        scale = torch.pow(2.0, e.double())[:, None]
        assert torch.equal((x.double() / scale).float().to(torch.float8_e4m3fn).double(), values)
        amax = x.double().abs().amax(-1, keepdim=True).clamp(max=po.LARGEST_KEPT[dtype])
        assert (amax <= 448 * scale).all() and (amax > 224 * scale).all()
        assert torch.equal((values * scale).to(dtype).double(), values * scale)


def test_oracle_attention_in_closed_form():
    """Equal keys: the mean of the values seen; one large key: its value; no key: zero."""
    v = torch.arange(12.0)[:, None, None].expand(12, 1, 64)
    q = torch.ones(3, 2, 64)
    out, _, _ = po.attention(q, torch.zeros(12, 1, 64), v, 0.1, True)
    assert torch.allclose(out[:, 0, 0], torch.tensor([4.5, 5.0, 5.5], dtype=torch.float64))
    k = torch.zeros(12, 1, 64)
    k[4] = 100
    out, _, _ = po.attention(q, k, v, 1.0, False)
    assert torch.allclose(out, torch.tensor(4.0, dtype=torch.float64))
    out, weight, _ = po.attention(torch.ones(15, 2, 64), torch.zeros(12, 1, 64), v, 0.1, True)
    assert not out[:3].any() and not weight[:3].any() and out[4].ne(0).all()


def host_program(tmp_path, body):
    src, exe = tmp_path / "plan.cpp", tmp_path / "plan"
    src.write_text('#include <cstdio>\n#include <vector>\n#include "paged_plan.h"\n' + body)
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-I", CSRC, str(src), "-o", str(exe)])
    return subprocess.run([str(exe)], stdout=subprocess.PIPE).stdout.decode()


def test_stretches_cover_every_tile_once(tmp_path):
    """Random batches: the items of all stretches, found one after the other as the kernel finds them, are each there whole; parts
    have places of their own, which are those that the item's first part says; stretches differ by no more than an item's rounding."""
    out = host_program(tmp_path, r"""
#include <map>
struct Seq { int n, keys; };
int main() {
  unsigned seed = 1;
  auto rnd = [&](int n) { seed = seed * 1664525u + 1013904223u; return (int)((seed >> 8) % (unsigned)n); };
  for (int round = 0; round < 3000; ++round) {
    const int batch = 1 + rnd(12), kv = 1 + rnd(4), group = 1 + rnd(9), rows_of_block = rnd(2) ? 32 : 128;
    const bool causal = rnd(2);
    std::vector<Seq> seqs(batch);
    std::vector<PagedLine> lines(batch);
    long all = 0;
    for (int b = 0; b < batch; ++b) {
      seqs[b] = {rnd(3) ? rnd(3) : rnd(300), rnd(3) ? rnd(500) : rnd(20000)};
      lines[b] = paged_line(seqs[b].keys, seqs[b].n, group, causal ? paged_step(rows_of_block, group, 4) : 0, rows_of_block, 64, 4);
      all += lines[b].all() * kv;
    }
    const long length = paged_stretch(all);
    const int stretches = paged_stretches(all, length);
    if (stretches * length < all || stretches > kPagedGroups) return puts("stretches"), 1;
    struct Item { int next = 0, tiles = -1, parts = 0, told = 0, first = 0; };
    std::map<std::vector<int>, Item> items;
    std::map<int, int> places;
    for (int s = 0; s < stretches; ++s) {
      long x = s * length;
      const long end = x + length < all ? x + length : all;
      while (x < end) {
        long before = 0;
        int b = 0;
        while (before + lines[b].all() * kv <= x) before += lines[b++].all() * kv;
        const int head = paged_divide(x - before, lines[b].all());
        const long from = before + head * lines[b].all();
        const int block = paged_block_at(lines[b], x - from);
        const long item = from + lines[b].before(block), weight = lines[b].of(block);
        if (weight <= 0 || item > x || item + weight <= x) return puts("block"), 1;
        const int rows = seqs[b].n * group, last = (rows < (block + 1) * rows_of_block ? rows : (block + 1) * rows_of_block) - 1;
        const int tiles = paged_tiles(paged_visible(seqs[b].keys, seqs[b].n, last / group, causal));
        const int t0 = paged_tile_at(tiles, x - item, weight), t1 = paged_tile_at(tiles, end - item, weight);
        const bool opens = item >= x, whole = opens && item + weight <= end;
        Item& it = items[{b, head, block}];
        if (opens != (it.parts == 0) || t0 != it.next || t1 < t0) return puts("gap"), 1;
        if (opens) {
          it.told = whole ? 1 : paged_divide(item + weight - 1, length) - s + 1;
          it.first = s;
        }
        if (!whole) {
          const int place = paged_place(s, opens ? 0 : 1) - (opens ? 0 : 2);
          if (place < 0 || place >= 2 * stretches || places[place]++) return puts("place"), 1;
          if (place != paged_place(it.first, it.parts)) return puts("place of the part"), 1;
        }
        it.next = t1, it.tiles = tiles, ++it.parts;
        x = item + weight;
      }
    }
    for (int b = 0; b < batch; ++b)
      for (int h = 0; h < kv; ++h)
        for (int k = 0; k < lines[b].blocks; ++k) {
          const Item it = items[{b, h, k}];
          if (it.next != it.tiles || it.parts != it.told) return puts("not whole"), 1;
        }
  }
  puts("ok");
}
""")
    assert out == "ok\n"


def test_parts_fit_their_places(tmp_path):
    """All that begin and end in one of the stretches, none that would go past the last one."""
    out = host_program(tmp_path, r"""
int main() {
  for (int rows : {16, 32, 128})
    for (int first = 0; first < kPagedGroups; ++first)
      for (int parts = 1; parts < kPagedGroups + 3; ++parts)
        for (int row : {0, 1, rows - 1}) {
          const bool fit = paged_parts_fit(2 * first * rows + row, parts, rows);
          if (fit != (parts > 1 && first + parts <= kPagedGroups)) return printf("%d %d %d\\n", rows, first, parts), 1;
          for (int p = 0; fit && p < parts; ++p)
            if (paged_place(first, p) >= 2 * kPagedGroups) return puts("past"), 1;
        }
  if (paged_parts_fit(-1, 2, 16) || paged_parts_fit(0, -5, 16) || paged_parts_fit(0x7fffffff, 0x7fffffff, 128)) return puts("nonsense"), 1;
  puts("ok");
}
""")
    assert out == "ok\n"


def test_division(tmp_path):
    out = host_program(tmp_path, r"""
int main() {
  unsigned long seed = 1;
  auto rnd = [&](int bits) { seed = seed * 6364136223846793005ul + 1442695040888963407ul; return (long)(seed >> (64 - bits)); };
  for (int i = 0; i < 4000000; ++i) {
    const long d = rnd(1 + i % 41) + 1, n = d * rnd(1 + i % 20) + rnd(1 + i % 41) % d;
    if (paged_divide(n, d) != n / d || paged_divide(n / d * d, d) != n / d) return puts("wrong"), 1;
    const int m = (int)(rnd(30)), e = (int)(rnd(20)) + 1 + m / (1 << 20);
    if (paged_divide(m, e) != m / e) return puts("wrong int"), 1;
  }
  puts("ok");
}
""")
    assert out == "ok\n"


def test_work_groups_take_every_stretch_once(tmp_path):
    out = host_program(tmp_path, r"""
int main() {
  for (int parts = 0; parts < 3000; ++parts) {
    std::vector<int> taken(parts + 1);
    for (int w = 0; w < (parts + 7) / 8 * 8 + 24; ++w) {
      const int number = paged_spread(w, parts);
      if (number < 0) return puts("negative"), 1;
      if (number < parts) ++taken[number];
    }
    for (int p = 0; p < parts; ++p)
      if (taken[p] != 1) return puts("not once"), 1;
  }
  puts("ok");
}
""")
    assert out == "ok\n"


def test_whole_items_are_taken_once(tmp_path):
    out = host_program(tmp_path, r"""
int main() {
  for (int items = 0; items < 6000; items += items < 700 ? 1 : 37) {
    std::vector<int> taken(items);
    for (int w = 0; w < kPagedGroups; ++w) {
      int last = -1;
      for (int round = 0;; ++round) {
        const int at = paged_whole(round, w, items);
        if (at >= items) break;
        if (at <= last) return puts("back"), 1;
        last = at;
        ++taken[at];
      }
    }
    for (int t : taken)
      if (t != 1) return puts("not once"), 1;
  }
  for (int blocks = 1; blocks < 20; ++blocks)
    for (int heads = 1; heads < 20; ++heads) {
      std::vector<int> taken(blocks * heads);
      for (int at = 0; at < blocks * heads; ++at) {
        int block, head;
        paged_whole_item(at, blocks, FmhaDivisor(heads), block, head);
        if (block < 0 || block >= blocks || head < 0 || head >= heads || taken[block * heads + head]++) return puts("item"), 1;
      }
    }
  puts("ok");
}
""")
    assert out == "ok\n"


def test_visible_keys(tmp_path):
    out = host_program(tmp_path, r"""
int main() {
  for (int keys = 0; keys < 40; ++keys)
    for (int n = 1; n < 40; ++n)
      for (int i = 0; i < n; ++i)
        for (int causal = 0; causal < 2; ++causal) {
          int seen = 0;
          for (int j = 0; j < keys; ++j) seen += !causal || j <= keys - n + i;
          if (paged_visible(keys, n, i, causal) != seen) return puts("wrong"), 1;
        }
  puts("ok");
}
""")
    assert out == "ok\n"
