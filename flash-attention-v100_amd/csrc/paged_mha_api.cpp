// PyTorch-ROCm extension `flash_attn_v100_paged_cuda`: validation, allocation, device guard and stream lookup around the C
// launchers declared in paged_mha.h.  Conventions of fused_mha_api.cpp: TORCH_CHECK ->
// RuntimeError, torch's current stream, no synchronisation.  What is in device memory (lengths, page numbers) is not looked at
// here: the kernels keep to their bounds by themselves.
#include <torch/extension.h>
#include <ATen/MemoryOverlap.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <array>
#include <cmath>

#include "api_common.h"
#include "paged_mha.h"

namespace {

using OptTensor = c10::optional<at::Tensor>;

void check_paged(int rc, const char* what) { TORCH_CHECK(rc == FUSED_MHA_OK, what, " failed: ", paged_mha_error_string(rc)); }

int type_code(at::ScalarType t, const char* what) {
  TORCH_CHECK(t == at::kHalf || t == at::kBFloat16, what, " must be fp16 or bf16");
  return t == at::kHalf ? PAGED_MHA_FP16 : PAGED_MHA_BF16;
}

void check_ints(const at::Tensor& x, const char* name, int64_t dims) {
  TORCH_CHECK(x.scalar_type() == at::kInt, name, " must be int32");
  TORCH_CHECK(x.dim() == dims, name, " must have ", dims, dims == 1 ? " dimension" : " dimensions");
  TORCH_CHECK(x.stride(-1) == 1 || x.size(-1) <= 1, name, " must have contiguous last dimension");
}

// All on one GPU, which this repository's kernels run on.
void check_devices(const at::Tensor& k_cache, std::initializer_list<const at::Tensor*> xs, std::initializer_list<const OptTensor*> ys) {
  TORCH_CHECK(k_cache.is_cuda(), "the cache must be on the GPU");
  for (const at::Tensor* x : xs) TORCH_CHECK(x->is_cuda() && x->get_device() == k_cache.get_device(), "all tensors must be on the GPU of the cache");
  for (const OptTensor* y : ys)
    TORCH_CHECK(!y->has_value() || ((*y)->is_cuda() && (*y)->get_device() == k_cache.get_device()), "all tensors must be on the GPU of the cache");
  api::check_arch(k_cache.get_device());
}

// There is no gradient through a cache: better an error than a result without one.
void check_no_grad(std::initializer_list<const at::Tensor*> xs, std::initializer_list<const OptTensor*> ys) {
  auto check = [](const at::Tensor& x) {
    TORCH_CHECK(!(at::GradMode::is_enabled() && x.requires_grad()) && !x._fw_grad(/*level=*/0).defined(),
                "the paged cache has no gradients: call it under torch.no_grad() or with detached tensors");
  };
  for (const at::Tensor* x : xs) check(*x);
  for (const OptTensor* y : ys)
    if (y->has_value()) check(**y);
  TORCH_CHECK(!torch::jit::tracer::isTracing(), "the paged cache is not supported under torch.jit.trace");
}

// A tensor that is written shares no memory with those that are read: work groups read lengths and pages at any time.
void check_apart(const at::Tensor& out, std::initializer_list<const at::Tensor*> xs, std::initializer_list<const OptTensor*> ys) {
  for (const at::Tensor* x : xs) at::assert_no_overlap(out, *x);
  for (const OptTensor* y : ys)
    if (y->has_value()) at::assert_no_overlap(out, **y);
}

// For autograd, which holds tensors that were saved before.
void written(const at::Tensor& x) {
  if (!x.is_inference()) x.unsafeGetTensorImpl()->bump_version();
}

// The stride of a dimension; torch says anything of those of size 1, which lead nowhere.
int64_t step(const at::Tensor& x, int64_t dim) { return x.size(dim) == 1 ? 0 : x.stride(dim); }

paged_mha_strides cache_strides(const at::Tensor& x) { return {step(x, 0), step(x, 1), step(x, 2)}; }

// Cache and batch as the C interface takes them.
struct Paged {
  paged_mha_cache cache{};
  paged_mha_batch batch{};
  at::ScalarType type;
  Paged(const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& page_table, const at::Tensor& cache_seqlens,
        const OptTensor& cu_seqlens, const OptTensor& k_scale, const OptTensor& v_scale, at::ScalarType type)
      : type(type) {
    const bool q8 = k_cache.scalar_type() == at::kFloat8_e4m3fn;
    cache.type = type_code(type, "queries, keys and values");
    cache.cache_type = q8 ? PAGED_MHA_E4M3 : cache.type;
    TORCH_CHECK(q8 || k_cache.scalar_type() == type, "the cache must have the dtype of the inputs or be float8_e4m3fn");
    TORCH_CHECK(v_cache.scalar_type() == k_cache.scalar_type(), "key and value cache must have the same dtype");
    TORCH_CHECK(k_cache.dim() == 4, "the cache must have 4 dimensions (pages, page_size, heads, head_size)");
    TORCH_CHECK(v_cache.sizes() == k_cache.sizes(), "key and value cache must have the same shape");
    TORCH_CHECK(k_cache.stride(3) == 1 && v_cache.stride(3) == 1, "the cache must have contiguous last dimension");
    TORCH_CHECK(k_cache.numel() > 0, "the cache must not be empty");
    for (int i = 0; i < 3; ++i) TORCH_CHECK(k_cache.size(i) < (int64_t(1) << 31), "the cache is too large");
    cache.key = k_cache.data_ptr(), cache.value = v_cache.data_ptr();
    cache.key_strides = cache_strides(k_cache), cache.value_strides = cache_strides(v_cache);
    cache.pages = (int)k_cache.size(0), cache.page_size = (int)k_cache.size(1), cache.kv_head = (int)k_cache.size(2);
    TORCH_CHECK(k_cache.size(3) == 64 || k_cache.size(3) == 128, "current repo only supports head dimension 64 or 128");
    cache.d = (int)k_cache.size(3);
    TORCH_CHECK(k_scale.has_value() == q8 && v_scale.has_value() == q8,
                q8 ? "a float8_e4m3fn cache needs k_scale and v_scale" : "k_scale and v_scale go with a float8_e4m3fn cache only");
    if (q8) {
      for (const at::Tensor* s : {&*k_scale, &*v_scale}) {
        TORCH_CHECK(s->scalar_type() == at::kFloat8_e8m0fnu, "k_scale and v_scale must be float8_e8m0fnu");
        TORCH_CHECK(s->sizes() == k_cache.sizes().slice(0, 3), "k_scale and v_scale must have shape (pages, page_size, heads)");
      }
      cache.key_scale = k_scale->data_ptr(), cache.value_scale = v_scale->data_ptr();
      cache.key_scale_strides = cache_strides(*k_scale), cache.value_scale_strides = cache_strides(*v_scale);
    }
    check_ints(page_table, "page_table", 2);
    check_ints(cache_seqlens, "cache_seqlens", 1);
    const int64_t n = cache_seqlens.size(0);
    TORCH_CHECK(n > 0 && n < (1 << 30), "batch size must be postive");
    TORCH_CHECK(page_table.size(0) == n, "page_table must have a row for each sequence");
    TORCH_CHECK(page_table.size(1) > 0 && page_table.size(1) < (1 << 30), "page_table must have columns");
    TORCH_CHECK(cache_seqlens.is_contiguous(), "cache_seqlens must be contiguous");
    batch.page_table = page_table.data_ptr<int>();
    batch.table_stride = page_table.stride(0), batch.table_width = (int)page_table.size(1);
    batch.cache_seqlens = cache_seqlens.data_ptr<int>();
    batch.batch = (int)n;
    if (cu_seqlens.has_value()) {
      check_ints(*cu_seqlens, "cu_seqlens", 1);
      TORCH_CHECK(cu_seqlens->is_contiguous(), "cu_seqlens must be contiguous");
      TORCH_CHECK(cu_seqlens->size(0) == n + 1, "cu_seqlens must have one element more than there are sequences");
      batch.cu_seqlens = cu_seqlens->data_ptr<int>();
    }
  }
  // Tokens of q, k or v, which is (batch, tokens, heads, head_size) or with cu_seqlens (tokens, heads, head_size).
  void set_tokens(const at::Tensor& x, const char* name, int64_t heads) {
    TORCH_CHECK(x.scalar_type() == type, name, " must have the same dtype as the other inputs");
    if (batch.cu_seqlens) {
      TORCH_CHECK(x.dim() == 3, name, " must have 3 dimensions (tokens, heads, head_size) with cu_seqlens");
    } else {
      TORCH_CHECK(x.dim() == 4, name, " must have 4 dimensions (batch, seqlen, heads, head_size)");
      TORCH_CHECK(x.size(0) == batch.batch, name, " must have the batch size of cache_seqlens");
    }
    TORCH_CHECK(x.size(-1) == cache.d, name, " must have the head size of the cache");
    TORCH_CHECK(heads == 0 || x.size(-2) == heads, name, " must have the heads of the cache");
    TORCH_CHECK(x.size(-2) > 0 && x.size(-2) < (1 << 30), name, " must have heads");
    TORCH_CHECK(x.size(-3) > 0 && x.size(-3) < (1 << 30), "seqlen must be positive");
    batch.tokens = (int)x.size(-3);
  }
};

// q, k or v with its strides where rows lie on 16-byte boundaries, otherwise a dense copy.
struct TokenOperand {
  at::Tensor x;
  fused_mha_strides st;
  explicit TokenOperand(const at::Tensor& in) : x(in) {
    auto of = [](const at::Tensor& t) { return fused_mha_strides{t.dim() == 4 ? step(t, 0) : 0, step(t, -3), step(t, -2)}; };
    st = of(x);
    if (x.stride(-1) != 1 || ((st.batch | st.seq | st.head) & 7) || (reinterpret_cast<uintptr_t>(x.data_ptr()) & 15u)) {
      x = x.clone(at::MemoryFormat::Contiguous);  // contiguous() may be the tensor itself, wherever it begins
      st = of(x);
    }
  }
};

}  // namespace

at::Tensor paged_attention(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& page_table,
                           const at::Tensor& cache_seqlens, c10::optional<double> softmax_scale, bool is_causal,
                           const OptTensor& cu_seqlens, c10::optional<int64_t> max_seqlen, const OptTensor& k_scale,
                           const OptTensor& v_scale, const OptTensor& out_) {
  check_no_grad({&q, &k_cache, &v_cache}, {&k_scale, &v_scale, &out_});
  Paged p(k_cache, v_cache, page_table, cache_seqlens, cu_seqlens, k_scale, v_scale, q.scalar_type());
  p.set_tokens(q, "query", 0);
  const int64_t heads = q.size(-2);
  TORCH_CHECK(heads % p.cache.kv_head == 0, "query heads must be a multiple of the cache's heads");
  TORCH_CHECK(!max_seqlen.has_value() || *max_seqlen > 0, "max_seqlen must be positive");
  const int max_new = (int)std::min<int64_t>(max_seqlen.value_or(0), (1 << 30) - 1);
  if (out_.has_value()) {
    TORCH_CHECK(out_->scalar_type() == q.scalar_type(), "Output must have the same dtype as inputs");
    TORCH_CHECK(out_->is_contiguous(), "Output tensor must be contiguous");
    TORCH_CHECK(out_->sizes() == q.sizes(), "out must have the shape of q");
    check_apart(*out_, {&q, &k_cache, &v_cache, &page_table, &cache_seqlens}, {&cu_seqlens, &k_scale, &v_scale});
  }
  check_devices(k_cache, {&q, &v_cache, &page_table, &cache_seqlens}, {&cu_seqlens, &k_scale, &v_scale, &out_});
  const api::OnDeviceOf device_guard(q);
  const TokenOperand qo(q);
  const at::Tensor out = out_.has_value() ? *out_ : api::gpu_empty(q.sizes(), q.scalar_type(), q);
  const float scale = (float)(softmax_scale.has_value() ? *softmax_scale : std::pow((double)p.cache.d, -0.5));
  const size_t bytes = paged_mha_forward_workspace_bytes(&p.cache, &p.batch, (int)heads, max_new);
  at::Tensor workspace;
  if (bytes) workspace = api::gpu_empty({(int64_t)bytes}, at::kByte, q);
  check_paged(paged_mha_forward(&p.cache, &p.batch, qo.x.data_ptr(), &qo.st, out.data_ptr(), (int)heads, max_new, scale,
                                is_causal ? 1 : 0, out_.has_value() ? 0 : 1, bytes ? workspace.data_ptr() : nullptr, bytes,
                                c10::hip::getCurrentHIPStream().stream()),
              "paged_mha_forward");
  if (out_.has_value()) written(out);
  return out;
}

void cache_write(const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_cache, const at::Tensor& v_cache,
                 const at::Tensor& page_table, const at::Tensor& cache_seqlens, const OptTensor& cu_seqlens, const OptTensor& k_scale,
                 const OptTensor& v_scale) {
  check_no_grad({&k, &v, &k_cache, &v_cache}, {&k_scale, &v_scale});
  Paged p(k_cache, v_cache, page_table, cache_seqlens, cu_seqlens, k_scale, v_scale, k.scalar_type());
  p.set_tokens(k, "key", p.cache.kv_head);
  p.set_tokens(v, "value", p.cache.kv_head);
  TORCH_CHECK(k.sizes() == v.sizes(), "key and value must have the same shape");
  for (const at::Tensor* x : {&k_cache, &v_cache}) at::assert_no_internal_overlap(*x);
  check_apart(k_cache, {&v_cache, &k, &v, &page_table, &cache_seqlens}, {&cu_seqlens, &k_scale, &v_scale});
  check_apart(v_cache, {&k, &v, &page_table, &cache_seqlens}, {&cu_seqlens, &k_scale, &v_scale});
  if (k_scale.has_value()) {
    for (const OptTensor* x : {&k_scale, &v_scale}) at::assert_no_internal_overlap(**x);
    check_apart(*k_scale, {&*v_scale, &k, &v, &page_table, &cache_seqlens}, {&cu_seqlens});
    check_apart(*v_scale, {&k, &v, &page_table, &cache_seqlens}, {&cu_seqlens});
  }
  check_devices(k_cache, {&k, &v, &v_cache, &page_table, &cache_seqlens}, {&cu_seqlens, &k_scale, &v_scale});
  const api::OnDeviceOf device_guard(k_cache);
  const TokenOperand ko(k), vo(v);
  check_paged(paged_mha_write(&p.cache, &p.batch, ko.x.data_ptr(), &ko.st, vo.x.data_ptr(), &vo.st,
                              c10::hip::getCurrentHIPStream().stream()),
              "paged_mha_write");
  written(k_cache), written(v_cache);
  if (k_scale.has_value()) written(*k_scale), written(*v_scale);
}

std::tuple<at::Tensor, at::Tensor> cache_read(const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& page_table,
                                              const at::Tensor& cache_seqlens, int64_t max_seqlen, const OptTensor& k_scale,
                                              const OptTensor& v_scale, c10::optional<at::ScalarType> dtype) {
  check_no_grad({&k_cache, &v_cache}, {&k_scale, &v_scale});
  const bool q8 = k_cache.scalar_type() == at::kFloat8_e4m3fn;
  Paged p(k_cache, v_cache, page_table, cache_seqlens, c10::nullopt, k_scale, v_scale,
          dtype.has_value() ? *dtype : q8 ? at::kHalf : k_cache.scalar_type());
  TORCH_CHECK(max_seqlen > 0 && max_seqlen < (1 << 30), "max_seqlen must be positive");
  p.batch.tokens = 1;
  check_devices(k_cache, {&v_cache, &page_table, &cache_seqlens}, {&k_scale, &v_scale});
  const api::OnDeviceOf device_guard(k_cache);
  const std::array<int64_t, 4> shape = {p.batch.batch, max_seqlen, p.cache.kv_head, p.cache.d};
  at::Tensor k = api::gpu_empty(shape, p.type, k_cache), v = api::gpu_empty(shape, p.type, k_cache);
  check_paged(paged_mha_read(&p.cache, &p.batch, (int)max_seqlen, k.data_ptr(), v.data_ptr(), c10::hip::getCurrentHIPStream().stream()),
              "paged_mha_read");
  return {k, v};
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "Attention over a paged cache for gfx950";
  m.def("attention", &paged_attention, "Attention of new tokens over a paged cache");
  m.def("write", &cache_write, "Keys and values of new tokens to their places in a paged cache");
  m.def("read", &cache_read, "Keys and values of a paged cache as dense tensors");
}
