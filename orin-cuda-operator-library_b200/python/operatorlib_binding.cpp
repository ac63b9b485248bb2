// TORCH_LIBRARY(operatorlib, ...) binding of the B200 operator library.
//
// Drop-in for the reference binding python/operatorlib_binding.cpp:190-206:
// the six schemas are identical; the CUDA dispatch key runs the kernels (and,
// beyond the reference, a Meta key gives shapes for FakeTensor tracing);
// inputs must be contiguous CUDA tensors (no implicit copies), outputs are
// allocated here, work goes on the input device's current stream under a
// device guard, and the user-facing error texts match the reference's
// (python/test_extension.py:124-168 checks them).  Every launch of these six
// goes through the C++ API of operatorlib/operators.h, which forwards to the
// C-ABI.
//
// Beyond the reference: rope, kv_append and paged_attention (decoding with a
// paged key-value cache) call the C-ABI.  Their tensors may be strided as long
// as the last dimension is contiguous, so that slices of a packed projection
// and either order of a cache's dimensions need no copy.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include <cmath>
#include <cstdint>
#include <limits>
#include <optional>
#include <type_traits>

#include "operatorlib/operators.h"
#include "operatorlib/opl_capi.h"

namespace {

using at::Tensor;

// Meta (shape-only) calls run the same checks minus the device check.
thread_local bool g_meta_call = false;

struct MetaCall {
  MetaCall() { g_meta_call = true; }
  ~MetaCall() { g_meta_call = false; }
};

void require_cuda_contiguous(const Tensor& t, const char* name) {
  if (!g_meta_call) TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

void require_matching(const Tensor& x, const Tensor& y, const char* xn,
                      const char* yn) {
  TORCH_CHECK(x.device() == y.device(), xn, " and ", yn,
              " must be on the same CUDA device");
  TORCH_CHECK(x.scalar_type() == y.scalar_type(), xn, " and ", yn,
              " must have the same dtype");
}

int as_positive_int(int64_t value, const char* what) {
  TORCH_CHECK(value > 0 && value <= std::numeric_limits<int>::max(), what,
              " must be in the positive int32 range");
  return static_cast<int>(value);
}

void raise_on_error(cudaError_t status, const char* op) {
  TORCH_CHECK(status == cudaSuccess, op, " launch failed: ",
              cudaGetErrorString(status));
}

cudaStream_t stream_of(const Tensor& t) {
  return at::cuda::getCurrentCUDAStream(t.get_device()).stream();
}

const __half* half_ptr(const Tensor& t) {
  return reinterpret_cast<const __half*>(t.data_ptr<at::Half>());
}

Tensor op_reduce_sum(const Tensor& input) {
  require_cuda_contiguous(input, "input");
  TORCH_CHECK(input.scalar_type() == at::kFloat,
              "reduce_sum supports float32 input only");
  TORCH_CHECK(input.numel() > 0, "input must be non-empty");
  if (g_meta_call) return at::empty({}, input.options());
  c10::cuda::CUDAGuard guard(input.device());
  Tensor out = at::empty({}, input.options());
  raise_on_error(operatorlib::reduce_sum_f32(
                     input.data_ptr<float>(), out.data_ptr<float>(),
                     static_cast<std::size_t>(input.numel()), stream_of(input)),
                 "reduce_sum");
  return out;
}

Tensor op_softmax(const Tensor& input) {
  require_cuda_contiguous(input, "input");
  TORCH_CHECK(input.scalar_type() == at::kFloat,
              "softmax supports float32 input only");
  TORCH_CHECK(input.dim() >= 1, "input must have at least one dimension");
  const int cols = as_positive_int(input.size(-1), "last dimension");
  const int rows = as_positive_int(input.numel() / input.size(-1), "row count");
  if (g_meta_call) return at::empty_like(input);
  c10::cuda::CUDAGuard guard(input.device());
  Tensor out = at::empty_like(input);
  raise_on_error(operatorlib::softmax_f32(input.data_ptr<float>(),
                                          out.data_ptr<float>(), rows, cols,
                                          stream_of(input)),
                 "softmax");
  return out;
}

Tensor op_transpose(const Tensor& input) {
  require_cuda_contiguous(input, "input");
  TORCH_CHECK(input.scalar_type() == at::kFloat,
              "transpose supports float32 input only");
  TORCH_CHECK(input.dim() == 2, "input must be a 2D matrix");
  const int rows = as_positive_int(input.size(0), "rows");
  const int cols = as_positive_int(input.size(1), "cols");
  if (g_meta_call) return at::empty({cols, rows}, input.options());
  c10::cuda::CUDAGuard guard(input.device());
  Tensor out = at::empty({cols, rows}, input.options());
  raise_on_error(operatorlib::transpose_f32(input.data_ptr<float>(),
                                            out.data_ptr<float>(), rows, cols,
                                            stream_of(input)),
                 "transpose");
  return out;
}

Tensor op_rmsnorm(const Tensor& input, const Tensor& weight, double epsilon) {
  require_cuda_contiguous(input, "input");
  require_cuda_contiguous(weight, "weight");
  require_matching(input, weight, "input", "weight");
  TORCH_CHECK(input.scalar_type() == at::kFloat,
              "rmsnorm supports float32 input only");
  TORCH_CHECK(input.dim() >= 1, "input must have at least one dimension");
  TORCH_CHECK(weight.dim() == 1, "weight must be 1D");
  TORCH_CHECK(std::isfinite(epsilon) && epsilon > 0.0,
              "epsilon must be finite and positive");
  const int hidden = as_positive_int(input.size(-1), "hidden size");
  TORCH_CHECK(weight.numel() == hidden,
              "weight length must equal the input hidden size");
  const int tokens =
      as_positive_int(input.numel() / input.size(-1), "token count");
  if (g_meta_call) return at::empty_like(input);
  c10::cuda::CUDAGuard guard(input.device());
  Tensor out = at::empty_like(input);
  raise_on_error(operatorlib::rmsnorm_f32(
                     input.data_ptr<float>(), weight.data_ptr<float>(),
                     out.data_ptr<float>(), tokens, hidden,
                     static_cast<float>(epsilon), stream_of(input)),
                 "rmsnorm");
  return out;
}

Tensor op_gemm(const Tensor& a, const Tensor& b) {
  require_cuda_contiguous(a, "a");
  require_cuda_contiguous(b, "b");
  require_matching(a, b, "a", "b");
  TORCH_CHECK(a.dim() == 2 && b.dim() == 2, "a and b must be 2D matrices");
  TORCH_CHECK(a.size(1) == b.size(0), "a.size(1) must equal b.size(0)");
  TORCH_CHECK(a.scalar_type() == at::kFloat || a.scalar_type() == at::kHalf,
              "gemm supports float32 or float16 inputs only");
  const int m = as_positive_int(a.size(0), "M");
  const int k = as_positive_int(a.size(1), "K");
  const int n = as_positive_int(b.size(1), "N");
  if (g_meta_call) return at::empty({m, n}, a.options().dtype(at::kFloat));
  c10::cuda::CUDAGuard guard(a.device());
  Tensor c = at::empty({m, n}, a.options().dtype(at::kFloat));
  const cudaError_t status =
      a.scalar_type() == at::kFloat
          ? operatorlib::gemm_f32(a.data_ptr<float>(), b.data_ptr<float>(),
                                  c.data_ptr<float>(), m, n, k, stream_of(a))
          : operatorlib::gemm_f16(half_ptr(a), half_ptr(b), c.data_ptr<float>(),
                                  m, n, k, stream_of(a));
  raise_on_error(status, "gemm");
  return c;
}

Tensor op_attention(const Tensor& q, const Tensor& k, const Tensor& v,
                    bool causal) {
  require_cuda_contiguous(q, "q");
  require_cuda_contiguous(k, "k");
  require_cuda_contiguous(v, "v");
  require_matching(q, k, "q", "k");
  require_matching(q, v, "q", "v");
  TORCH_CHECK(q.dim() == 4, "q, k and v must use [B,H,S,D] layout");
  TORCH_CHECK(q.sizes() == k.sizes() && q.sizes() == v.sizes(),
              "q, k and v must have identical shapes");
  TORCH_CHECK(q.scalar_type() == at::kFloat || q.scalar_type() == at::kHalf,
              "attention supports float32 or float16 inputs only");
  const int batch = as_positive_int(q.size(0), "batch");
  const int heads = as_positive_int(q.size(1), "heads");
  const int sequence = as_positive_int(q.size(2), "sequence");
  const int head_dim = as_positive_int(q.size(3), "head dimension");
  TORCH_CHECK(head_dim <= 128, "head dimension must be at most 128");
  TORCH_CHECK(static_cast<int64_t>(batch) * heads <=
                  std::numeric_limits<int>::max(),
              "batch * heads exceeds the supported int32 range");
  if (g_meta_call) return at::empty(q.sizes(), q.options().dtype(at::kFloat));
  c10::cuda::CUDAGuard guard(q.device());
  Tensor out = at::empty(q.sizes(), q.options().dtype(at::kFloat));
  const cudaError_t status =
      q.scalar_type() == at::kFloat
          ? operatorlib::attention_f32(q.data_ptr<float>(), k.data_ptr<float>(),
                                       v.data_ptr<float>(), out.data_ptr<float>(),
                                       batch, heads, sequence, head_dim, causal,
                                       stream_of(q))
          : operatorlib::attention_f16(half_ptr(q), half_ptr(k), half_ptr(v),
                                       out.data_ptr<float>(), batch, heads,
                                       sequence, head_dim, causal, stream_of(q));
  raise_on_error(status, "attention");
  return out;
}

// ------------------------------------------- decoding with a paged cache

constexpr int64_t kMaxHeadDim = 256;

void require_cuda_rows(const Tensor& t, const char* name, int64_t dims) {
  if (!g_meta_call) TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.dim() == dims, name, " must have ", dims, " dimensions");
  TORCH_CHECK(t.stride(-1) == 1 || t.size(-1) == 1, name,
              " must be contiguous in its last dimension");
}

void require_type(const Tensor& t, const Tensor& like, at::ScalarType type, const char* name,
                  const char* text) {
  TORCH_CHECK(t.device() == like.device(), name, " must be on the other tensors' device");
  TORCH_CHECK(t.scalar_type() == type, name, " must be ", text);
}

void require_float_type(const Tensor& t, const char* op) {
  TORCH_CHECK(t.scalar_type() == at::kFloat || t.scalar_type() == at::kHalf ||
                  t.scalar_type() == at::kBFloat16,
              op, " supports float32, float16 or bfloat16 inputs only");
}

int as_head_dim(int64_t value) {
  TORCH_CHECK(value <= kMaxHeadDim, "head dimension must be at most 256");
  return as_positive_int(value, "head dimension");
}

// Two elements of `t` at the same address would be written by two threads.
void require_no_overlap(const Tensor& t, const char* name) {
  for (int64_t d = 0; d < t.dim(); ++d)
    TORCH_CHECK(t.size(d) == 1 || t.stride(d) != 0, name,
                " is written and must not be expanded");
}

opl_rope_spec make_rope(const Tensor& like, const Tensor& positions, const Tensor& inv_freq,
                        at::IntArrayRef sections, bool adjacent, bool inverse, int64_t tokens,
                        int64_t head_dim) {
  require_cuda_contiguous(positions, "positions");
  require_cuda_contiguous(inv_freq, "inv_freq");
  require_type(positions, like, at::kLong, "positions", "int64");
  require_type(inv_freq, like, at::kFloat, "inv_freq", "float32");
  TORCH_CHECK(inv_freq.dim() == 1, "inv_freq must be 1D");
  const int64_t pairs = inv_freq.numel();
  TORCH_CHECK(2 * pairs <= head_dim,
              "inv_freq must have at most head_dim / 2 elements");
  const int64_t axes = sections.empty() ? 1 : static_cast<int64_t>(sections.size());
  TORCH_CHECK(axes <= 4, "sections must name at most 4 position axes");
  opl_rope_spec spec = {};
  int64_t sum = 0;
  for (int64_t s = 0; s < axes; ++s) {
    const int64_t section = sections.empty() ? pairs : sections[s];
    TORCH_CHECK(section >= 0 && section <= pairs, "sections must be pairs of inv_freq");
    spec.sections[s] = static_cast<int>(section);
    sum += section;
  }
  TORCH_CHECK(sum == pairs, "sections must add up to the length of inv_freq");
  TORCH_CHECK(positions.dim() == 1 ? axes == 1 : positions.dim() == 2 && positions.size(0) == axes,
              "positions must be [tokens], or [axes, tokens] with an axis for each section");
  TORCH_CHECK(positions.size(-1) == tokens, "positions must have one column for each token");
  spec.axes = static_cast<int>(axes);
  spec.rot_dim = static_cast<int>(2 * pairs);
  spec.adjacent = adjacent ? 1 : 0;
  spec.inverse = inverse ? 1 : 0;
  if (!g_meta_call) {
    spec.positions = positions.data_ptr<int64_t>();
    spec.inv_freq = inv_freq.data_ptr<float>();
  }
  return spec;
}

opl_kv_cache make_cache(const Tensor& like, const Tensor& k_cache, const Tensor& v_cache,
                        int64_t head_dim) {
  require_cuda_rows(k_cache, "k_cache", 4);
  require_cuda_rows(v_cache, "v_cache", 4);
  require_matching(like, k_cache, "q", "k_cache");
  require_matching(like, v_cache, "q", "v_cache");
  TORCH_CHECK(k_cache.sizes() == v_cache.sizes(), "k_cache and v_cache must have identical shapes");
  TORCH_CHECK(k_cache.size(3) == head_dim,
              "the caches must be [pages, page_size, kv_heads, head_dim] with q's head_dim");
  opl_kv_cache cache = {};
  cache.pages = as_positive_int(k_cache.size(0), "pages");
  cache.page_size = as_positive_int(k_cache.size(1), "page size");
  cache.kv_heads = as_positive_int(k_cache.size(2), "key-value heads");
  cache.head_dim = as_head_dim(head_dim);
  cache.k_page = k_cache.stride(0);
  cache.k_token = k_cache.stride(1);
  cache.k_head = k_cache.stride(2);
  cache.v_page = v_cache.stride(0);
  cache.v_token = v_cache.stride(1);
  cache.v_head = v_cache.stride(2);
  if (!g_meta_call) {
    cache.k = k_cache.data_ptr();
    cache.v = v_cache.data_ptr();
  }
  return cache;
}

template <typename T>
T* typed(const Tensor& t) {
  return static_cast<T*>(t.data_ptr());
}

int rope_call(const Tensor& x, Tensor& out, int tokens, int heads, int head_dim,
              const opl_rope_spec& spec, cudaStream_t stream) {
  const auto run = [&](auto entry, auto* type) {
    using T = std::remove_pointer_t<decltype(type)>;
    return entry(typed<T>(x), typed<T>(out), tokens, heads, head_dim, x.stride(0), x.stride(1),
                 out.stride(0), out.stride(1), &spec, stream);
  };
  if (x.scalar_type() == at::kFloat) return run(opl_rope_f32, static_cast<float*>(nullptr));
  if (x.scalar_type() == at::kHalf) return run(opl_rope_f16, static_cast<opl_half_t*>(nullptr));
  return run(opl_rope_bf16, static_cast<opl_bf16_t*>(nullptr));
}

Tensor op_rope(const Tensor& x, const Tensor& positions, const Tensor& inv_freq,
               at::IntArrayRef sections, bool adjacent, bool inverse) {
  require_cuda_rows(x, "x", 3);
  require_float_type(x, "rope");
  const int tokens = as_positive_int(x.size(0), "token count");
  const int heads = as_positive_int(x.size(1), "heads");
  const int head_dim = as_head_dim(x.size(2));
  const opl_rope_spec spec =
      make_rope(x, positions, inv_freq, sections, adjacent, inverse, tokens, head_dim);
  if (g_meta_call) return at::empty(x.sizes(), x.options());
  c10::cuda::CUDAGuard guard(x.device());
  Tensor out = at::empty(x.sizes(), x.options());
  raise_on_error(static_cast<cudaError_t>(
                     rope_call(x, out, tokens, heads, head_dim, spec, stream_of(x))),
                 "rope");
  return out;
}

Tensor op_kv_append(const Tensor& q, const Tensor& k, const Tensor& v, Tensor& k_cache,
                    Tensor& v_cache, const Tensor& slots, const Tensor& positions,
                    const Tensor& inv_freq, at::IntArrayRef sections, bool adjacent) {
  require_cuda_rows(q, "q", 3);
  require_cuda_rows(k, "k", 3);
  require_cuda_rows(v, "v", 3);
  require_float_type(q, "kv_append");
  require_matching(q, k, "q", "k");
  require_matching(q, v, "q", "v");
  TORCH_CHECK(k.sizes() == v.sizes(), "k and v must have identical shapes");
  TORCH_CHECK(k.size(0) == q.size(0) && k.size(2) == q.size(2),
              "k and v must have q's tokens and head_dim");
  const int tokens = as_positive_int(q.size(0), "token count");
  const int heads = as_positive_int(q.size(1), "heads");
  const opl_kv_cache cache = make_cache(q, k_cache, v_cache, q.size(2));
  TORCH_CHECK(k.size(1) == cache.kv_heads, "k and v must have the caches' key-value heads");
  require_no_overlap(k_cache, "k_cache");
  require_no_overlap(v_cache, "v_cache");
  TORCH_CHECK(g_meta_call || cache.k != cache.v, "k_cache and v_cache must not share memory");
  require_cuda_contiguous(slots, "slots");
  require_type(slots, q, at::kLong, "slots", "int64");
  TORCH_CHECK(slots.dim() == 1 && slots.size(0) == tokens, "slots must have one element a token");
  const opl_rope_spec spec = make_rope(q, positions, inv_freq, sections, adjacent, false, tokens,
                                       cache.head_dim);
  if (g_meta_call) return at::empty(q.sizes(), q.options());
  c10::cuda::CUDAGuard guard(q.device());
  Tensor out = at::empty(q.sizes(), q.options());
  const auto run = [&](auto entry, auto* type) {
    using T = std::remove_pointer_t<decltype(type)>;
    return entry(typed<T>(q), q.stride(0), q.stride(1), typed<T>(k), k.stride(0), k.stride(1),
                 typed<T>(v), v.stride(0), v.stride(1), typed<T>(out), out.stride(0),
                 out.stride(1), &cache, slots.data_ptr<int64_t>(), tokens, heads, &spec,
                 stream_of(q));
  };
  int status;
  if (q.scalar_type() == at::kFloat)
    status = run(opl_kv_append_f32, static_cast<float*>(nullptr));
  else if (q.scalar_type() == at::kHalf)
    status = run(opl_kv_append_f16, static_cast<opl_half_t*>(nullptr));
  else
    status = run(opl_kv_append_bf16, static_cast<opl_bf16_t*>(nullptr));
  raise_on_error(static_cast<cudaError_t>(status), "kv_append");
  return out;
}

Tensor op_paged_attention(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache,
                          const Tensor& block_table, const Tensor& seq_lens,
                          std::optional<double> scale) {
  require_cuda_rows(q, "q", 3);
  require_float_type(q, "paged_attention");
  const int batch = as_positive_int(q.size(0), "batch");
  const int heads = as_positive_int(q.size(1), "heads");
  const opl_kv_cache cache = make_cache(q, k_cache, v_cache, q.size(2));
  TORCH_CHECK(heads % cache.kv_heads == 0, "q's heads must be a multiple of the key-value heads");
  require_cuda_rows(block_table, "block_table", 2);
  require_type(block_table, q, at::kInt, "block_table", "int32");
  require_cuda_contiguous(seq_lens, "seq_lens");
  require_type(seq_lens, q, at::kInt, "seq_lens", "int32");
  TORCH_CHECK(block_table.size(0) == batch, "block_table must have one row a sequence");
  TORCH_CHECK(seq_lens.dim() == 1 && seq_lens.size(0) == batch,
              "seq_lens must have one element a sequence");
  const int max_pages = as_positive_int(block_table.size(1), "block_table columns");
  const int64_t room = block_table.size(1) * cache.page_size;
  TORCH_CHECK(room <= int64_t{1} << 30 && room <= (int64_t{1} << 34) / batch,
              "block_table has room for more than 2^30 keys a sequence, or 2^34 in all");
  const double s = scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(cache.head_dim));
  TORCH_CHECK(std::isfinite(static_cast<float>(s)), "scale must be finite");
  if (g_meta_call) return at::empty(q.sizes(), q.options());
  c10::cuda::CUDAGuard guard(q.device());
  Tensor out = at::empty(q.sizes(), q.options());
  std::size_t bytes = 0;
  raise_on_error(static_cast<cudaError_t>(opl_paged_attention_workspace(
                     heads, cache.kv_heads, cache.head_dim, &bytes)),
                 "paged_attention");
  Tensor workspace = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
  const auto run = [&](auto entry, auto* type) {
    using T = std::remove_pointer_t<decltype(type)>;
    return entry(typed<T>(q), q.stride(0), q.stride(1), &cache, block_table.data_ptr<int>(),
                 block_table.stride(0), max_pages, seq_lens.data_ptr<int>(), typed<T>(out), batch,
                 heads, static_cast<float>(s), workspace.data_ptr(), bytes, stream_of(q));
  };
  int status;
  if (q.scalar_type() == at::kFloat)
    status = run(opl_paged_attention_f32, static_cast<float*>(nullptr));
  else if (q.scalar_type() == at::kHalf)
    status = run(opl_paged_attention_f16, static_cast<opl_half_t*>(nullptr));
  else
    status = run(opl_paged_attention_bf16, static_cast<opl_bf16_t*>(nullptr));
  raise_on_error(static_cast<cudaError_t>(status), "paged_attention");
  return out;
}

// Meta kernels: output shape/dtype only, after the same argument checks, so
// FakeTensor tracing (torch.compile, torch.export) sees the ops.  The
// reference registers the CUDA key only.
Tensor meta_reduce_sum(const Tensor& input) {
  MetaCall meta;
  return op_reduce_sum(input);
}
Tensor meta_softmax(const Tensor& input) {
  MetaCall meta;
  return op_softmax(input);
}
Tensor meta_transpose(const Tensor& input) {
  MetaCall meta;
  return op_transpose(input);
}
Tensor meta_rmsnorm(const Tensor& input, const Tensor& weight, double epsilon) {
  MetaCall meta;
  return op_rmsnorm(input, weight, epsilon);
}
Tensor meta_gemm(const Tensor& a, const Tensor& b) {
  MetaCall meta;
  return op_gemm(a, b);
}
Tensor meta_attention(const Tensor& q, const Tensor& k, const Tensor& v, bool causal) {
  MetaCall meta;
  return op_attention(q, k, v, causal);
}

Tensor meta_rope(const Tensor& x, const Tensor& positions, const Tensor& inv_freq,
                 at::IntArrayRef sections, bool adjacent, bool inverse) {
  MetaCall meta;
  return op_rope(x, positions, inv_freq, sections, adjacent, inverse);
}
Tensor meta_kv_append(const Tensor& q, const Tensor& k, const Tensor& v, Tensor& k_cache,
                      Tensor& v_cache, const Tensor& slots, const Tensor& positions,
                      const Tensor& inv_freq, at::IntArrayRef sections, bool adjacent) {
  MetaCall meta;
  return op_kv_append(q, k, v, k_cache, v_cache, slots, positions, inv_freq, sections, adjacent);
}
Tensor meta_paged_attention(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache,
                            const Tensor& block_table, const Tensor& seq_lens,
                            std::optional<double> scale) {
  MetaCall meta;
  return op_paged_attention(q, k_cache, v_cache, block_table, seq_lens, scale);
}

}  // namespace

TORCH_LIBRARY(operatorlib, m) {
  m.def("reduce_sum(Tensor input) -> Tensor");
  m.def("softmax(Tensor input) -> Tensor");
  m.def("transpose(Tensor input) -> Tensor");
  m.def("rmsnorm(Tensor input, Tensor weight, float epsilon=1e-5) -> Tensor");
  m.def("gemm(Tensor a, Tensor b) -> Tensor");
  m.def("attention(Tensor q, Tensor k, Tensor v, bool causal=False) -> Tensor");
  m.def(
      "rope(Tensor x, Tensor positions, Tensor inv_freq, int[] sections=[], bool adjacent=False, "
      "bool inverse=False) -> Tensor");
  m.def(
      "kv_append(Tensor q, Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, "
      "Tensor slots, Tensor positions, Tensor inv_freq, int[] sections=[], "
      "bool adjacent=False) -> Tensor");
  m.def(
      "paged_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, "
      "Tensor seq_lens, float? scale=None) -> Tensor");
}

TORCH_LIBRARY_IMPL(operatorlib, CUDA, m) {
  m.impl("reduce_sum", &op_reduce_sum);
  m.impl("softmax", &op_softmax);
  m.impl("transpose", &op_transpose);
  m.impl("rmsnorm", &op_rmsnorm);
  m.impl("gemm", &op_gemm);
  m.impl("attention", &op_attention);
  m.impl("rope", &op_rope);
  m.impl("kv_append", &op_kv_append);
  m.impl("paged_attention", &op_paged_attention);
}

TORCH_LIBRARY_IMPL(operatorlib, Meta, m) {
  m.impl("reduce_sum", &meta_reduce_sum);
  m.impl("softmax", &meta_softmax);
  m.impl("transpose", &meta_transpose);
  m.impl("rmsnorm", &meta_rmsnorm);
  m.impl("gemm", &meta_gemm);
  m.impl("attention", &meta_attention);
  m.impl("rope", &meta_rope);
  m.impl("kv_append", &meta_kv_append);
  m.impl("paged_attention", &meta_paged_attention);
}
