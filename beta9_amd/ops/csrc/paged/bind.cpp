// The paged cache's operators as torch functions: every shape, type and stride that a kernel assumes is checked here,
// before its launch. What lies on the GPU (lengths, tables, slots) is bounded by the kernels themselves.

#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <torch/extension.h>

#include <cmath>

#include "paged.h"

namespace {

using at::Tensor;
using paged::Type;

#define REQUIRE(cond, ...) TORCH_CHECK_VALUE(cond, __VA_ARGS__)

constexpr double kLog2E = 1.4426950408889634;

hipStream_t current_stream() { return at::hip::getCurrentHIPStreamMasqueradingAsCUDA(); }

void launched(hipError_t status, const char* name) {
  TORCH_CHECK(status == hipSuccess, name, ": ", hipGetErrorString(status));
}

void check_gpu(const Tensor& t, const Tensor& like, const char* name) {
  REQUIRE(t.is_cuda() && t.device() == like.device(), name, " must be on ", like.device(), ", is on ", t.device());
  TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), name,
              " requires a gradient: the paged cache's operators have none (use torch.no_grad or inference_mode)");
}

void check_ints(const Tensor& t, const Tensor& like, int64_t dims, const char* name) {
  check_gpu(t, like, name);
  TORCH_CHECK_TYPE(t.scalar_type() == at::kInt, name, " must be int32, is ", t.scalar_type());
  REQUIRE(t.dim() == dims && (t.numel() == 0 || t.stride(dims - 1) == 1), name, " must have ", dims,
          " dimension(s), the last without gaps");
}

int page_log2(int64_t page_size) {
  REQUIRE(page_size >= 16 && page_size <= 256 && (page_size & (page_size - 1)) == 0,
          "page_size must be 16, 32, 64, 128 or 256, is ", page_size);
  int log2 = 0;
  while ((1LL << log2) < page_size) log2++;
  return log2;
}

Type type_of(const Tensor& t, const char* name) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, name, " must be bfloat16 or float16, is ",
                   t.scalar_type());
  return t.scalar_type() == at::kBFloat16 ? Type::kBF16 : Type::kFP16;
}

Type check_caches(const Tensor& k, const Tensor& v, const Tensor& like, Type type) {
  check_gpu(k, like, "k_cache");
  check_gpu(v, like, "v_cache");
  REQUIRE(k.dim() == 4 && k.sizes() == v.sizes(), "k_cache and v_cache must be [pages, kv heads, page size, head dim] of one shape");
  REQUIRE(k.is_contiguous() && v.is_contiguous(), "k_cache and v_cache must be contiguous");
  REQUIRE(((uintptr_t)k.data_ptr() | (uintptr_t)v.data_ptr()) % 16 == 0, "k_cache and v_cache must begin on 16 bytes");
  TORCH_CHECK_TYPE(k.scalar_type() == v.scalar_type() &&
                       (k.scalar_type() == like.scalar_type() || k.scalar_type() == at::kFloat8_e4m3fn),
                   "k_cache and v_cache must both be ", like.scalar_type(), " or float8_e4m3fn");
  REQUIRE(k.size(0) >= 1 && k.size(1) >= 1, "the cache must have a page and a head");
  REQUIRE(k.size(0) * k.size(2) < (1LL << 31), "the cache must have fewer than 2^31 slots");
  REQUIRE(k.size(0) * k.size(2) * k.size(1) < (1LL << 32), "the cache must have fewer than 2^32 rows of a head");
  REQUIRE(k.size(3) % 8 == 0 && k.size(3) >= 8 && k.size(3) <= paged::kMaxHeadDim, "head dim must be a multiple of 8, at most ",
          paged::kMaxHeadDim, ", is ", k.size(3));
  return k.scalar_type() == at::kFloat8_e4m3fn ? Type::kE4M3 : type;
}

void check_table(const Tensor& tables, const Tensor& like, int64_t page_size) {
  check_ints(tables, like, 2, "tables");
  REQUIRE(tables.size(0) <= paged::kMaxRequests, "at most ", paged::kMaxRequests, " requests, got ", tables.size(0));
  REQUIRE(tables.size(1) >= 1 && tables.size(1) * page_size <= (1LL << 30), "a table row must name at least 1 and at most 2^30 slots");
}

// The kernels multiply by it and by its inverse, in 32 bits.
void check_scale(double x, const char* name) {
  REQUIRE(x >= 0x1p-126 && x <= 0x1p126, name, " must be a positive number that fits 32 bits, and its inverse too, is ", x);
}

// A view of n values of a one-dimensional buffer, made directly: six of them by the dispatcher cost more than the launch.
Tensor part_of(const Tensor& buffer, int64_t first, int64_t n) {
  Tensor t = at::detail::make_tensor<at::TensorImpl>(c10::Storage(buffer.storage()), buffer.key_set(), buffer.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(first);
  t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  return t;
}

std::vector<Tensor> plan_step(const Tensor& tables, const Tensor& lens, const Tensor& new_lens, const Tensor& free_pages,
                              const Tensor& free_count, int64_t page_size, int64_t num_tokens) {
  paged::PlanArgs a;
  a.page_log2 = page_log2(page_size);
  check_table(tables, tables, page_size);
  int64_t n = tables.size(0);
  REQUIRE(n >= 1, "tables must have a row");
  REQUIRE(n == 1 || tables.stride(0) >= tables.size(1), "the rows of tables must not overlap");
  check_ints(lens, tables, 1, "lens");
  check_ints(new_lens, tables, 1, "new_lens");
  check_ints(free_pages, tables, 1, "free_pages");
  check_ints(free_count, tables, 1, "free_count");
  REQUIRE(lens.size(0) == n && new_lens.size(0) == n, "lens and new_lens must have one value for each of the ", n, " rows of tables");
  REQUIRE(free_count.size(0) == 1, "free_count must have one value");
  REQUIRE(free_pages.size(0) * page_size < (1LL << 31), "the cache must have fewer than 2^31 slots");
  REQUIRE(num_tokens >= 0 && num_tokens < (1LL << 31), "num_tokens must be 0 or more and fit 31 bits, is ", num_tokens);
  c10::DeviceGuard guard(tables.device());
  // one buffer: slots and positions, then lens and free_count next to each other, cu_new, kv_lens
  int64_t at_lens = 2 * num_tokens, at_cu = at_lens + n + 1, at_kv = at_cu + n + 1;
  Tensor all = at::empty({at_kv + n}, tables.options());
  int* base = all.data_ptr<int>();
  a.tables = tables.data_ptr<int>(), a.lens = lens.data_ptr<int>(), a.new_lens = new_lens.data_ptr<int>();
  a.free_pages = free_pages.data_ptr<int>(), a.free_count = free_count.data_ptr<int>();
  a.slots = base, a.positions = base + num_tokens;
  a.lens_out = base + at_lens, a.free_out = a.lens_out + n, a.cu_new = base + at_cu, a.kv_lens = base + at_kv;
  a.requests = (int)n, a.width = (int)tables.size(1), a.pages = (int)free_pages.size(0), a.tokens = (int)num_tokens;
  a.table_stride = tables.stride(0);
  launched(paged::launch_plan(a, current_stream()), "plan_step");
  return {part_of(all, 0, num_tokens), part_of(all, num_tokens, num_tokens), part_of(all, at_cu, n + 1),
          part_of(all, at_kv, n), part_of(all, at_lens, n), part_of(all, at_lens + n, 1)};
}

std::vector<Tensor> release_pages(const Tensor& tables, const Tensor& lens, const Tensor& done, const Tensor& free_pages,
                                  const Tensor& free_count, int64_t page_size) {
  paged::ReleaseArgs a;
  a.page_log2 = page_log2(page_size);
  check_table(tables, tables, page_size);
  int64_t n = tables.size(0);
  REQUIRE(n >= 1, "tables must have a row");
  REQUIRE(n == 1 || tables.stride(0) >= tables.size(1), "the rows of tables must not overlap");
  check_ints(lens, tables, 1, "lens");
  check_ints(free_pages, tables, 1, "free_pages");
  check_ints(free_count, tables, 1, "free_count");
  check_gpu(done, tables, "done");
  TORCH_CHECK_TYPE(done.scalar_type() == at::kBool, "done must be bool, is ", done.scalar_type());
  REQUIRE(done.dim() == 1 && done.is_contiguous() && lens.size(0) == n && done.size(0) == n,
          "lens and done must have one value for each of the ", n, " rows of tables");
  REQUIRE(free_count.size(0) == 1, "free_count must have one value");
  REQUIRE(free_pages.size(0) * page_size < (1LL << 31), "the cache must have fewer than 2^31 slots");
  c10::DeviceGuard guard(tables.device());
  Tensor state = at::empty({n + 1}, tables.options());
  a.tables = tables.data_ptr<int>(), a.lens = lens.data_ptr<int>(), a.done = (const uint8_t*)done.data_ptr();
  a.free_pages = free_pages.data_ptr<int>(), a.free_count = free_count.data_ptr<int>();
  a.lens_out = state.data_ptr<int>(), a.free_out = a.lens_out + n;
  a.requests = (int)n, a.width = (int)tables.size(1), a.pages = (int)free_pages.size(0), a.table_stride = tables.stride(0);
  launched(paged::launch_release(a, current_stream()), "release_pages");
  return {part_of(state, 0, n), part_of(state, n, 1)};
}

void write_kv(const Tensor& k, const Tensor& v, const Tensor& k_cache, const Tensor& v_cache, const Tensor& slots, double k_scale,
              double v_scale) {
  paged::WriteArgs a;
  check_gpu(k, k, "k");
  check_gpu(v, k, "v");
  a.type = type_of(k, "k");
  TORCH_CHECK_TYPE(v.scalar_type() == k.scalar_type(), "v must be ", k.scalar_type(), " like k, is ", v.scalar_type());
  a.cache = check_caches(k_cache, v_cache, k, a.type);
  a.page_log2 = page_log2(k_cache.size(2));
  REQUIRE(k.dim() == 3 && k.sizes() == v.sizes() && k.size(1) == k_cache.size(1) && k.size(2) == k_cache.size(3),
          "k and v must be [tokens, ", k_cache.size(1), ", ", k_cache.size(3), "] for this cache");
  // a grid's threads are counted in 32 bits
  REQUIRE(k.size(0) < (1LL << 31) && k.size(0) < (1LL << 32) / (k.size(1) * (k.size(2) / 8)), "too many tokens");
  REQUIRE(k.numel() == 0 || (k.stride(2) == 1 && v.stride(2) == 1), "k and v must have no gaps along the head dim");
  check_ints(slots, k, 1, "slots");
  REQUIRE(slots.size(0) == k.size(0), "slots must have one value for each of the ", k.size(0), " tokens, has ", slots.size(0));
  check_scale(k_scale, "k_scale");
  check_scale(v_scale, "v_scale");
  REQUIRE(a.cache == Type::kE4M3 || (k_scale == 1.0 && v_scale == 1.0), "only a float8_e4m3fn cache has scales");
  c10::DeviceGuard guard(k.device());
  a.k = k.data_ptr(), a.v = v.data_ptr(), a.k_cache = k_cache.data_ptr(), a.v_cache = v_cache.data_ptr();
  a.slots = slots.data_ptr<int>();
  a.k_row = k.stride(0), a.k_head = k.stride(1), a.v_row = v.stride(0), a.v_head = v.stride(1);
  a.tokens = (int)k.size(0), a.kv_heads = (int)k.size(1), a.dim = (int)k.size(2);
  a.slots_in_cache = k_cache.size(0) * k_cache.size(2);
  a.k_inverse = 1.f / (float)k_scale, a.v_inverse = 1.f / (float)v_scale;
  launched(paged::launch_write(a, current_stream()), "write_kv");
}

Tensor attend(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& tables, const Tensor& kv_lens,
              const Tensor* cu_new, double scale, double k_scale, double v_scale, const c10::optional<Tensor>& out_given) {
  paged::AttendArgs a;
  check_gpu(q, q, "q");
  a.type = type_of(q, "q");
  a.cache = check_caches(k_cache, v_cache, q, a.type);
  int64_t page_size = k_cache.size(2), kv_heads = k_cache.size(1), dim = k_cache.size(3);
  a.page_log2 = page_log2(page_size);
  REQUIRE(q.dim() == 3 && q.size(2) == dim, "q must be [rows, heads, ", dim, "] for this cache");
  REQUIRE(q.size(1) >= 1 && q.size(1) % kv_heads == 0, "q's ", q.size(1), " heads must be a multiple of the cache's ", kv_heads);
  REQUIRE(q.numel() == 0 || q.stride(2) == 1, "q must have no gaps along the head dim");
  REQUIRE(q.size(0) < (1LL << 31) / q.size(1) && q.size(1) <= 65535, "too many rows or heads");
  check_table(tables, q, page_size);
  check_ints(kv_lens, q, 1, "kv_lens");
  int64_t requests = tables.size(0);
  REQUIRE(kv_lens.size(0) == requests, "kv_lens must have one value for each of the ", requests, " rows of tables");
  if (cu_new) {
    check_ints(*cu_new, q, 1, "cu_new");
    REQUIRE(cu_new->size(0) == requests + 1, "cu_new must have ", requests + 1, " values, has ", cu_new->size(0));
  } else {
    REQUIRE(q.size(0) == requests, "q must have one row for each of the ", requests, " rows of tables");
  }
  REQUIRE(std::isfinite((float)(scale * k_scale * kLog2E)), "scale must be finite, also by k_scale in 32 bits");
  check_scale(k_scale, "k_scale");
  check_scale(v_scale, "v_scale");
  REQUIRE(a.cache == Type::kE4M3 || (k_scale == 1.0 && v_scale == 1.0), "only a float8_e4m3fn cache has scales");
  c10::DeviceGuard guard(q.device());
  Tensor out;
  if (out_given) {
    out = *out_given;
    check_gpu(out, q, "out");
    TORCH_CHECK_TYPE(out.scalar_type() == q.scalar_type(), "out must be ", q.scalar_type(), " like q, is ", out.scalar_type());
    REQUIRE(out.sizes() == q.sizes() && out.is_contiguous(), "out must be contiguous and of q's shape");
    REQUIRE((uintptr_t)out.data_ptr() % 16 == 0, "out must begin on 16 bytes");
    auto begin = [](const Tensor& t) { return (const char*)t.data_ptr(); };
    int64_t q_span = q.numel() ? ((q.size(0) - 1) * q.stride(0) + (q.size(1) - 1) * q.stride(1) + dim) * 2 : 0;
    REQUIRE(begin(out) + out.numel() * 2 <= begin(q) || begin(q) + q_span <= begin(out) || !out.numel(), "out must not overlap q");
  } else {
    out = at::empty(q.sizes(), q.options());
  }
  if (q.numel() == 0) return out;
  a.q = q.data_ptr(), a.out = out.data_ptr(), a.k_cache = k_cache.data_ptr(), a.v_cache = v_cache.data_ptr();
  a.tables = tables.data_ptr<int>(), a.kv_lens = kv_lens.data_ptr<int>(), a.cu_new = cu_new ? cu_new->data_ptr<int>() : nullptr;
  a.q_row = q.stride(0), a.q_head = q.stride(1), a.out_row = out.stride(0), a.out_head = out.stride(1), a.table_stride = tables.stride(0);
  a.rows = (int)q.size(0), a.requests = (int)requests, a.heads = (int)q.size(1), a.kv_heads = (int)kv_heads, a.dim = (int)dim;
  a.width = (int)tables.size(1), a.pages = (int)k_cache.size(0);
  a.score_scale = (float)(scale * k_scale * kLog2E), a.value_scale = (float)v_scale;
  a.clear_rest = out_given ? 0 : 1;
  REQUIRE(!cu_new || paged::prompt_fits(a), "too many rows, requests or heads");
  int64_t floats = cu_new ? paged::prompt_workspace(a) : paged::decode_workspace(a);
  Tensor workspace;
  if (floats) workspace = at::empty({floats}, q.options().dtype(at::kFloat));
  float* space = floats ? workspace.data_ptr<float>() : nullptr;
  launched(cu_new ? paged::launch_prompt(a, space, current_stream()) : paged::launch_decode(a, space, current_stream()),
           cu_new ? "prompt_attention" : "decode_attention");
  return out;
}

Tensor decode_attention(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& tables, const Tensor& kv_lens,
                        double scale, double k_scale, double v_scale, const c10::optional<Tensor>& out) {
  return attend(q, k_cache, v_cache, tables, kv_lens, nullptr, scale, k_scale, v_scale, out);
}

Tensor prompt_attention(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& tables, const Tensor& kv_lens,
                        const Tensor& cu_new, double scale, double k_scale, double v_scale, const c10::optional<Tensor>& out) {
  return attend(q, k_cache, v_cache, tables, kv_lens, &cu_new, scale, k_scale, v_scale, out);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("plan_step", &plan_step);
  m.def("release_pages", &release_pages);
  m.def("write_kv", &write_kv);
  m.def("decode_attention", &decode_attention);
  m.def("prompt_attention", &prompt_attention);
}
