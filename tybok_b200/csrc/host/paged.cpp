// The paged cache: page plan, head norms with rotation and store, attention over pages.
#include <ATen/cuda/EmptyTensor.h>

#include <algorithm>

#include "native.h"

namespace tbn {

static void need_ints(const Tensor& t, int64_t n, const char* what, const char* name) {
  if (!is_vector(t, at::kInt, n)) type_error(std::string(what) + ": " + name + " must be contiguous int32 [" + std::to_string(n) + "]");
}

// A new tensor on the device of another, without the dispatcher's half a microsecond (the calls here are bound by the host).
static Tensor new_tensor(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
}

// Tensors of one allocation, 16-byte aligned pieces of it (an allocation each would cost a call as much as its launch); or, `apart`, of
// their own.
class Pieces {
 public:
  Pieces(const Tensor& like, bool apart) : like_(like), apart_(apart) {}
  void add(int64_t n) { size_ += (n + 3) & ~int64_t(3); }
  void allocate() {
    if (!apart_) buf_ = new_tensor({size_}, at::kInt, like_);
  }
  Tensor take(at::IntArrayRef sizes) {
    if (apart_) return new_tensor(sizes, at::kInt, like_);
    int64_t n = 1;
    for (const int64_t s : sizes) n *= s;
    Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buf_.storage()), buf_.key_set(), buf_.dtype());
    t.unsafeGetTensorImpl()->set_storage_offset(at_);
    t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
    at_ += (n + 3) & ~int64_t(3);
    return t;
  }

 private:
  Tensor like_, buf_;
  bool apart_;
  int64_t size_ = 0, at_ = 0;
};

using Plan = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>;

// (lengths, table, stack, count, cu_tokens, pos, slots, missing); the first four are the given tensors themselves in place.  What is new
// lies in one allocation (a second one costs a small plan 7.9 us instead of 7.1), or, `apart`, in one for each.
static Plan page_plan(const Tensor& lens, const Tensor& fresh, const Tensor& table, const Tensor& stack, const Tensor& count, int64_t tokens,
                      int64_t page, const OptTensor& finished, bool in_place, bool apart) {
  const char* what = in_place ? "page_plan_" : "page_plan";
  if (lens.dim() != 1 || lens.numel() < 1) type_error(std::string(what) + ": key_lens must be int32 [B] with one request at least");
  const int64_t b = lens.numel();
  need_ints(lens, b, what, "key_lens");
  need_ints(fresh, b, what, "new_lens");
  if (table.scalar_type() != at::kInt || table.dim() != 2 || table.size(0) != b || table.size(1) < 1 || !table.is_contiguous())
    type_error(std::string(what) + ": block_table must be contiguous int32 [B, width]");
  if (stack.dim() != 1 || stack.numel() < 1) type_error(std::string(what) + ": free_pages must be int32 [pages]");
  need_ints(stack, stack.numel(), what, "free_pages");
  need_ints(count, 1, what, "free_count");
  if (finished && ((finished->scalar_type() != at::kBool && finished->scalar_type() != at::kByte) || finished->numel() != b || !finished->is_contiguous()))
    type_error(std::string(what) + ": finished must be contiguous bool or uint8 [B]");
  if (tokens < 0 || tokens > 0x7fffffff || page < 1 || page > 0x40000000 || table.size(1) > 0x7fffffff || stack.numel() > 0x7fffffff)
    value_error(std::string(what) + ": tokens and page_size must be 31-bit numbers, tokens not negative");
  same_device(lens.device(), what, {&fresh, &table, &stack, &count, opt(finished)});
  require_cuda(lens, what);
  const c10::cuda::CUDAGuard guard(lens.device());
  const int64_t width = table.size(1), pages = stack.numel();
  Pieces mem(lens, apart);
  if (!in_place)
    for (const int64_t n : {b, b * width, pages, int64_t(1)}) mem.add(n);
  for (const int64_t n : {b + 1, tokens, tokens, int64_t(1)}) mem.add(n);
  mem.allocate();
  Tensor lens2 = in_place ? lens : mem.take({b}), table2 = in_place ? table : mem.take({b, width});
  Tensor stack2 = in_place ? stack : mem.take({pages}), count2 = in_place ? count : mem.take({1});
  Tensor cu = mem.take({b + 1}), pos = mem.take({tokens}), slots = mem.take({tokens}), missing = mem.take({1});
  const auto ip = [](const Tensor& t) { return static_cast<int*>(t.data_ptr()); };
  check(tybok_page_plan(ip(lens), ip(fresh), ptr(finished), ip(table), ip(stack), ip(count), ip(lens2), ip(table2), ip(stack2), ip(count2), ip(cu),
                        ip(pos), ip(slots), ip(missing), b, width, pages, tokens, page, stream_of(lens)),
        "tybok_page_plan");
  return {lens2, table2, stack2, count2, cu, pos, slots, missing};
}

// A pool of pages [P, G, page, D]: any strides that the kernels' 16-byte accesses take.
static void need_pool(const Tensor& t, const char* what, const char* name) {
  const std::string who = std::string(what) + ": " + name;
  if (!is_bf16(t) || t.dim() != 4 || t.numel() == 0) type_error(who + " must be bf16 [pages, kv heads, page size, head dim]");
  bool ok = t.stride(3) == 1 && !(reinterpret_cast<uintptr_t>(t.data_ptr()) & 15);
  for (int i = 0; i < 3; ++i) ok = ok && t.stride(i) % 8 == 0 && (t.stride(i) > 0 || t.size(i) == 1);
  if (!ok) type_error(who + " must have unit stride along the head, other strides positive multiples of 8 elements and a 16-byte aligned start");
  if (t.size(0) > 0x7fffffff || t.size(2) > 0x7fffffff) value_error(who + ": pages and their size must be 31-bit numbers");
}

// Whether a pool's rows share no element: each stride, from the smallest up, passes over all that lies inside it.
static bool rows_apart(const Tensor& t) {
  int order[3] = {0, 1, 2};
  std::sort(order, order + 3, [&](int a, int b) { return t.stride(a) < t.stride(b); });
  int64_t inside = t.size(3);
  for (const int i : order) {
    if (t.size(i) == 1) continue;
    if (t.stride(i) < inside) return false;
    inside += t.stride(i) * (t.size(i) - 1);
  }
  return true;
}

static Tensor head_norm_rope_store(const Tensor& qkv, const Tensor& pos, const Tensor& slots, const Tensor& cos, const Tensor& sin, const Tensor& kp,
                                   const Tensor& vp, int64_t heads, const OptTensor& norm_q, const OptTensor& norm_k, double eps, bool paired) {
  const char* what = "head_norm_rope_store";
  need_pool(kp, what, "k_pages");
  need_pool(vp, what, "v_pages");
  if (kp.sizes() != vp.sizes()) value_error("head_norm_rope_store: key and value pages differ in shape");
  if (!rows_apart(kp) || !rows_apart(vp) || kp.data_ptr() == vp.data_ptr()) value_error("head_norm_rope_store: rows of the pools must not overlap");
  const int64_t g = kp.size(1), page = kp.size(2), d = kp.size(3);
  if (!is_bf16(qkv) || qkv.dim() != 2) type_error("head_norm_rope_store: qkv must be bf16 [tokens, (H + 2G) * D]");
  if (heads < 1 || qkv.size(1) != (heads + 2 * g) * d) value_error("head_norm_rope_store: the rows of qkv must hold H + 2G heads");
  const int64_t t = qkv.size(0);
  need_ints(pos, t, what, "pos");
  need_ints(slots, t, what, "slots");
  if (cos.scalar_type() != at::kFloat || cos.dim() != 2 || !cos.is_contiguous() || sin.scalar_type() != at::kFloat || !sin.is_contiguous() ||
      sin.sizes() != cos.sizes())
    type_error("head_norm_rope_store: cos and sin must be contiguous fp32 [positions, rotated channels / 2]");
  if (t > 0x7fffffff || cos.size(0) > 0x7fffffff || cos.size(1) > d) value_error("head_norm_rope_store: sizes must be 31-bit numbers, rotated channels at most the head's");
  for (const Tensor* w : {opt(norm_q), opt(norm_k)})
    if (w && !is_vector(*w, at::kFloat, d)) type_error("head_norm_rope_store: norm weights must be contiguous fp32 [head dim]");
  same_device(qkv.device(), what, {&pos, &slots, &cos, &sin, &kp, &vp, opt(norm_q), opt(norm_k)});
  require_cuda(qkv, what);
  const c10::cuda::CUDAGuard guard(qkv.device());
  const Tensor x = vector_rows_of(qkv);
  Tensor q = new_tensor({t, heads * d}, at::kBFloat16, x);
  if (t == 0) return q;
  const int64_t ks[3] = {kp.stride(0), kp.stride(1), kp.stride(2)}, vs[3] = {vp.stride(0), vp.stride(1), vp.stride(2)};
  check(tybok_head_norm_rope_store(ptr(x), x.stride(0), static_cast<const int*>(pos.data_ptr()), static_cast<const int*>(slots.data_ptr()), f32(cos),
                                   f32(sin), cos.size(0), 2 * cos.size(1), paired, norm_q ? f32(*norm_q) : nullptr, norm_k ? f32(*norm_k) : nullptr,
                                   eps, ptr(q), ptr(kp), ks, ptr(vp), vs, t, heads, g, d, kp.size(0), page, status_ptr(qkv.get_device()),
                                   stream_of(qkv)),
        "tybok_head_norm_rope_store");
  return q;
}

static std::tuple<Tensor, Tensor> paged_attention(const Tensor& q, const Tensor& kp, const Tensor& vp, const Tensor& table, const Tensor& cu,
                                                  const Tensor& lens, double scale, bool causal, std::optional<int64_t> max_tokens, bool out_bf16,
                                                  bool out_planes, int out_shift) {
  const char* what = "paged_attention";
  need_pool(kp, what, "k_pages");
  need_pool(vp, what, "v_pages");
  if (kp.sizes() != vp.sizes()) value_error("paged_attention: key and value pages differ in shape");
  const int64_t g = kp.size(1), page = kp.size(2), d = kp.size(3), b = lens.numel();
  if (!is_bf16(q) || q.dim() != 2) type_error("paged_attention: q must be bf16 [tokens, H * D]");
  const int64_t t = q.size(0), h = q.size(1) / d;
  if (h < 1 || q.size(1) != h * d || h % g != 0) value_error("paged_attention: the rows of q must hold whole heads, a multiple of the key heads");
  if (b < 1) value_error("paged_attention: one request at least");
  need_ints(lens, b, what, "key_lens");
  need_ints(cu, b + 1, what, "cu_tokens");
  if (table.scalar_type() != at::kInt || table.dim() != 2 || table.size(0) != b || table.size(1) < 1 || table.stride(1) != 1)
    type_error("paged_attention: block_table must be int32 [B, width] with unit inner stride");
  if (b > 0x7fffffff || t > 0x7fffffff || table.size(1) > 0x7fffffff) value_error("paged_attention: sizes must be 31-bit numbers");
  if (!out_bf16 && !out_planes) value_error("at least one of out_bf16 / out_planes must be set");
  if (max_tokens && *max_tokens < 1) value_error("paged_attention: max_tokens must be positive");
  same_device(q.device(), what, {&kp, &vp, &table, &cu, &lens});
  require_cuda(q, what);
  const c10::cuda::CUDAGuard guard(q.device());
  const Tensor x = vector_rows_of(q);
  Tensor y = out_bf16 ? new_tensor({t, h * d}, at::kBFloat16, x) : new_tensor({0}, at::kBFloat16, x);
  Tensor yp = out_planes ? new_tensor({3, t, h * d}, at::kByte, x) : new_tensor({0}, at::kByte, x);
  if (t == 0) return {y, yp};
  const int64_t most = std::min(t, max_tokens.value_or(t));
  const size_t need = tybok_paged_attention_workspace_bytes(h, g, d, most);
  const Tensor ws = new_tensor({static_cast<int64_t>(need ? need : 1)}, at::kByte, x);
  const int64_t ks[3] = {kp.stride(0), kp.stride(1), kp.stride(2)}, vs[3] = {vp.stride(0), vp.stride(1), vp.stride(2)};
  check(tybok_paged_attention(ptr(x), x.stride(0), ptr(kp), ks, ptr(vp), vs, static_cast<const int*>(table.data_ptr()), table.stride(0),
                              static_cast<const int*>(cu.data_ptr()), static_cast<const int*>(lens.data_ptr()), out_bf16 ? ptr(y) : nullptr,
                              out_planes ? ptr(yp) : nullptr, out_shift, t, b, h, g, d, kp.size(0), page, table.size(1), most, causal, scale,
                              ptr(ws), need, status_ptr(q.get_device()), stream_of(q)),
        "tybok_paged_attention");
  return {y, yp};
}

void bind_paged(py::module_& m) {
  // (a registered op: its results share no memory)
  m.def(
      "page_plan_op",
      [](const Tensor& lens, const Tensor& fresh, const Tensor& table, const Tensor& stack, const Tensor& count, int64_t tokens, int64_t page,
         const OptTensor& finished, bool in_place) { return page_plan(lens, fresh, table, stack, count, tokens, page, finished, in_place, true); },
      NoGil());
  m.def("head_norm_rope_store_op", &head_norm_rope_store, NoGil());
  m.def("paged_attention_op", &paged_attention, NoGil());
  m.def(
      "page_plan",
      [](const Tensor& lens, const Tensor& fresh, const Tensor& table, const Tensor& stack, const Tensor& count, int64_t tokens, int64_t page,
         const OptTensor& finished, bool in_place) -> std::optional<Plan> {
        if (!plain({&lens, &fresh, &table, &stack, &count, opt(finished)})) return std::nullopt;
        return page_plan(lens, fresh, table, stack, count, tokens, page, finished, in_place, false);
      },
      NoGil());
  m.def(
      "head_norm_rope_store",
      [](const Tensor& qkv, const Tensor& pos, const Tensor& slots, const Tensor& cos, const Tensor& sin, const Tensor& kp, const Tensor& vp,
         int64_t heads, const OptTensor& norm_q, const OptTensor& norm_k, double eps, bool paired) -> OptTensor {
        if (!plain({&qkv, &pos, &slots, &cos, &sin, &kp, &vp, opt(norm_q), opt(norm_k)})) return std::nullopt;
        return head_norm_rope_store(qkv, pos, slots, cos, sin, kp, vp, heads, norm_q, norm_k, eps, paired);
      },
      NoGil());
  m.def(
      "paged_attention",
      [](const Tensor& q, const Tensor& kp, const Tensor& vp, const Tensor& table, const Tensor& cu, const Tensor& lens, double scale, bool causal,
         std::optional<int64_t> max_tokens, bool out_bf16, bool out_planes, int out_shift) -> std::optional<std::tuple<Tensor, Tensor>> {
        if (!plain({&q, &kp, &vp, &table, &cu, &lens})) return std::nullopt;
        return paged_attention(q, kp, vp, table, cu, lens, scale, causal, max_tokens, out_bf16, out_planes, out_shift);
      },
      NoGil());
}

}  // namespace tbn
