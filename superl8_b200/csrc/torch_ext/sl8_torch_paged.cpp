// Rotary positions and the paged int8 K/V cache of the torch extension: checks, allocation and the
// C-ABI calls (include/superl8_b200_paged.h).  The same checks, in the same words, as the ctypes twin
// in superl8_b200/_C.py.
#include <torch/extension.h>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <tuple>

#include "../../../include/superl8_b200.h"

namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;

void* stream_of(const Tensor& t) { return static_cast<void*>(at::cuda::getCurrentCUDAStream(t.get_device()).stream()); }

void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == SL8_OK, "superl8_b200 ", what, ": ", sl8_status_string(rc), " (status ", std::to_string(rc), ")");
}

int code_of(const Tensor& t, bool f32, const char* what, const char* name) {
  if (t.scalar_type() == at::kHalf) return SL8_F16;
  if (t.scalar_type() == at::kBFloat16) return SL8_BF16;
  if (f32 && t.scalar_type() == at::kFloat) return SL8_F32;
  TORCH_CHECK(false, "superl8_b200 ", what, ": ", name, " must be float16", f32 ? ", bfloat16 or float32" : " or bfloat16");
  return -1;
}

void check_on(const Tensor& t, const Tensor& like, const char* what) {
  TORCH_CHECK(t.is_cuda(), "superl8_b200 ", what, ": all inputs must be CUDA tensors");
  TORCH_CHECK(t.get_device() == like.get_device(), "superl8_b200 ", what, ": all inputs must be on the same device");
}

// Rows the kernels can take in place: contiguous channels (and, for the 16-byte loads of the cache kernels,
// aligned rows); anything else is copied.  So are rows that overlap with a step of one element: a result laid out
// like them would not have contiguous channels.
Tensor rows(const Tensor& t, bool aligned) {
  bool ok = t.stride(3) == 1 || t.size(3) == 1;
  for (int d = 0; d < 3; ++d) ok = ok && (t.size(d) <= 1 || t.stride(d) != 1);
  if (aligned && ok) {
    ok = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    for (int d = 0; d < 3; ++d) ok = ok && (t.size(d) <= 1 || t.stride(d) % 8 == 0);
  }
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

int64_t step(const Tensor& t, int d) { return t.size(d) == 1 ? 0 : t.stride(d); }

struct Freq {
  int rot = 0, n_axes = 1, pos64 = 0;
  const void* positions = nullptr;
  int64_t sa = 0, sb = 0, ss = 0;
  const float* inv_freq = nullptr;
  const uint8_t* axis = nullptr;
};

// positions [S], [B, S] or [axes, B, S] (a batch of 1 is shared); inv_freq fp32 [rot / 2]; freq_axis uint8.
Freq freq_of(const OptTensor& positions, const Tensor& inv_freq, const OptTensor& freq_axis, const Tensor& like, int64_t B, int64_t S,
             int64_t D, const char* what) {
  Freq f;
  check_on(inv_freq, like, what);
  TORCH_CHECK(inv_freq.scalar_type() == at::kFloat && inv_freq.dim() == 1 && inv_freq.is_contiguous(), "superl8_b200 ", what,
              ": inv_freq must be a contiguous float32 [rot / 2] tensor");
  TORCH_CHECK(2 * inv_freq.size(0) <= D, "superl8_b200 ", what, ": 2 * len(inv_freq) must not exceed the head dim");
  f.rot = (int)(2 * inv_freq.size(0));
  f.inv_freq = inv_freq.data_ptr<float>();
  if (positions.has_value()) {
    const Tensor& p = *positions;
    check_on(p, like, what);
    TORCH_CHECK(p.scalar_type() == at::kInt || p.scalar_type() == at::kLong, "superl8_b200 ", what, ": positions must be int32 or int64");
    TORCH_CHECK(p.dim() >= 1 && p.dim() <= 3, "superl8_b200 ", what, ": positions must be [S], [B, S] or [axes, B, S]");
    const int d = (int)p.dim();
    TORCH_CHECK(p.size(d - 1) == S && (d < 2 || p.size(d - 2) == B || p.size(d - 2) == 1) && (d < 3 || (p.size(0) >= 1 && p.size(0) <= 255)),
                "superl8_b200 ", what, ": positions must be [S], [B, S] or [axes, B, S]");
    f.positions = p.data_ptr();
    f.pos64 = p.scalar_type() == at::kLong;
    f.ss = p.stride(d - 1);
    f.sb = d >= 2 ? step(p, d - 2) : 0;
    f.sa = d == 3 ? p.stride(0) : 0;
    f.n_axes = d == 3 ? (int)p.size(0) : 1;
  }
  if (freq_axis.has_value()) {
    check_on(*freq_axis, like, what);
    TORCH_CHECK(freq_axis->scalar_type() == at::kByte && freq_axis->dim() == 1 && freq_axis->is_contiguous() &&
                    freq_axis->size(0) == inv_freq.size(0),
                "superl8_b200 ", what, ": freq_axis must be a contiguous uint8 [rot / 2] tensor");
    f.axis = freq_axis->data_ptr<uint8_t>();
  }
  TORCH_CHECK(f.n_axes == 1 || f.axis != nullptr, "superl8_b200 ", what, ": positions with several axes need freq_axis");
  return f;
}

std::tuple<Tensor, OptTensor> rope(const Tensor& q_in, const OptTensor& k_in, const Tensor& positions, const Tensor& inv_freq,
                                   const OptTensor& freq_axis, bool interleaved, bool inverse) {
  const char* what = "apply_rope";
  TORCH_CHECK(q_in.is_cuda(), "superl8_b200 ", what, ": all inputs must be CUDA tensors");
  TORCH_CHECK(q_in.dim() == 4, "superl8_b200 ", what, ": expect [B,H,S,D]");
  sl8_rope_params p{};
  p.dtype = code_of(q_in, true, what, "q");
  const int64_t B = q_in.size(0), S = q_in.size(2), D = q_in.size(3);
  TORCH_CHECK(D % 2 == 0 && D > 0, "superl8_b200 ", what, ": the head dim must be even");
  const c10::cuda::CUDAGuard guard(q_in.device());
  const Tensor q = rows(q_in, false);
  Tensor q_out = at::empty_like(q), k, k_out;
  if (k_in.has_value()) {
    check_on(*k_in, q_in, what);
    TORCH_CHECK(k_in->dim() == 4 && k_in->size(0) == B && k_in->size(2) == S && k_in->size(3) == D, "superl8_b200 ", what,
                ": q and k must agree in batch, length and head dim");
    TORCH_CHECK(k_in->scalar_type() == q_in.scalar_type(), "superl8_b200 ", what, ": q and k must share one dtype");
    k = rows(*k_in, false);
    k_out = at::empty_like(k);
    p.k = k.data_ptr(); p.k_out = k_out.data_ptr(); p.Hkv = (int)k.size(1);
    p.k_stride_b = step(k, 0); p.k_stride_h = step(k, 1); p.k_stride_s = step(k, 2);
    p.k_out_stride_b = step(k_out, 0); p.k_out_stride_h = step(k_out, 1); p.k_out_stride_s = step(k_out, 2);
  }
  const Freq f = freq_of(positions, inv_freq, freq_axis, q_in, B, S, D, what);
  p.q = q.data_ptr(); p.q_out = q_out.data_ptr();
  p.q_stride_b = step(q, 0); p.q_stride_h = step(q, 1); p.q_stride_s = step(q, 2);
  p.q_out_stride_b = step(q_out, 0); p.q_out_stride_h = step(q_out, 1); p.q_out_stride_s = step(q_out, 2);
  p.positions = f.positions; p.pos_stride_axis = f.sa; p.pos_stride_b = f.sb; p.pos_stride_s = f.ss; p.pos_is_64 = f.pos64;
  p.inv_freq = f.inv_freq; p.freq_axis = f.axis; p.n_axes = f.n_axes;
  p.B = (int)B; p.Hq = (int)q.size(1); p.S = (int)S; p.D = (int)D; p.rot = f.rot;
  p.interleaved = interleaved; p.inverse = inverse;
  if (q.numel() + (k.defined() ? k.numel() : 0) > 0) check_rc(sl8_rope(&p, stream_of(q)), what);
  return {q_out, k_in.has_value() ? OptTensor(k_out) : OptTensor()};
}

// The rotation is linear and orthogonal: its gradient is the rotation by the opposite angle, itself
// differentiable the same way.
struct RopeFunction : public torch::autograd::Function<RopeFunction> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const OptTensor& k,
                                                const Tensor& positions, const Tensor& inv_freq, const OptTensor& freq_axis,
                                                bool interleaved, bool inverse) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({positions, inv_freq, freq_axis.has_value() ? *freq_axis : Tensor()});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["inverse"] = inverse;
    const auto r = rope(q, k, positions, inv_freq, freq_axis, interleaved, inverse);
    if (!k.has_value()) return {std::get<0>(r)};
    return {std::get<0>(r), *std::get<1>(r)};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, const torch::autograd::variable_list& grads) {
    const auto saved = ctx->get_saved_variables();
    const bool interleaved = ctx->saved_data["interleaved"].toBool(), inverse = ctx->saved_data["inverse"].toBool();
    const OptTensor axis = saved[2].defined() ? OptTensor(saved[2]) : OptTensor();
    Tensor dq = grads[0], dk = grads.size() > 1 ? grads[1] : Tensor();
    if (dq.defined() || dk.defined()) {
      const bool both = dq.defined() && dk.defined();
      const auto r = RopeFunction::apply(dq.defined() ? dq : dk, both ? OptTensor(dk) : OptTensor(), saved[0], saved[1], axis, interleaved,
                                         !inverse);
      if (both) { dq = r[0]; dk = r[1]; }
      else if (dq.defined()) dq = r[0];
      else dk = r[0];
    }
    return {dq, dk, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, OptTensor> apply_rope(const Tensor& q, const OptTensor& k, const Tensor& positions, const Tensor& inv_freq,
                                         const OptTensor& freq_axis, bool interleaved) {
  TORCH_CHECK(!inv_freq.requires_grad(), "superl8_b200 apply_rope: inv_freq is a constant (no gradient is computed for it)");
  if (!(at::GradMode::is_enabled() && (q.requires_grad() || (k.has_value() && k->requires_grad()))))
    return rope(q, k, positions, inv_freq, freq_axis, interleaved, false);
  const auto r = RopeFunction::apply(q, k, positions, inv_freq, freq_axis, interleaved, false);
  return {r[0], k.has_value() ? OptTensor(r[1]) : OptTensor()};
}

// The cache's tensors and a batch's table and lengths.
sl8_paged_cache cache_of(const Tensor& k_i8, const Tensor& k_scale, const Tensor& v_i8, const Tensor& v_scale, const Tensor& table,
                         const Tensor& lens, const char* what) {
  TORCH_CHECK(k_i8.is_cuda(), "superl8_b200 ", what, ": all inputs must be CUDA tensors");
  for (const Tensor* t : {&k_scale, &v_i8, &v_scale, &table, &lens}) check_on(*t, k_i8, what);
  TORCH_CHECK(k_i8.scalar_type() == at::kChar && v_i8.scalar_type() == at::kChar, "superl8_b200 ", what, ": the cache's codes must be int8");
  TORCH_CHECK(k_i8.dim() == 4 && k_i8.sizes() == v_i8.sizes() && k_i8.is_contiguous() && v_i8.is_contiguous(), "superl8_b200 ", what,
              ": the cache's codes must be contiguous [pages, H_kv, page_size, D], K like V");
  TORCH_CHECK(k_scale.scalar_type() == at::kFloat && v_scale.scalar_type() == at::kFloat, "superl8_b200 ", what, ": scales must be float32");
  TORCH_CHECK(k_scale.dim() == 2 && k_scale.size(0) == k_i8.size(0) && k_scale.size(1) == k_i8.size(1) && k_scale.sizes() == v_scale.sizes() &&
                  k_scale.is_contiguous() && v_scale.is_contiguous(),
              "superl8_b200 ", what, ": scales must be contiguous [pages, H_kv]");
  const int64_t page = k_i8.size(2), D = k_i8.size(3);
  TORCH_CHECK(page == 16 || page == 32 || page == 64 || page == 128 || page == 256, "superl8_b200 ", what,
              ": page size must be 16/32/64/128/256, got ", std::to_string(page));
  TORCH_CHECK(D == 32 || D == 64 || D == 128 || D == 256, "superl8_b200 ", what, ": head dim must be 32/64/128/256, got ", std::to_string(D));
  TORCH_CHECK(table.scalar_type() == at::kInt && table.dim() == 2 && (table.size(1) <= 1 || table.stride(1) == 1), "superl8_b200 ", what,
              ": block_table must be int32 [B, pages per sequence] with contiguous rows");
  TORCH_CHECK(lens.scalar_type() == at::kInt && lens.dim() == 1 && lens.is_contiguous() && lens.size(0) == table.size(0), "superl8_b200 ", what,
              ": context_lens must be a contiguous int32 [B] tensor");
  sl8_paged_cache c{};
  c.k = k_i8.data_ptr<int8_t>(); c.v = v_i8.data_ptr<int8_t>();
  c.k_scale = k_scale.data_ptr<float>(); c.v_scale = v_scale.data_ptr<float>();
  c.block_table = table.data_ptr<int32_t>(); c.table_stride = table.stride(0); c.context_lens = lens.data_ptr<int32_t>();
  c.num_pages = (int)k_i8.size(0); c.Hkv = (int)k_i8.size(1); c.page_size = (int)page; c.D = (int)D; c.max_pages = (int)table.size(1);
  return c;
}

const int32_t* lens_of(const OptTensor& t, const Tensor& like, int64_t B, const char* name, const char* what) {
  if (!t.has_value()) return nullptr;
  check_on(*t, like, what);
  TORCH_CHECK(t->scalar_type() == at::kInt && t->dim() == 1 && t->is_contiguous() && t->size(0) == B, "superl8_b200 ", what, ": ", name,
              " must be a contiguous int32 [B] tensor");
  return t->data_ptr<int32_t>();
}

OptTensor kv_append_paged(const Tensor& k_in, const Tensor& v_in, const Tensor& k_i8, const Tensor& k_scale, const Tensor& v_i8,
                          const Tensor& v_scale, const Tensor& table, const Tensor& lens, const OptTensor& new_lens, const OptTensor& q_in,
                          const OptTensor& positions, const OptTensor& inv_freq, const OptTensor& freq_axis, bool interleaved) {
  const at::NoGradGuard no_grad;   // the cache operators carry no gradient
  const char* what = "kv_append_paged";
  const sl8_paged_cache c = cache_of(k_i8, k_scale, v_i8, v_scale, table, lens, what);
  check_on(k_in, k_i8, what);
  check_on(v_in, k_i8, what);
  sl8_append_params p{};
  p.dtype = code_of(k_in, false, what, "k");
  TORCH_CHECK(v_in.scalar_type() == k_in.scalar_type(), "superl8_b200 ", what, ": k and v must share one dtype");
  TORCH_CHECK(k_in.dim() == 4 && k_in.sizes() == v_in.sizes(), "superl8_b200 ", what, ": expect k and v [B,H,S,D] of one shape");
  const int64_t B = k_in.size(0), M = k_in.size(2), D = k_in.size(3);
  TORCH_CHECK(B == lens.size(0) && k_in.size(1) == c.Hkv && D == c.D, "superl8_b200 ", what,
              ": k and v must match the cache and block_table in batch, heads and head dim");
  p.new_lens = lens_of(new_lens, k_i8, B, "new_lens", what);
  TORCH_CHECK(inv_freq.has_value() || (!q_in.has_value() && !positions.has_value() && !freq_axis.has_value()), "superl8_b200 ", what,
              ": q, positions and freq_axis need inv_freq");
  const c10::cuda::CUDAGuard guard(k_i8.device());
  p.n_axes = 1;
  if (inv_freq.has_value()) {
    const Freq f = freq_of(positions, *inv_freq, freq_axis, k_i8, B, M, D, what);
    TORCH_CHECK(f.rot % 16 == 0, "superl8_b200 ", what, ": 2 * len(inv_freq) must be a multiple of 16");
    p.positions = f.positions; p.pos_stride_axis = f.sa; p.pos_stride_b = f.sb; p.pos_stride_s = f.ss; p.pos_is_64 = f.pos64;
    p.inv_freq = f.inv_freq; p.freq_axis = f.axis; p.n_axes = f.n_axes; p.rot = f.rot;
  }
  const Tensor k = rows(k_in, true), v = rows(v_in, true);
  p.k_new = k.data_ptr(); p.v_new = v.data_ptr();
  p.k_stride_b = step(k, 0); p.k_stride_h = step(k, 1); p.k_stride_s = step(k, 2);
  p.v_stride_b = step(v, 0); p.v_stride_h = step(v, 1); p.v_stride_s = step(v, 2);
  p.B = (int)B; p.M = (int)M; p.interleaved = interleaved;
  Tensor q, q_out;
  if (q_in.has_value()) {
    check_on(*q_in, k_i8, what);
    TORCH_CHECK(q_in->scalar_type() == k_in.scalar_type(), "superl8_b200 ", what, ": q must have the dtype of k and v");
    TORCH_CHECK(q_in->dim() == 4 && q_in->size(0) == B && q_in->size(2) == M && q_in->size(3) == D, "superl8_b200 ", what,
                ": q must be [B,H_q,S,D] with the batch, length and head dim of k");
    q = rows(*q_in, true);
    q_out = at::empty_like(q);
    p.q = q.data_ptr(); p.q_out = q_out.data_ptr(); p.Hq = (int)q.size(1);
    p.q_stride_b = step(q, 0); p.q_stride_h = step(q, 1); p.q_stride_s = step(q, 2);
    p.q_out_stride_b = step(q_out, 0); p.q_out_stride_h = step(q_out, 1); p.q_out_stride_s = step(q_out, 2);
  }
  if (k.numel() + (q.defined() ? q.numel() : 0) > 0) check_rc(sl8_kv_append_paged(&c, &p, stream_of(k_i8)), what);
  return q_in.has_value() ? OptTensor(q_out) : OptTensor();
}

std::tuple<Tensor, Tensor> kv_read_paged(const Tensor& k_i8, const Tensor& k_scale, const Tensor& v_i8, const Tensor& v_scale,
                                         const Tensor& table, const Tensor& lens, int64_t num_tokens, const OptTensor& first, bool bf16) {
  const char* what = "kv_read_paged";
  const sl8_paged_cache c = cache_of(k_i8, k_scale, v_i8, v_scale, table, lens, what);
  TORCH_CHECK(num_tokens >= 0 && num_tokens <= 0x7fffffff, "superl8_b200 ", what, ": num_tokens must not be negative");
  const int32_t* from = lens_of(first, k_i8, lens.size(0), "first", what);
  const c10::cuda::CUDAGuard guard(k_i8.device());
  const auto opt = k_i8.options().dtype(bf16 ? at::kBFloat16 : at::kHalf);
  Tensor k = at::empty({lens.size(0), c.Hkv, num_tokens, c.D}, opt), v = at::empty_like(k);
  if (k.numel() > 0)
    check_rc(sl8_kv_read_paged(&c, (int)lens.size(0), from, (int)num_tokens, bf16 ? SL8_BF16 : SL8_F16, k.data_ptr(), v.data_ptr(),
                               stream_of(k_i8)), what);
  return {k, v};
}

Tensor attn_paged(const Tensor& q_in, const Tensor& k_i8, const Tensor& k_scale, const Tensor& v_i8, const Tensor& v_scale,
                  const Tensor& table, const Tensor& lens, const c10::optional<double>& scale, bool causal, int64_t window_left,
                  const OptTensor& query_lens, int64_t max_context_len, int64_t backend) {
  const at::NoGradGuard no_grad;   // the cache operators carry no gradient
  const char* what = "attn_paged_cached";
  const sl8_paged_cache c = cache_of(k_i8, k_scale, v_i8, v_scale, table, lens, what);
  check_on(q_in, k_i8, what);
  sl8_paged_attn_params p{};
  p.dtype = code_of(q_in, false, what, "q");
  TORCH_CHECK(q_in.dim() == 4, "superl8_b200 ", what, ": expect q [B,H,S,D]");
  const int64_t B = q_in.size(0), Hq = q_in.size(1), M = q_in.size(2);
  TORCH_CHECK(B == lens.size(0) && q_in.size(3) == c.D, "superl8_b200 ", what, ": q must match the cache and block_table in batch and head dim");
  TORCH_CHECK(c.Hkv > 0 && Hq % c.Hkv == 0, "superl8_b200 ", what, ": H_q must be divisible by H_kv (GQA)");
  p.query_lens = lens_of(query_lens, k_i8, B, "query_lens", what);
  const c10::cuda::CUDAGuard guard(k_i8.device());
  const Tensor q = rows(q_in, true);
  Tensor out = at::empty_like(q);
  if (out.numel() == 0) return out;
  p.q = q.data_ptr(); p.out = out.data_ptr();
  p.q_stride_b = step(q, 0); p.q_stride_h = step(q, 1); p.q_stride_s = step(q, 2);
  p.out_stride_b = step(out, 0); p.out_stride_h = step(out, 1); p.out_stride_s = step(out, 2);
  p.B = (int)B; p.Hq = (int)Hq; p.M = (int)M; p.causal = causal;
  p.window_left = window_left < 0 ? -1 : (int)std::min<int64_t>(window_left, 0x7fffffff);
  p.max_context_len = (int)std::max<int64_t>(0, std::min<int64_t>(max_context_len, 0x7fffffff));
  p.softmax_scale = (float)(scale.has_value() ? *scale : 1.0 / std::sqrt((double)c.D));
  p.backend = (int)backend;
  const size_t bytes = sl8_attn_paged_workspace(&c, &p);
  Tensor ws = at::empty({(int64_t)bytes}, k_i8.options().dtype(at::kByte));
  check_rc(sl8_attn_paged(&c, &p, ws.data_ptr(), bytes, stream_of(k_i8)), what);
  return out;
}

}  // namespace

void bind_paged(pybind11::module_& m) {
  namespace py = pybind11;
  m.def("rope", &rope, py::arg("q"), py::arg("k"), py::arg("positions"), py::arg("inv_freq"), py::arg("freq_axis"), py::arg("interleaved"),
        py::arg("inverse"));
  m.def("apply_rope", &apply_rope, py::arg("q"), py::arg("k"), py::arg("positions"), py::arg("inv_freq"), py::arg("freq_axis"),
        py::arg("interleaved"));
  m.def("kv_append_paged", &kv_append_paged, py::arg("k"), py::arg("v"), py::arg("k_i8"), py::arg("k_scale"), py::arg("v_i8"),
        py::arg("v_scale"), py::arg("block_table"), py::arg("context_lens"), py::arg("new_lens"), py::arg("q"), py::arg("positions"),
        py::arg("inv_freq"), py::arg("freq_axis"), py::arg("interleaved"));
  m.def("kv_read_paged", &kv_read_paged, py::arg("k_i8"), py::arg("k_scale"), py::arg("v_i8"), py::arg("v_scale"), py::arg("block_table"),
        py::arg("context_lens"), py::arg("num_tokens"), py::arg("first"), py::arg("bf16"));
  m.def("attn_paged", &attn_paged, py::arg("q"), py::arg("k_i8"), py::arg("k_scale"), py::arg("v_i8"), py::arg("v_scale"),
        py::arg("block_table"), py::arg("context_lens"), py::arg("scale"), py::arg("causal"), py::arg("window_left"), py::arg("query_lens"),
        py::arg("max_context_len"), py::arg("backend"));
}
