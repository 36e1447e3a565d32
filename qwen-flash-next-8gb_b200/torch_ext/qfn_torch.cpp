// The thin torch extension over libqfn's C ABI: the parts of the hot path
// as torch operators (torch.ops.qfn.*), so that PyTorch callers reach the
// kernels through one dispatcher call instead of ctypes.  Each operator
// checks its tensors (type errors raise TypeError, shape / device errors
// ValueError, as the Python wrappers did), makes the tensors' device current,
// and calls the C entry point on torch's current stream; a non-zero status
// raises RuntimeError with the library's message.  No computation happens
// here: a missing libqfn.so fails at load time.
//
//   qfn::moe_decode  -> qfn_moe_decode_variant  (qmoe.moe_decode, qmoe.py:77-83)
//   qfn::moe_prefill -> qfn_moe_prefill         (the expert loop of QwenEngine.moe, qwen_engine.py:835-852)
//   qfn::gemv        -> qfn_gemv_e4m3           (fp8gemv.gemv, fp8gemv.py:5-26)
//   qfn::linear      -> qfn_linear_e4m3         (Lin.__call__ for T > 1, qwen_engine.py:79-83)
//   qfn::deltanet_chunk  -> qfn_deltanet_chunk      (the gated delta rule over prompts)
//   qfn::deltanet_step   -> qfn_deltanet_step_batch (one token for each request of a batch)
//   qfn::gated_norm      -> qfn_gated_norm
//   qfn::norm_residual   -> qfn_norm_residual
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <initializer_list>
#include <utility>

#include "qfn.h"

namespace {

void req_cuda(const at::Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a CUDA tensor (libqfn has no CPU path)");
  TORCH_CHECK_VALUE(t.is_contiguous(), name, " must be contiguous");
}

void req_type(const at::Tensor& t, const char* name, at::ScalarType dt) {
  TORCH_CHECK_TYPE(t.scalar_type() == dt, name, " must be ", dt, ", got ", t.scalar_type());
}

void same_device(const at::Tensor& t, const char* name, const at::Tensor& ref, const char* ref_name) {
  TORCH_CHECK_VALUE(t.device() == ref.device(), name, " is on ", t.device(), ", ", ref_name, " on ", ref.device());
}

void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == QFN_OK, what, ": ", qfn_strerror(rc), " (", qfn_last_error(), ")");
}

void* stream_of(const at::Tensor& t) {
  return static_cast<void*>(c10::cuda::getCurrentCUDAStream(t.device().index()).stream());
}

at::Tensor moe_decode(const at::Tensor& slots, const at::Tensor& sidx, const at::Tensor& s2, const at::Tensor& coef,
                      const at::Tensor& x, at::Tensor h_buf, int64_t variant) {
  const std::pair<const at::Tensor*, const char*> all[] = {
      {&slots, "slots_u8"}, {&sidx, "sidx"}, {&s2, "s2"}, {&coef, "coef"}, {&x, "x"}, {&h_buf, "h_buf"}};
  for (const auto& a : all) req_cuda(*a.first, a.second);
  req_type(slots, "slots_u8", at::kByte);
  req_type(sidx, "sidx", at::kInt);
  req_type(s2, "s2", at::kFloat);
  req_type(coef, "coef", at::kFloat);
  req_type(h_buf, "h_buf", at::kFloat);
  const int64_t K = sidx.numel();
  TORCH_CHECK_VALUE(slots.dim() == 2 && slots.size(1) == QFN_BLOCK_BYTES, "slots_u8 must be [S, ", QFN_BLOCK_BYTES,
                    "], got ", slots.sizes());
  TORCH_CHECK_VALUE(sidx.dim() == 1 && K >= 1 && K <= QFN_MAX_TOPK, "sidx must be int32[K] with 1 <= K <= ",
                    QFN_MAX_TOPK);
  TORCH_CHECK_VALUE(s2.dim() == 2 && s2.size(0) == K && s2.size(1) == 3 && coef.dim() == 1 && coef.size(0) == K,
                    "s2 must be [K,3] and coef [K]; got ", s2.sizes(), ", ", coef.sizes());
  TORCH_CHECK_VALUE(x.numel() == QFN_HID && (x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kFloat),
                    "x must be bf16/fp32 with ", QFN_HID, " elements");
  TORCH_CHECK_VALUE(h_buf.dim() == 2 && h_buf.size(0) >= K && h_buf.size(1) == QFN_INTER, "h_buf must be f32[>=K, ",
                    QFN_INTER, "]");
  for (const auto& a : all) same_device(*a.first, a.second, slots, "slots_u8");
  c10::cuda::CUDAGuard guard(slots.device());
  at::Tensor out = at::empty({QFN_HID}, slots.options().dtype(at::kFloat));
  check_rc(qfn_moe_decode_variant(slots.data_ptr<uint8_t>(), slots.size(0), sidx.data_ptr<int32_t>(),
                                  s2.data_ptr<float>(), coef.data_ptr<float>(), x.data_ptr(),
                                  x.scalar_type() == at::kFloat ? QFN_DTYPE_F32 : QFN_DTYPE_BF16,
                                  h_buf.data_ptr<float>(), out.data_ptr<float>(), static_cast<int>(K),
                                  static_cast<int>(variant), stream_of(out)),
           "qfn_moe_decode");
  return out;
}

at::Tensor moe_prefill(const at::Tensor& x, const at::Tensor& ti, const at::Tensor& tv, const at::Tensor& table,
                       const at::Tensor& s2, int64_t L) {
  const std::pair<const at::Tensor*, const char*> all[] = {
      {&x, "x"}, {&ti, "ti"}, {&tv, "tv"}, {&table, "table"}, {&s2, "s2"}};
  for (const auto& a : all) req_cuda(*a.first, a.second);
  req_type(x, "x", at::kBFloat16);
  req_type(table, "table", at::kByte);
  req_type(s2, "s2", at::kFloat);
  TORCH_CHECK_VALUE(x.dim() == 2 && x.size(1) == QFN_HID, "x must be bf16[T, ", QFN_HID, "], got ", x.sizes());
  const int64_t T = x.size(0);
  TORCH_CHECK_VALUE(ti.dim() == 2 && ti.size(0) == T && tv.sizes() == ti.sizes(),
                    "ti and tv must be [T, topk] with T=", T, "; got ", ti.sizes(), ", ", tv.sizes());
  TORCH_CHECK_TYPE(ti.scalar_type() == at::kLong || ti.scalar_type() == at::kInt, "ti must be int64 or int32");
  TORCH_CHECK_TYPE(tv.scalar_type() == at::kBFloat16 || tv.scalar_type() == at::kFloat, "tv must be bf16 or fp32");
  TORCH_CHECK_VALUE(s2.dim() == 2 && s2.size(1) == 3, "s2 must be f32[n_experts, 3], got ", s2.sizes());
  TORCH_CHECK_VALUE(table.dim() == 2 && table.size(1) == QFN_BLOCK_BYTES, "table must be [NB, ", QFN_BLOCK_BYTES,
                    "]");
  for (const auto& a : all) same_device(*a.first, a.second, x, "x");
  c10::cuda::CUDAGuard guard(x.device());
  const int topk = static_cast<int>(ti.size(1));
  const int E = static_cast<int>(s2.size(0));
  at::Tensor out = at::empty({T, QFN_HID}, x.options().dtype(at::kFloat));
  if (T == 0) return out;
  const size_t nbytes = qfn_moe_prefill_workspace(T, topk, E);
  at::Tensor ws = at::empty({static_cast<int64_t>(nbytes)}, x.options().dtype(at::kByte));
  check_rc(qfn_moe_prefill(x.data_ptr(), T, ti.data_ptr(), ti.scalar_type() == at::kLong ? 1 : 0, tv.data_ptr(),
                           tv.scalar_type() == at::kBFloat16 ? QFN_DTYPE_BF16 : QFN_DTYPE_F32, topk,
                           table.data_ptr<uint8_t>(), table.size(0), L * E, s2.data_ptr<float>(), E,
                           out.data_ptr<float>(), ws.data_ptr(), nbytes, stream_of(out)),
           "qfn_moe_prefill");
  return out;
}

at::Tensor gemv(const at::Tensor& q, const at::Tensor& s, const at::Tensor& x, bool out_f32) {
  req_cuda(q, "q");
  TORCH_CHECK_TYPE(q.scalar_type() == at::kFloat8_e4m3fn || q.scalar_type() == at::kByte,
                   "q must be float8_e4m3fn (or its raw uint8 bytes), got ", q.scalar_type());
  req_cuda(s, "s");
  req_type(s, "s", at::kFloat);
  req_cuda(x, "x");
  req_type(x, "x", at::kBFloat16);
  TORCH_CHECK_VALUE(q.dim() == 2, "q must be [N, K]");
  const int64_t N = q.size(0), K = q.size(1);
  TORCH_CHECK_VALUE(s.numel() == N && x.numel() == K, "s must have ", N, " and x ", K, " elements; got ", s.numel(),
                    ", ", x.numel());
  same_device(s, "s", q, "q");
  same_device(x, "x", q, "q");
  c10::cuda::CUDAGuard guard(q.device());
  at::Tensor y = at::empty({N}, q.options().dtype(out_f32 ? at::kFloat : at::kBFloat16));
  check_rc(qfn_gemv_e4m3(static_cast<const uint8_t*>(q.data_ptr()), s.data_ptr<float>(),
                         static_cast<const uint16_t*>(x.data_ptr()), y.data_ptr(),
                         out_f32 ? QFN_DTYPE_F32 : QFN_DTYPE_BF16, N, K, stream_of(y)),
           "qfn_gemv_e4m3");
  return y;
}

// Lin.__call__ for T > 1 (qwen_engine.py:79-83): x [T, K] bf16 -> [T, N] bf16.
at::Tensor linear(const at::Tensor& x, const at::Tensor& q, const at::Tensor& s) {
  req_cuda(q, "q");
  TORCH_CHECK_TYPE(q.scalar_type() == at::kFloat8_e4m3fn || q.scalar_type() == at::kByte,
                   "q must be float8_e4m3fn (or its raw uint8 bytes), got ", q.scalar_type());
  req_cuda(s, "s");
  req_type(s, "s", at::kFloat);
  req_cuda(x, "x");
  req_type(x, "x", at::kBFloat16);
  TORCH_CHECK_VALUE(q.dim() == 2 && x.dim() == 2, "q must be [N, K] and x [T, K]");
  const int64_t N = q.size(0), K = q.size(1), T = x.size(0);
  TORCH_CHECK_VALUE(x.size(1) == K && s.numel() == N, "x must be [T, ", K, "] and s have ", N, " elements; got ",
                    x.sizes(), ", ", s.numel());
  same_device(s, "s", q, "q");
  same_device(x, "x", q, "q");
  c10::cuda::CUDAGuard guard(q.device());
  // the kernel's TMA reads x from a 16-byte aligned base (a view may start anywhere)
  const at::Tensor xa = reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 ? x.clone() : x;
  at::Tensor y = at::empty({T, N}, x.options());
  if (T == 0 || N == 0) return y;
  check_rc(qfn_linear_e4m3(static_cast<const uint8_t*>(q.data_ptr()), s.data_ptr<float>(),
                           static_cast<const uint16_t*>(xa.data_ptr()), static_cast<uint16_t*>(y.data_ptr()), T, N, K,
                           stream_of(y)),
           "qfn_linear_e4m3");
  return y;
}

const at::Tensor* given(const std::optional<at::Tensor>& t) { return t ? &*t : nullptr; }

// Forward only: a result without its gradient would look like one with it.
void req_no_grad(const char* what, std::initializer_list<std::pair<const at::Tensor*, const char*>> tensors) {
  if (!at::GradMode::is_enabled()) return;
  for (const auto& t : tensors)
    TORCH_CHECK(!t.first || !t.first->requires_grad(), what, " is forward only and ", t.second,
                " requires a gradient (call it under torch.no_grad(), or detach it)");
}

// A CUDA tensor of type dt on ref's device; views pass.
void req_view(const at::Tensor& t, const char* name, at::ScalarType dt, const at::Tensor& ref, const char* ref_name) {
  TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a CUDA tensor (libqfn has no CPU path)");
  req_type(t, name, dt);
  same_device(t, name, ref, ref_name);
}

int dtype_code(const at::Tensor& t, const char* name) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16, name,
                   " must be bf16 or fp32, got ", t.scalar_type());
  return t.scalar_type() == at::kFloat ? QFN_DTYPE_F32 : QFN_DTYPE_BF16;
}

// Whether two tensors' memory (as dense as their sizes say) shares a byte.  Most tensors have storages of their own,
// which is told without their sizes (asking for those of a call's ten pairs took 0.3 us).
bool overlap(const at::Tensor& a, const at::Tensor& b) {
  const c10::StorageImpl *sa = a.storage().unsafeGetStorageImpl(), *sb = b.storage().unsafeGetStorageImpl();
  const uintptr_t pa = reinterpret_cast<uintptr_t>(sa->data()), pb = reinterpret_cast<uintptr_t>(sb->data());
  if (pa >= pb + sb->nbytes() || pb >= pa + sa->nbytes()) return false;
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.data_ptr()), y = reinterpret_cast<uintptr_t>(b.data_ptr());
  int64_t na = 0, nb = 0;
  if (a.numel() == 0 || b.numel() == 0) return false;
  for (int64_t i = 0; i < a.dim(); ++i) na += (a.size(i) - 1) * a.stride(i);
  for (int64_t i = 0; i < b.dim(); ++i) nb += (b.size(i) - 1) * b.stride(i);
  return x < y + (nb + 1) * b.element_size() && y < x + (na + 1) * a.element_size();
}

// `t` is written while others are still read.
void req_apart(const at::Tensor& t, const char* name,
               std::initializer_list<std::pair<const at::Tensor*, const char*>> others) {
  for (const auto& o : others)
    TORCH_CHECK_VALUE(!o.first || !o.first->defined() || !overlap(t, *o.first), name, " overlaps ", o.second);
}
// One operand of the batched delta rule as rows: [.., heads(, d)] after one or two leading dimensions that
// count as one.  Views are taken as they are if their last dimension is dense and their leading ones can be
// counted as one; others are copied.
struct DeltaOperand {
  at::Tensor t;
  int64_t row, head;
  DeltaOperand(const at::Tensor& x, int lead, bool vectors) : t(x) {
    const int64_t d = lead + 1;   // the vectors' dimension
    const bool dense = !vectors || t.stride(d) == 1;
    const bool merge = lead == 1 || t.size(0) <= 1 || t.size(1) <= 1 || t.stride(0) == t.size(1) * t.stride(1);
    if (!dense || !merge) t = t.contiguous();
    row = lead == 2 && t.size(1) <= 1 && t.size(0) > 1 ? t.stride(0) : t.stride(lead - 1);
    head = t.stride(lead);
  }
};

// q, k [.., Hq, dk], v [.., H, dv], g, beta [.., H] with the same one or two leading dimensions.
struct DeltaRows {
  const at::Tensor& q_;
  int lead;
  int64_t rows;
  int H, Hq, dk, dv;
  DeltaOperand q, k, v, g, beta;
  int64_t strides[10];
  static const at::Tensor& checked(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& g,
                                   const at::Tensor& beta, int lead) {
    TORCH_CHECK_VALUE(q.dim() == lead + 2, "query must be [", lead == 2 ? "B, T, " : "R, ", "heads, dk], got ", q.sizes());
    TORCH_CHECK_VALUE(k.sizes() == q.sizes(), "key must have query's shape ", q.sizes(), ", got ", k.sizes());
    TORCH_CHECK_VALUE(v.dim() == lead + 2 && v.sizes().slice(0, lead) == q.sizes().slice(0, lead) && q.size(lead) >= 1 &&
                          v.size(lead) >= 1 && v.size(lead) % q.size(lead) == 0,
                      "value must be ", q.sizes().slice(0, lead), " x a multiple of query's ", q.size(lead),
                      " heads x dv, got ", v.sizes());
    TORCH_CHECK_VALUE(g.dim() == lead + 1 && g.sizes() == v.sizes().slice(0, lead + 1), "g must be ",
                      v.sizes().slice(0, lead + 1), ", got ", g.sizes());
    TORCH_CHECK_VALUE(beta.sizes() == g.sizes(), "beta must be ", g.sizes(), ", got ", beta.sizes());
    req_view(q, "query", at::kBFloat16, q, "query");
    req_view(k, "key", at::kBFloat16, q, "query");
    req_view(v, "value", at::kBFloat16, q, "query");
    req_view(g, "g", at::kFloat, q, "query");
    req_view(beta, "beta", at::kBFloat16, q, "query");
    return q;
  }
  DeltaRows(const at::Tensor& q0, const at::Tensor& k0, const at::Tensor& v0, const at::Tensor& g0,
            const at::Tensor& beta0, int lead_)
      : q_(checked(q0, k0, v0, g0, beta0, lead_)), lead(lead_), rows(lead == 2 ? q0.size(0) * q0.size(1) : q0.size(0)),
        H(static_cast<int>(v0.size(lead))), Hq(static_cast<int>(q0.size(lead))), dk(static_cast<int>(q0.size(lead + 1))),
        dv(static_cast<int>(v0.size(lead + 1))), q(q0, lead, true), k(k0, lead, true), v(v0, lead, true),
        g(g0, lead, false), beta(beta0, lead, false) {
    const DeltaOperand* all[] = {&q, &k, &v, &g, &beta};
    for (int i = 0; i < 5; ++i) {
      strides[2 * i] = all[i]->row;
      strides[2 * i + 1] = all[i]->head;
    }
  }
};

const uint16_t* u16(const at::Tensor& t) { return static_cast<const uint16_t*>(t.data_ptr()); }

void req_state(const at::Tensor& S, const char* name, int64_t n, const DeltaRows& r) {
  req_view(S, name, at::kFloat, r.q_, "query");
  TORCH_CHECK_VALUE(S.dim() == 4 && (n < 0 || S.size(0) == n) && S.size(1) == r.H && S.size(2) == r.dk &&
                        S.size(3) == r.dv && S.is_contiguous(),
                    name, " must be a contiguous fp32 [", n < 0 ? std::string("slots") : std::to_string(n), ", ", r.H, ", ",
                    r.dk, ", ", r.dv, "], got ", S.sizes());
}

// A state to be written.  It may be the state that is read, whose overlap the library checks.
void req_new_state(const at::Tensor& S, const char* name, const DeltaRows& r, const std::optional<at::Tensor>& plan,
                   const char* plan_name) {
  req_apart(S, name, {{&r.q.t, "query"}, {&r.k.t, "key"}, {&r.v.t, "value"}, {&r.g.t, "g"}, {&r.beta.t, "beta"},
                      {given(plan), plan_name}});
}

at::Tensor req_out(const std::optional<at::Tensor>& out, const at::Tensor& value, const DeltaRows& r,
                   const std::optional<at::Tensor>& plan, const char* plan_name) {
  if (!out) return at::empty(value.sizes(), r.q_.options());
  req_view(*out, "out", at::kBFloat16, r.q_, "query");
  TORCH_CHECK_VALUE(out->is_contiguous() && out->sizes() == value.sizes(), "out must be a contiguous ", value.sizes(),
                    ", got ", out->sizes());
  req_apart(*out, "out", {{&r.q.t, "query"}, {&r.k.t, "key"}, {&r.v.t, "value"}, {&r.g.t, "g"}, {&r.beta.t, "beta"},
                          {given(plan), plan_name}});   // states: the library
  return *out;
}

// What an operator returns in the place of a tensor that its caller gave to be written: a returned tensor shares no
// memory with an argument and is returned once, as the schemas say.
at::Tensor written(const at::Tensor& like) { return at::empty({0}, like.options()); }

// query, key [B, T, Hq, dk], value [B, T, H, dv], g, beta [B, T, H]: B sequences, or (B = 1) those of cu_seqlens.
std::tuple<at::Tensor, at::Tensor> deltanet_chunk(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                  const at::Tensor& g, const at::Tensor& beta,
                                                  const std::optional<at::Tensor>& cu,
                                                  const std::optional<at::Tensor>& s_in,
                                                  const std::optional<at::Tensor>& s_out,
                                                  const std::optional<at::Tensor>& out_) {
  req_no_grad("deltanet_chunk", {{&q, "query"}, {&k, "key"}, {&v, "value"}, {&g, "g"}, {&beta, "beta"},
                                 {given(s_in), "initial_state"}, {given(s_out), "final_state"}, {given(out_), "out"}});
  TORCH_CHECK_VALUE(!cu || (q.dim() == 4 && q.size(0) == 1),
                    "cu_seqlens takes one batch row holding every sequence, got query ", q.sizes());
  TORCH_CHECK_VALUE(!out_ || out_->sizes() == v.sizes(), "out must be a contiguous ", v.sizes());
  const DeltaRows r(q, k, v, g, beta, 2);
  int64_t n_seqs = q.size(0);
  if (cu) {
    req_cuda(*cu, "cu_seqlens");
    req_type(*cu, "cu_seqlens", at::kInt);
    same_device(*cu, "cu_seqlens", q, "query");
    TORCH_CHECK_VALUE(cu->dim() == 1 && cu->size(0) >= 1, "cu_seqlens must be int32 [sequences + 1], got ",
                      cu->sizes());
    n_seqs = cu->size(0) - 1;
  }
  if (s_in) req_state(*s_in, "initial_state", n_seqs, r);
  if (s_out) {
    req_state(*s_out, "final_state", n_seqs, r);
    req_new_state(*s_out, "final_state", r, cu, "cu_seqlens");
  }
  c10::cuda::CUDAGuard guard(q.device());
  at::Tensor out = req_out(out_, v, r, cu, "cu_seqlens");
  at::Tensor S = s_out ? *s_out : at::empty({n_seqs, r.H, r.dk, r.dv}, g.options());
  // equal sequences need no workspace where one of them alone needs none
  const size_t nbytes = !cu && qfn_deltanet_chunk_workspace(q.size(1), 1, r.H, r.Hq, r.dk, r.dv) == 0
                            ? 0
                            : qfn_deltanet_chunk_workspace(r.rows, n_seqs, r.H, r.Hq, r.dk, r.dv);
  at::Tensor ws;
  if (nbytes) ws = at::empty({static_cast<int64_t>(nbytes)}, q.options().dtype(at::kByte));
  check_rc(qfn_deltanet_chunk(u16(r.q.t), u16(r.k.t), u16(r.v.t), r.g.t.data_ptr<float>(), u16(r.beta.t), r.strides,
                              cu ? cu->data_ptr<int32_t>() : nullptr, n_seqs, r.rows,
                              s_in ? s_in->data_ptr<float>() : nullptr, S.data_ptr<float>(),
                              static_cast<uint16_t*>(out.data_ptr()), r.H, r.Hq, r.dk, r.dv,
                              nbytes ? ws.data_ptr() : nullptr, nbytes, stream_of(q)),
           "qfn_deltanet_chunk");
  return {out_ ? written(out) : out, s_out ? written(S) : S};
}

at::Tensor deltanet_step(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& g,
                         const at::Tensor& beta, const at::Tensor& state, const std::optional<at::Tensor>& index,
                         at::Tensor out_state, const std::optional<at::Tensor>& out_) {
  req_no_grad("deltanet_step", {{&q, "query"}, {&k, "key"}, {&v, "value"}, {&g, "g"}, {&beta, "beta"}, {&state, "state"},
                                {&out_state, "out_state"}, {given(out_), "out"}});
  const DeltaRows r(q, k, v, g, beta, 1);
  const int64_t R = r.rows;
  req_state(state, "state", -1, r);
  req_state(out_state, "out_state", state.size(0), r);
  TORCH_CHECK_VALUE(R == 0 || state.size(0) >= 1, "state has no slots");
  if (index) {
    req_cuda(*index, "state_index");
    req_type(*index, "state_index", at::kInt);
    same_device(*index, "state_index", q, "query");
    TORCH_CHECK_VALUE(index->dim() == 1 && index->size(0) == R, "state_index must be int32 [", R, "], got ",
                      index->sizes());
  }
  TORCH_CHECK_VALUE(index || R <= state.size(0), "state has ", state.size(0), " slots for ", R,
                    " tokens (pass state_index)");
  req_new_state(out_state, "out_state", r, index, "state_index");
  c10::cuda::CUDAGuard guard(q.device());
  at::Tensor out = req_out(out_, v, r, index, "state_index");
  if (R == 0) return out_ ? written(out) : out;
  check_rc(qfn_deltanet_step_batch(u16(r.q.t), u16(r.k.t), u16(r.v.t), r.g.t.data_ptr<float>(), u16(r.beta.t), r.strides,
                                   index ? index->data_ptr<int32_t>() : nullptr, state.size(0),
                                   state.data_ptr<float>(), out_state.data_ptr<float>(),
                                   static_cast<uint16_t*>(out.data_ptr()), R, r.H, r.Hq, r.dk, r.dv, stream_of(q)),
           "qfn_deltanet_step_batch");
  return out_ ? written(out) : out;
}

// x, z [R, H, D], w [D] -> [R, H, D]
at::Tensor gated_norm(const at::Tensor& x_, const at::Tensor& z_, const at::Tensor& w, double eps) {
  at::Tensor x = x_, z = z_;
  req_no_grad("gated_norm", {{&x, "x"}, {&z, "z"}, {&w, "weight"}});
  req_view(x, "x", at::kBFloat16, x, "x");
  req_view(z, "z", at::kBFloat16, x, "x");
  req_cuda(w, "weight");
  same_device(w, "weight", x, "x");
  TORCH_CHECK_VALUE(x.dim() == 3 && z.sizes() == x.sizes() && w.dim() == 1 && w.size(0) == x.size(2),
                    "x and z must have the same shape and weight their last size; got ", x.sizes(), ", ", z.sizes(),
                    ", ", w.sizes());
  if (x.stride(2) != 1) x = x.contiguous();
  if (z.stride(2) != 1) z = z.contiguous();
  const int wd = dtype_code(w, "weight");
  c10::cuda::CUDAGuard guard(x.device());
  at::Tensor y = at::empty(x.sizes(), x.options());
  if (y.numel() == 0) return y;
  check_rc(qfn_gated_norm(u16(x), x.stride(0), x.stride(1), u16(z), z.stride(0), z.stride(1), w.data_ptr(), wd,
                          static_cast<uint16_t*>(y.data_ptr()), x.size(0), static_cast<int>(x.size(1)),
                          static_cast<int>(x.size(2)), static_cast<float>(eps), stream_of(y)),
           "qfn_gated_norm");
  return y;
}

// block, residual [T, D]; gate [T, 1] or [T, D]; residual_out: residual's type, contiguous.  Without next the second
// tensor is empty.
std::tuple<at::Tensor, at::Tensor> norm_residual(const at::Tensor& block_, const at::Tensor& residual_,
                                                 const std::optional<at::Tensor>& post,
                                                 const std::optional<at::Tensor>& gate_, bool sigmoid, double scale,
                                                 const std::optional<at::Tensor>& next, double eps,
                                                 const std::optional<at::Tensor>& r_out) {
  at::Tensor block = block_, residual = residual_, gate;
  req_no_grad("norm_residual", {{&block, "block"}, {&residual, "residual"}, {given(post), "post_weight"},
                                {given(gate_), "gate"}, {given(next), "next_weight"}, {given(r_out), "out"}});
  TORCH_CHECK_VALUE(block.is_cuda(), "block must be a CUDA tensor (libqfn has no CPU path)");
  TORCH_CHECK_VALUE(residual.is_cuda(), "residual must be a CUDA tensor (libqfn has no CPU path)");
  same_device(residual, "residual", block, "block");
  TORCH_CHECK_VALUE(block.dim() == 2 && residual.sizes() == block.sizes(),
                    "block and residual must have the same shape; got ", block.sizes(), ", ", residual.sizes());
  const int64_t T = block.size(0), D = block.size(1);
  const int bd = dtype_code(block, "block"), rd = dtype_code(residual, "residual");
  if (block.stride(1) != 1) block = block.contiguous();
  if (residual.stride(1) != 1) residual = residual.contiguous();
  int kind = 0, gd = QFN_DTYPE_BF16, pd = QFN_DTYPE_BF16, nd = QFN_DTYPE_BF16;
  if (gate_) {
    gate = *gate_;
    TORCH_CHECK_VALUE(gate.is_cuda(), "gate must be a CUDA tensor (libqfn has no CPU path)");
    same_device(gate, "gate", block, "block");
    gd = dtype_code(gate, "gate");
    TORCH_CHECK_VALUE(gate.dim() == 2 && gate.size(0) == T && (gate.size(1) == 1 || gate.size(1) == D),
                      "gate must be [", T, ", 1] or [", T, ", ", D, "], got ", gate.sizes());
    kind = gate.size(1) == D ? 2 : 1;
    if (kind == 2 && D > 1 && gate.stride(1) != 1) gate = gate.contiguous();
  }
  for (const auto& w : {std::make_pair(&post, "post_weight"), std::make_pair(&next, "next_weight")}) {
    if (!*w.first) continue;
    req_cuda(**w.first, w.second);
    same_device(**w.first, w.second, block, "block");
    TORCH_CHECK_VALUE((*w.first)->dim() == 1 && (*w.first)->size(0) == D, w.second, " must be [", D, "], got ",
                      (*w.first)->sizes());
  }
  if (post) pd = dtype_code(*post, "post_weight");
  if (next) nd = dtype_code(*next, "next_weight");
  c10::cuda::CUDAGuard guard(block.device());
  at::Tensor r = r_out ? *r_out : at::empty({T, D}, residual.options());
  if (r_out) {
    req_view(r, "out", residual.scalar_type(), block, "block");
    TORCH_CHECK_VALUE(r.is_contiguous() && r.sizes() == block.sizes(), "out must be a contiguous [", T, ", ", D,
                      "], got ", r.sizes());
    // in place of the residual itself is fine: a thread writes what it has read
    TORCH_CHECK_VALUE((r.data_ptr() == residual.data_ptr() && residual.is_contiguous()) || !overlap(r, residual),
                      "out overlaps the residual without being it");
    req_apart(r, "out", {{&block, "block"}, {&gate, "gate"}, {given(post), "post_weight"}, {given(next), "next_weight"}});
  }
  at::Tensor n = at::empty(next ? at::IntArrayRef{T, D} : at::IntArrayRef{0}, block.options().dtype(at::kBFloat16));
  if (T == 0 || D == 0) return {r_out ? written(r) : r, n};
  check_rc(qfn_norm_residual(block.data_ptr(), bd, block.stride(0), residual.data_ptr(), rd, residual.stride(0),
                             post ? post->data_ptr() : nullptr, pd, kind ? gate.data_ptr() : nullptr, kind, gd,
                             kind ? gate.stride(0) : 0, sigmoid, static_cast<float>(scale),
                             next ? next->data_ptr() : nullptr, nd, r.data_ptr(),
                             next ? static_cast<uint16_t*>(n.data_ptr()) : nullptr, T, static_cast<int>(D),
                             static_cast<float>(eps), stream_of(r)),
           "qfn_norm_residual");
  return {r_out ? written(r) : r, n};
}

}  // namespace

// Catch-all kernels (not per dispatch key): a CPU tensor reaches the checks
// above and raises ValueError rather than a missing-kernel error.
TORCH_LIBRARY(qfn, m) {
  m.def("moe_decode(Tensor slots, Tensor sidx, Tensor s2, Tensor coef, Tensor x, Tensor(a!) h_buf, int variant) -> Tensor",
        &moe_decode);
  m.def("moe_prefill(Tensor x, Tensor ti, Tensor tv, Tensor table, Tensor s2, int L) -> Tensor", &moe_prefill);
  m.def("gemv(Tensor q, Tensor s, Tensor x, bool out_f32) -> Tensor", &gemv);
  m.def("linear(Tensor x, Tensor q, Tensor s) -> Tensor", &linear);
  m.def("deltanet_chunk(Tensor q, Tensor k, Tensor v, Tensor g, Tensor beta, Tensor? cu_seqlens, "
        "Tensor? initial_state, Tensor(a!)? final_state, Tensor(b!)? out) -> (Tensor, Tensor)",
        &deltanet_chunk);
  m.def("deltanet_step(Tensor q, Tensor k, Tensor v, Tensor g, Tensor beta, Tensor state, Tensor? state_index, "
        "Tensor(a!) out_state, Tensor(b!)? out) -> Tensor",
        &deltanet_step);
  m.def("gated_norm(Tensor x, Tensor z, Tensor weight, float eps) -> Tensor", &gated_norm);
  m.def("norm_residual(Tensor block, Tensor residual, Tensor? post_weight, Tensor? gate, bool sigmoid, float scale, "
        "Tensor? next_weight, float eps, Tensor(a!)? out) -> (Tensor, Tensor)",
        &norm_residual);
}
