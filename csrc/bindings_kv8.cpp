// Torch op registrations of the key/value cache in 8 bits (csrc/kernels/kv8.hip, kv8_attn.hip) and of the norms of
// query and key heads with the rotation (csrc/kernels/qk_norm.hip).
#include "bindings_util.h"
#include "kernels/kv8_pages.h"

#include <ATen/core/dispatch/Dispatcher.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

namespace {

using OptTensor = c10::optional<at::Tensor>;

bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

void check_table(const at::Tensor& cos, const at::Tensor& sin, int64_t D, const at::Tensor& like) {
  check_f32(cos, "cos");
  check_f32(sin, "sin");
  MX_CHECK(cos.dim() == 2 && cos.size(1) == D / 2 && cos.size(0) >= 1 && sin.sizes() == cos.sizes() &&
               cos.size(0) <= INT32_MAX && cos.device() == like.device() && sin.device() == like.device(),
           "cos, sin: f32 [positions, D / 2] on the rows' device");
}

const int32_t* check_ints(const at::Tensor& t, at::IntArrayRef shape, const at::Tensor& like, const char* name) {
  MX_CHECK(t.device() == like.device() && t.scalar_type() == at::kInt && t.is_contiguous() && t.sizes() == shape, name,
           ": contiguous int32 ", shape, " on the device of the others, got ", t.scalar_type(), " ", t.sizes());
  return t.data_ptr<int32_t>();
}

const uint16_t* check_weight(const OptTensor& w, int64_t D, const at::Tensor& like, const char* name) {
  if (!given(w)) return nullptr;
  check_bf16(*w, name);
  MX_CHECK(w->dim() == 1 && w->size(0) == D && w->device() == like.device(), name, ": bf16 [", D, "] on the rows' device");
  return bf(*w);
}

void check_heads(int64_t Hq, int64_t Hkv, int64_t D) {
  MX_CHECK(D == 32 || D == 64 || D == 128, "heads of 32, 64 or 128 channels, got ", D);
  MX_CHECK(Hkv >= 1 && Hq >= Hkv && Hq % Hkv == 0 && Hq <= 4096, "query heads in whole groups of a key head, got ", Hq, " of ", Hkv);
}

// t if its rows are what the kernels read (16-byte pieces, row strides of such), else a copy of it; the checks say what is no rows
at::Tensor rows16(const at::Tensor& t) {
  if (t.dim() != 2 || (t.stride(1) == 1 && t.stride(0) >= t.size(1) && t.stride(0) % 8 == 0 &&
                       reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0))
    return t;
  return t.clone(at::MemoryFormat::Contiguous);
}

// t, or a copy of it at a multiple of 16 bytes
at::Tensor placed(const at::Tensor& t) {
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 || !t.is_contiguous() ? t : t.clone();
}
OptTensor placed(const OptTensor& t) { return given(t) ? OptTensor(placed(*t)) : c10::nullopt; }

// A backward pass takes each leaf's gradient on the stream of the leaf's accumulator, which lives as long as any graph of the leaf
// does: captured, it would pull the default stream of a graph from before into the capture, and that ends the process.
void check_capture(at::TensorList leaves) {
  if (!cur_stream()) return;  // the default stream is never captured
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  MX_OK((int)hipStreamIsCapturing(cur_stream(), &status));
  if (status == hipStreamCaptureStatusNone) return;
  for (const at::Tensor& t : leaves) {
    if (!t.requires_grad() || !t.is_leaf()) continue;
    const auto kept = torch::autograd::impl::try_get_grad_accumulator(t);
    const auto stream = kept ? kept->stream() : std::nullopt;
    MX_CHECK(!stream || c10::hip::HIPStreamMasqueradingAsCUDA(*stream).stream() != nullptr,
             "qk_norm_rope: its backward cannot be captured while another graph of the same leaf lives on the default stream; let "
             "go of that one's outputs first, or give the captured one detached leaves");
  }
}

int64_t check_qkv(const at::Tensor& qkv, int64_t Hq, int64_t Hkv, int64_t D) {
  const int64_t ld = check_rows_bf16(qkv, "qkv");
  MX_CHECK(qkv.size(1) == (Hq + 2 * Hkv) * D, "qkv [T, (Hq + 2 Hkv) D], got ", qkv.sizes());
  MX_CHECK(reinterpret_cast<uintptr_t>(qkv.data_ptr()) % 16 == 0, "qkv: rows start at multiples of 16 bytes");
  return ld;
}

// ---------------------------------------------------------------- norms of query and key heads, rotated
// q [B, Hq, S, D], k, v [B, Hkv, S, D] of qkv rows [B * S, (Hq + 2 Hkv) D]
std::tuple<at::Tensor, at::Tensor, at::Tensor> qk_norm_rope(const at::Tensor& any, const at::Tensor& wq_any,
                                                            const at::Tensor& wk_any, const at::Tensor& cos_any,
                                                            const at::Tensor& sin_any, int64_t B, int64_t S, int64_t Hq,
                                                            int64_t Hkv, int64_t D, double eps, const OptTensor& positions) {
  MX_CHECK(any.is_cuda(), "qkv must be a GPU tensor");
  DevGuard g(any.device());
  const at::Tensor qkv = rows16(any), wq = placed(wq_any), wk = placed(wk_any), cos = placed(cos_any), sin = placed(sin_any);
  check_heads(Hq, Hkv, D);
  const int64_t ld = check_qkv(qkv, Hq, Hkv, D);
  MX_CHECK(B >= 0 && S >= 0 && qkv.size(0) == B * S, "qkv has ", qkv.size(0), " rows, B * S = ", B * S);
  check_table(cos, sin, D, qkv);
  MX_CHECK(given(positions) || cos.size(0) >= S, "the table has ", cos.size(0), " positions, rows up to ", S);
  auto q = at::empty({B, Hq, S, D}, qkv.options()), k = at::empty({B, Hkv, S, D}, qkv.options()), v = at::empty_like(k);
  const int rc = mx_qk_norm_rope(bf(qkv), ld, check_weight(wq, D, qkv, "q_norm"), check_weight(wk, D, qkv, "k_norm"),
                                 cos.data_ptr<float>(), sin.data_ptr<float>(),
                                 given(positions) ? check_ints(*positions, {B * S}, qkv, "positions") : nullptr,
                                 (int)cos.size(0), bfm(q), bfm(k), bfm(v), (int)B, (int)S, (int)Hq, (int)Hkv, (int)D,
                                 (float)eps, cur_stream());
  MX_CHECK(rc != -1, "qk_norm_rope: too many rows");
  MX_OK(rc);
  return {q, k, v};
}

// gradients [B, H, S, D] of q, k, v, all bf16 or all f32; those of k and v as whole numbers of summands a head
std::tuple<at::Tensor, at::Tensor, at::Tensor> qk_norm_rope_bwd(const at::Tensor& dq_any, const at::Tensor& dk_any,
                                                                const at::Tensor& dv_any, const at::Tensor& any,
                                                                const at::Tensor& wq_any, const at::Tensor& wk_any,
                                                                const at::Tensor& cos_any, const at::Tensor& sin_any,
                                                                int64_t Hkv, double eps, const OptTensor& positions,
                                                                int64_t out_pad, bool need_dw, bool dw32) {
  MX_CHECK(any.is_cuda(), "qkv must be a GPU tensor");
  DevGuard g(any.device());
  const at::Tensor qkv = rows16(any), wq = placed(wq_any), wk = placed(wk_any), cos = placed(cos_any), sin = placed(sin_any);
  const at::Tensor dq = placed(dq_any), dk = placed(dk_any), dv = placed(dv_any);
  MX_CHECK(dq.dim() == 4 && dk.dim() == 4 && dv.sizes() == dk.sizes(), "gradients [B, H, S, D]");
  const int64_t B = dq.size(0), Hq = dq.size(1), S = dq.size(2), D = dq.size(3);
  check_heads(Hq, Hkv, D);
  const int64_t ld = check_qkv(qkv, Hq, Hkv, D);
  const bool g32 = dq.scalar_type() == at::kFloat;
  for (const at::Tensor& t : {dq, dk, dv}) {
    if (g32) check_f32(t, "gradients of q, k, v");
    else check_bf16(t, "gradients of q, k, v");
    MX_CHECK(t.device() == qkv.device(), "gradients on the rows' device");
  }
  MX_CHECK(dk.size(0) == B && dk.size(2) == S && dk.size(3) == D && dk.size(1) >= Hkv && dk.size(1) % Hkv == 0 &&
               qkv.size(0) == B * S && (g32 || dk.size(1) == Hkv),
           "gradients of k, v [B, n Hkv, S, D] (bf16: n = 1) beside rows [B S, ..]");
  MX_CHECK(out_pad >= 0 && out_pad % 8 == 0, "out_pad must be a non-negative multiple of 8");
  check_table(cos, sin, D, qkv);
  MX_CHECK(given(positions) || cos.size(0) >= S, "the table has ", cos.size(0), " positions, rows up to ", S);
  const uint16_t *pq = check_weight(wq, D, qkv, "q_norm"), *pk = check_weight(wk, D, qkv, "k_norm");
  const int64_t NHD = (Hq + 2 * Hkv) * D;
  auto dqkv = empty_rows(B * S, NHD, out_pad, qkv.options());
  const auto wo = qkv.options().dtype(dw32 ? at::kFloat : at::kBFloat16);
  const int64_t W = need_dw ? D : 0;
  auto dwq = B * S ? at::empty({W}, wo) : at::zeros({W}, wo), dwk = B * S ? at::empty({W}, wo) : at::zeros({W}, wo);
  MX_CHECK(B * S <= INT32_MAX, "qk_norm_rope_bwd: too many rows");
  auto part = at::empty({mx_qk_norm_rope_bwd_parts((int)B, (int)S, (int)Hq, (int)Hkv, (int)D), D},
                        qkv.options().dtype(at::kFloat));
  const int rc = mx_qk_norm_rope_bwd(dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), g32 ? 1 : 0, (int)(dk.size(1) / Hkv), bf(qkv),
                                     ld, pq, pk, cos.data_ptr<float>(), sin.data_ptr<float>(),
                                     given(positions) ? check_ints(*positions, {B * S}, qkv, "positions") : nullptr,
                                     (int)cos.size(0), bfm(dqkv), NHD + out_pad, part.data_ptr<float>(),
                                     need_dw ? dwq.data_ptr() : nullptr, need_dw ? dwk.data_ptr() : nullptr, dw32 ? 1 : 0,
                                     (int)B, (int)S, (int)Hq, (int)Hkv, (int)D, (float)eps, cur_stream());
  MX_CHECK(rc != -1, "qk_norm_rope_bwd: too many rows");
  MX_OK(rc);
  return {dqkv, dwq, dwk};
}

// The ops for autograd's kernel, which calls them through the dispatcher: whatever records, batches or stands in for calls
// (tracers, dispatch modes, batches of backwards) then meets the op and not the allocations inside it.
const auto& forward_op() {
  static const auto op =
      c10::Dispatcher::singleton().findSchemaOrThrow("mxllm::qk_norm_rope", "").typed<decltype(qk_norm_rope)>();
  return op;
}
const auto& backward_op() {
  static const auto op =
      c10::Dispatcher::singleton().findSchemaOrThrow("mxllm::qk_norm_rope_bwd", "").typed<decltype(qk_norm_rope_bwd)>();
  return op;
}

// The same for autograd, here as its Python form (mxllm/ops/attention.py, which a weight with an owner takes) costs 40 us of the host's
// time a step more, as much as 2,048 rows of 48 heads of 128 take forward and backward.  (Rows that the kernels cannot read as
// they lie are copied by either op: only below the dispatcher is there an address to look at.)
struct QKNormRope : torch::autograd::Function<QKNormRope> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& qkv,
                                                const at::Tensor& wq, const at::Tensor& wk, const at::Tensor& cos,
                                                const at::Tensor& sin, int64_t B, int64_t S, int64_t Hq, int64_t Hkv, int64_t D,
                                                double eps, const OptTensor& positions) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [q, k, v] = forward_op().call(qkv, wq, wk, cos, sin, B, S, Hq, Hkv, D, eps, positions);
    ctx->save_for_backward({qkv, wq, wk, cos, sin, given(positions) ? *positions : at::Tensor()});
    ctx->saved_data["Hkv"] = Hkv;
    ctx->saved_data["eps"] = eps;
    return {q, k, v};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 const torch::autograd::variable_list& g) {
    const auto saved = ctx->get_saved_variables();
    const bool need_q = ctx->needs_input_grad(1), need_k = ctx->needs_input_grad(2);
    torch::autograd::variable_list out(12);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      auto [dqkv, dwq, dwk] = backward_op().call(
          g[0].contiguous(), g[1].contiguous(), g[2].contiguous(), saved[0], saved[1], saved[2], saved[3], saved[4],
          ctx->saved_data["Hkv"].toInt(), ctx->saved_data["eps"].toDouble(),
          saved[5].defined() ? OptTensor(saved[5]) : c10::nullopt, 0, need_q || need_k, false);
      out[0] = dqkv;
      if (need_q) out[1] = dwq;
      if (need_k) out[2] = dwk;
    }
    if (at::GradMode::is_enabled()) {  // its own gradient is not known: whoever asks for it is told
      torch::autograd::variable_list in;
      for (int i = 0; i < 3; ++i)
        if (out[i].defined()) in.push_back(out[i].detach().requires_grad_());
      const auto told = (*std::make_shared<torch::autograd::DelayedError>("qk_norm_rope is differentiable once",
                                                                          (int64_t)in.size()))(std::move(in));
      for (int i = 0, j = 0; i < 3; ++i)
        if (out[i].defined()) out[i] = told[j++];
    }
    return out;
  }
};

std::tuple<at::Tensor, at::Tensor, at::Tensor> qk_norm_rope_grad(const at::Tensor& qkv, const at::Tensor& wq,
                                                                 const at::Tensor& wk, const at::Tensor& cos,
                                                                 const at::Tensor& sin, int64_t B, int64_t S, int64_t Hq,
                                                                 int64_t Hkv, int64_t D, double eps, const OptTensor& positions) {
  bool recorded = false;
  for (const at::Tensor* t : {&qkv, &wq, &wk})
    recorded = recorded || (at::GradMode::is_enabled() && t->requires_grad()) || t->_fw_grad(0).defined();
  if (!recorded) {
    at::AutoDispatchBelowADInplaceOrView below;
    return forward_op().call(qkv, wq, wk, cos, sin, B, S, Hq, Hkv, D, eps, positions);
  }
  if (at::GradMode::is_enabled()) {
    DevGuard g(qkv.device());
    check_capture({qkv, wq, wk});
  }
  const auto out = QKNormRope::apply(qkv, wq, wk, cos, sin, B, S, Hq, Hkv, D, eps, positions);
  return {out[0], out[1], out[2]};
}

// ---------------------------------------------------------------- the cache in 8 bits
// k, v uint8 [pages, Hkv, block, D], ke, ve uint8 [pages, Hkv, block / 16], table int32 [slots, max_pages]
mx::Kv8Pages check_pages(const at::Tensor& k, const at::Tensor& v, const at::Tensor& ke, const at::Tensor& ve,
                         const at::Tensor& table, const at::Tensor& like) {
  for (const at::Tensor& t : {k, v, ke, ve}) {
    MX_CHECK(t.device() == like.device() && t.scalar_type() == at::kByte && t.is_contiguous(),
             "8-bit cache: contiguous uint8 tensors on the device of the rows");
  }
  MX_CHECK(k.dim() == 4 && k.size(0) >= 1 && k.size(1) >= 1 && k.size(2) >= 16 && k.size(2) % 16 == 0 && k.size(3) >= 1 &&
               v.sizes() == k.sizes(),
           "8-bit cache: codes [pages, Hkv, block, D] with blocks of a multiple of 16 positions, got ", k.sizes(), " and ",
           v.sizes());
  MX_CHECK(ke.sizes() == at::IntArrayRef({k.size(0), k.size(1), k.size(2) / 16}) && ve.sizes() == ke.sizes(),
           "8-bit cache: exponents [pages, Hkv, block / 16], got ", ke.sizes(), " and ", ve.sizes());
  MX_CHECK(k.numel() / k.size(3) / 16 <= INT32_MAX, "8-bit cache: too many pages");
  for (const at::Tensor& t : {k, v}) MX_CHECK(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, "8-bit cache: alignment");
  MX_CHECK(table.device() == like.device() && table.scalar_type() == at::kInt && table.dim() == 2 && table.is_contiguous() &&
               table.size(0) >= 1 && table.size(1) >= 1 && table.size(0) <= INT32_MAX &&
               table.size(1) * k.size(2) <= INT32_MAX,
           "block table: contiguous int32 [slots, max_pages]");
  const auto at8 = [](const at::Tensor& t) { return reinterpret_cast<uint8_t*>(t.data_ptr()); };
  return {at8(k), at8(v), at8(ke), at8(ve), table.data_ptr<int32_t>(), (int)table.size(0), (int)table.size(1),
          (int)k.size(2), (int)k.size(0), (int)k.size(1)};
}

struct Appended {
  at::Tensor q, k, v;
};
Appended append(const at::Tensor& qkv_any, const at::Tensor& cos_any, const at::Tensor& sin_any, const at::Tensor& index_any,
                const OptTensor& slots, bool runs, const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ke,
                const at::Tensor& ve, const at::Tensor& table, int64_t Hq, const OptTensor& wq_any, const OptTensor& wk_any,
                double eps) {
  MX_CHECK(qkv_any.is_cuda() && qkv_any.dim() == 2, "qkv: [T, (Hq + 2 Hkv) D] on the GPU");
  DevGuard g(qkv_any.device());
  const at::Tensor qkv = rows16(qkv_any), cos = placed(cos_any), sin = placed(sin_any);
  const at::Tensor index = runs ? placed(index_any) : index_any;
  const OptTensor wq = placed(wq_any), wk = placed(wk_any);
  const mx::Kv8Pages pg = check_pages(kc, vc, ke, ve, table, qkv);
  const int64_t Hkv = kc.size(1), D = kc.size(3), T = qkv.size(0);
  check_heads(Hq, Hkv, D);
  const int64_t ld = check_qkv(qkv, Hq, Hkv, D);
  check_table(cos, sin, D, qkv);
  MX_CHECK(given(wq) == given(wk), "weights of both norms, or of none");
  MX_CHECK(T <= INT32_MAX, "too many rows");
  const int64_t n = runs ? index.size(0) : T;
  const int32_t* ix = runs ? check_ints(index, {n, 4}, qkv, "runs") : check_ints(index, {T}, qkv, "pos");
  const int32_t* sl = given(slots) ? check_ints(*slots, {T}, qkv, "slots") : nullptr;
  Appended out;
  if (runs) {
    out.q = at::empty({Hq, T, D}, qkv.options());
    out.k = at::empty({Hkv, T, D}, qkv.options());
    out.v = at::empty_like(out.k);
  } else {
    out.q = at::empty({T, Hq, D}, qkv.options());
  }
  const int rc = mx_kv8_append(bf(qkv), ld, cos.data_ptr<float>(), sin.data_ptr<float>(), (int)cos.size(0), runs ? 1 : 0, ix,
                               sl, (int)n, (int)T, check_weight(wq, D, qkv, "q_norm"), check_weight(wk, D, qkv, "k_norm"),
                               eps, bfm(out.q), runs ? bfm(out.k) : nullptr, runs ? bfm(out.v) : nullptr, &pg,
                               (int)Hq, (int)D, cur_stream());
  MX_CHECK(rc != -1, "kv8_append: too many rows");
  MX_OK(rc);
  return out;
}

at::Tensor kv8_append_tokens(const at::Tensor& qkv, const at::Tensor& cos, const at::Tensor& sin, const at::Tensor& pos,
                             const OptTensor& slots, at::Tensor kc, at::Tensor vc, at::Tensor ke, at::Tensor ve,
                             const at::Tensor& table, int64_t Hq, const OptTensor& wq, const OptTensor& wk, double eps) {
  return append(qkv, cos, sin, pos, slots, false, kc, vc, ke, ve, table, Hq, wq, wk, eps).q;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> kv8_append_prompts(const at::Tensor& qkv, const at::Tensor& cos,
                                                                  const at::Tensor& sin, const at::Tensor& runs,
                                                                  at::Tensor kc, at::Tensor vc, at::Tensor ke, at::Tensor ve,
                                                                  const at::Tensor& table, int64_t Hq, const OptTensor& wq,
                                                                  const OptTensor& wk, double eps) {
  MX_CHECK(runs.dim() == 2 && runs.size(1) == 4, "runs int32 [n, 4] = first row, rows, slot, first position");
  const Appended a = append(qkv, cos, sin, runs, c10::nullopt, true, kc, vc, ke, ve, table, Hq, wq, wk, eps);
  return {a.q, a.k, a.v};
}

std::tuple<at::Tensor, at::Tensor> kv8_read(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ke,
                                            const at::Tensor& ve, const at::Tensor& table, const OptTensor& slots,
                                            const at::Tensor& starts, const at::Tensor& ends, int64_t n) {
  const mx::Kv8Pages pg = check_pages(kc, vc, ke, ve, table, kc);
  const int64_t Hkv = kc.size(1), D = kc.size(3);
  check_heads(Hkv, Hkv, D);
  MX_CHECK(starts.dim() == 1 && n >= 0 && n <= INT32_MAX - 16, "starts int32 [B], n >= 0");
  const int64_t B = starts.size(0);
  const int32_t *from = check_ints(starts, {B}, kc, "starts"), *to = check_ints(ends, {B}, kc, "ends");
  const int32_t* sl = given(slots) ? check_ints(*slots, {B}, kc, "slots") : nullptr;
  DevGuard g(kc.device());
  auto k = at::empty({B, Hkv, n, D}, kc.options().dtype(at::kBFloat16)), v = at::empty_like(k);
  const int rc = mx_kv8_read(&pg, sl, from, to, bfm(k), bfm(v), (int)B, (int)n, (int)D, cur_stream());
  MX_CHECK(rc != -1, "kv8_read: too many positions");
  MX_OK(rc);
  return {k, v};
}

at::Tensor kv8_decode_attn(const at::Tensor& q_any, const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ke,
                           const at::Tensor& ve, const at::Tensor& table, const at::Tensor& pos, const OptTensor& slots,
                           int64_t max_len, double scale) {
  MX_CHECK(q_any.is_cuda(), "q: on the GPU");
  DevGuard g(q_any.device());
  const bool as_is = q_any.is_contiguous() && reinterpret_cast<uintptr_t>(q_any.data_ptr()) % 16 == 0;
  const at::Tensor q = as_is ? q_any : q_any.clone(at::MemoryFormat::Contiguous);
  check_bf16(q, "q");
  const mx::Kv8Pages pg = check_pages(kc, vc, ke, ve, table, q);
  MX_CHECK(q.dim() == 3 && q.size(2) == kc.size(3), "q [B, Hq, D], got ", q.sizes());
  const int64_t B = q.size(0), Hq = q.size(1), D = q.size(2), Hkv = kc.size(1);
  check_heads(Hq, Hkv, D);
  MX_CHECK(Hq / Hkv <= 16, "up to 16 query heads a key head, got ", Hq / Hkv);
  MX_CHECK(max_len >= 1, "max_len: at least one position, got ", max_len);
  MX_CHECK(scale > 0 && scale <= 3.4028234663852886e38, "scale: a positive number, got ", scale);
  const int32_t* p = check_ints(pos, {B}, q, "pos");
  const int32_t* sl = given(slots) ? check_ints(*slots, {B}, q, "slots") : nullptr;
  const int64_t cap = std::min<int64_t>(max_len, (int64_t)pg.maxp * pg.block);
  auto out = at::empty({B, Hq * D}, q.options());
  const int64_t parts = mx_kv8_attn_parts((int)B, (int)Hkv, (int)D, (int)cap);
  at::Tensor work;  // outputs of the parts [Hq, parts, D], then their maxima and sums [Hq, parts, 2]
  float *po = nullptr, *ml = nullptr;
  if (parts) {
    work = at::empty({Hq * parts * (D + 2)}, q.options().dtype(at::kFloat));
    po = work.data_ptr<float>(), ml = po + Hq * parts * D;
  }
  const int rc = mx_kv8_attn(bf(q), &pg, p, sl, ml, po, bfm(out), (int)B, (int)Hq, (int)D, (int)cap, (float)scale,
                             cur_stream());
  MX_CHECK(rc != -1, "kv8_decode_attn: sizes not taken");
  MX_OK(rc);
  return out;
}

// causal attention inside each segment of blocks [n, 4] (mxllm/ops/hybrid.py PromptRows.attn_blocks), which name every row: q
// [Hq, T, D], k, v [Hkv, T, D] -> [T, Hq * D]
at::Tensor prompt_rows_attention(const at::Tensor& q_any, const at::Tensor& k_any, const at::Tensor& v_any,
                                 const at::Tensor& blocks_any, double scale) {
  MX_CHECK(q_any.is_cuda(), "q: on the GPU");
  DevGuard g(q_any.device());
  const at::Tensor q = placed(q_any.contiguous()), k = placed(k_any.contiguous()), v = placed(v_any.contiguous()),
                   blocks = placed(blocks_any);
  check_bf16(q, "q");
  check_bf16(k, "k");
  check_bf16(v, "v");
  MX_CHECK(q.dim() == 3 && k.dim() == 3 && v.sizes() == k.sizes() && k.size(1) == q.size(1) && k.size(2) == q.size(2) &&
               k.device() == q.device() && v.device() == q.device(),
           "q [Hq, T, D], k, v [Hkv, T, D] on one device");
  const int64_t Hq = q.size(0), T = q.size(1), D = q.size(2), Hkv = k.size(0);
  check_heads(Hq, Hkv, D);
  MX_CHECK(T * D * 2 < INT32_MAX, "prompt_rows_attention: too many rows");
  MX_CHECK(blocks.dim() == 2, "blocks int32 [n, 4]");
  const int32_t* bl = check_ints(blocks, {blocks.size(0), 4}, q, "blocks");
  auto o = at::empty({T, Hq * D}, q.options());
  const int rc = mx_attn_fwd_prompts(bf(q), bf(k), bf(v), bl, (int)blocks.size(0), bfm(o), (int)T, (int)Hq, (int)Hkv, (int)D,
                                     (float)scale, cur_stream());
  MX_CHECK(rc != -1, "prompt_rows_attention: sizes not taken");
  MX_OK(rc);
  return o;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(mxllm, m) {
  m.def("prompt_rows_attention(Tensor q, Tensor k, Tensor v, Tensor blocks, float scale) -> Tensor");
  m.def("qk_norm_rope(Tensor qkv, Tensor wq, Tensor wk, Tensor cos, Tensor sin, int B, int S, int Hq, int Hkv, int D, float eps, Tensor? positions=None) -> (Tensor, Tensor, Tensor)");
  m.def("grads_capturable(Tensor[] leaves) -> ()");
  m.def("qk_norm_rope_bwd(Tensor dq, Tensor dk, Tensor dv, Tensor qkv, Tensor wq, Tensor wk, Tensor cos, Tensor sin, int Hkv, float eps, Tensor? positions=None, int out_pad=0, bool need_dw=True, bool dw32=False) -> (Tensor, Tensor, Tensor)");
  m.def("kv8_append_tokens(Tensor qkv, Tensor cos, Tensor sin, Tensor pos, Tensor? slots, Tensor(a!) k, Tensor(b!) v, Tensor(c!) ke, Tensor(d!) ve, Tensor table, int Hq, Tensor? wq, Tensor? wk, float eps) -> Tensor");
  m.def("kv8_append_prompts(Tensor qkv, Tensor cos, Tensor sin, Tensor runs, Tensor(a!) k, Tensor(b!) v, Tensor(c!) ke, Tensor(d!) ve, Tensor table, int Hq, Tensor? wq, Tensor? wk, float eps) -> (Tensor, Tensor, Tensor)");
  m.def("kv8_read(Tensor k, Tensor v, Tensor ke, Tensor ve, Tensor table, Tensor? slots, Tensor starts, Tensor ends, int n) -> (Tensor, Tensor)");
  m.def("kv8_decode_attn(Tensor q, Tensor k, Tensor v, Tensor ke, Tensor ve, Tensor table, Tensor pos, Tensor? slots, int max_len, float scale) -> Tensor");
}

TORCH_LIBRARY_IMPL(mxllm, CUDA, m) {
  m.impl("qk_norm_rope", &qk_norm_rope);
  m.impl("qk_norm_rope_bwd", &qk_norm_rope_bwd);
  m.impl("grads_capturable", &check_capture);
  m.impl("kv8_append_tokens", &kv8_append_tokens);
  m.impl("kv8_append_prompts", &kv8_append_prompts);
  m.impl("prompt_rows_attention", &prompt_rows_attention);
  m.impl("kv8_read", &kv8_read);
  m.impl("kv8_decode_attn", &kv8_decode_attn);
}

TORCH_LIBRARY_IMPL(mxllm, AutogradCUDA, m) { m.impl("qk_norm_rope", &qk_norm_rope_grad); }
