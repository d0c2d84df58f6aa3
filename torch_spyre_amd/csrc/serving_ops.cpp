// PyTorch-ROCm kernels of the rotary, 8-bit cache and drafted-token ops, as
// torch_ops.cpp has those of attention: each checks its tensors, allocates its
// outputs and workspace from the caching allocator and calls the C ABI on the
// current stream.
//
//   spyre::rotary                  positions rotated into q and k, with its gradient
//   spyre::kv_quant_append         K / V rows quantised into the 8-bit paged cache
//   spyre::rotary_kv_quant_append  the same, q and k rotated first
//   spyre::kv_quant_read           tokens of the 8-bit cache as dense fp16 K / V
//   spyre::quant_paged_decode_attention   one query a sequence over the 8-bit cache
//   spyre::paged_tree_attention    drafted tokens over the paged cache (fp16 or 8-bit)
// No reference counterparts.

#include <torch/csrc/autograd/custom_function.h>

#include <cmath>
#include <cstdint>
#include <limits>

#include "torch_checks.h"

namespace {

using namespace spyre_torch;

constexpr int64_t kPage = 64;

int as_int(int64_t x, const char* name) {
  TORCH_CHECK_VALUE(x >= 0 && x <= std::numeric_limits<int>::max(), name, " ", x, " does not fit 31 bits");
  return static_cast<int>(x);
}

// ---------------------------------------------------------------- rotary --

int rotary_type(at::ScalarType t) {
  TORCH_CHECK_TYPE(t == at::kHalf || t == at::kBFloat16 || t == at::kFloat,
                   "q and k must be float16, bfloat16 or float32 (got ", t, ")");
  return t == at::kHalf ? SPYRE_DT_FLOAT16 : t == at::kBFloat16 ? SPYRE_DT_BFLOAT16 : SPYRE_DT_FLOAT32;
}

// Positions [rows] or [B, rows] as (tensor, bytes, strides), frequencies [pairs].
struct Angles {
  at::Tensor positions, frequencies;
  int bytes, pairs;
  int64_t sb, ss;
};

Angles angles_of(const at::Tensor& positions, const at::Tensor& frequencies, int64_t B, int64_t S, int64_t D,
                 const c10::Device& dev) {
  require_on(positions, dev, "positions");
  require_on(frequencies, dev, "frequencies");
  TORCH_CHECK_TYPE(positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong,
                   "positions must be int32 or int64 (got ", positions.scalar_type(), ")");
  TORCH_CHECK_TYPE(frequencies.scalar_type() == at::kDouble, "frequencies must be float64 (got ",
                   frequencies.scalar_type(), ")");
  TORCH_CHECK_VALUE(!frequencies.requires_grad(), "frequencies take no gradient");
  TORCH_CHECK_VALUE(frequencies.dim() == 1 && frequencies.is_contiguous(), "frequencies must be contiguous [pairs]");
  TORCH_CHECK_VALUE(frequencies.size(0) > 0 && 2 * frequencies.size(0) <= D, "2 x ", frequencies.size(0),
                    " rotated features do not fit head_dim ", D);
  const bool flat = positions.dim() == 1;
  TORCH_CHECK_VALUE((flat && positions.size(0) == S) ||
                        (positions.dim() == 2 && positions.size(1) == S && (positions.size(0) == B || positions.size(0) == 1)),
                    "positions must be [", S, "] or [", B, ", ", S, "] (got ", positions.sizes(), ")");
  return {positions, frequencies, positions.scalar_type() == at::kLong ? 8 : 4, as_int(frequencies.size(0), "pairs"),
          flat || positions.size(0) != B ? 0 : positions.stride(0), positions.stride(-1)};
}

at::Tensor unit_feature_stride(const at::Tensor& t) {
  return t.stride(-1) == 1 || t.numel() == 0 ? t : t.clone(at::MemoryFormat::Contiguous);
}

std::tuple<at::Tensor, at::Tensor> rotary(const at::Tensor& query, const std::optional<at::Tensor>& key,
                                          const at::Tensor& positions, const at::Tensor& frequencies, double amplitude,
                                          bool interleaved, bool inverse) {
  TORCH_CHECK_VALUE(query.is_cuda(), "q must be a CUDA (HIP) tensor; there is no CPU path");
  TORCH_CHECK_VALUE(query.dim() == 4, "q must be 4-D [B, H, S, D]");
  const int type = rotary_type(query.scalar_type());
  const int64_t B = query.size(0), Hq = query.size(1), S = query.size(2), D = query.size(3);
  if (key.has_value()) {
    require_on(*key, query.device(), "k");
    TORCH_CHECK_VALUE(key->dim() == 4 && key->size(0) == B && key->size(2) == S && key->size(3) == D,
                      "k must be [", B, ", Hkv, ", S, ", ", D, "] (got ", key->sizes(), ")");
    TORCH_CHECK_TYPE(key->scalar_type() == query.scalar_type(), "q and k differ in dtype");
  }
  const Angles an = angles_of(positions, frequencies, B, S, D, query.device());
  const c10::OptionalDeviceGuard guard(query.device());
  const at::Tensor q = unit_feature_stride(query);
  const at::Tensor k = key.has_value() ? unit_feature_stride(*key) : at::Tensor();
  at::Tensor qo = at::empty_like(q);
  at::Tensor ko = key.has_value() ? at::empty_like(k) : at::empty({0}, q.options());
  if (qo.stride(-1) != 1 && qo.numel()) qo = at::empty(q.sizes(), q.options());
  if (key.has_value() && ko.stride(-1) != 1 && ko.numel()) ko = at::empty(k.sizes(), k.options());
  const int64_t Hkv = key.has_value() ? k.size(1) : 0;
  auto st = [](const at::Tensor& t) { return std::array<int64_t, 3>{t.stride(0), t.stride(1), t.stride(2)}; };
  const auto qs = st(q), qos = st(qo);
  const auto ks = Hkv ? st(k) : qs, kos = Hkv ? st(ko) : qos;
  check_rc("spyre_rotary",
           spyre_rotary(q.data_ptr(), qs.data(), qo.data_ptr(), qos.data(), as_int(Hq, "heads"),
                        Hkv ? k.data_ptr() : nullptr, ks.data(), Hkv ? ko.data_ptr() : nullptr, kos.data(),
                        as_int(Hkv, "heads"), type, an.positions.data_ptr(), an.bytes, an.sb, an.ss,
                        an.frequencies.data_ptr<double>(), an.pairs, static_cast<float>(amplitude), interleaved, inverse,
                        as_int(B, "batch"), as_int(S, "length"), as_int(D, "head_dim"), stream_of(q)));
  return {qo, ko};
}

std::tuple<at::Tensor, at::Tensor> call_rotary(const at::Tensor& q, const std::optional<at::Tensor>& k,
                                               const at::Tensor& positions, const at::Tensor& frequencies,
                                               double amplitude, bool interleaved, bool inverse) {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("spyre::rotary", "")
                             .typed<std::tuple<at::Tensor, at::Tensor>(const at::Tensor&, const std::optional<at::Tensor>&,
                                                                       const at::Tensor&, const at::Tensor&, double, bool,
                                                                       bool)>();
  return op.call(q, k, positions, frequencies, amplitude, interleaved, inverse);
}

// The rotation is orthogonal but for the amplitude, so the gradient is the
// rotation back, by the same kernel; in forward mode (rotary_autograd) the
// tangent is rotated as the operand is.
struct Rotary : torch::autograd::Function<Rotary> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& q,
                                                const std::optional<at::Tensor>& k, const at::Tensor& positions,
                                                const at::Tensor& frequencies, double amplitude, bool interleaved,
                                                bool inverse) {
    ctx->save_for_backward({positions, frequencies});
    ctx->saved_data["amplitude"] = amplitude;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["inverse"] = inverse;
    ctx->set_materialize_grads(false);
    at::AutoDispatchBelowADInplaceOrView below;
    auto [qo, ko] = call_rotary(q, k, positions, frequencies, amplitude, interleaved, inverse);
    if (!k.has_value()) ctx->mark_non_differentiable({ko});
    return {qo, ko};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const double amplitude = ctx->saved_data["amplitude"].toDouble();
    const bool interleaved = ctx->saved_data["interleaved"].toBool(), inverse = ctx->saved_data["inverse"].toBool();
    at::Tensor dq, dk;
    auto back = [&](const at::Tensor& x, const std::optional<at::Tensor>& y) {
      return call_rotary(x, y, saved[0], saved[1], amplitude, interleaved, !inverse);
    };
    if (grads[0].defined() && grads[1].defined())
      std::tie(dq, dk) = back(grads[0], grads[1]);
    else if (grads[0].defined())
      dq = std::get<0>(back(grads[0], std::nullopt));
    else if (grads[1].defined())
      dk = std::get<0>(back(grads[1], std::nullopt));
    return {dq, dk, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

std::tuple<at::Tensor, at::Tensor> rotary_autograd(const at::Tensor& q, const std::optional<at::Tensor>& k,
                                                   const at::Tensor& positions, const at::Tensor& frequencies,
                                                   double amplitude, bool interleaved, bool inverse) {
  TORCH_CHECK_VALUE(!frequencies._fw_grad(0).defined(), "frequencies take no gradient");
  const at::Tensor tq = q._fw_grad(0), tk = k.has_value() ? k->_fw_grad(0) : at::Tensor();
  if (tq.defined() || tk.defined()) {
    // Forward mode: the rotation is linear, so a result's tangent is the
    // rotation of its operand's.
    auto plain = [](const at::Tensor& t) { return t._fw_primal(0); };
    auto [qo, ko] = rotary_autograd(plain(q), k.has_value() ? std::make_optional(plain(*k)) : std::nullopt, positions,
                                    frequencies, amplitude, interleaved, inverse);
    auto along = [&](const at::Tensor& x, const std::optional<at::Tensor>& y) {
      return rotary_autograd(x, y, positions, frequencies, amplitude, interleaved, inverse);
    };
    at::Tensor dq, dk;
    if (tq.defined() && tk.defined())
      std::tie(dq, dk) = along(tq, tk);
    else if (tq.defined())
      dq = std::get<0>(along(tq, std::nullopt));
    else
      dk = std::get<0>(along(tk, std::nullopt));
    if (dq.defined()) qo._set_fw_grad(dq, 0, false);
    if (dk.defined()) ko._set_fw_grad(dk, 0, false);
    return {qo, ko};
  }
  if (!at::GradMode::is_enabled() || !(q.requires_grad() || (k.has_value() && k->requires_grad()))) {
    at::AutoDispatchBelowADInplaceOrView below;
    return call_rotary(q, k, positions, frequencies, amplitude, interleaved, inverse);
  }
  auto out = Rotary::apply(q, k, positions, frequencies, amplitude, interleaved, inverse);
  return {out[0], out[1]};
}

// ----------------------------------------------------------------- cache --

struct Cache {
  int kind;
  int64_t pages, Hkv, D;
};

Cache check_cache8(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks, const at::Tensor& vs,
                   const c10::Device& dev) {
  require_on(kc, dev, "k_cache");
  require_on(vc, dev, "v_cache");
  require_on(ks, dev, "k_scale");
  require_on(vs, dev, "v_scale");
  TORCH_CHECK_TYPE((kc.scalar_type() == at::kFloat8_e4m3fn || kc.scalar_type() == at::kChar) &&
                       vc.scalar_type() == kc.scalar_type(),
                   "8-bit caches must both be float8_e4m3fn or int8 (got ", kc.scalar_type(), " and ", vc.scalar_type(), ")");
  TORCH_CHECK_TYPE(ks.scalar_type() == at::kFloat && vs.scalar_type() == at::kFloat, "k_scale and v_scale must be float32");
  TORCH_CHECK_VALUE(kc.dim() == 5 && kc.size(3) == kPage && kc.size(4) == 16 && kc.is_contiguous(),
                    "k_cache must be contiguous [pages, Hkv, D/16, 64, 16] (got ", kc.sizes(), ")");
  const int64_t P = kc.size(0), H = kc.size(1), D = kc.size(2) * 16;
  TORCH_CHECK_VALUE(vc.sizes() == at::IntArrayRef({P, H, 4, D, 16}) && vc.is_contiguous(), "v_cache must be contiguous [", P,
                    ", ", H, ", 4, ", D, ", 16] (got ", vc.sizes(), ")");
  for (const at::Tensor* s : {&ks, &vs})
    TORCH_CHECK_VALUE(s->sizes() == at::IntArrayRef({P, H, kPage}) && s->is_contiguous(),
                      "k_scale and v_scale must be contiguous [", P, ", ", H, ", 64] (got ", s->sizes(), ")");
  return {kc.scalar_type() == at::kChar ? SPYRE_CODES_INT8 : SPYRE_CODES_E4M3, P, H, D};
}

void check_table(const at::Tensor& t, int64_t B, const c10::Device& dev) {
  require_on(t, dev, "block_table");
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.dim() == 2 && t.size(0) == B && (t.size(1) <= 1 || t.stride(1) == 1),
                    "block_table must be int32 [B, pages_per_seq] with unit column stride");
}

void check_lens(const at::Tensor& t, int64_t B, const c10::Device& dev, const char* name) {
  require_on(t, dev, name);
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == B && t.is_contiguous(), name,
                    " must be contiguous int32 [B]");
}

// fp16 rows that the kernels read as 16-byte vectors: feature stride 1, other
// strides multiples of 8, 16-byte aligned; anything else is copied into that form.
at::Tensor rows_operand(const at::Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a CUDA (HIP) tensor; there is no CPU path");
  TORCH_CHECK_TYPE(t.scalar_type() == at::kHalf, name, " must be float16 (got ", t.scalar_type(), ")");
  TORCH_CHECK_VALUE(t.dim() == 4, name, " must be 4-D [B, T, H, D]");
  const auto st = t.strides();
  const bool ready = st[3] == 1 && st[0] % 8 == 0 && st[1] % 8 == 0 && st[2] % 8 == 0 &&
                     reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  return ready ? t : t.clone(at::MemoryFormat::Contiguous);
}

at::Tensor quant_append(const std::optional<at::Tensor>& query, const at::Tensor& k_new, const at::Tensor& v_new,
                        const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks, const at::Tensor& vs,
                        const at::Tensor& block_table, const at::Tensor& slots,
                        const std::optional<at::Tensor>& positions, const std::optional<at::Tensor>& frequencies,
                        double amplitude, bool interleaved) {
  const at::Tensor k = rows_operand(k_new, "k_new"), v = rows_operand(v_new, "v_new");
  const auto dev = k.device();
  const int64_t B = k.size(0), T = k.size(1), Hkv = k.size(2), D = k.size(3);
  require_on(v, dev, "v_new");
  TORCH_CHECK_VALUE(v.sizes() == k.sizes(), "k_new and v_new shapes differ");
  const Cache c = check_cache8(kc, vc, ks, vs, dev);
  TORCH_CHECK_VALUE(c.Hkv == Hkv && c.D == D, "the cache holds ", c.Hkv, " KV heads of ", c.D, " features, k_new ", Hkv,
                    " of ", D);
  check_table(block_table, B, dev);
  require_on(slots, dev, "slots");
  TORCH_CHECK_VALUE(slots.scalar_type() == at::kInt && slots.dim() == 2 && slots.size(0) == B && slots.size(1) == T,
                    "slots must be int32 [", B, ", ", T, "] (got ", slots.scalar_type(), " ", slots.sizes(), ")");
  at::Tensor q, q_out;
  Angles an{};
  int64_t Hq = 0;
  if (query.has_value()) {
    q = rows_operand(*query, "q");
    require_on(q, dev, "q");
    TORCH_CHECK_VALUE(q.size(0) == B && q.size(1) == T && q.size(3) == D, "q must be [", B, ", ", T, ", Hq, ", D, "] (got ",
                      q.sizes(), ")");
    Hq = q.size(2);
    an = angles_of(*positions, *frequencies, B, T, D, dev);
    TORCH_CHECK_VALUE(an.pairs % 8 == 0, "rotated features must be a multiple of 16 (got ", 2 * an.pairs, ")");
  }
  const c10::OptionalDeviceGuard guard(dev);
  if (query.has_value()) q_out = at::empty({B, T, Hq, D}, q.options());
  auto st = [](const at::Tensor& t) { return std::array<int64_t, 3>{t.stride(0), t.stride(1), t.stride(2)}; };
  const auto k3 = st(k), v3 = st(v), q3 = query.has_value() ? st(q) : k3;
  check_rc("spyre_kv_quant_append",
           spyre_kv_quant_append(Hq ? q.data_ptr() : nullptr, q3.data(), Hq ? q_out.data_ptr() : nullptr, as_int(Hq, "heads"),
                                 k.data_ptr(), k3.data(), v.data_ptr(), v3.data(), kc.data_ptr(), vc.data_ptr(),
                                 ks.data_ptr<float>(), vs.data_ptr<float>(), c.kind, block_table.data_ptr<int32_t>(),
                                 block_table.stride(0), block_table.size(1), slots.data_ptr<int32_t>(), slots.stride(0),
                                 slots.stride(1), an.pairs ? an.positions.data_ptr() : nullptr, an.bytes, an.sb, an.ss,
                                 an.pairs ? an.frequencies.data_ptr<double>() : nullptr, an.pairs,
                                 static_cast<float>(amplitude), interleaved, as_int(B, "batch"), as_int(T, "tokens"),
                                 as_int(Hkv, "heads"), as_int(D, "head_dim"), kPage, c.pages, stream_of(k)));
  return q_out;
}

void kv_quant_append(const at::Tensor& k_new, const at::Tensor& v_new, const at::Tensor& kc, const at::Tensor& vc,
                     const at::Tensor& ks, const at::Tensor& vs, const at::Tensor& block_table, const at::Tensor& slots) {
  quant_append(std::nullopt, k_new, v_new, kc, vc, ks, vs, block_table, slots, std::nullopt, std::nullopt, 1.0, false);
}

at::Tensor rotary_kv_quant_append(const at::Tensor& q, const at::Tensor& k_new, const at::Tensor& v_new,
                                  const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks, const at::Tensor& vs,
                                  const at::Tensor& block_table, const at::Tensor& slots, const at::Tensor& positions,
                                  const at::Tensor& frequencies, double amplitude, bool interleaved) {
  return quant_append(q, k_new, v_new, kc, vc, ks, vs, block_table, slots, positions, frequencies, amplitude, interleaved);
}

std::tuple<at::Tensor, at::Tensor> kv_quant_read(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks,
                                                 const at::Tensor& vs, const at::Tensor& block_table,
                                                 const at::Tensor& lens, int64_t length,
                                                 const std::optional<at::Tensor>& start) {
  TORCH_CHECK_VALUE(kc.is_cuda(), "k_cache must be a CUDA (HIP) tensor; there is no CPU path");
  const auto dev = kc.device();
  const Cache c = check_cache8(kc, vc, ks, vs, dev);
  TORCH_CHECK_VALUE(length >= 0, "length ", length, " is negative");
  TORCH_CHECK_VALUE(block_table.dim() == 2, "block_table must be int32 [B, pages_per_seq] with unit column stride");
  const int64_t B = block_table.size(0);
  check_table(block_table, B, dev);
  check_lens(lens, B, dev, "lens");
  if (start.has_value()) check_lens(*start, B, dev, "start");
  const c10::OptionalDeviceGuard guard(dev);
  at::Tensor k = at::empty({B, c.Hkv, length, c.D}, kc.options().dtype(at::kHalf));
  at::Tensor v = at::empty_like(k);
  check_rc("spyre_kv_quant_read",
           spyre_kv_quant_read(kc.data_ptr(), vc.data_ptr(), ks.data_ptr<float>(), vs.data_ptr<float>(), c.kind,
                               block_table.data_ptr<int32_t>(), block_table.stride(0), block_table.size(1),
                               lens.data_ptr<int32_t>(), start.has_value() ? start->data_ptr<int32_t>() : nullptr,
                               k.data_ptr(), v.data_ptr(), as_int(B, "batch"), as_int(c.Hkv, "heads"),
                               as_int(length, "length"), as_int(c.D, "head_dim"), kPage, c.pages, stream_of(kc)));
  return {k, v};
}

// ------------------------------------------------------------- attention --

std::tuple<at::Tensor, at::Tensor> attend(const at::Tensor& query, const at::Tensor& kc, const at::Tensor& vc,
                                          const std::optional<at::Tensor>& ks, const std::optional<at::Tensor>& vs,
                                          const at::Tensor& block_table, const at::Tensor& context_lens,
                                          const std::optional<at::Tensor>& tree_mask,
                                          const std::optional<at::Tensor>& draft_lens, bool draft_keys,
                                          std::optional<double> scale, int64_t max_context_len) {
  const at::Tensor q = rows_operand(query, "q");
  const auto dev = q.device();
  const int64_t B = q.size(0), T = q.size(1), Hq = q.size(2), D = q.size(3);
  Cache c{SPYRE_CACHE_F16, 0, 0, D};
  TORCH_CHECK_VALUE(ks.has_value() == vs.has_value(), "k_scale and v_scale go together");
  if (ks.has_value()) {
    c = check_cache8(kc, vc, *ks, *vs, dev);
    TORCH_CHECK_VALUE(c.D == D, "the cache holds heads of ", c.D, " features, q of ", D);
  } else {
    require_on(kc, dev, "k_cache");
    require_on(vc, dev, "v_cache");
    TORCH_CHECK_TYPE(kc.scalar_type() == at::kHalf && vc.scalar_type() == at::kHalf,
                     "caches without scales must be float16 (got ", kc.scalar_type(), " and ", vc.scalar_type(), ")");
    TORCH_CHECK_VALUE(kc.dim() == 5 && kc.size(3) == kPage && kc.size(4) == 64 && kc.size(2) * 64 == D && kc.is_contiguous(),
                      "k_cache must be contiguous [pages, Hkv, ", D / 64, ", 64, 64] (got ", kc.sizes(), ")");
    c.pages = kc.size(0), c.Hkv = kc.size(1);
    TORCH_CHECK_VALUE(vc.sizes() == at::IntArrayRef({c.pages, c.Hkv, D, kPage}) && vc.is_contiguous(),
                      "v_cache must be contiguous [", c.pages, ", ", c.Hkv, ", ", D, ", 64] (got ", vc.sizes(), ")");
  }
  TORCH_CHECK_VALUE(c.Hkv > 0 && Hq > 0 && Hq % c.Hkv == 0, "Hq=", Hq, " is not a multiple of Hkv=", c.Hkv);
  check_table(block_table, B, dev);
  check_lens(context_lens, B, dev, "context_lens");
  if (draft_lens.has_value()) check_lens(*draft_lens, B, dev, "draft_lens");
  at::Tensor mask;
  int64_t ms[3] = {0, 0, 0};
  if (tree_mask.has_value()) {
    require_on(*tree_mask, dev, "tree_mask");
    TORCH_CHECK_TYPE(tree_mask->scalar_type() == at::kBool, "tree_mask must be bool (got ", tree_mask->scalar_type(), ")");
    TORCH_CHECK_VALUE((tree_mask->dim() == 2 || (tree_mask->dim() == 3 && (tree_mask->size(0) == B || tree_mask->size(0) == 1))) &&
                          tree_mask->size(-1) == T && tree_mask->size(-2) == T,
                      "tree_mask must be [", T, ", ", T, "] or [", B, ", ", T, ", ", T, "] (got ", tree_mask->sizes(), ")");
    mask = *tree_mask;
    ms[0] = mask.dim() == 3 && mask.size(0) == B ? mask.stride(0) : 0;
    ms[1] = mask.stride(-2), ms[2] = mask.stride(-1);
  }
  const c10::OptionalDeviceGuard guard(dev);
  if (max_context_len < 0) max_context_len = B ? std::max(context_lens.max().item<int32_t>(), 0) : 0;  // synchronises
  TORCH_CHECK_VALUE(max_context_len <= block_table.size(1) * kPage, "max_context_len ", max_context_len,
                    " exceeds the block table's ", block_table.size(1), " pages");
  const double s = scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(D));
  at::Tensor out = at::empty({B, T, Hq, D}, q.options());
  at::Tensor lse = at::empty({B, T, Hq}, q.options().dtype(at::kFloat));
  const int iB = as_int(B, "batch"), iT = as_int(T, "tokens"), iHq = as_int(Hq, "heads"), iHkv = as_int(c.Hkv, "heads"),
            iD = as_int(D, "head_dim"), iM = as_int(max_context_len, "max_context_len");
  const size_t need = spyre_paged_tree_attn_workspace_bytes(c.kind, iB, iT, iHq, iHkv, iD, iM, draft_keys);
  const at::Tensor ws = need ? at::empty({static_cast<int64_t>(need)}, q.options().dtype(at::kByte)) : at::Tensor();
  const int64_t qs[3] = {q.stride(0), q.stride(1), q.stride(2)};
  check_rc("spyre_paged_tree_attn",
           spyre_paged_tree_attn(q.data_ptr(), qs, kc.data_ptr(), vc.data_ptr(), ks.has_value() ? ks->data_ptr<float>() : nullptr,
                                 vs.has_value() ? vs->data_ptr<float>() : nullptr, c.kind, block_table.data_ptr<int32_t>(),
                                 block_table.stride(0), block_table.size(1), context_lens.data_ptr<int32_t>(),
                                 draft_lens.has_value() ? draft_lens->data_ptr<int32_t>() : nullptr, draft_keys,
                                 mask.defined() ? mask.data_ptr() : nullptr, ms, out.data_ptr(), lse.data_ptr<float>(),
                                 need ? ws.data_ptr() : nullptr, need, iB, iT, iHq, iHkv, iD, kPage, c.pages, iM,
                                 static_cast<float>(s), stream_of(q)));
  return {out, lse};
}

std::tuple<at::Tensor, at::Tensor> paged_tree_attention(const at::Tensor& q, const at::Tensor& kc, const at::Tensor& vc,
                                                        const at::Tensor& block_table, const at::Tensor& context_lens,
                                                        const std::optional<at::Tensor>& tree_mask,
                                                        const std::optional<at::Tensor>& draft_lens,
                                                        const std::optional<at::Tensor>& ks,
                                                        const std::optional<at::Tensor>& vs, std::optional<double> scale,
                                                        int64_t max_context_len) {
  return attend(q, kc, vc, ks, vs, block_table, context_lens, tree_mask, draft_lens, true, scale, max_context_len);
}

std::tuple<at::Tensor, at::Tensor> quant_paged_decode_attention(const at::Tensor& q, const at::Tensor& kc,
                                                                const at::Tensor& vc, const at::Tensor& ks,
                                                                const at::Tensor& vs, const at::Tensor& block_table,
                                                                const at::Tensor& context_lens, std::optional<double> scale,
                                                                int64_t max_context_len) {
  TORCH_CHECK_VALUE(q.dim() == 3, "q must be float16 [B, Hq, D]");
  auto [out, lse] = attend(q.unsqueeze(1), kc, vc, ks, vs, block_table, context_lens, std::nullopt, std::nullopt, false,
                           scale, max_context_len);
  return {out.squeeze(1), lse.squeeze(1)};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(spyre, m) {
  m.def("rotary(Tensor q, Tensor? k, Tensor positions, Tensor frequencies, float amplitude=1.0, "
        "bool interleaved=False, bool inverse=False) -> (Tensor, Tensor)");
  m.def("kv_quant_append(Tensor k_new, Tensor v_new, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scale, "
        "Tensor(d!) v_scale, Tensor block_table, Tensor slots) -> ()");
  m.def("rotary_kv_quant_append(Tensor q, Tensor k_new, Tensor v_new, Tensor(a!) k_cache, Tensor(b!) v_cache, "
        "Tensor(c!) k_scale, Tensor(d!) v_scale, Tensor block_table, Tensor slots, Tensor positions, "
        "Tensor frequencies, float amplitude=1.0, bool interleaved=False) -> Tensor");
  m.def("kv_quant_read(Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, Tensor block_table, "
        "Tensor lens, int length, Tensor? start=None) -> (Tensor, Tensor)");
  m.def("quant_paged_decode_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, "
        "Tensor block_table, Tensor context_lens, float? scale=None, int max_context_len=-1) -> (Tensor, Tensor)");
  m.def("paged_tree_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, Tensor context_lens, "
        "Tensor? tree_mask=None, Tensor? draft_lens=None, Tensor? k_scale=None, Tensor? v_scale=None, "
        "float? scale=None, int max_context_len=-1) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(spyre, CUDA, m) {
  m.impl("rotary", &rotary);
  m.impl("kv_quant_append", &kv_quant_append);
  m.impl("rotary_kv_quant_append", &rotary_kv_quant_append);
  m.impl("kv_quant_read", &kv_quant_read);
  m.impl("quant_paged_decode_attention", &quant_paged_decode_attention);
  m.impl("paged_tree_attention", &paged_tree_attention);
}

TORCH_LIBRARY_IMPL(spyre, Autograd, m) {
  m.impl("rotary", &rotary_autograd);
}
