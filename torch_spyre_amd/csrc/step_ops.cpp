// PyTorch-ROCm kernels of the page, draft verification and latent attention ops,
// as serving_ops.cpp has those of the ops beside them.
//
//   spyre::plan_pages              a block table extended from the sequences' lengths, slots of new tokens
//   spyre::release_pages           pages back to the free ones
//   spyre::verify_drafts           drafted tokens against the target's probabilities
//   spyre::latent_append           rows into the paged latent cache
//   spyre::latent_read             tokens of it as dense rows
//   spyre::paged_latent_attention  attention over it, all heads on one row a token
//   spyre::latent_attention        causal attention with expanded keys and values
// No reference counterparts.

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "torch_checks.h"

namespace {

using namespace spyre_torch;

constexpr int64_t kRope = 64;

void check_i32(const at::Tensor& t, at::IntArrayRef size, const c10::Device& dev, const char* name) {
  require_on(t, dev, name);
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.sizes() == size && t.is_contiguous(), name, " must be contiguous int32 ", size,
                    " (got ", t.scalar_type(), " ", t.sizes(), ")");
}

// The ring of free pages and its cursor.
void check_ring(const at::Tensor& free_pages, const at::Tensor& cursor, const c10::Device& dev) {
  require_on(free_pages, dev, "free_pages");
  require_on(cursor, dev, "cursor");
  TORCH_CHECK_VALUE(free_pages.scalar_type() == at::kInt && free_pages.dim() == 1 && free_pages.is_contiguous(),
                    "free_pages must be contiguous int32 [pages] (got ", free_pages.scalar_type(), " ", free_pages.sizes(), ")");
  TORCH_CHECK_VALUE(cursor.scalar_type() == at::kLong && cursor.sizes() == at::IntArrayRef({2}) && cursor.is_contiguous(),
                    "cursor must be contiguous int64 [2], taken and returned (got ", cursor.scalar_type(), " ", cursor.sizes(), ")");
}

int64_t table_rows(const at::Tensor& t) {
  TORCH_CHECK_VALUE(t.is_cuda(), "block_table must be a CUDA (HIP) tensor; there is no CPU path");
  TORCH_CHECK_VALUE(t.dim() == 2, "block_table must be int32 [B, pages_per_seq] with unit column stride");
  return t.size(0);
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> plan_pages(
    const at::Tensor& block_table, const at::Tensor& held, const at::Tensor& context_lens, const at::Tensor& new_lens,
    const at::Tensor& free_pages, const at::Tensor& cursor, int64_t length, int64_t tokens) {
  const int64_t B = table_rows(block_table);
  const auto dev = block_table.device();
  check_table(block_table, B, dev);
  check_i32(held, {B}, dev, "held");
  check_i32(context_lens, {B}, dev, "context_lens");
  check_i32(new_lens, {B}, dev, "new_lens");
  check_ring(free_pages, cursor, dev);
  TORCH_CHECK_VALUE((length >= 0) != (tokens >= 0), "either length or tokens is given (got ", length, " and ", tokens, ")");
  TORCH_CHECK_VALUE(B <= 1 || block_table.stride(0) >= block_table.size(1), "rows of block_table overlap");
  const c10::OptionalDeviceGuard guard(dev);
  const bool packed = tokens >= 0;
  const auto i32 = held.options();
  at::Tensor positions = packed ? at::empty({tokens}, i32) : at::empty({B, length}, i32);
  at::Tensor slots = at::empty_like(positions, cursor.options());
  at::Tensor starts = at::empty({packed ? B + 1 : 0}, i32);
  at::Tensor held_out = at::empty({B}, i32), cursor_out = at::empty({2}, cursor.options());
  check_rc("spyre_plan_pages",
           spyre_plan_pages(block_table.data_ptr<int32_t>(), block_table.stride(0), block_table.size(1), held.data_ptr<int32_t>(),
                            context_lens.data_ptr<int32_t>(), new_lens.data_ptr<int32_t>(), free_pages.data_ptr<int32_t>(),
                            free_pages.numel(), cursor.data_ptr<int64_t>(), packed ? -1 : as_int(length, "length"),
                            packed ? tokens : -1, positions.data_ptr<int32_t>(), slots.data_ptr<int64_t>(),
                            starts.data_ptr<int32_t>(), held_out.data_ptr<int32_t>(), cursor_out.data_ptr<int64_t>(),
                            as_int(B, "sequences"), stream_of(block_table)));
  return {positions, slots, held_out, cursor_out, starts};
}

std::tuple<at::Tensor, at::Tensor> release_pages(const at::Tensor& block_table, const at::Tensor& held, const at::Tensor& lens,
                                                 const at::Tensor& free_pages, const at::Tensor& cursor) {
  const int64_t B = table_rows(block_table);
  const auto dev = block_table.device();
  check_table(block_table, B, dev);
  check_i32(held, {B}, dev, "held");
  check_i32(lens, {B}, dev, "lens");
  check_ring(free_pages, cursor, dev);
  const c10::OptionalDeviceGuard guard(dev);
  at::Tensor held_out = at::empty({B}, held.options()), cursor_out = at::empty({2}, cursor.options());
  check_rc("spyre_release_pages",
           spyre_release_pages(block_table.data_ptr<int32_t>(), block_table.stride(0), block_table.size(1), held.data_ptr<int32_t>(),
                               lens.data_ptr<int32_t>(), free_pages.data_ptr<int32_t>(), free_pages.numel(),
                               cursor.data_ptr<int64_t>(), held_out.data_ptr<int32_t>(), cursor_out.data_ptr<int64_t>(),
                               as_int(B, "sequences"), stream_of(block_table)));
  return {held_out, cursor_out};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> verify_drafts(const at::Tensor& tokens, const at::Tensor& target_probs,
                                                             const at::Tensor& uniforms, const std::optional<at::Tensor>& draft_probs,
                                                             const std::optional<at::Tensor>& parents,
                                                             const std::optional<at::Tensor>& draft_lens) {
  TORCH_CHECK_VALUE(target_probs.is_cuda(), "target_probs must be a CUDA (HIP) tensor; there is no CPU path");
  const auto dev = target_probs.device();
  require_on(tokens, dev, "draft_tokens");
  require_on(uniforms, dev, "uniforms");
  TORCH_CHECK_VALUE((tokens.scalar_type() == at::kInt || tokens.scalar_type() == at::kLong) && tokens.dim() == 2,
                    "draft_tokens must be int32 or int64 [B, T] (got ", tokens.scalar_type(), " ", tokens.sizes(), ")");
  const int64_t B = tokens.size(0), T = tokens.size(1);
  const auto type = target_probs.scalar_type();
  TORCH_CHECK_TYPE(type == at::kFloat || type == at::kHalf || type == at::kBFloat16,
                   "target_probs must be float32, float16 or bfloat16 (got ", type, ")");
  TORCH_CHECK_VALUE(target_probs.dim() == 3 && target_probs.size(0) == B && target_probs.size(1) == T + 1 && target_probs.size(2) > 0,
                    "target_probs must be [", B, ", ", T + 1, ", V] (got ", target_probs.sizes(), ")");
  const int64_t V = target_probs.size(2);
  TORCH_CHECK_VALUE(uniforms.scalar_type() == at::kFloat && uniforms.sizes() == at::IntArrayRef({B, T + 1}),
                    "uniforms must be float32 [", B, ", ", T + 1, "] (got ", uniforms.scalar_type(), " ", uniforms.sizes(), ")");
  if (draft_probs.has_value()) {
    require_on(*draft_probs, dev, "draft_probs");
    TORCH_CHECK_TYPE(draft_probs->scalar_type() == type, "draft_probs and target_probs differ in dtype");
    TORCH_CHECK_VALUE(draft_probs->sizes() == at::IntArrayRef({B, T, V}), "draft_probs must be [", B, ", ", T, ", ", V, "] (got ",
                      draft_probs->sizes(), ")");
    TORCH_CHECK_VALUE(!parents.has_value(), "draft_probs are those of a chain: a tree (parents) takes none");
  }
  if (parents.has_value()) {
    require_on(*parents, dev, "parents");
    TORCH_CHECK_VALUE(parents->scalar_type() == at::kInt && parents->sizes() == at::IntArrayRef({B, T}), "parents must be int32 [", B,
                      ", ", T, "] (got ", parents->scalar_type(), " ", parents->sizes(), ")");
  }
  if (draft_lens.has_value()) check_lens(*draft_lens, B, dev, "draft_lens");
  const c10::OptionalDeviceGuard guard(dev);
  auto rows = [](const at::Tensor& t) { return t.stride(2) == 1 || t.size(2) == 1 ? t : t.contiguous(); };
  const at::Tensor p = rows(target_probs), q = draft_probs.has_value() ? rows(*draft_probs) : at::Tensor();
  at::Tensor out = at::empty({B, T + 1}, tokens.options());
  at::Tensor accepted = at::empty({B}, tokens.options().dtype(at::kInt)), path = at::empty({B, T}, accepted.options());
  const int iB = as_int(B, "batch"), iT = as_int(T, "drafted tokens"), iV = as_int(V, "vocabulary");
  const size_t need = spyre_verify_drafts_workspace_bytes(iB, iV);
  const at::Tensor ws = at::empty({static_cast<int64_t>(need)}, tokens.options().dtype(at::kByte));
  const int64_t ps[2] = {p.stride(0), p.stride(1)};
  const int64_t qs[2] = {q.defined() ? q.stride(0) : 0, q.defined() ? q.stride(1) : 0};
  check_rc("spyre_verify_drafts",
           spyre_verify_drafts(tokens.data_ptr(), static_cast<int>(tokens.element_size()), tokens.stride(0), tokens.stride(1),
                               p.data_ptr(), ps, q.defined() && T ? q.data_ptr() : nullptr, qs,
                               type == at::kFloat ? SPYRE_DT_FLOAT32 : type == at::kHalf ? SPYRE_DT_FLOAT16 : SPYRE_DT_BFLOAT16,
                               uniforms.data_ptr<float>(), uniforms.stride(0), uniforms.stride(1),
                               parents.has_value() ? parents->data_ptr<int32_t>() : nullptr,
                               parents.has_value() ? parents->stride(0) : 0, parents.has_value() ? parents->stride(1) : 0,
                               draft_lens.has_value() ? draft_lens->data_ptr<int32_t>() : nullptr, out.data_ptr(),
                               accepted.data_ptr<int32_t>(), path.data_ptr<int32_t>(), ws.data_ptr(), need, iB, iT, iV,
                               stream_of(p)));
  return {out, accepted, path};
}

// ---------------------------------------------------------------- latent --

struct Latent {
  int64_t pages, rank;
};

Latent check_latent(const at::Tensor& cache, const c10::Device& dev) {
  require_on(cache, dev, "cache");
  TORCH_CHECK_TYPE(cache.scalar_type() == at::kHalf, "cache must be float16 (got ", cache.scalar_type(), ")");
  TORCH_CHECK_VALUE(cache.dim() == 4 && cache.size(1) > 1 && cache.size(2) == kPage && cache.size(3) == 64 && cache.is_contiguous(),
                    "cache must be contiguous [pages, (rank + 64) / 64, 64, 64] (got ", cache.sizes(), ")");
  return {cache.size(0), cache.size(1) * 64 - kRope};
}

// fp16 rows [.., features] as a matrix that the kernels read as 16-byte vectors.
at::Tensor matrix(const at::Tensor& t, int64_t features, const char* name) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kHalf, name, " must be float16 (got ", t.scalar_type(), ")");
  TORCH_CHECK_VALUE(t.dim() >= 2 && t.size(-1) == features, name, " must be [..., ", features, "] (got ", t.sizes(), ")");
  const at::Tensor x = t.reshape({-1, features});
  const bool ready = x.stride(1) == 1 && x.stride(0) % 8 == 0 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
  return ready ? x : x.clone(at::MemoryFormat::Contiguous);
}

void latent_append(const at::Tensor& latent, const at::Tensor& k_rope, const at::Tensor& cache, const at::Tensor& slots) {
  TORCH_CHECK_VALUE(cache.is_cuda(), "cache must be a CUDA (HIP) tensor; there is no CPU path");
  const auto dev = cache.device();
  const Latent c = check_latent(cache, dev);
  require_on(latent, dev, "latent");
  require_on(k_rope, dev, "k_rope");
  require_on(slots, dev, "slots");
  TORCH_CHECK_VALUE(slots.scalar_type() == at::kLong, "slots must be int64 (got ", slots.scalar_type(), ")");
  TORCH_CHECK_VALUE(latent.sizes().slice(0, latent.dim() - (latent.dim() > 0)) == slots.sizes() &&
                        k_rope.sizes().slice(0, k_rope.dim() - (k_rope.dim() > 0)) == slots.sizes(),
                    "latent and k_rope must have a row for each of the slots ", slots.sizes(), " (got ", latent.sizes(), " and ",
                    k_rope.sizes(), ")");
  const c10::OptionalDeviceGuard guard(dev);
  if (slots.numel() == 0) return;
  const at::Tensor x = matrix(latent, c.rank, "latent"), r = matrix(k_rope, kRope, "k_rope");
  const at::Tensor s = slots.contiguous();
  check_rc("spyre_latent_append_f16",
           spyre_latent_append_f16(x.data_ptr(), x.stride(0), r.data_ptr(), r.stride(0), cache.data_ptr(), s.data_ptr<int64_t>(),
                                   s.numel(), as_int(c.rank, "rank"), c.pages, stream_of(cache)));
}

std::tuple<at::Tensor, at::Tensor> latent_read(const at::Tensor& cache, const at::Tensor& block_table, const at::Tensor& lens,
                                               int64_t length, const std::optional<at::Tensor>& start) {
  TORCH_CHECK_VALUE(cache.is_cuda(), "cache must be a CUDA (HIP) tensor; there is no CPU path");
  const auto dev = cache.device();
  const Latent c = check_latent(cache, dev);
  TORCH_CHECK_VALUE(length >= 0, "length ", length, " is negative");
  const int64_t B = table_rows(block_table);
  check_table(block_table, B, dev);
  check_lens(lens, B, dev, "lens");
  if (start.has_value()) check_lens(*start, B, dev, "start");
  const c10::OptionalDeviceGuard guard(dev);
  at::Tensor latent = at::empty({B, length, c.rank}, cache.options()), rope = at::empty({B, length, kRope}, cache.options());
  check_rc("spyre_latent_read_f16",
           spyre_latent_read_f16(cache.data_ptr(), block_table.data_ptr<int32_t>(), block_table.stride(0), block_table.size(1),
                                 lens.data_ptr<int32_t>(), start.has_value() ? start->data_ptr<int32_t>() : nullptr,
                                 latent.data_ptr(), rope.data_ptr(), as_int(B, "batch"), as_int(length, "length"),
                                 as_int(c.rank, "rank"), c.pages, stream_of(cache)));
  return {latent, rope};
}

// Queries [B, T, H, D] of which 64 of a sequence's (t, h) lie within the 2^30 elements that the
// kernel reaches: those of a product batched over heads, [H, B, T, D], are copied from B T = 16513 on
// with 128 heads of 512 features.
at::Tensor near_rows(const at::Tensor& t) {
  const int64_t T = t.size(1), H = t.size(2);
  if (t.numel() == 0) return t;
  const double reach = static_cast<double>(std::min(T - 1, (64 + H - 2) / H)) * t.stride(1) + static_cast<double>(H - 1) * t.stride(2);
  return reach < (1 << 30) - 512 ? t : t.clone(at::MemoryFormat::Contiguous);
}

std::tuple<at::Tensor, at::Tensor> paged_latent_attention(const at::Tensor& query, const at::Tensor& query_rope,
                                                          const at::Tensor& cache, const at::Tensor& block_table,
                                                          const at::Tensor& context_lens, double scale,
                                                          const std::optional<at::Tensor>& tree_mask,
                                                          const std::optional<at::Tensor>& draft_lens, int64_t max_context_len) {
  const at::Tensor q = near_rows(rows_operand(query, "q")), qr = near_rows(rows_operand(query_rope, "q_rope"));
  const auto dev = q.device();
  const Latent c = check_latent(cache, dev);
  const int64_t B = q.size(0), T = q.size(1), H = q.size(2);
  TORCH_CHECK_VALUE(q.size(3) == c.rank, "the cache holds latent vectors of ", c.rank, " features, q has ", q.size(3));
  require_on(qr, dev, "q_rope");
  TORCH_CHECK_VALUE(qr.sizes() == at::IntArrayRef({B, T, H, kRope}), "q_rope must be [", B, ", ", T, ", ", H, ", 64] (got ", qr.sizes(), ")");
  TORCH_CHECK_VALUE(H > 0, "q has no heads");
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
  at::Tensor out = at::empty({B, T, H, c.rank}, q.options());
  at::Tensor lse = at::empty({B, T, H}, q.options().dtype(at::kFloat));
  const int iB = as_int(B, "batch"), iT = as_int(T, "tokens"), iH = as_int(H, "heads"), iR = as_int(c.rank, "rank"),
            iM = as_int(max_context_len, "max_context_len");
  const size_t need = spyre_paged_latent_attn_workspace_bytes(iB, iT, iH, iR, iM);
  const at::Tensor ws = need ? at::empty({static_cast<int64_t>(need)}, q.options().dtype(at::kByte)) : at::Tensor();
  const int64_t qs[3] = {q.stride(0), q.stride(1), q.stride(2)}, qrs[3] = {qr.stride(0), qr.stride(1), qr.stride(2)};
  check_rc("spyre_paged_latent_attn",
           spyre_paged_latent_attn(q.data_ptr(), qs, qr.data_ptr(), qrs, cache.data_ptr(), block_table.data_ptr<int32_t>(),
                                   block_table.stride(0), block_table.size(1), context_lens.data_ptr<int32_t>(),
                                   draft_lens.has_value() ? draft_lens->data_ptr<int32_t>() : nullptr,
                                   mask.defined() ? mask.data_ptr() : nullptr, ms, out.data_ptr(), lse.data_ptr<float>(),
                                   need ? ws.data_ptr() : nullptr, need, iB, iT, iH, iR, c.pages, iM, static_cast<float>(scale),
                                   stream_of(q)));
  return {out, lse};
}

// Keys or values [B, keys, H, D] whose tokens are less than the 2^23 elements apart that the kernel
// takes (those of a tile in 31 bits): of [keys, B, H, D] with B H D beyond, a copy.
at::Tensor near_keys(const at::Tensor& t) { return t.stride(1) < (1 << 23) ? t : t.clone(at::MemoryFormat::Contiguous); }

std::tuple<at::Tensor, at::Tensor> latent_attention(const at::Tensor& query, const at::Tensor& query_rope, const at::Tensor& key,
                                                    const at::Tensor& key_rope, const at::Tensor& value,
                                                    const at::Tensor& context_lens, const std::optional<at::Tensor>& new_lens,
                                                    std::optional<double> scale) {
  const at::Tensor q = rows_operand(query, "q"), qr = rows_operand(query_rope, "q_rope");
  const at::Tensor k = near_keys(rows_operand(key, "k")), v = near_keys(rows_operand(value, "v"));
  const auto dev = q.device();
  const int64_t B = q.size(0), T = q.size(1), H = q.size(2), D = q.size(3), n = k.size(1);
  require_on(qr, dev, "q_rope");
  require_on(k, dev, "k");
  require_on(v, dev, "v");
  require_on(key_rope, dev, "k_rope");
  TORCH_CHECK_VALUE(H > 0, "q has no heads");
  TORCH_CHECK_VALUE(qr.sizes() == at::IntArrayRef({B, T, H, kRope}), "q_rope must be [", B, ", ", T, ", ", H, ", 64] (got ", qr.sizes(), ")");
  TORCH_CHECK_VALUE(k.sizes() == at::IntArrayRef({B, n, H, D}) && v.sizes() == k.sizes(), "k and v must be [", B, ", keys, ", H, ", ", D,
                    "] (got ", k.sizes(), " and ", v.sizes(), ")");
  TORCH_CHECK_TYPE(key_rope.scalar_type() == at::kHalf, "k_rope must be float16 (got ", key_rope.scalar_type(), ")");
  TORCH_CHECK_VALUE(key_rope.sizes() == at::IntArrayRef({B, n, kRope}), "k_rope must be [", B, ", ", n, ", 64] (got ", key_rope.sizes(), ")");
  check_lens(context_lens, B, dev, "context_lens");
  if (new_lens.has_value()) check_lens(*new_lens, B, dev, "new_lens");
  const c10::OptionalDeviceGuard guard(dev);
  const at::Tensor kr = near_keys(rows_operand(key_rope.unsqueeze(2), "k_rope"));
  const double s = scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(D + kRope));
  at::Tensor out = at::empty({B, T, H, D}, q.options());
  at::Tensor lse = at::empty({B, T, H}, q.options().dtype(at::kFloat));
  auto st = [](const at::Tensor& t) { return std::array<int64_t, 3>{t.stride(0), t.stride(1), t.stride(2)}; };
  const auto qs = st(q), qrs = st(qr), ks = st(k), krs = st(kr), vs = st(v);
  const int iB = as_int(B, "batch"), iT = as_int(T, "tokens"), iH = as_int(H, "heads"), iD = as_int(D, "head_dim"),
            iN = as_int(n, "keys");
  const size_t need = spyre_latent_attn_workspace_bytes(iB, iT, iH, iD, iN);
  const at::Tensor ws = need ? at::empty({static_cast<int64_t>(need)}, q.options().dtype(at::kByte)) : at::Tensor();
  check_rc("spyre_latent_attn",
           spyre_latent_attn(q.data_ptr(), qs.data(), qr.data_ptr(), qrs.data(), k.data_ptr(), ks.data(), kr.data_ptr(), krs.data(),
                             v.data_ptr(), vs.data(), context_lens.data_ptr<int32_t>(),
                             new_lens.has_value() ? new_lens->data_ptr<int32_t>() : nullptr, out.data_ptr(), lse.data_ptr<float>(),
                             need ? ws.data_ptr() : nullptr, need, iB, iT, iH, iD, iN, static_cast<float>(s), stream_of(q)));
  return {out, lse};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(spyre, m) {
  m.def("plan_pages(Tensor(a!) block_table, Tensor held, Tensor context_lens, Tensor new_lens, Tensor free_pages, "
        "Tensor cursor, int length=-1, int tokens=-1) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("release_pages(Tensor block_table, Tensor held, Tensor lens, Tensor(a!) free_pages, Tensor cursor) -> (Tensor, Tensor)");
  m.def("verify_drafts(Tensor draft_tokens, Tensor target_probs, Tensor uniforms, Tensor? draft_probs=None, "
        "Tensor? parents=None, Tensor? draft_lens=None) -> (Tensor, Tensor, Tensor)");
  m.def("latent_append(Tensor latent, Tensor k_rope, Tensor(a!) cache, Tensor slots) -> ()");
  m.def("latent_read(Tensor cache, Tensor block_table, Tensor lens, int length, Tensor? start=None) -> (Tensor, Tensor)");
  m.def("paged_latent_attention(Tensor q, Tensor q_rope, Tensor cache, Tensor block_table, Tensor context_lens, float scale, "
        "Tensor? tree_mask=None, Tensor? draft_lens=None, int max_context_len=-1) -> (Tensor, Tensor)");
  m.def("latent_attention(Tensor q, Tensor q_rope, Tensor k, Tensor k_rope, Tensor v, Tensor context_lens, "
        "Tensor? new_lens=None, float? scale=None) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(spyre, CUDA, m) {
  m.impl("plan_pages", &plan_pages);
  m.impl("release_pages", &release_pages);
  m.impl("verify_drafts", &verify_drafts);
  m.impl("latent_append", &latent_append);
  m.impl("latent_read", &latent_read);
  m.impl("paged_latent_attention", &paged_latent_attention);
  m.impl("latent_attention", &latent_attention);
}
