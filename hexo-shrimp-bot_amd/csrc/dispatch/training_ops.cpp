// The training operators of the mantisnet:: namespace on torch's dispatcher:
// fused_attention_relative, policy_log_probs, residual_dropout and their
// backwards, over the C entry points of libmantis_hip.so (include/mantis_hip.h).
//
// Their checks, outputs, workspaces and gradients live here and not in Python
// because a training step calls them between other host-bound work: a call
// with its backward of 1,464 x 128 rows takes 60 us against 128 through
// Python functions, whose backward runs in torch's device thread, cold, at
// twice the time of the same code in the caller's.
//
// Errors follow ops.py: ValueError for arguments, RuntimeError for a CPU tensor
// (there is no CPU path) or a failed launch; indices are checked on the device
// and recorded in the device's error words, which ops.raise_on_device_error reads.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <array>
#include <atomic>
#include <memory>
#include <mutex>
#include <utility>

#include "../../../include/mantis_hip.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ------------------------------------------------------------- devices, streams, errors

at::Device on_gpu(std::initializer_list<const Tensor*> tensors) {
  optional<at::Device> dev;
  for (const Tensor* t : tensors) {
    if (!t || !t->defined()) continue;
    TORCH_CHECK(t->is_cuda(),
                "the MantisNet kernels run on the MI355X only (got a CPU tensor); there is no CPU path");
    if (!dev) dev = t->device();
    TORCH_CHECK_VALUE(t->device() == *dev, "all inputs must be on one device");
  }
  return *dev;
}

void* stream_of(at::Device dev) { return c10::hip::getCurrentHIPStream(dev.index()).stream(); }

// The devices' error words (ops.error_flag), held until the process ends.
constexpr int kMaxDevices = 64;
std::mutex words_lock;
std::atomic<const Tensor*> words_of[kMaxDevices] = {};

// Made on the first use, filled, and only then seen by anyone else: another thread's or stream's
// kernels write them next.  On a stream of their own and outside any capture, whose
// memory would be the graph's, cleared by its replays.
const Tensor& words(int64_t device) {
  TORCH_CHECK(device >= 0 && device < kMaxDevices, "device index past ", kMaxDevices);
  if (const Tensor* w = words_of[device].load(std::memory_order_acquire)) return *w;
  std::lock_guard<std::mutex> hold(words_lock);
  if (const Tensor* w = words_of[device].load(std::memory_order_acquire)) return *w;
  const c10::impl::ExcludeDispatchKeyGuard no_modes(
      c10::DispatchKeySet({c10::DispatchKey::Python, c10::DispatchKey::PythonTLSSnapshot}));
  const c10::InferenceMode ordinary(false);  // (they are cleared outside of one too)
  const at::Device dev(at::kCUDA, c10::DeviceIndex(device));
  const c10::DeviceGuard on(dev);
  const c10::hip::HIPStreamCaptureModeGuard apart(hipStreamCaptureModeRelaxed);
  const c10::hip::HIPStream stream = c10::hip::getStreamFromPool(false, c10::DeviceIndex(device));
  const c10::hip::HIPStreamGuard beside(stream);
  auto made = std::make_unique<const Tensor>(at::zeros({2}, at::TensorOptions(at::kInt).device(dev)));
  stream.synchronize();
  words_of[device].store(made.get(), std::memory_order_release);
  return *made.release();
}

// The words, made if need be or (make false) none where no one has asked for them.
optional<Tensor> error_words(int64_t device, bool make) {
  if (make) return words(device);
  const Tensor* w = device >= 0 && device < kMaxDevices ? words_of[device].load(std::memory_order_acquire) : nullptr;
  return w ? optional<Tensor>(*w) : std::nullopt;
}

int32_t* error_flag(at::Device dev) { return words(dev.index()).data_ptr<int32_t>(); }

void check_status(int32_t status, const char* what) {
  TORCH_CHECK_VALUE(status != MANTIS_E_ARG, what, ": unsupported shape, dtype, alignment or null input");
  TORCH_CHECK(status == MANTIS_OK, what, ": HIP launch failed (status ", status, ")");
}

int32_t dtype_of(at::ScalarType t) {
  if (t == at::kBFloat16) return MANTIS_BF16;
  if (t == at::kHalf) return MANTIS_F16;
  TORCH_CHECK_VALUE(t == at::kFloat, "unsupported dtype ", t, "; expected float16, bfloat16 or float32");
  return MANTIS_F32;
}

template <typename T = float>
T* ptr(const optional<Tensor>& t) {
  return t && t->defined() ? static_cast<T*>(t->data_ptr()) : nullptr;
}

// (a tangent would be lost below autograd)
bool wants_grad(std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    TORCH_CHECK_NOT_IMPLEMENTED(!t || !t->defined() || !t->_fw_grad(/*level=*/0).defined(),
                                "forward-mode differentiation of the MantisNet operators is not implemented");
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors)
    if (t && t->defined() && t->requires_grad()) return true;
  return false;
}

// ------------------------------------------------------------- relative attention

struct HeadRows {  // a (P, A, T, D) operand and its element strides as the kernels take them
  Tensor t;
  int64_t strides[4] = {};
};

// whether t's rows are dense, 16-byte aligned and within their descriptors (a
// dimension of one entry has no stride of its own)
bool row_strides(const Tensor& t, int64_t (&s)[4]) {
  const auto sizes = t.sizes(), st = t.strides();
  s[0] = sizes[0] == 1 ? 0 : st[0];
  s[1] = sizes[1] == 1 ? 0 : st[1];
  s[2] = sizes[2] == 1 ? sizes[3] : st[2];
  s[3] = 1;
  return st[3] == 1 && (s[0] | s[1] | s[2]) % 8 == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 &&
         s[2] >= sizes[3] && s[2] < 8192 && sizes[2] * s[2] * 2 <= 0x7FFFFFFF;
}

HeadRows head_rows(const Tensor& t) {
  HeadRows r{t};
  if (row_strides(t, r.strides)) return r;
  r.t = t.clone(at::MemoryFormat::Contiguous);
  TORCH_CHECK_VALUE(row_strides(r.t, r.strides), "a position's rows are past the kernel's 2 GiB");
  return r;
}

// An empty result beside the operand t (P, A, T, D), kernels and fakes alike: whole rows in the
// order that t's own lie in memory (heads inside rows for a projection's view, packed or not),
// without its gaps; contiguous where t has no such order (a repeated dimension, D not innermost)
// or the kernels do not take its rows.
Tensor empty_rows_like(const Tensor& t) {
  const auto n = t.sym_sizes(), s = t.sym_strides();
  std::array<c10::SymInt, 4> strides{n[1] * n[2] * n[3], n[2] * n[3], n[3], 1};
  // outermost first; a dimension of one entry has no place of its own and stands before the others
  std::array<int, 3> order{0, 1, 2};
  const auto before = [&](int a, int b) {
    if (n[a] == 1 || n[b] == 1) return n[a] == 1 && n[b] != 1;
    return s[a] > s[b];
  };
  for (int i = 1; i < 3; ++i)
    for (int j = i; j > 0 && before(order[j], order[j - 1]); --j) std::swap(order[j], order[j - 1]);
  bool ordered = s[3] == 1;
  for (int i = 0; i < 3 && ordered; ++i) ordered = n[i] == 1 || s[i] != 0;
  if (ordered) {
    std::array<c10::SymInt, 4> own = strides;
    c10::SymInt step = n[3];
    for (int i = 2; i >= 0; --i) {
      own[order[i]] = step;
      step = step * n[order[i]];
    }
    if (n[2] == 1 || (own[2] < 8192 && n[2] * own[2] * 2 <= 0x7FFFFFFF)) strides = own;
  }
  return at::empty_strided_symint(n, strides, t.options());
}

HeadRows head_rows_like(const Tensor& t) {
  HeadRows r{empty_rows_like(t)};
  row_strides(r.t, r.strides);
  return r;
}

// (a conversion that is none costs a dispatch)
Tensor as(const Tensor& t, at::ScalarType dtype) { return t.scalar_type() == dtype ? t : t.to(dtype); }

// (sizes as symbols here and in the fakes, which see them where a trace leaves them open)
void check_relative(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& bias, const Tensor& coords,
                    const Tensor& buckets, const Tensor& seq_lens, int64_t n_latents) {
  TORCH_CHECK_VALUE(q.dim() == 4 && k.sym_sizes() == q.sym_sizes() && v.sym_sizes() == q.sym_sizes(),
                    "q, k and v must have the same (P, A, T, D) shape");
  const auto p = q.sym_size(0), heads = q.sym_size(1), t = q.sym_size(2), hd = q.sym_size(3);
  TORCH_CHECK_VALUE((q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16) &&
                        k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
                    "relative attention runs 16-bit MFMA: q, k and v must share float16 or bfloat16");
  TORCH_CHECK_VALUE(hd == 16 || hd == 32 || hd == 64, "relative attention supports head_dim 16, 32 and 64");
  TORCH_CHECK_VALUE(seq_lens.dim() == 1 && seq_lens.sym_size(0) == p && seq_lens.scalar_type() == at::kInt,
                    "seq_lens must be int32 with shape (P,)");
  TORCH_CHECK_VALUE(bias.dim() == 2 && bias.sym_size(0) == heads && bias.is_floating_point(),
                    "bias must be floating point with shape (heads, buckets)");
  TORCH_CHECK_VALUE(bias.sym_size(1) >= 1 && bias.sym_size(1) <= 384, "bias must hold 1 to 384 buckets");
  TORCH_CHECK_VALUE(coords.dim() == 3 && coords.sym_size(0) == p && coords.sym_size(1) == t && coords.sym_size(2) == 2 &&
                        coords.scalar_type() == at::kInt,
                    "coords must be int32 with shape (P, T, 2)");
  TORCH_CHECK_VALUE(buckets.dim() == 2 && buckets.scalar_type() == at::kInt && buckets.sym_size(0) % 2 == 1 &&
                        buckets.sym_size(1) % 2 == 1,
                    "buckets must be int32 with an odd number of rows and of columns");
  TORCH_CHECK_VALUE(buckets.sym_numel() <= 4096, "buckets must hold at most 4096 displacements");
  TORCH_CHECK_VALUE(n_latents >= 0 && n_latents <= t && (n_latents == 0 || bias.sym_size(1) >= 2),
                    "n_latents must lie in [0, T], with two buckets of their own");
}

// contiguous coordinates whose pairs are 8-byte aligned
Tensor coord_pairs(const Tensor& coords) {
  Tensor c = coords.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 8 ? c.clone() : c;
}

using Three = std::tuple<Tensor, Tensor, Tensor>;
using Four = std::tuple<Tensor, Tensor, Tensor, Tensor>;

Three relative_meta(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& bias, const Tensor& coords,
                    const Tensor& buckets, const Tensor& seq_lens, int64_t n_latents) {
  check_relative(q, k, v, bias, coords, buckets, seq_lens, n_latents);
  const auto f32 = q.options().dtype(at::kFloat);
  const auto n = q.sym_sizes();
  return {empty_rows_like(q), at::empty_symint({n[0], n[1], n[2]}, f32), at::empty_symint({n[0], n[1], n[2], 2}, f32)};
}

Three relative(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& bias_, const Tensor& coords_,
               const Tensor& buckets_, const Tensor& seq_lens_, int64_t n_latents) {
  const at::Device dev = on_gpu({&q_, &k_, &v_, &bias_, &coords_, &buckets_, &seq_lens_});
  check_relative(q_, k_, v_, bias_, coords_, buckets_, seq_lens_, n_latents);
  const c10::DeviceGuard guard(dev);
  const int64_t p = q_.size(0), heads = q_.size(1), t = q_.size(2), hd = q_.size(3);
  const HeadRows out = head_rows_like(q_);
  const auto f32 = q_.options().dtype(at::kFloat);
  Tensor lse = at::empty({p, heads, t}, f32), stats = at::empty({p, heads, t, 2}, f32);
  if (out.t.numel() == 0) return {out.t, lse, stats};
  const HeadRows q = head_rows(q_), k = head_rows(k_), v = head_rows(v_);
  const Tensor bias = as(bias_, at::kFloat).contiguous(), coords = coord_pairs(coords_),
               buckets = buckets_.contiguous(), seq_lens = seq_lens_.contiguous();
  check_status(mantis_relative_attention(
                   q.t.data_ptr(), q.strides, k.t.data_ptr(), k.strides, v.t.data_ptr(), v.strides,
                   dtype_of(q_.scalar_type()), bias.data_ptr<float>(), bias.size(1), coords.data_ptr<int32_t>(),
                   buckets.data_ptr<int32_t>(), buckets.size(0), buckets.size(1), n_latents,
                   seq_lens.data_ptr<int32_t>(), p, int32_t(heads), t, int32_t(hd), out.t.data_ptr(), out.strides,
                   lse.data_ptr<float>(), stats.data_ptr<float>(), error_flag(dev), stream_of(dev)),
               "relative_attention");
  return {out.t, lse, stats};
}

void check_relative_backward(const Tensor& q, const Tensor& stats, const Tensor& grad_out) {
  TORCH_CHECK_VALUE(grad_out.sym_sizes() == q.sym_sizes(), "grad_out must have q's shape");
  TORCH_CHECK_VALUE(stats.dim() == 4 && stats.sym_size(0) == q.sym_size(0) && stats.sym_size(1) == q.sym_size(1) &&
                        stats.sym_size(2) == q.sym_size(2) && stats.sym_size(3) == 2 && stats.scalar_type() == at::kFloat,
                    "stats must be the forward's (P, A, T, 2) fp32 statistics");
}

Four relative_backward_meta(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& bias,
                            const Tensor& coords, const Tensor& buckets, const Tensor& seq_lens, int64_t n_latents,
                            const Tensor& stats, const Tensor& grad_out) {
  check_relative(q, k, v, bias, coords, buckets, seq_lens, n_latents);
  check_relative_backward(q, stats, grad_out);
  return {empty_rows_like(q), empty_rows_like(k), empty_rows_like(v), at::empty_symint(bias.sym_sizes(), bias.options())};
}

Four relative_backward(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& bias_,
                       const Tensor& coords_, const Tensor& buckets_, const Tensor& seq_lens_, int64_t n_latents,
                       const Tensor& stats_, const Tensor& grad_out_) {
  const at::Device dev = on_gpu({&q_, &k_, &v_, &bias_, &coords_, &buckets_, &seq_lens_, &stats_, &grad_out_});
  check_relative(q_, k_, v_, bias_, coords_, buckets_, seq_lens_, n_latents);
  check_relative_backward(q_, stats_, grad_out_);
  const c10::DeviceGuard guard(dev);
  const int64_t p = q_.size(0), heads = q_.size(1), t = q_.size(2), hd = q_.size(3), n_buckets = bias_.size(1);
  const HeadRows dq = head_rows_like(q_), dk = head_rows_like(k_), dv = head_rows_like(v_);
  if (dq.t.numel() == 0) return {dq.t, dk.t, dv.t, at::zeros(bias_.sizes(), bias_.options())};
  const HeadRows q = head_rows(q_), k = head_rows(k_), v = head_rows(v_),
                 go = head_rows(as(grad_out_, q_.scalar_type()));
  const Tensor bias = as(bias_, at::kFloat).contiguous(), coords = coord_pairs(coords_),
               buckets = buckets_.contiguous(), seq_lens = seq_lens_.contiguous(), stats = stats_.contiguous();
  Tensor dbias = at::empty({heads, n_buckets}, q_.options().dtype(at::kFloat));
  const int64_t bytes = mantis_relative_attention_backward_workspace(p, int32_t(heads), t, n_buckets);
  const Tensor ws = at::empty({bytes}, q_.options().dtype(at::kByte));
  check_status(mantis_relative_attention_backward(
                   q.t.data_ptr(), q.strides, k.t.data_ptr(), k.strides, v.t.data_ptr(), v.strides, go.t.data_ptr(),
                   go.strides, stats.data_ptr<float>(), dtype_of(q_.scalar_type()), bias.data_ptr<float>(), n_buckets,
                   coords.data_ptr<int32_t>(), buckets.data_ptr<int32_t>(), buckets.size(0), buckets.size(1),
                   n_latents, seq_lens.data_ptr<int32_t>(), p, int32_t(heads), t, int32_t(hd), ws.data_ptr(), bytes,
                   dq.t.data_ptr(), dq.strides, dk.t.data_ptr(), dk.strides, dv.t.data_ptr(), dv.strides,
                   dbias.data_ptr<float>(), error_flag(dev), stream_of(dev)),
               "relative_attention_backward");
  return {dq.t, dk.t, dv.t, as(dbias, bias_.scalar_type())};
}

// ------------------------------------------------------------- policy

void check_policy(const Tensor& logits, const Tensor& offsets, const Tensor& moves, int64_t top) {
  TORCH_CHECK_VALUE(logits.dim() == 1, "logits must be flat (N,)");
  dtype_of(logits.scalar_type());
  TORCH_CHECK_VALUE(offsets.dim() == 1 && offsets.sym_size(0) >= 1, "offsets must hold P + 1 entries");
  TORCH_CHECK_VALUE(offsets.scalar_type() == at::kLong, "offsets must have dtype int64");
  TORCH_CHECK_VALUE(moves.dim() == 2 && moves.sym_size(0) == offsets.sym_size(0) - 1, "moves must have shape (P, moves)");
  TORCH_CHECK_VALUE(moves.scalar_type() == at::kLong, "moves must have dtype int64");
  TORCH_CHECK_VALUE(moves.sym_size(1) <= 1024, "at most 1024 moves of a position");
  TORCH_CHECK_VALUE(top >= 0 && top <= 64, "top must lie in [0, 64], got ", top);
}

struct Runs {  // the logits' stride and the index tables as the kernels take them
  Tensor logits;
  int64_t stride;
  Tensor offsets, moves;
  Runs(const Tensor& logits_, const Tensor& offsets_, const Tensor& moves_)
      : logits(logits_), stride(logits_.numel() > 1 ? logits_.stride(0) : 1), offsets(offsets_.contiguous()),
        moves(moves_.contiguous()) {
    if (stride < 1) logits = logits_.contiguous(), stride = 1;
  }
};

using Six = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>;

Six policy_outputs(const Tensor& logits, const Tensor& moves, int64_t top) {
  const auto p = moves.sym_size(0);
  const c10::SymInt k = top;
  const auto f32 = logits.options().dtype(at::kFloat);
  return {at::empty_symint({p, moves.sym_size(1)}, f32), at::empty_symint({p}, f32), at::empty_symint({p}, f32),
          at::empty_symint({p, k}, f32), at::empty_symint({p, k}, moves.options()), at::empty_symint({p, 2}, f32)};
}

Six policy_meta(const Tensor& logits, const Tensor& offsets, const Tensor& moves, int64_t top) {
  check_policy(logits, offsets, moves, top);
  return policy_outputs(logits, moves, top);
}

Six policy(const Tensor& logits, const Tensor& offsets, const Tensor& moves, int64_t top) {
  const at::Device dev = on_gpu({&logits, &offsets, &moves});
  const c10::DeviceGuard guard(dev);
  check_policy(logits, offsets, moves, top);
  const Runs r(logits, offsets, moves);
  Six res = policy_outputs(logits, moves, top);
  const int64_t p = moves.size(0), n = logits.numel();
  if (p == 0) return res;
  const int64_t bytes = mantis_policy_log_probs_workspace(p, n, int32_t(top));
  const Tensor ws = bytes ? at::empty({bytes}, logits.options().dtype(at::kByte)) : Tensor();
  auto& [log_probs, entropy, lse, top_log, top_moves, norm] = res;
  check_status(mantis_policy_log_probs(r.logits.data_ptr(), dtype_of(logits.scalar_type()), r.stride,
                                       r.offsets.data_ptr<int64_t>(), p, n, r.moves.data_ptr<int64_t>(), moves.size(1),
                                       int32_t(top), log_probs.data_ptr<float>(), entropy.data_ptr<float>(),
                                       lse.data_ptr<float>(), top_log.data_ptr<float>(),
                                       top_moves.data_ptr<int64_t>(), norm.data_ptr<float>(),
                                       bytes ? ws.data_ptr() : nullptr, bytes, error_flag(dev), stream_of(dev)),
               "policy_log_probs");
  return res;
}

struct PolicyGrads {
  optional<Tensor> log_probs, entropy, lse, top;
};

void check_policy_backward(const Tensor& logits, const Tensor& offsets, const Tensor& moves, const Tensor& top_moves,
                           const Tensor& entropy, const Tensor& norm, const PolicyGrads& g) {
  TORCH_CHECK_VALUE(top_moves.dim() == 2 && top_moves.scalar_type() == at::kLong, "top_moves must be the forward's");
  const auto p = top_moves.sym_size(0), k = top_moves.sym_size(1);
  TORCH_CHECK_VALUE(k <= 64, "top_moves must be the forward's");
  check_policy(logits, offsets, moves, 0);
  TORCH_CHECK_VALUE(moves.sym_size(0) == p && entropy.dim() == 1 && entropy.sym_size(0) == p && norm.dim() == 2 &&
                        norm.sym_size(0) == p && norm.sym_size(1) == 2 && entropy.scalar_type() == at::kFloat &&
                        norm.scalar_type() == at::kFloat,
                    "top_moves, entropy and norm must be the forward's");
  const auto check = [](const optional<Tensor>& grad, c10::SymIntArrayRef shape, const char* name) {
    TORCH_CHECK_VALUE(!grad || !grad->defined() || grad->sym_sizes() == shape, "the gradient of ", name,
                      " must have shape ", shape);
  };
  check(g.log_probs, {p, moves.sym_size(1)}, "log_probs");
  check(g.entropy, {p}, "entropy");
  check(g.lse, {p}, "lse");
  check(g.top, {p, k}, "top_log_probs");
}

Tensor policy_backward_meta(const Tensor& logits, const Tensor& offsets, const Tensor& moves, const Tensor& top_moves,
                            const Tensor& entropy, const Tensor& norm, const optional<Tensor>& g_log,
                            const optional<Tensor>& g_ent, const optional<Tensor>& g_lse,
                            const optional<Tensor>& g_top) {
  check_policy_backward(logits, offsets, moves, top_moves, entropy, norm, {g_log, g_ent, g_lse, g_top});
  return at::empty_symint(logits.sym_sizes(), logits.options());
}

Tensor policy_backward(const Tensor& logits, const Tensor& offsets, const Tensor& moves, const Tensor& top_moves_,
                       const Tensor& entropy_, const Tensor& norm_, const optional<Tensor>& g_log,
                       const optional<Tensor>& g_ent, const optional<Tensor>& g_lse, const optional<Tensor>& g_top) {
  PolicyGrads g{g_log, g_ent, g_lse, g_top};
  auto given = [](const optional<Tensor>& t) { return t ? &*t : nullptr; };
  const at::Device dev = on_gpu({&logits, &offsets, &moves, &top_moves_, &entropy_, &norm_, given(g_log), given(g_ent),
                                 given(g_lse), given(g_top)});
  const c10::DeviceGuard guard(dev);
  check_policy_backward(logits, offsets, moves, top_moves_, entropy_, norm_, g);
  for (optional<Tensor>* grad : {&g.log_probs, &g.entropy, &g.lse, &g.top})
    if (*grad && (*grad)->defined()) *grad = as(**grad, at::kFloat).contiguous();
  const Runs r(logits, offsets, moves);
  const int64_t p = moves.size(0), n = logits.numel();
  if (p == 0) return at::zeros({n}, logits.options());
  Tensor out = at::empty({n}, logits.options());
  if (n == 0) return out;
  const Tensor top_moves = top_moves_.contiguous(), entropy = entropy_.contiguous(), norm = norm_.contiguous();
  check_status(mantis_policy_log_probs_backward(
                   r.logits.data_ptr(), dtype_of(logits.scalar_type()), r.stride, r.offsets.data_ptr<int64_t>(), p, n,
                   r.moves.data_ptr<int64_t>(), moves.size(1), int32_t(top_moves.size(1)),
                   top_moves.data_ptr<int64_t>(), entropy.data_ptr<float>(), norm.data_ptr<float>(), ptr(g.log_probs),
                   ptr(g.entropy), ptr(g.lse), ptr(g.top), out.data_ptr(), error_flag(dev), stream_of(dev)),
               "policy_log_probs_backward");
  return out;
}

// ------------------------------------------------------------- dropout

void check_dropout(const Tensor& x, const optional<Tensor>& residual, const Tensor& rng, double p, int64_t salt) {
  dtype_of(x.scalar_type());
  if (residual) {
    dtype_of(residual->scalar_type());
    TORCH_CHECK_VALUE(residual->sym_sizes() == x.sym_sizes(), "x and residual must have one shape");
  }
  TORCH_CHECK_VALUE(rng.dim() == 1 && rng.sym_size(0) == 2 && rng.scalar_type() == at::kLong,
                    "rng must hold two int64, (seed, step)");
  TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, "the dropout probability must lie in [0, 1], got ", p);
  TORCH_CHECK_VALUE(salt >= 0 && salt <= 0xFFFFFFFFLL, "salt must lie in [0, 2^32), got ", salt);
}

Tensor dropout_meta(const Tensor& x, const optional<Tensor>& residual, const Tensor& rng, double p, int64_t salt) {
  check_dropout(x, residual, rng, p, salt);
  return at::empty_symint(x.sym_sizes(), (residual ? *residual : x).options());
}

Tensor dropout_into(const Tensor& x_, const optional<Tensor>& residual_, const Tensor& rng_, double p, int64_t salt,
                    at::ScalarType dtype) {
  const at::Device dev = on_gpu({&x_, residual_ ? &*residual_ : nullptr, &rng_});
  check_dropout(x_, residual_, rng_, p, salt);
  const int32_t out_dtype = dtype_of(dtype);
  const c10::DeviceGuard guard(dev);
  Tensor out = at::empty(x_.sizes(), x_.options().dtype(dtype));
  if (out.numel() == 0) return out;
  const Tensor x = x_.contiguous(), rng = rng_.contiguous();
  const optional<Tensor> residual = residual_ ? optional<Tensor>(residual_->contiguous()) : std::nullopt;
  check_status(mantis_residual_dropout(x.data_ptr(), dtype_of(x.scalar_type()), ptr<void>(residual),
                                       rng.data_ptr<int64_t>(), x.numel(), p, salt, out.data_ptr(), out_dtype,
                                       stream_of(dev)),
               "residual_dropout");
  return out;
}

Tensor dropout(const Tensor& x, const optional<Tensor>& residual, const Tensor& rng, double p, int64_t salt) {
  return dropout_into(x, residual, rng, p, salt, (residual ? *residual : x).scalar_type());
}

Tensor dropout_backward_meta(const Tensor& grad_out, const Tensor& rng, double p, int64_t salt, at::ScalarType dtype) {
  check_dropout(grad_out, std::nullopt, rng, p, salt);
  dtype_of(dtype);
  return at::empty_symint(grad_out.sym_sizes(), grad_out.options().dtype(dtype));
}

Tensor dropout_backward(const Tensor& grad_out, const Tensor& rng, double p, int64_t salt, at::ScalarType dtype) {
  return dropout_into(grad_out, std::nullopt, rng, p, salt, dtype);
}

// ------------------------------------------------------------- gradients

// the operators through the dispatcher, so that tracing and other modes see them
#define MANTIS_OPERATOR(name, function)                                                                       \
  auto call_##name() {                                                                                        \
    static const auto op =                                                                                    \
        c10::Dispatcher::singleton().findSchemaOrThrow("mantisnet::" #name, "").typed<decltype(function)>();   \
    return op;                                                                                                \
  }
MANTIS_OPERATOR(fused_attention_relative, relative)
MANTIS_OPERATOR(fused_attention_relative_backward, relative_backward)
MANTIS_OPERATOR(policy_log_probs, policy)
MANTIS_OPERATOR(policy_log_probs_backward, policy_backward)
MANTIS_OPERATOR(residual_dropout, dropout)
MANTIS_OPERATOR(residual_dropout_backward, dropout_backward)
#undef MANTIS_OPERATOR

// In a backward without create_graph the operators' Autograd keys have nothing to do.
struct BelowAutograd {
  optional<at::AutoDispatchBelowADInplaceOrView> below;
  BelowAutograd() {
    if (!at::GradMode::is_enabled()) below.emplace();
  }
};

struct RelativeAttention : torch::autograd::Function<RelativeAttention> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                               const Tensor& bias, const Tensor& coords, const Tensor& buckets,
                               const Tensor& seq_lens, int64_t n_latents) {
    const at::AutoDispatchBelowADInplaceOrView below;
    auto [out, lse, stats] = call_fused_attention_relative().call(q, k, v, bias, coords, buckets, seq_lens, n_latents);
    ctx->save_for_backward({q, k, v, bias, coords, buckets, seq_lens, stats});
    ctx->saved_data["n_latents"] = n_latents;
    ctx->mark_non_differentiable({lse, stats});
    ctx->set_materialize_grads(false);
    return {out, lse, stats};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list res(8);
    if (!grads[0].defined()) return res;
    const BelowAutograd below;
    const auto s = ctx->get_saved_variables();
    std::tie(res[0], res[1], res[2], res[3]) = call_fused_attention_relative_backward().call(
        s[0], s[1], s[2], s[3], s[4], s[5], s[6], ctx->saved_data["n_latents"].toInt(), s[7], grads[0]);
    return res;
  }
};

Three relative_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& bias, const Tensor& coords,
                        const Tensor& buckets, const Tensor& seq_lens, int64_t n_latents) {
  if (!wants_grad({&q, &k, &v, &bias})) {
    const at::AutoDispatchBelowADInplaceOrView below;
    return call_fused_attention_relative().call(q, k, v, bias, coords, buckets, seq_lens, n_latents);
  }
  const variable_list r = RelativeAttention::apply(q, k, v, bias, coords, buckets, seq_lens, n_latents);
  return {r[0], r[1], r[2]};
}

struct PolicyLogProbs : torch::autograd::Function<PolicyLogProbs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& offsets, const Tensor& moves,
                               int64_t top) {
    const at::AutoDispatchBelowADInplaceOrView below;
    auto [log_probs, entropy, lse, top_log, top_moves, norm] = call_policy_log_probs().call(logits, offsets, moves, top);
    ctx->save_for_backward({logits, offsets, moves, top_moves, entropy, norm});
    ctx->mark_non_differentiable({top_moves, norm});
    ctx->set_materialize_grads(false);
    return {log_probs, entropy, lse, top_log, top_moves, norm};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list res(4);
    auto given = [](const Tensor& t) { return t.defined() ? optional<Tensor>(t) : std::nullopt; };
    const BelowAutograd below;
    const auto s = ctx->get_saved_variables();
    res[0] = call_policy_log_probs_backward().call(s[0], s[1], s[2], s[3], s[4], s[5], given(grads[0]),
                                                   given(grads[1]), given(grads[2]), given(grads[3]));
    return res;
  }
};

Six policy_autograd(const Tensor& logits, const Tensor& offsets, const Tensor& moves, int64_t top) {
  if (!wants_grad({&logits})) {
    const at::AutoDispatchBelowADInplaceOrView below;
    return call_policy_log_probs().call(logits, offsets, moves, top);
  }
  const variable_list r = PolicyLogProbs::apply(logits, offsets, moves, top);
  return {r[0], r[1], r[2], r[3], r[4], r[5]};
}

struct ResidualDropout : torch::autograd::Function<ResidualDropout> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& residual, const Tensor& rng,
                        double p, int64_t salt) {
    const at::AutoDispatchBelowADInplaceOrView below;
    Tensor out = call_residual_dropout().call(x, residual, rng, p, salt);
    ctx->save_for_backward({rng});  // (a step counted on before the backward is an error there)
    ctx->saved_data["p"] = p;
    ctx->saved_data["salt"] = salt;
    ctx->saved_data["dtype"] = int64_t(x.scalar_type());
    ctx->saved_data["residual"] = residual.has_value();
    ctx->set_materialize_grads(false);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list res(5);
    if (!grads[0].defined()) return res;
    const BelowAutograd below;
    if (ctx->needs_input_grad(0))
      res[0] = call_residual_dropout_backward().call(grads[0], ctx->get_saved_variables()[0],
                                                     ctx->saved_data["p"].toDouble(), ctx->saved_data["salt"].toInt(),
                                                     at::ScalarType(ctx->saved_data["dtype"].toInt()));
    if (ctx->saved_data["residual"].toBool()) res[1] = grads[0];
    return res;
  }
};

Tensor dropout_autograd(const Tensor& x, const optional<Tensor>& residual, const Tensor& rng, double p, int64_t salt) {
  if (!wants_grad({&x, residual ? &*residual : nullptr})) {
    const at::AutoDispatchBelowADInplaceOrView below;
    return call_residual_dropout().call(x, residual, rng, p, salt);
  }
  return ResidualDropout::apply(x, residual, rng, p, salt);
}

}  // namespace

// (the operators' schemas are defined in mantisnet/library.py)
TORCH_LIBRARY_FRAGMENT(mantisnet, m) {
  m.def("error_words(int device, bool make) -> Tensor?", error_words);
}

namespace {
void kernels(torch::Library& m) {  // (a CPU tensor reaches them too, and is refused)
  m.impl("fused_attention_relative", relative);
  m.impl("fused_attention_relative_backward", relative_backward);
  m.impl("policy_log_probs", policy);
  m.impl("policy_log_probs_backward", policy_backward);
  m.impl("residual_dropout", dropout);
  m.impl("residual_dropout_backward", dropout_backward);
}
}  // namespace

TORCH_LIBRARY_IMPL(mantisnet, CUDA, m) { kernels(m); }
TORCH_LIBRARY_IMPL(mantisnet, CPU, m) { kernels(m); }

TORCH_LIBRARY_IMPL(mantisnet, Meta, m) {
  m.impl("fused_attention_relative", relative_meta);
  m.impl("fused_attention_relative_backward", relative_backward_meta);
  m.impl("policy_log_probs", policy_meta);
  m.impl("policy_log_probs_backward", policy_backward_meta);
  m.impl("residual_dropout", dropout_meta);
  m.impl("residual_dropout_backward", dropout_backward_meta);
}

// the backwards have no gradients of their own: asking for one is an error
TORCH_LIBRARY_IMPL(mantisnet, Autograd, m) {
  m.impl("fused_attention_relative", relative_autograd);
  m.impl("policy_log_probs", policy_autograd);
  m.impl("residual_dropout", dropout_autograd);
  m.impl("fused_attention_relative_backward", torch::autograd::autogradNotImplementedFallback());
  m.impl("policy_log_probs_backward", torch::autograd::autogradNotImplementedFallback());
  m.impl("residual_dropout_backward", torch::autograd::autogradNotImplementedFallback());
}
