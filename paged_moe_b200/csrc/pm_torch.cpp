// pm_torch.cpp -- the thin PyTorch extension over the C ABI of
// libpm_sample.so (include/pm_sample.h).
//
// The Python layer resolves the sampler / processor settings once (a cached
// device array of pm_row_params) and hands tensors to these functions; they
// pack the C structs, allocate the outputs on the logits' device, call the C
// ABI on the current CUDA stream and raise on a bad status.  No arithmetic
// happens here: every kernel is in libpm_sample.so.
#include <ATen/cuda/CUDAContext.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <optional>
#include <string>
#include <vector>

#include "../../include/pm_sample.h"

namespace {

using OptT = std::optional<torch::Tensor>;

const void* ptr(const OptT& t) { return t.has_value() ? t->data_ptr() : nullptr; }

void check(int rc, const char* what) {
  if (rc == PM_OK) return;
  std::string msg = std::string(what) + ": ";
  switch (rc) {
    case PM_ERR_ARG: msg += "invalid argument"; break;
    case PM_ERR_CUDA: msg += "CUDA error " + std::to_string(pm_last_cuda_error()); break;
    case PM_ERR_UNSUPPORTED: msg += "outside this build's limits"; break;
    case PM_ERR_WORKSPACE: msg += "workspace too small"; break;
    default: msg += "status " + std::to_string(rc);
  }
  if (rc == PM_ERR_ARG) throw std::invalid_argument(msg);
  throw std::runtime_error(msg);
}

int dtype_code(const torch::Tensor& t) {
  if (t.scalar_type() == torch::kFloat32) return PM_DTYPE_F32;
  if (t.scalar_type() == torch::kBFloat16) return PM_DTYPE_BF16;
  throw std::invalid_argument("logits must be float32 or bfloat16");
}

// The rows struct over prepared tensors (contiguous, on the device, except
// logits / mask, which may be pinned host memory for the masked pass).
pm_rows make_rows(const torch::Tensor& logits, const torch::Tensor& params, bool per_row, int64_t flags_any,
                  int64_t top_k_max, const OptT& hist, const OptT& hist_len, const OptT& feed, int64_t feed_group,
                  const OptT& bias_tok, const OptT& bias_val, const OptT& mask, const OptT& forced) {
  if (logits.dim() != 2 || logits.stride(1) != 1) throw std::invalid_argument("logits must be [rows, vocab], unit stride");
  pm_rows r;
  std::memset(&r, 0, sizeof(r));
  r.logits = logits.data_ptr();
  r.dtype = dtype_code(logits);
  r.rows = logits.size(0);
  r.vocab = logits.size(1);
  r.row_stride = logits.stride(0);
  r.params = reinterpret_cast<const pm_row_params*>(params.data_ptr());
  r.params_per_row = per_row ? 1 : 0;
  r.flags_any = (uint32_t)flags_any;
  r.top_k_max = (int32_t)top_k_max;
  if (hist.has_value()) {
    r.hist = reinterpret_cast<const int32_t*>(hist->data_ptr());
    r.hist_stride = hist->size(1);
    r.hist_len = reinterpret_cast<const int32_t*>(ptr(hist_len));
  }
  if (feed.has_value()) {
    r.feed = reinterpret_cast<const int32_t*>(feed->data_ptr());
    r.feed_group = (int32_t)feed_group;
  }
  if (bias_tok.has_value()) {
    r.bias_tokens = reinterpret_cast<const int32_t*>(bias_tok->data_ptr());
    r.bias_values = reinterpret_cast<const float*>(ptr(bias_val));
    r.n_bias = (int32_t)bias_tok->numel();
  }
  if (mask.has_value()) {
    r.mask = reinterpret_cast<const uint32_t*>(mask->data_ptr());
    r.mask_stride = mask->size(1);
  }
  r.forced = reinterpret_cast<const int32_t*>(ptr(forced));
  return r;
}

pm_noise make_noise(int64_t seed, int64_t offset, int64_t row_base, const OptT& gumbel, const OptT& uniform) {
  pm_noise n;
  std::memset(&n, 0, sizeof(n));
  n.mode = (gumbel.has_value() || uniform.has_value()) ? PM_NOISE_INJECTED : PM_NOISE_PHILOX;
  n.seed = (uint64_t)seed;
  n.offset = (uint64_t)offset;
  n.row_base = (uint32_t)row_base;
  if (gumbel.has_value()) {
    n.gumbel = reinterpret_cast<const float*>(gumbel->data_ptr());
    n.gumbel_stride = gumbel->size(1);
  }
  n.uniform = reinterpret_cast<const double*>(ptr(uniform));
  return n;
}

void* stream_of(const torch::Device& dev) {
  return reinterpret_cast<void*>(at::cuda::getCurrentCUDAStream(dev.index()).stream());
}

// pm_sample_rows: [tokens, lse?, logprob?, surv_ids?, surv_probs?, n_surv?]
// (absent outputs are empty tensors; all are views of one allocation).
std::vector<torch::Tensor> sample_rows(torch::Tensor logits, torch::Tensor params, bool per_row, int64_t flags_any,
                                       int64_t top_k_max, OptT hist, OptT hist_len, OptT bias_tok, OptT bias_val,
                                       OptT mask, OptT forced, int64_t seed, int64_t offset, int64_t row_base,
                                       OptT gumbel, OptT uniform, bool want_lse, bool want_logprob,
                                       int64_t survivors, torch::Tensor workspace) {
  const torch::Device dev = params.device();
  const c10::cuda::CUDAGuard guard(dev);
  pm_rows r = make_rows(logits, params, per_row, flags_any, top_k_max, hist, hist_len, std::nullopt, 0, bias_tok,
                        bias_val, mask, forced);
  pm_noise nz = make_noise(seed, offset, row_base, gumbel, uniform);
  const int64_t B = r.rows;
  const int64_t S = survivors > 0 ? survivors : 0;
  // every output in one device allocation (32-bit words), handed out as views
  const int64_t words = B + (want_lse ? B : 0) + (want_logprob ? B : 0) + (S ? 2 * B * S + B : 0);
  torch::Tensor buf = torch::empty({words}, torch::TensorOptions().dtype(torch::kInt32).device(dev));
  torch::Tensor none = buf.narrow(0, 0, 0);
  int64_t at = 0;
  auto take = [&](int64_t n) {
    torch::Tensor t = buf.narrow(0, at, n);
    at += n;
    return t;
  };
  std::vector<torch::Tensor> res(6, none);
  pm_sample_out out;
  std::memset(&out, 0, sizeof(out));
  res[0] = take(B);
  out.tokens = res[0].data_ptr<int32_t>();
  if (want_lse) {
    res[1] = take(B).view(torch::kFloat32);
    out.lse = res[1].data_ptr<float>();
  }
  if (want_logprob) {
    res[2] = take(B).view(torch::kFloat32);
    out.token_logprob = res[2].data_ptr<float>();
  }
  if (S) {
    res[3] = take(B * S).view({B, S});
    res[4] = take(B * S).view(torch::kFloat32).view({B, S});
    res[5] = take(B);
    out.surv_ids = res[3].data_ptr<int32_t>();
    out.surv_probs = res[4].data_ptr<float>();
    out.n_surv = res[5].data_ptr<int32_t>();
    out.surv_cap = (int32_t)S;
  }
  check(pm_sample_rows(&r, &nz, &out, workspace.data_ptr(), (size_t)workspace.numel(), stream_of(dev)),
        "pm_sample_rows");
  return res;
}

// Workspace bytes pm_sample_rows needs for these rows (0: unsupported).
int64_t sample_workspace_bytes(torch::Tensor logits, torch::Tensor params, bool per_row, int64_t flags_any,
                               int64_t top_k_max, OptT hist, OptT mask) {
  pm_rows r = make_rows(logits, params, per_row, flags_any, top_k_max, hist, std::nullopt, std::nullopt, 0,
                        std::nullopt, std::nullopt, mask, std::nullopt);
  return (int64_t)pm_sample_workspace_bytes(&r);
}

// pm_verify: [tokens [B, k+1], n_accepted [B], row_tokens [B, k+1] or empty]
std::vector<torch::Tensor> verify(torch::Tensor logits, torch::Tensor params, bool per_row, int64_t flags_any,
                                  int64_t top_k_max, OptT hist, OptT hist_len, OptT feed, int64_t feed_group,
                                  OptT bias_tok, OptT bias_val, OptT mask, int64_t seed, int64_t offset,
                                  int64_t row_base, OptT gumbel, OptT uniform, int64_t mode, torch::Tensor drafts,
                                  OptT draft_logits, OptT u_accept, OptT u_residual, bool want_row_tokens,
                                  torch::Tensor workspace_cache) {
  const torch::Device dev = params.device();
  const c10::cuda::CUDAGuard guard(dev);
  pm_rows r = make_rows(logits, params, per_row, flags_any, top_k_max, hist, hist_len, feed, feed_group, bias_tok,
                        bias_val, mask, std::nullopt);
  pm_noise nz = make_noise(seed, offset, row_base, gumbel, uniform);
  const int64_t B = drafts.size(0), k = drafts.size(1);
  // every output in one device allocation, handed out as views
  const int64_t K1 = k + 1;
  torch::Tensor buf = torch::empty({B * K1 + B + (want_row_tokens ? B * K1 : 0)},
                                   torch::TensorOptions().dtype(torch::kInt32).device(dev));
  std::vector<torch::Tensor> res(3);
  res[0] = buf.narrow(0, 0, B * K1).view({B, K1});
  res[1] = buf.narrow(0, B * K1, B);
  res[2] = want_row_tokens ? buf.narrow(0, B * K1 + B, B * K1).view({B, K1}) : buf.narrow(0, 0, 0);
  pm_verify_args va;
  std::memset(&va, 0, sizeof(va));
  va.mode = (int32_t)mode;
  va.drafts = reinterpret_cast<const int32_t*>(drafts.data_ptr());
  va.n_draft = (int32_t)k;
  if (draft_logits.has_value()) {
    va.draft_logits = draft_logits->data_ptr();
    va.draft_dtype = dtype_code(*draft_logits);
    va.draft_row_stride = draft_logits->stride(0);
  }
  va.u_accept = reinterpret_cast<const double*>(ptr(u_accept));
  va.u_residual = reinterpret_cast<const double*>(ptr(u_residual));
  va.tokens = res[0].data_ptr<int32_t>();
  va.n_accepted = res[1].data_ptr<int32_t>();
  if (want_row_tokens) va.row_tokens = res[2].data_ptr<int32_t>();
  const size_t need = pm_verify_workspace_bytes(&r, &va);
  if (need == 0) check(PM_ERR_UNSUPPORTED, "pm_verify_workspace_bytes");
  if ((size_t)workspace_cache.numel() < need) check(PM_ERR_WORKSPACE, "pm_verify");
  check(pm_verify(&r, &nz, &va, workspace_cache.data_ptr(), (size_t)workspace_cache.numel(), stream_of(dev)),
        "pm_verify");
  return res;
}

int64_t verify_workspace_bytes(torch::Tensor logits, torch::Tensor params, bool per_row, int64_t flags_any,
                               int64_t top_k_max, OptT hist, OptT feed, int64_t feed_group, OptT mask, int64_t mode,
                               torch::Tensor drafts) {
  pm_rows r = make_rows(logits, params, per_row, flags_any, top_k_max, hist, std::nullopt, feed, feed_group,
                        std::nullopt, std::nullopt, mask, std::nullopt);
  pm_verify_args va;
  std::memset(&va, 0, sizeof(va));
  va.mode = (int32_t)mode;
  va.n_draft = (int32_t)drafts.size(1);
  return (int64_t)pm_verify_workspace_bytes(&r, &va);
}

// ---------------------------------------------------------------------------
// Top log-probabilities and beam search.  Arguments are checked here, before
// any CUDA call: shapes and types first, devices last.
// ---------------------------------------------------------------------------
[[noreturn]] void bad_value(const std::string& what) { throw std::invalid_argument(what); }
[[noreturn]] void bad_type(const std::string& what) { throw pybind11::type_error(what); }

int logits_code(const torch::Tensor& t) {
  if (t.scalar_type() == torch::kFloat32) return PM_DTYPE_F32;
  if (t.scalar_type() == torch::kBFloat16) return PM_DTYPE_BF16;
  bad_type("logits must be float32 or bfloat16, got " + std::string(torch::toString(t.scalar_type())));
}

// [rows, vocab] with unit stride: the tensor itself where it lies so.
torch::Tensor as_rows(const torch::Tensor& t) {
  if (t.dim() < 2) bad_value("logits must have at least two dimensions, the vocabulary last");
  torch::Tensor r = t;
  const int64_t V = t.size(-1);
  if (V < 1) bad_value("the vocabulary is empty");
  if (t.dim() > 2) {
    int64_t rows = 1;
    for (int64_t d = 0; d + 1 < t.dim(); ++d) rows *= t.size(d);
    r = t.reshape({rows, V});
  }
  // a single row's stride says nothing: one that is below V would be refused
  if ((V > 1 && r.stride(1) != 1) || (r.size(0) > 1 && r.stride(0) < V)) r = r.contiguous();
  return r;
}

int64_t row_stride(const torch::Tensor& rows) {
  return rows.size(0) > 1 ? rows.stride(0) : std::max(rows.stride(0), rows.size(1));
}

void on_device(const torch::Tensor& t, const torch::Device& dev, const char* name) {
  if (t.device() != dev) bad_value(std::string(name) + " must be on " + dev.str() + ", got " + t.device().str());
}

void need_cuda(const torch::Tensor& t, const char* name) {
  if (!t.is_cuda()) bad_value(std::string(name) + " must be a CUDA tensor");
}

// Whether a forward-mode derivative (a dual tensor's tangent) rides on t.
bool has_tangent(const torch::Tensor& t) {
  return c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(/*level=*/0).defined();
}

// A temperature whose inverse the kernels' fp32 exponents can hold.
void check_temp(double temp) {
  if (!(temp > 0.0) || std::isinf(temp)) bad_value("temp must be positive");
  if (temp < 4.3e-39 || temp > 2e45) bad_value("temp must lie within [4.3e-39, 2e45]");
}

// The allowed-token words of `rows` rows: contiguous [rows, words], or [words]
// for every row (stride 0).
struct Mask {
  torch::Tensor t;
  const uint32_t* words = nullptr;
  int64_t stride = 0;
};
Mask check_mask(const OptT& mask, int64_t rows, int64_t V) {
  Mask m;
  if (!mask.has_value()) return m;
  if (mask->scalar_type() != torch::kInt32 && mask->scalar_type() != torch::kUInt32)
    bad_type("mask must be packed 32-bit words (int32 or uint32)");
  if (mask->dim() < 1 || mask->size(-1) < (V + 31) / 32) bad_value("mask has fewer than ceil(vocab/32) words per row");
  m.t = mask->contiguous();
  if (m.t.dim() > 1) {
    m.stride = m.t.size(-1);
    if (m.t.numel() != rows * m.stride) bad_value("mask must be [words] or one row of words per row of logits");
  }
  m.words = reinterpret_cast<const uint32_t*>(m.t.data_ptr());
  return m;
}

// Bytes [at, ...) of a call's own output buffer as a tensor, without the time of
// the dispatched narrow() and view().
torch::Tensor piece(const torch::Tensor& buf, int64_t at, torch::ScalarType type, torch::IntArrayRef sizes) {
  torch::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buf.storage()), buf.key_set(),
                                                             c10::scalarTypeToTypeMeta(type));
  t.unsafeGetTensorImpl()->set_storage_offset(at / (int64_t)c10::elementSize(type));
  t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
  return t;
}

// pm_top_logprobs: [ids [N, k], logprobs [N, k], lse [N] or empty]
std::vector<torch::Tensor> top_logprobs(torch::Tensor logits, int64_t k, double temp, OptT mask, bool want_lse) {
  pm_top_rows t;
  std::memset(&t, 0, sizeof(t));
  t.dtype = logits_code(logits);
  if (logits.dim() != 2) bad_value("logits must be [rows, vocab]");
  if (k < 1) bad_value("k must be at least 1");
  check_temp(temp);
  torch::Tensor x = as_rows(logits);
  const Mask m = check_mask(mask, x.size(0), x.size(1));
  need_cuda(x, "logits");
  if (m.words) on_device(m.t, x.device(), "mask");
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t N = x.size(0);
  t.logits = x.data_ptr();
  t.rows = N;
  t.vocab = x.size(1);
  t.row_stride = row_stride(x);
  t.mask = m.words;
  t.mask_stride = m.stride;
  t.k = (int32_t)std::min<int64_t>(k, 0x7fffffff);
  t.inv_temperature = 1.0 / temp;
  if (k > 256) check(PM_ERR_UNSUPPORTED, "pm_top_logprobs");  // before any allocation
  torch::Tensor buf = torch::empty({N * (2 * k + (want_lse ? 1 : 0))}, x.options().dtype(torch::kInt32));
  torch::Tensor ids = piece(buf, 0, torch::kInt32, {N, k});
  torch::Tensor lp = piece(buf, 4 * N * k, torch::kFloat32, {N, k});
  torch::Tensor lse = piece(buf, 8 * N * k, torch::kFloat32, {want_lse ? N : 0});
  check(pm_top_logprobs(&t, ids.data_ptr<int32_t>(), lp.data_ptr<float>(), want_lse ? lse.data_ptr<float>() : nullptr,
                        stream_of(x.device())),
        "pm_top_logprobs");
  return {ids, lp, lse};
}

// pm_beam_select: [scores, parents, tokens, lengths or empty, done or empty]
std::vector<torch::Tensor> beam_select(torch::Tensor logits, torch::Tensor scores, int64_t n, OptT mask, OptT done,
                                       int64_t eos, OptT lengths, double length_penalty, bool keep_slots) {
  pm_beam b;
  std::memset(&b, 0, sizeof(b));
  b.dtype = logits_code(logits);
  if (scores.dim() != 2) bad_value("scores must be [items, beams]");
  if (scores.scalar_type() != torch::kFloat32) bad_type("scores must be float32");
  const int64_t B = scores.size(0), W = scores.size(1);
  if (W < 1) bad_value("there must be at least one beam");
  torch::Tensor x = as_rows(logits);
  if (x.size(0) != B * W || (logits.dim() == 3 && logits.size(0) != B) || logits.dim() > 3)
    bad_value("logits must be [items, beams, vocab] or [items * beams, vocab]");
  const int64_t V = x.size(1);
  if (n < 1) bad_value("n must be at least 1");
  if (keep_slots && n != W) bad_value("keep_slots needs n equal to the number of beams");
  if (eos < -1 || eos > 0x7fffffff) bad_value("eos must be a token id");
  if (!(std::fabs(length_penalty) <= 16.0)) bad_value("length_penalty must lie within [-16, 16]");
  if (length_penalty != 0.0 && !lengths.has_value()) bad_value("length_penalty needs lengths");
  if (done.has_value()) {
    if (eos < 0) bad_value("done needs eos, the token that finished beams go on with");
    if (done->scalar_type() != torch::kBool && done->scalar_type() != torch::kUInt8) bad_type("done must be bool");
    if (done->dim() != 2 || done->size(0) != B || done->size(1) != W) bad_value("done must be [items, beams]");
    done = done->contiguous();
  }
  if (lengths.has_value()) {
    if (lengths->scalar_type() != torch::kInt32) bad_type("lengths must be int32");
    if (lengths->dim() != 2 || lengths->size(0) != B || lengths->size(1) != W)
      bad_value("lengths must be [items, beams]");
    lengths = lengths->contiguous();
  }
  const Mask m = check_mask(mask, B * W, V);
  need_cuda(x, "logits");
  scores = scores.contiguous();
  on_device(scores, x.device(), "scores");
  if (m.words) on_device(m.t, x.device(), "mask");
  if (done.has_value()) on_device(*done, x.device(), "done");
  if (lengths.has_value()) on_device(*lengths, x.device(), "lengths");
  const c10::cuda::CUDAGuard guard(x.device());
  b.logits = x.data_ptr();
  b.items = B;
  b.beams = (int32_t)std::min<int64_t>(W, 0x7fffffff);
  b.vocab = V;
  b.row_stride = row_stride(x);
  b.mask = m.words;
  b.mask_stride = m.stride;
  b.scores = scores.data_ptr<float>();
  b.done = reinterpret_cast<const uint8_t*>(ptr(done));
  b.lengths = reinterpret_cast<const int32_t*>(ptr(lengths));
  b.eos = (int32_t)eos;
  b.length_penalty = length_penalty;
  b.n = (int32_t)std::min<int64_t>(n, 0x7fffffff);
  b.keep_slots = keep_slots ? 1 : 0;
  const size_t need = pm_beam_select_workspace_bytes(&b);
  if (need == 0) check(PM_ERR_UNSUPPORTED, "pm_beam_select");
  // workspace and outputs are allocated per call: two captured graphs, or
  // two streams, never share them
  torch::Tensor ws = torch::empty({(int64_t)need}, x.options().dtype(torch::kUInt8));
  const int64_t E = B * n;
  torch::Tensor buf = torch::empty({E * 3 + (lengths.has_value() ? E : 0) + (eos >= 0 ? (E + 3) / 4 : 0)},
                                   x.options().dtype(torch::kInt32));
  std::vector<torch::Tensor> res(5);
  int64_t at = 0;
  auto take = [&](torch::ScalarType type) {
    torch::Tensor t = piece(buf, at, type, {B, n});
    at += E * 4;
    return t;
  };
  pm_beam_out o;
  std::memset(&o, 0, sizeof(o));
  res[0] = take(torch::kFloat32);
  res[1] = take(torch::kInt32);
  res[2] = take(torch::kInt32);
  o.scores = res[0].data_ptr<float>();
  o.parents = res[1].data_ptr<int32_t>();
  o.tokens = res[2].data_ptr<int32_t>();
  if (lengths.has_value()) {
    res[3] = take(torch::kInt32);
    o.lengths = res[3].data_ptr<int32_t>();
  }
  if (eos >= 0) {
    res[4] = take(torch::kBool);
    o.done = reinterpret_cast<uint8_t*>(res[4].data_ptr());
  }
  check(pm_beam_select(&b, &o, ws.data_ptr(), need, stream_of(x.device())), "pm_beam_select");
  return res;
}

// One state of beam_reorder as (row, run) geometry.  dim: the dimension of
// positions, or -1.  The dimensions from `dim` on have to be dense; those
// between the rows and it have to collapse into one.  No two rows share memory.
void state_geometry(const torch::Tensor& t, int64_t dim, const std::string& name, int64_t* outer, int64_t* outer_stride,
                    int64_t* run, int64_t* pos) {
  const int64_t size = t.element_size(), D = t.dim();
  for (int64_t d = 0; d < D; ++d)
    if (t.size(d) > 1 && t.stride(d) == 0) bad_value(name + " has rows or elements that share memory (expanded)");
  // dense from the last dimension up to `first`
  int64_t first = D, n = 1;
  while (first > 1 && (t.size(first - 1) == 1 || t.stride(first - 1) == n)) n *= t.size(--first);
  if (dim >= 0 && first > dim) bad_value(name + " must be dense from its position dimension on");
  const int64_t split = dim >= 0 ? dim : first;
  int64_t dense = 1;
  for (int64_t d = split; d < D; ++d) dense *= t.size(d);
  *run = dense * size;
  *pos = dim >= 0 ? (t.size(dim) ? dense / t.size(dim) * size : size) : 0;
  *outer = 1;
  *outer_stride = 0;
  for (int64_t d = split - 1; d >= 1; --d) {
    if (t.size(d) == 1) continue;
    if (*outer == 1) {
      *outer_stride = t.stride(d) * size;
    } else if (t.stride(d) * size != *outer_stride * *outer) {
      bad_value(name + " has dimensions between its rows and its dense part that do not collapse into one");
    }
    *outer *= t.size(d);
  }
  if (*outer == 0) { *outer = 1; *run = 0; }
  // rows and runs behind one another, whichever of them lies closer together
  if (t.numel() == 0) return;
  int64_t near = t.size(0), near_stride = t.stride(0) * size, far = *outer, far_stride = *outer_stride;
  if (near == 1 || (far > 1 && far_stride < near_stride)) {
    std::swap(near, far);
    std::swap(near_stride, far_stride);
  }
  if ((near > 1 && near_stride < *run) || (far > 1 && far_stride < near_stride * (near - 1) + *run))
    bad_value(name + " has rows or elements that share memory (overlapping windows)");
}

// pm_beam_reorder over any number of states, PM_MAX_STATES a launch.
void beam_reorder(std::vector<torch::Tensor> states, torch::Tensor parents,
                  std::optional<std::vector<torch::Tensor>> out, OptT lengths, std::vector<int64_t> dims) {
  if (parents.dim() != 2) bad_value("parents must be [items, beams]");
  if (parents.scalar_type() != torch::kInt32) bad_type("parents must be int32");
  const int64_t B = parents.size(0), W = parents.size(1);
  if (W < 1) bad_value("there must be at least one beam");
  if (out.has_value() && out->size() != states.size()) bad_value("out must hold one tensor per state");
  if (dims.size() != states.size()) bad_value("seq_dim must be one dimension, or one per state");
  if (lengths.has_value()) {
    if (lengths->scalar_type() != torch::kInt32) bad_type("lengths must be int32");
    if (lengths->numel() != B * W || lengths->dim() > 2 || (lengths->dim() == 2 && lengths->size(1) != W))
      bad_value("lengths must be [items, beams] or [items * beams]");
    lengths = lengths->contiguous();
  }
  const bool graded = at::GradMode::is_enabled();
  std::vector<pm_state> s(states.size());
  struct Extent {  // of a tensor that fills it, or of its first byte
    const char *from, *to;
    bool written;
  };
  std::vector<Extent> extents;
  extents.reserve(2 * states.size() + 2);
  auto add_extent = [&](const torch::Tensor& t, const void* at, bool write) {
    const char* from = reinterpret_cast<const char*>(at);
    extents.push_back({from, from + (t.is_non_overlapping_and_dense() ? t.numel() * t.element_size() : 1), write});
  };
  for (size_t i = 0; i < states.size(); ++i) {
    const torch::Tensor& a = states[i];
    const std::string name = "state " + std::to_string(i);
    const torch::Tensor& b = out.has_value() ? (*out)[i] : a;
    if (graded && (a.requires_grad() || b.requires_grad()))
      bad_value(name + " requires a gradient, which the reorder does not carry; call it under torch.no_grad()");
    if (has_tangent(a) || has_tangent(b)) bad_value(name + " has a tangent, which the reorder does not carry");
    if (a.dim() < 1 || a.size(0) != B * W) bad_value(name + " must have items * beams rows");
    int64_t dim = dims[i];
    if (dim >= 0 && !lengths.has_value()) bad_value("seq_dim needs lengths");
    if (dim == 0 || dim >= a.dim()) bad_value(name + ": seq_dim must lie behind the row dimension");
    std::memset(&s[i], 0, sizeof(pm_state));
    state_geometry(a, dim, name, &s[i].outer, &s[i].src_outer_stride, &s[i].run_bytes, &s[i].pos_bytes);
    const int64_t size = a.element_size();
    s[i].src = a.data_ptr();
    s[i].src_row_stride = a.stride(0) * size;
    s[i].dst = b.data_ptr();
    s[i].dst_row_stride = b.stride(0) * size;
    s[i].dst_outer_stride = s[i].src_outer_stride;
    if (out.has_value()) {
      if (b.sizes() != a.sizes() || b.scalar_type() != a.scalar_type())
        bad_value("out of " + name + " must have its shape and type");
      // bytes are moved: a conjugation or a sign that is still to be taken is not
      if (b.is_conj() != a.is_conj() || b.is_neg() != a.is_neg())
        bad_value("out of " + name + " must be conjugated or negated lazily where it is");
      int64_t outer, run, pos;
      state_geometry(b, dim, "out of " + name, &outer, &s[i].dst_outer_stride, &run, &pos);
      if (run != s[i].run_bytes || outer != s[i].outer) {
        // one of the two is dense where the other has several runs: its runs
        // follow one another
        const bool shorter = run < s[i].run_bytes;
        if ((shorter ? s[i].outer : outer) != 1) bad_value("out of " + name + " must be laid out like it");
        s[i].run_bytes = std::min(run, s[i].run_bytes);
        s[i].outer = std::max(outer, s[i].outer);
        (shorter ? s[i].src_outer_stride : s[i].dst_outer_stride) = s[i].run_bytes;
      }
    }
    if (a.numel() == 0) { s[i].run_bytes = 0; continue; }
    add_extent(a, s[i].src, !out.has_value());
    if (out.has_value()) add_extent(b, s[i].dst, true);
  }
  // parents and lengths are read while states are written
  if (parents.numel()) add_extent(parents, parents.data_ptr(), false);
  if (lengths.has_value() && lengths->numel()) add_extent(*lengths, lengths->data_ptr(), false);
  // the same memory twice would be moved twice, or read after it was written
  std::sort(extents.begin(), extents.end(), [](const Extent& a, const Extent& b) { return a.from < b.from; });
  const char *end = nullptr, *written_end = nullptr;  // of those that begin before
  for (const Extent& e : extents) {
    if (e.from < (e.written ? end : written_end))
      bad_value(out.has_value() ? "out shares its memory with a state or another out, or overlaps it"
                                : "two states (or a state and parents or lengths) share their memory or overlap");
    end = std::max(end, e.to);
    if (e.written) written_end = std::max(written_end, e.to);
  }
  need_cuda(parents, "parents");
  const torch::Device dev = parents.device();
  if (lengths.has_value()) on_device(*lengths, dev, "lengths");
  for (size_t i = 0; i < states.size(); ++i) {
    on_device(states[i], dev, "states");
    if (out.has_value()) on_device((*out)[i], dev, "out");
  }
  if ((W > 1 && parents.stride(1) != 1) || (B > 1 && parents.stride(0) < W)) parents = parents.contiguous();
  const c10::cuda::CUDAGuard guard(dev);
  for (size_t i = 0; i < s.size(); i += PM_MAX_STATES)
    check(pm_beam_reorder(s.data() + i, (int32_t)std::min<size_t>(PM_MAX_STATES, s.size() - i),
                          parents.data_ptr<int32_t>(), B > 1 ? parents.stride(0) : W,
                          reinterpret_cast<const int32_t*>(ptr(lengths)), B, (int32_t)std::min<int64_t>(W, 0x7fffffff),
                          stream_of(dev)),
          "pm_beam_reorder");
  for (const torch::Tensor& t : out.has_value() ? *out : states)  // as an operation in place does
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// pm_distill_loss over logits [..., V] viewed as rows: [loss or empty, grad or
// empty].  The gradient is [N, V], dense where the logits are.
std::vector<torch::Tensor> distill(torch::Tensor logits, torch::Tensor ids, torch::Tensor logprobs, double temp,
                                   int64_t tail, OptT weights, int64_t reduction, bool want_loss, bool want_grad,
                                   OptT grad_loss) {
  pm_distill d;
  std::memset(&d, 0, sizeof(d));
  d.dtype = logits_code(logits);
  check_temp(temp);
  torch::Tensor x = as_rows(logits.detach());
  const int64_t N = x.size(0), V = x.size(1);
  if (ids.dim() < 1 || ids.size(-1) < 1 || ids.numel() != N * ids.size(-1))
    bad_value("teacher_ids must be [rows, k], one row per row of logits");
  const int64_t K = ids.size(-1);
  if (logprobs.sizes() != ids.sizes()) bad_value("teacher_logprobs must have the shape of teacher_ids");
  if (ids.scalar_type() != torch::kInt32 && ids.scalar_type() != torch::kInt64) bad_type("teacher_ids must be int32 or int64");
  if (logprobs.scalar_type() != torch::kFloat32 && logprobs.scalar_type() != torch::kBFloat16)
    bad_type("teacher_logprobs must be float32 or bfloat16");
  if (weights.has_value()) {
    if (weights->scalar_type() != torch::kFloat32) bad_type("weights must be float32");
    if (weights->numel() != N) bad_value("weights must hold one value per row");
  }
  if (grad_loss.has_value()) {
    if (grad_loss->numel() != (reduction == PM_REDUCE_NONE ? N : 1)) bad_value("the loss's gradient has another size");
  }
  need_cuda(x, "logits");
  const torch::Device dev = x.device();
  on_device(ids, dev, "teacher_ids");
  on_device(logprobs, dev, "teacher_logprobs");
  if (weights.has_value()) on_device(*weights, dev, "weights");
  if (grad_loss.has_value()) on_device(*grad_loss, dev, "the loss's gradient");
  const c10::cuda::CUDAGuard guard(dev);
  if (ids.scalar_type() == torch::kInt64)  // ids past 32 bits are no entries either
    ids = torch::where((ids >= 0).logical_and(ids < V), ids, torch::full({}, -1, ids.options())).to(torch::kInt32);
  ids = ids.contiguous();
  logprobs = logprobs.detach().to(torch::kFloat32).contiguous();
  if (weights.has_value()) weights = weights->detach().contiguous();
  if (grad_loss.has_value()) grad_loss = grad_loss->detach().to(torch::kFloat32).contiguous();
  d.logits = x.data_ptr();
  d.rows = N;
  d.vocab = V;
  d.row_stride = row_stride(x);
  d.ids = ids.data_ptr<int32_t>();
  d.logprobs = logprobs.data_ptr<float>();
  d.k = (int32_t)std::min<int64_t>(K, 0x7fffffff);
  d.inv_temperature = 1.0 / temp;
  d.tail = (int32_t)tail;
  d.reduction = (int32_t)reduction;
  d.weights = reinterpret_cast<const float*>(ptr(weights));
  const size_t need = pm_distill_workspace_bytes(&d);
  if (need == 0) check(PM_ERR_UNSUPPORTED, "pm_distill_loss");
  torch::Tensor ws = torch::empty({(int64_t)need}, x.options().dtype(torch::kUInt8));
  torch::Tensor loss, grad;
  if (want_loss)
    loss = torch::empty(reduction == PM_REDUCE_NONE ? std::vector<int64_t>{N} : std::vector<int64_t>{},
                        x.options().dtype(torch::kFloat32));
  if (want_grad) {
    // rows as far from a 16-byte boundary as the logits', so that the kernel
    // reads and writes whole vectors; dense where the logits are
    const int64_t unit = 16 / x.element_size();
    const int64_t first = (int64_t)(reinterpret_cast<uintptr_t>(x.data_ptr()) % 16) / x.element_size();
    const int64_t step = N > 1 ? V + ((x.stride(0) - V) % unit + unit) % unit : V;
    if (first == 0 && step == V)
      grad = torch::empty({N, V}, x.options());
    else
      grad = torch::empty({first + N * step}, x.options()).as_strided({N, V}, {step, 1}, first);
  }
  check(pm_distill_loss(&d, want_loss ? loss.data_ptr<float>() : nullptr, want_grad ? grad.data_ptr() : nullptr,
                        want_grad && N > 1 ? grad.stride(0) : V,
                        reinterpret_cast<const float*>(ptr(grad_loss)), ws.data_ptr(), need, stream_of(dev)),
        "pm_distill_loss");
  return {loss, grad};
}

// grad [N, V] *= factor (one value on the device), in place.
void distill_scale(torch::Tensor grad, torch::Tensor factor) {
  const c10::cuda::CUDAGuard guard(grad.device());
  factor = factor.detach().to(torch::kFloat32).contiguous();
  check(pm_distill_scale(grad.data_ptr(), logits_code(grad), grad.size(0), grad.size(1), row_stride(grad),
                         factor.data_ptr<float>(), stream_of(grad.device())),
        "pm_distill_scale");
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// A gradient that cannot be differentiated once more says so when it is.
variable_list once(torch::Tensor grad, const torch::Tensor& grad_loss, size_t inputs) {
  if (at::GradMode::is_enabled() && grad_loss.requires_grad())
    grad = (*std::make_shared<torch::autograd::DelayedError>(
        "distill_loss has no second derivative", 1))({grad.detach().requires_grad_()})[0];
  variable_list grads(inputs);
  grads[0] = std::move(grad);
  return grads;
}

// Sum and mean: the loss and its gradient in one pass over the logits, in the
// forward; the backward multiplies by the loss's own gradient, in place, and
// hands the buffer on.
struct DistillWithGrad : torch::autograd::Function<DistillWithGrad> {
  static torch::Tensor forward(AutogradContext* ctx, const torch::Tensor& logits, const torch::Tensor& ids,
                               const torch::Tensor& logprobs, double temp, int64_t tail, const OptT& weights,
                               int64_t reduction) {
    std::vector<torch::Tensor> r = distill(logits, ids, logprobs, temp, tail, weights, reduction, true, true, OptT());
    ctx->saved_data["grad"] = r[1];
    ctx->saved_data["shape"] = logits.sizes();
    return r[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto it = ctx->saved_data.find("grad");
    TORCH_CHECK(it != ctx->saved_data.end(),
                "distill_loss keeps its gradient for one backward pass; call it again for another");
    torch::Tensor grad = it->second.toTensor();
    ctx->saved_data.erase(it);
    {
      const at::NoGradGuard off;
      distill_scale(grad, grads[0]);
      grad = grad.view(ctx->saved_data["shape"].toIntVector());
    }
    return once(std::move(grad), grads[0], 7);
  }
};

// No reduction: the gradient waits for the rows' own, so the backward reads
// the logits again.
struct DistillPerRow : torch::autograd::Function<DistillPerRow> {
  static torch::Tensor forward(AutogradContext* ctx, const torch::Tensor& logits, const torch::Tensor& ids,
                               const torch::Tensor& logprobs, double temp, int64_t tail, const OptT& weights,
                               int64_t reduction) {
    torch::Tensor loss = distill(logits, ids, logprobs, temp, tail, weights, reduction, true, false, OptT())[0];
    ctx->save_for_backward({logits, ids, logprobs, weights.has_value() ? *weights : torch::Tensor()});
    ctx->saved_data["temp"] = temp;
    ctx->saved_data["tail"] = tail;
    ctx->saved_data["reduction"] = reduction;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    torch::Tensor grad;
    {
      const at::NoGradGuard off;
      grad = distill(saved[0], saved[1], saved[2], ctx->saved_data["temp"].toDouble(),
                     ctx->saved_data["tail"].toInt(), saved[3].defined() ? OptT(saved[3]) : OptT(),
                     ctx->saved_data["reduction"].toInt(), false, true, OptT(grads[0]))[1];
      grad = grad.view(saved[0].sizes());
    }
    return once(std::move(grad), grads[0], 7);
  }
};

// The loss of logits [..., V]: one value, or one per row [N] without a reduction.
torch::Tensor distill_loss(torch::Tensor logits, torch::Tensor ids, torch::Tensor logprobs, double temp, int64_t tail,
                           OptT weights, int64_t reduction) {
  // its loss would come back without a tangent, as if it did not depend on the logits
  if (has_tangent(logits)) bad_value("distill_loss has no forward-mode derivative; its gradient comes from backward");
  if (at::GradMode::is_enabled() && logits.requires_grad()) {
    if (reduction == PM_REDUCE_NONE)
      return DistillPerRow::apply(logits, ids, logprobs, temp, tail, weights, reduction);
    return DistillWithGrad::apply(logits, ids, logprobs, temp, tail, weights, reduction);
  }
  return distill(logits, ids, logprobs, temp, tail, weights, reduction, true, false, OptT())[0];
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "PyTorch binding of libpm_sample.so (C ABI: include/pm_sample.h)";
  m.def("sample_rows", &sample_rows);
  m.def("sample_workspace_bytes", &sample_workspace_bytes);
  m.def("verify", &verify);
  m.def("verify_workspace_bytes", &verify_workspace_bytes);
  m.def("top_logprobs", &top_logprobs);
  m.def("beam_select", &beam_select);
  m.def("beam_reorder", &beam_reorder);
  m.def("distill_loss", &distill_loss);
  m.def("version", [] { return std::string(pm_version()); });
}
