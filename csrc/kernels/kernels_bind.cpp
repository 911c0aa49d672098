// Bindings of the SIMT / warp-MMA kernels.  Tensors are validated here; the
// current CUDA stream is used; every launch failure raises.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/ops/as_strided_native.h>
#include <c10/cuda/CUDAGuard.h>

#include "kernels_api.h"

namespace k = tn5b::kernels;

namespace {
cudaStream_t cur() { return at::cuda::getCurrentCUDAStream().stream(); }
void ok(int r, const char* what) {
  TORCH_CHECK(r == 0, what, " failed: ", r < 0 ? "bad arguments" : cudaGetErrorString(cudaError_t(r)));
}
void need(const at::Tensor& t, at::ScalarType dt, const char* name, bool contiguous = true) {
  TORCH_CHECK(t.is_cuda(), name, " must be on CUDA");
  TORCH_CHECK(t.scalar_type() == dt, name, " has the wrong dtype");
  if (contiguous) TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}
const void* opt_ptr(const c10::optional<at::Tensor>& t) { return t ? t->data_ptr() : nullptr; }

void taco_encode(const at::Tensor& in, at::Tensor& packet) {
  need(in, at::kBFloat16, "input"); need(packet, at::kByte, "packet");
  TORCH_CHECK(packet.numel() == in.numel() / 128 * 136, "packet size must be elements/128*136");
  const c10::cuda::CUDAGuard g(in.device());
  ok(k::taco_encode(in.data_ptr(), packet.data_ptr(), in.numel(), cur()), "taco_encode");
}
void taco_decode(const at::Tensor& packet, at::Tensor& out) {
  need(out, at::kBFloat16, "out"); need(packet, at::kByte, "packet");
  TORCH_CHECK(packet.numel() == out.numel() / 128 * 136, "packet size must be elements/128*136");
  const c10::cuda::CUDAGuard g(out.device());
  ok(k::taco_decode(packet.data_ptr(), out.data_ptr(), out.numel(), cur()), "taco_decode");
}
void taco_decode_reduce(const at::Tensor& local, const at::Tensor& packets, at::Tensor& out, int64_t rank,
                        int64_t world) {
  need(local, at::kBFloat16, "local"); need(packets, at::kByte, "packets"); need(out, at::kBFloat16, "out");
  TORCH_CHECK(packets.numel() == (world - 1) * (local.numel() / 128 * 136), "packets size");
  const c10::cuda::CUDAGuard g(out.device());
  ok(k::taco_decode_reduce(local.data_ptr(), packets.data_ptr(), out.data_ptr(), local.numel(), int(rank),
                           int(world), cur()), "taco_decode_reduce");
}
void ordered_reduce(const at::Tensor& local, const at::Tensor& remote, at::Tensor& out, int64_t rank,
                    int64_t world) {
  need(local, at::kBFloat16, "local"); need(remote, at::kBFloat16, "remote"); need(out, at::kBFloat16, "out");
  TORCH_CHECK(remote.numel() == (world - 1) * local.numel(), "remote size");
  const c10::cuda::CUDAGuard g(out.device());
  ok(k::ordered_reduce(local.data_ptr(), remote.data_ptr(), out.data_ptr(), local.numel(), int(rank),
                       int(world), cur()), "ordered_reduce");
}
void diagnostic_delay(int64_t cycles) { ok(k::diagnostic_delay(uint64_t(cycles), cur()), "diagnostic_delay"); }

void layernorm_fwd(const at::Tensor& x, const at::Tensor& w, const at::Tensor& b, at::Tensor& y,
                   at::Tensor& mean, at::Tensor& rstd, double eps) {
  need(x, at::kBFloat16, "x", false); need(y, at::kBFloat16, "y", false);
  need(w, at::kBFloat16, "w"); need(b, at::kBFloat16, "b");
  need(mean, at::kFloat, "mean"); need(rstd, at::kFloat, "rstd");
  TORCH_CHECK(x.dim() == 2 && x.stride(1) == 1 && y.stride(1) == 1);
  const c10::cuda::CUDAGuard g(x.device());
  ok(k::layernorm_fwd(x.data_ptr(), w.data_ptr(), b.data_ptr(), y.data_ptr(), mean.data_ptr<float>(),
                      rstd.data_ptr<float>(), int(x.size(0)), int(x.size(1)), x.stride(0), y.stride(0),
                      float(eps), cur()), "layernorm_fwd");
}
int64_t layernorm_bwd_workspace(int64_t rows, int64_t H) { return 2 * int64_t(k::layernorm_bwd_parts(int(rows))) * H; }
void layernorm_bwd(const at::Tensor& dy, const at::Tensor& x, const at::Tensor& w, const at::Tensor& mean,
                   const at::Tensor& rstd, at::Tensor& dx, at::Tensor& dw, at::Tensor& db,
                   at::Tensor& workspace, const c10::optional<at::Tensor>& dres) {
  need(dy, at::kBFloat16, "dy"); need(x, at::kBFloat16, "x"); need(dx, at::kBFloat16, "dx");
  need(workspace, at::kFloat, "workspace");
  TORCH_CHECK(workspace.numel() >= layernorm_bwd_workspace(x.size(0), x.size(1)), "workspace too small");
  const c10::cuda::CUDAGuard g(x.device());
  ok(k::layernorm_bwd(dy.data_ptr(), x.data_ptr(), w.data_ptr(), mean.data_ptr<float>(),
                      rstd.data_ptr<float>(), dx.data_ptr(), dw.data_ptr(), db.data_ptr(),
                      workspace.data_ptr<float>(), int(x.size(0)), int(x.size(1)), opt_ptr(dres), cur()),
     "layernorm_bwd");
}
void column_sum(const at::Tensor& gm, at::Tensor& out, at::Tensor& workspace) {
  need(gm, at::kBFloat16, "g", false); need(out, at::kBFloat16, "out"); need(workspace, at::kFloat, "ws");
  TORCH_CHECK(gm.dim() == 2 && gm.stride(1) == 1);
  TORCH_CHECK(workspace.numel() >= int64_t(k::layernorm_bwd_parts(int(gm.size(0)))) * gm.size(1));
  const c10::cuda::CUDAGuard g(gm.device());
  ok(k::column_sum(gm.data_ptr(), gm.stride(0), int(gm.size(0)), int(gm.size(1)), out.data_ptr(),
                   workspace.data_ptr<float>(), cur()), "column_sum");
}
void gelu_bwd(const at::Tensor& dy, const at::Tensor& pre, at::Tensor& dx) {
  need(dy, at::kBFloat16, "dy"); need(pre, at::kBFloat16, "pre"); need(dx, at::kBFloat16, "dx");
  const c10::cuda::CUDAGuard g(dy.device());
  ok(k::gelu_bwd(dy.data_ptr(), pre.data_ptr(), dx.data_ptr(), dy.numel(), cur()), "gelu_bwd");
}

void ce_stats(const at::Tensor& logits, const at::Tensor& targets, int64_t start, at::Tensor& rowmax,
              at::Tensor& selected) {
  need(logits, at::kBFloat16, "logits", false); need(targets, at::kLong, "targets");
  const c10::cuda::CUDAGuard g(logits.device());
  ok(k::ce_stats(logits.data_ptr(), logits.stride(0), int(logits.size(0)), int(logits.size(1)),
                 targets.data_ptr<int64_t>(), start, rowmax.data_ptr<float>(), selected.data_ptr<float>(),
                 cur()), "ce_stats");
}
void ce_sumexp(const at::Tensor& logits, const at::Tensor& gmax, at::Tensor& sumexp) {
  const c10::cuda::CUDAGuard g(logits.device());
  ok(k::ce_sumexp(logits.data_ptr(), logits.stride(0), int(logits.size(0)), int(logits.size(1)),
                  gmax.data_ptr<float>(), sumexp.data_ptr<float>(), cur()), "ce_sumexp");
}
void ce_loss(const at::Tensor& gmax, const at::Tensor& sumexp, const at::Tensor& selected,
             const c10::optional<at::Tensor>& row_loss, at::Tensor& mean_loss, double scale) {
  const c10::cuda::CUDAGuard g(gmax.device());
  ok(k::ce_loss(gmax.data_ptr<float>(), sumexp.data_ptr<float>(), selected.data_ptr<float>(),
                int(gmax.numel()), row_loss ? row_loss->data_ptr<float>() : nullptr,
                mean_loss.data_ptr<float>(), float(scale), cur()), "ce_loss");
}
void ce_bwd(at::Tensor& logits, const at::Tensor& targets, int64_t start, const at::Tensor& gmax,
            const at::Tensor& sumexp, double scale, const c10::optional<at::Tensor>& scale_t) {
  need(logits, at::kBFloat16, "logits", false);
  const c10::cuda::CUDAGuard g(logits.device());
  ok(k::ce_bwd(logits.data_ptr(), logits.stride(0), int(logits.size(0)), int(logits.size(1)),
               targets.data_ptr<int64_t>(), start, gmax.data_ptr<float>(), sumexp.data_ptr<float>(),
               float(scale), scale_t ? scale_t->data_ptr<float>() : nullptr, cur()), "ce_bwd");
}

int64_t grad_sqsum_parts(int64_t n) { return k::grad_sqsum_parts(n); }
void grad_sqsum(const at::Tensor& grad, at::Tensor& partial, at::Tensor& out, bool accumulate) {
  TORCH_CHECK(grad.is_cuda() && grad.is_contiguous());
  need(partial, at::kDouble, "partial"); need(out, at::kDouble, "out");
  TORCH_CHECK(partial.numel() >= k::grad_sqsum_parts(grad.numel()), "partial workspace too small");
  const bool fp32 = grad.scalar_type() == at::kFloat;
  TORCH_CHECK(fp32 || grad.scalar_type() == at::kBFloat16);
  const c10::cuda::CUDAGuard g(grad.device());
  ok(k::grad_sqsum(grad.data_ptr(), fp32, grad.numel(), partial.data_ptr<double>(), out.data_ptr<double>(),
                   accumulate, cur()), "grad_sqsum");
}
void adamw_step(at::Tensor& master, at::Tensor& m, at::Tensor& v, const at::Tensor& grad, at::Tensor& param,
                int64_t n_decay, const at::Tensor& norm2, double max_norm, double lr, double wd, double beta1,
                double beta2, double eps, int64_t step, const at::Tensor& status) {
  need(master, at::kFloat, "master"); need(m, at::kFloat, "m"); need(v, at::kFloat, "v");
  need(param, at::kBFloat16, "param"); need(norm2, at::kDouble, "norm2");
  const bool fp32 = grad.scalar_type() == at::kFloat;
  TORCH_CHECK(grad.numel() == master.numel() && param.numel() == master.numel() && m.numel() == master.numel());
  const c10::cuda::CUDAGuard g(master.device());
  ok(k::adamw_step(master.data_ptr<float>(), m.data_ptr<float>(), v.data_ptr<float>(), grad.data_ptr(), fp32,
                   param.data_ptr(), master.numel(), n_decay, norm2.data_ptr<double>(), float(max_norm),
                   float(lr), float(wd), float(beta1), float(beta2), float(eps), int(step),
                   status.data_ptr<int>(), cur()), "adamw_step");
}

void embed_fwd(const at::Tensor& tok, const at::Tensor& E, at::Tensor& out, int64_t start) {
  need(tok, at::kLong, "tokens"); need(E, at::kBFloat16, "E"); need(out, at::kBFloat16, "out");
  const c10::cuda::CUDAGuard g(E.device());
  ok(k::embed_fwd(tok.data_ptr<int64_t>(), E.data_ptr(), out.data_ptr(), int(tok.numel()), int(E.size(1)),
                  start, E.size(0), cur()), "embed_fwd");
}
void add_position(at::Tensor& x, const at::Tensor& P, int64_t row0) {
  need(x, at::kBFloat16, "x"); need(P, at::kBFloat16, "P");
  const c10::cuda::CUDAGuard g(x.device());
  ok(k::add_position(x.data_ptr(), P.data_ptr(), int(x.size(0)), int(x.size(1)), row0, int(P.size(0)), cur()),
     "add_position");
}
void position_bwd(const at::Tensor& gr, at::Tensor& dP, int64_t row0) {
  need(gr, at::kBFloat16, "g"); need(dP, at::kBFloat16, "dP");
  const c10::cuda::CUDAGuard g(gr.device());
  ok(k::position_bwd(gr.data_ptr(), dP.data_ptr(), int(gr.size(0)), int(gr.size(1)), row0, int(dP.size(0)),
                     cur()), "position_bwd");
}
int64_t embed_bwd_workspace(int64_t M, int64_t V) { return k::embed_bwd_workspace_ints(int(M), V); }
void embed_bwd(const at::Tensor& tok, const at::Tensor& gr, at::Tensor& dE, int64_t start, at::Tensor& ws,
               bool accumulate) {
  need(tok, at::kLong, "tokens"); need(gr, at::kBFloat16, "g"); need(dE, at::kBFloat16, "dE");
  need(ws, at::kInt, "workspace");
  TORCH_CHECK(ws.numel() >= k::embed_bwd_workspace_ints(int(tok.numel()), dE.size(0)));
  const c10::cuda::CUDAGuard g(gr.device());
  ok(k::embed_bwd(tok.data_ptr<int64_t>(), gr.data_ptr(), dE.data_ptr(), int(tok.numel()), int(dE.size(1)),
                  start, dE.size(0), ws.data_ptr<int>(), accumulate, cur()), "embed_bwd");
}

void attention_fwd_tc(const at::Tensor& qkv, at::Tensor& out, at::Tensor& lse, int64_t B, int64_t S, int64_t H,
                      double scale, const at::Tensor& status, int64_t timeout_ns, int64_t trace) {
  need(qkv, at::kBFloat16, "qkv", false); need(out, at::kBFloat16, "out", false); need(lse, at::kFloat, "lse");
  TORCH_CHECK(qkv.stride(1) == 1 && out.stride(1) == 1);
  TORCH_CHECK(qkv.size(0) == B * S && qkv.size(1) == 3 * H * 128 && out.size(1) == H * 128);
  const c10::cuda::CUDAGuard g(qkv.device());
  ok(k::attention_fwd_tc(qkv.data_ptr(), qkv.stride(0), out.data_ptr(), out.stride(0), lse.data_ptr<float>(),
                         int(B), int(S), int(H), float(scale), status.data_ptr<int>(), uint64_t(timeout_ns), cur(),
                         reinterpret_cast<unsigned long long*>(trace)),
     "attention_fwd_tc");
}
// Optional [2, CTAs, 8] int64 cycle counters of the backward kernels (dK/dV, dQ).
unsigned long long* dbg_words(const c10::optional<at::Tensor>& dbg, int kernel, int64_t ctas) {
  if (!dbg) return nullptr;
  TORCH_CHECK(dbg->is_cuda() && dbg->scalar_type() == at::kLong && dbg->is_contiguous() &&
                  dbg->numel() == 2 * ctas * 8,
              "attention debug counters must be a contiguous int64 [2, B*H*S/128, 8] CUDA tensor");
  return reinterpret_cast<unsigned long long*>(dbg->data_ptr<int64_t>()) + kernel * ctas * 8;
}
void attention_bwd_tc(const at::Tensor& qkv, const at::Tensor& out, const at::Tensor& dout, const at::Tensor& lse,
                      at::Tensor& Dvec, at::Tensor& dqkv, int64_t B, int64_t S, int64_t H, double scale,
                      const at::Tensor& status, int64_t timeout_ns, const c10::optional<at::Tensor>& dbg) {
  need(qkv, at::kBFloat16, "qkv", false); need(out, at::kBFloat16, "out", false);
  need(dout, at::kBFloat16, "dout", false); need(dqkv, at::kBFloat16, "dqkv", false);
  need(lse, at::kFloat, "lse"); need(Dvec, at::kFloat, "D");
  TORCH_CHECK(qkv.stride(1) == 1 && dout.stride(1) == 1 && dqkv.stride(1) == 1 && out.stride(1) == 1);
  const c10::cuda::CUDAGuard g(qkv.device());
  ok(k::attention_bwd_pre(out.data_ptr(), out.stride(0), dout.data_ptr(), dout.stride(0), Dvec.data_ptr<float>(),
                          int(B), int(S), int(H), cur()), "attention_bwd_pre");
  ok(k::attention_bwd_tc(qkv.data_ptr(), qkv.stride(0), dout.data_ptr(), dout.stride(0), lse.data_ptr<float>(),
                         Dvec.data_ptr<float>(), dqkv.data_ptr(), dqkv.stride(0), int(B), int(S), int(H), float(scale),
                         status.data_ptr<int>(), uint64_t(timeout_ns), cur(), dbg_words(dbg, 0, B * H * (S / 128)),
                         dbg_words(dbg, 1, B * H * (S / 128))),
     "attention_bwd_tc");
}

// Numbers go into messages as text: c10's message stream crashes on integers where
// the extension and libtorch were linked against different C++ runtimes.
std::string shape_text(int64_t rows, int64_t cols) {
  return "[" + std::to_string(rows) + ", " + std::to_string(cols) + "]";
}
// Row kernels: storage type code, and the checks shared by their bindings.
int type_code(const at::Tensor& t, bool half, const char* name) {
  if (t.scalar_type() == at::kBFloat16) return k::kTypeBF16;
  if (t.scalar_type() == at::kFloat) return k::kTypeFP32;
  TORCH_CHECK(half && t.scalar_type() == at::kHalf, name, " has the wrong dtype");
  return k::kTypeFP16;
}
void need_like(const at::Tensor& t, const at::Tensor& like, at::ScalarType dt, const char* name) {
  TORCH_CHECK(t.device() == like.device(), name, " must be on ", like.device());
  TORCH_CHECK(t.scalar_type() == dt, name, " has the wrong dtype");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}
void need_rows(const at::Tensor& t, const at::Tensor& like, int64_t rows, int64_t cols, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name, " must be on ", like.device());
  TORCH_CHECK(t.scalar_type() == like.scalar_type(), name, " has the wrong dtype");
  TORCH_CHECK(t.dim() == 2 && t.size(0) == rows && t.size(1) == cols && (t.stride(1) == 1 || cols == 1), name,
              " must be ", shape_text(rows, cols), " with contiguous rows");
}
void need_vector(const at::Tensor& t, const at::Tensor& like, int64_t n, const char* name) {
  need_like(t, like, like.scalar_type(), name);
  TORCH_CHECK(t.dim() == 1 && t.numel() == n, name, " must hold ", std::to_string(n), " values");
}
void need_floats(const at::Tensor& t, const at::Tensor& like, int64_t n, const char* name) {
  need_like(t, like, at::kFloat, name);
  TORCH_CHECK(t.numel() >= n, name, " must hold ", std::to_string(n), " values");
}

void need_vocabulary(int64_t vocab, int64_t vocab_total, int64_t top_k) {
  TORCH_CHECK(vocab > 0 && vocab_total <= 0x7fffffff, "the vocabulary must have 1 to 2^31 - 1 ids");
  TORCH_CHECK(top_k >= 0 && top_k <= 32 && top_k <= vocab, "top_k is out of range");
}
// Calls without rows are checked like others; there is nothing to launch for them then.
void score_fwd(const at::Tensor& logits, const at::Tensor& targets, int64_t start, int64_t vocab_total, int64_t top_k,
               const c10::optional<at::Tensor>& out, const c10::optional<at::Tensor>& top_ids,
               const c10::optional<at::Tensor>& record) {
  // out: FP32 [5 + top_k rows' worth]: logprob, entropy, state[3], then the alternatives' log probabilities.
  const int type = type_code(logits, true, "logits");
  const int64_t rows = logits.size(0), vocab = logits.size(1);
  need_rows(logits, logits, rows, vocab, "logits");
  need_vocabulary(vocab, vocab_total, top_k);
  need_like(targets, logits, at::kLong, "targets");
  TORCH_CHECK(targets.dim() == 1 && targets.numel() == rows, "targets must hold one id a row");
  float* f = nullptr;
  int64_t* ids = nullptr;
  float* rec = nullptr;
  if (record) {
    need_floats(*record, logits, rows * (4 + 2 * top_k), "record");
    rec = record->data_ptr<float>();
  } else {
    TORCH_CHECK(out && (top_ids || !top_k), "out and top_ids are needed without a record");
    need_floats(*out, logits, rows * (5 + top_k), "out");
    f = out->data_ptr<float>();
    if (top_k) {
      need_like(*top_ids, logits, at::kLong, "top_ids");
      TORCH_CHECK(top_ids->numel() == rows * top_k, "top_ids must hold top_k ids a row");
      ids = top_ids->data_ptr<int64_t>();
    }
  }
  if (!rows) return;
  const c10::cuda::CUDAGuard g(logits.device());
  ok(k::score_fwd(logits.data_ptr(), type, logits.stride(0), rows, vocab, targets.data_ptr<int64_t>(), start,
                  vocab_total, int(top_k), f, f + rows, f + 2 * rows, f + 5 * rows, ids, rec, cur()), "score_fwd");
}
void score_merge(const at::Tensor& records, const at::Tensor& targets, int64_t vocab, int64_t top_k, at::Tensor& out,
                 at::Tensor& top_ids) {
  const int64_t rows = targets.numel(), parts = records.size(0);
  need_like(targets, records, at::kLong, "targets");
  need_floats(records, records, parts * rows * (4 + 2 * top_k), "records");
  need_floats(out, records, rows * (5 + top_k), "out");
  need_like(top_ids, records, at::kLong, "top_ids");
  TORCH_CHECK(records.is_cuda() && top_ids.numel() == rows * top_k, "top_ids must hold top_k ids a row");
  float* f = out.data_ptr<float>();
  const c10::cuda::CUDAGuard g(records.device());
  ok(k::score_merge(records.data_ptr<float>(), int(parts), rows, vocab, targets.data_ptr<int64_t>(), int(top_k), f,
                    f + rows, f + 2 * rows, f + 5 * rows, top_ids.data_ptr<int64_t>(), cur()), "score_merge");
}
void score_bwd(const at::Tensor& logits, const at::Tensor& targets, int64_t start, int64_t vocab_total,
               const at::Tensor& state, const at::Tensor& dlogprob, const c10::optional<at::Tensor>& dentropy,
               at::Tensor& out) {
  const int type = type_code(logits, true, "logits");
  const int64_t rows = logits.size(0), vocab = logits.size(1);
  need_rows(logits, logits, rows, vocab, "logits");
  need_rows(out, logits, rows, vocab, "out");
  need_vocabulary(vocab, vocab_total, 0);
  need_like(targets, logits, at::kLong, "targets");
  TORCH_CHECK(targets.dim() == 1 && targets.numel() == rows, "targets must hold one id a row");
  need_floats(state, logits, 3 * rows, "state");
  need_floats(dlogprob, logits, rows, "dlogprob");
  if (dentropy) need_floats(*dentropy, logits, rows, "dentropy");
  if (!rows) return;
  const c10::cuda::CUDAGuard g(logits.device());
  ok(k::score_bwd(logits.data_ptr(), type, logits.stride(0), rows, vocab, targets.data_ptr<int64_t>(), start,
                  vocab_total, state.data_ptr<float>(), dlogprob.data_ptr<float>(),
                  dentropy ? dentropy->data_ptr<float>() : nullptr, out.data_ptr(), out.stride(0), cur()),
     "score_bwd");
}

void need_packed(const at::Tensor& data, const at::Tensor& like, int64_t rows, int64_t cols, const char* name) {
  TORCH_CHECK(data.is_cuda() && data.device() == like.device(), name, " must be on ", like.device());
  TORCH_CHECK(data.scalar_type() == at::kByte && data.dim() == 2 && data.is_contiguous() && data.size(0) == rows &&
                  data.size(1) == k::act_pack_row_bytes(cols),
              name, " is not the packed form of ", shape_text(rows, cols));
  TORCH_CHECK(reinterpret_cast<uintptr_t>(data.data_ptr()) % 16 == 0, name, " must start on a 16-byte boundary");
}
void act_pack(const at::Tensor& x, at::Tensor& data) {
  const int type = type_code(x, false, "x");
  need_rows(x, x, x.size(0), x.size(1), "x");
  TORCH_CHECK(x.size(1) > 0, "x needs at least one column");
  need_packed(data, x, x.size(0), x.size(1), "data");
  if (!x.size(0)) return;
  const c10::cuda::CUDAGuard g(x.device());
  ok(k::act_pack(x.data_ptr(), type, x.stride(0), data.data_ptr(), x.size(0), x.size(1), cur()), "act_pack");
}
void act_unpack(const at::Tensor& data, at::Tensor& out, const c10::optional<at::Tensor>& act) {
  const int type = type_code(out, false, "out");
  const int64_t rows = out.size(0), cols = out.size(1);
  need_like(out, data, out.scalar_type(), "out");
  need_packed(data, out, rows, cols, "data");
  if (act) {
    need_like(*act, out, out.scalar_type(), "act");
    TORCH_CHECK(act->sizes() == out.sizes(), "act and out differ in shape");
  }
  if (!out.numel()) return;
  const c10::cuda::CUDAGuard g(out.device());
  ok(k::act_unpack(data.data_ptr(), out.data_ptr(), act ? act->data_ptr() : nullptr, type, rows, cols, cur()),
     "act_unpack");
}

void need_width(int64_t cols) {
  TORCH_CHECK(cols > 0 && cols <= k::join_max_cols(), "the hidden size is out of range");
}
void join_fwd(const at::Tensor& x, const at::Tensor& y, const at::Tensor& pw, const at::Tensor& pb,
              const at::Tensor& gate, const at::Tensor& w, const at::Tensor& b, at::Tensor& u, at::Tensor& h,
              at::Tensor& stats, double alpha, double eps) {
  const int type = type_code(x, false, "x");
  const int64_t rows = x.size(0), cols = x.size(1);
  need_rows(x, x, rows, cols, "x"); need_rows(y, x, rows, cols, "y");
  need_rows(h, x, rows, cols, "h"); need_rows(u, x, rows, cols, "x_out");
  TORCH_CHECK(u.is_contiguous(), "x_out must be contiguous");
  need_vector(pw, x, cols, "post_weight"); need_vector(pb, x, cols, "post_bias"); need_vector(gate, x, cols, "gate");
  need_vector(w, x, cols, "pre_weight"); need_vector(b, x, cols, "pre_bias");
  need_floats(stats, x, 4 * rows, "stats");
  need_width(cols);
  if (!rows) return;
  const c10::cuda::CUDAGuard g(x.device());
  ok(k::join_fwd(x.data_ptr(), x.stride(0), y.data_ptr(), y.stride(0), type, pw.data_ptr(), pb.data_ptr(),
                 gate.data_ptr(), w.data_ptr(), b.data_ptr(), u.data_ptr(), h.data_ptr(), h.stride(0),
                 stats.data_ptr<float>(), rows, cols, float(alpha), float(eps), cur()), "block_join_fwd");
}
int64_t join_bwd_workspace(int64_t rows, int64_t cols, bool branch) {
  return k::join_bwd_parts(rows, cols) * (branch ? 4 : 2) * cols;
}
// Gradients of the joint, or of LayerNorm alone where `y` is absent.  `u` and `y` are
// both packed (bytes) or both of dh's type.  grads: dpre_weight, dpre_bias and, with a
// branch, dpost_weight, dpost_bias, dgate, [2 or 5, cols].
struct RowStats {  // FP32 [rows] each; *_y without a branch: null
  const float *mean_u, *rstd_u, *mean_y, *rstd_y;
};
void run_join_bwd(const at::Tensor& dh, const c10::optional<at::Tensor>& du, const at::Tensor& u,
                  const c10::optional<at::Tensor>& y, const RowStats& stats, const c10::optional<at::Tensor>& pw,
                  const c10::optional<at::Tensor>& pb, const c10::optional<at::Tensor>& gate, const at::Tensor& w,
                  const c10::optional<at::Tensor>& b, const at::Tensor& dx, const c10::optional<at::Tensor>& dy,
                  const c10::optional<at::Tensor>& h, const at::Tensor& grads, const at::Tensor& workspace,
                  double alpha) {
  k::JoinBwdCall c = {};
  c.type = type_code(dh, false, "dh");
  const int64_t rows = dh.size(0), cols = dh.size(1);
  c.rows = rows;
  c.cols = cols;
  c.packed = u.scalar_type() == at::kByte;
  c.alpha = float(alpha);
  need_rows(dh, dh, rows, cols, "dh"); need_rows(dx, dh, rows, cols, "dx");
  auto kept = [&](const at::Tensor& t, const char* name) {
    if (c.packed) need_packed(t, dh, rows, cols, name);
    else need_rows(t, dh, rows, cols, name);
  };
  kept(u, "x_out");
  need_vector(w, dh, cols, "pre_weight");
  c.dh = dh.data_ptr(); c.ld_dh = dh.stride(0);
  c.dx = dx.data_ptr(); c.ld_dx = dx.stride(0);
  c.u = u.data_ptr(); c.ld_u = u.stride(0);
  c.mean_u = stats.mean_u; c.rstd_u = stats.rstd_u;
  c.w = w.data_ptr();
  if (du) {
    need_rows(*du, dh, rows, cols, "dx_out");
    c.du = du->data_ptr(); c.ld_du = du->stride(0);
  }
  if (h) {
    TORCH_CHECK(b, "the norm's output needs its bias");
    need_rows(*h, dh, rows, cols, "h");
    TORCH_CHECK(h->is_contiguous(), "h must be contiguous");
    need_vector(*b, dh, cols, "pre_bias");
    c.h = h->data_ptr(); c.b = b->data_ptr();
  }
  const bool branch = y.has_value();
  need_like(grads, dh, dh.scalar_type(), "grads");
  TORCH_CHECK(grads.numel() == (branch ? 5 : 2) * cols, "grads must be ", shape_text(branch ? 5 : 2, cols));
  const int64_t step = cols * grads.element_size();
  char* gp = static_cast<char*>(grads.data_ptr());
  c.dw = gp; c.db = gp + step;
  if (branch) {
    TORCH_CHECK(dy && pw && pb && gate && (!rows || (stats.mean_y && stats.rstd_y)), "the branch's tensors go together");
    kept(*y, "y");
    need_rows(*dy, dh, rows, cols, "dy");
    need_vector(*pw, dh, cols, "post_weight"); need_vector(*pb, dh, cols, "post_bias");
    need_vector(*gate, dh, cols, "gate");
    c.y = y->data_ptr(); c.ld_y = y->stride(0);
    c.dy = dy->data_ptr(); c.ld_dy = dy->stride(0);
    c.mean_y = stats.mean_y; c.rstd_y = stats.rstd_y;
    c.pw = pw->data_ptr(); c.pb = pb->data_ptr(); c.gate = gate->data_ptr();
    c.dpw = gp + 2 * step; c.dpb = gp + 3 * step; c.dgate = gp + 4 * step;
  }
  need_floats(workspace, dh, join_bwd_workspace(rows, cols, branch), "workspace");
  c.workspace = workspace.data_ptr<float>();
  if (!rows) {
    grads.zero_();
    return;
  }
  const c10::cuda::CUDAGuard g(dh.device());
  ok(k::join_bwd(c, cur()), branch ? "block_join_bwd" : "layer_norm_bwd_packed");
}
void join_bwd(const at::Tensor& dh, const c10::optional<at::Tensor>& du, const at::Tensor& u,
              const c10::optional<at::Tensor>& y, const at::Tensor& mean_u, const at::Tensor& rstd_u,
              const c10::optional<at::Tensor>& mean_y, const c10::optional<at::Tensor>& rstd_y,
              const c10::optional<at::Tensor>& pw, const c10::optional<at::Tensor>& pb,
              const c10::optional<at::Tensor>& gate, const at::Tensor& w, const c10::optional<at::Tensor>& b,
              at::Tensor& dx, const c10::optional<at::Tensor>& dy, const c10::optional<at::Tensor>& h,
              at::Tensor& grads, at::Tensor& workspace, double alpha) {
  const int64_t rows = dh.size(0);
  need_floats(mean_u, dh, rows, "mean"); need_floats(rstd_u, dh, rows, "rstd");
  RowStats stats{mean_u.data_ptr<float>(), rstd_u.data_ptr<float>(), nullptr, nullptr};
  if (mean_y && rstd_y) {
    need_floats(*mean_y, dh, rows, "mean_y"); need_floats(*rstd_y, dh, rows, "rstd_y");
    stats.mean_y = mean_y->data_ptr<float>(); stats.rstd_y = rstd_y->data_ptr<float>();
  }
  run_join_bwd(dh, du, u, y, stats, pw, pb, gate, w, b, dx, dy, h, grads, workspace, alpha);
}

// The operators' public forms: outputs are allocated here, so that a call costs one
// crossing from Python.  Arguments are checked by the functions above.
// Outputs and their parts are made without the dispatcher, which would cost more than a
// small kernel: they are plain tensors on `like`'s device.
at::Tensor fresh(const at::Tensor& like, at::IntArrayRef sizes, at::ScalarType type) {
  return at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt);
}
at::Tensor rows_like(const at::Tensor& t) { return fresh(t, {t.size(0), t.size(1)}, t.scalar_type()); }
at::Tensor part(const at::Tensor& t, at::IntArrayRef sizes, int64_t offset) {
  const int64_t inner = sizes.size() == 2 ? std::max<int64_t>(sizes[1], 1) : 1;
  if (sizes.size() == 2) return at::native::as_strided_tensorimpl(t, sizes, {inner, 1}, offset);
  return at::native::as_strided_tensorimpl(t, sizes, {1}, offset);
}
void need_matrix(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.dim() == 2, name, " must be a matrix on CUDA");
}
void need_own_rows(const c10::optional<at::Tensor>& t, const char* name) {
  if (t) TORCH_CHECK(t->dim() == 2 && (t->size(0) < 2 || t->stride(0) >= t->size(1)), name, " needs rows of its own");
}
using Tensors = std::vector<c10::optional<at::Tensor>>;

Tensors token_logprobs(const at::Tensor& logits, const at::Tensor& targets, int64_t top_k) {
  need_matrix(logits, "logits");
  need_vocabulary(logits.size(1), logits.size(1), top_k);
  const int64_t rows = logits.size(0);
  at::Tensor out = fresh(logits, {rows * (5 + top_k)}, at::kFloat);
  at::Tensor ids = fresh(logits, {rows, top_k}, at::kLong);
  score_fwd(logits, targets.contiguous(), 0, logits.size(1), top_k, out, ids, c10::nullopt);
  return {part(out, {rows}, 0), part(out, {rows}, rows), part(out, {rows, top_k}, 5 * rows), ids,
          part(out, {3, rows}, 2 * rows)};
}
at::Tensor token_logprobs_backward(const at::Tensor& logits, const at::Tensor& targets, int64_t start,
                                   int64_t vocab_total, const at::Tensor& state, const at::Tensor& dlogprob,
                                   const c10::optional<at::Tensor>& dentropy, const c10::optional<at::Tensor>& out) {
  need_matrix(logits, "logits");
  need_own_rows(out, "out");
  const int64_t rows = logits.size(0);
  TORCH_CHECK(state.dim() == 2 && state.size(0) == 3 && state.size(1) == rows, "the state belongs to other logits");
  TORCH_CHECK(dlogprob.dim() == 1 && dlogprob.numel() == rows, "dlogprob must hold one value a row");
  TORCH_CHECK(!dentropy || (dentropy->dim() == 1 && dentropy->numel() == rows), "dentropy must hold one value a row");
  at::Tensor to = out ? *out : rows_like(logits);
  c10::optional<at::Tensor> de;
  if (dentropy) de = dentropy->contiguous();
  score_bwd(logits, targets.contiguous(), start, vocab_total, state, dlogprob.contiguous(), de, to);
  return to;
}
at::Tensor pack(const at::Tensor& x) {
  need_matrix(x, "x");
  at::Tensor data = fresh(x, {x.size(0), k::act_pack_row_bytes(x.size(1))}, at::kByte);
  act_pack(x, data);
  return data;
}
Tensors unpack(const at::Tensor& data, int64_t cols, bool fp32, bool gelu) {
  need_matrix(data, "data");
  const at::ScalarType type = fp32 ? at::kFloat : at::kBFloat16;
  at::Tensor out = fresh(data, {data.size(0), cols}, type);
  c10::optional<at::Tensor> act;
  if (gelu) act = fresh(data, {data.size(0), cols}, type);
  act_unpack(data, out, act);
  return {out, act};
}
Tensors block_join_fwd(const at::Tensor& x, const at::Tensor& y, const at::Tensor& pw, const at::Tensor& pb,
                       const at::Tensor& gate, const at::Tensor& w, const at::Tensor& b, double alpha, double eps,
                       const c10::optional<at::Tensor>& out) {
  need_matrix(x, "x");
  need_own_rows(out, "out");
  at::Tensor u = rows_like(x);
  at::Tensor h = out ? *out : rows_like(x);
  at::Tensor stats = fresh(x, {4, x.size(0)}, at::kFloat);
  join_fwd(x, y, pw, pb, gate, w, b, u, h, stats, alpha, eps);
  return {u, h, stats};
}
struct Spare {  // gradients of the parameters, and a workspace that is large enough
  at::Tensor grads, workspace;
  Spare(const at::Tensor& dh, bool branch, const c10::optional<at::Tensor>& given) {
    const int64_t rows = dh.size(0), cols = dh.size(1);
    need_width(cols);
    grads = fresh(dh, {branch ? 5 : 2, cols}, dh.scalar_type());
    const int64_t size = join_bwd_workspace(rows, cols, branch);
    workspace = given && given->numel() >= size ? *given : fresh(dh, {size}, at::kFloat);
  }
};
// (dx, dy, dpost_weight, dpost_bias, dgate, dpre_weight, dpre_bias, h)
Tensors block_join_bwd(const at::Tensor& dh, const c10::optional<at::Tensor>& du, const at::Tensor& u,
                       const at::Tensor& y, const at::Tensor& stats, const at::Tensor& pw, const at::Tensor& pb,
                       const at::Tensor& gate, const at::Tensor& w, const c10::optional<at::Tensor>& b,
                       const c10::optional<at::Tensor>& out, const c10::optional<at::Tensor>& workspace, double alpha) {
  need_matrix(dh, "dh");
  need_own_rows(out, "out");
  const int64_t rows = dh.size(0);
  need_like(stats, dh, at::kFloat, "stats");
  TORCH_CHECK(stats.dim() == 2 && stats.size(0) == 4 && stats.size(1) == rows, "stats must be [4, rows]");
  TORCH_CHECK(u.scalar_type() == y.scalar_type(), "x_out and y are kept in the same form");
  Spare spare(dh, true, workspace);
  at::Tensor dx = rows_like(dh);
  c10::optional<at::Tensor> dy = out ? *out : rows_like(dh), h;
  if (b) h = rows_like(dh);
  const float* s = stats.data_ptr<float>();
  run_join_bwd(dh, du, u, y, RowStats{s + 2 * rows, s + 3 * rows, s, s + rows}, pw, pb, gate, w, b, dx, dy, h,
               spare.grads, spare.workspace, alpha);
  const int64_t cols = dh.size(1);
  auto grad = [&](int i) { return part(spare.grads, {cols}, i * cols); };
  return {dx, dy, grad(2), grad(3), grad(4), grad(0), grad(1), h};
}
// (dx, dweight, dbias, y)
Tensors layer_norm_bwd_packed(const at::Tensor& dy, const c10::optional<at::Tensor>& dres, const at::Tensor& x,
                              const at::Tensor& mean, const at::Tensor& rstd, const at::Tensor& w,
                              const c10::optional<at::Tensor>& b, const c10::optional<at::Tensor>& out,
                              const c10::optional<at::Tensor>& workspace) {
  need_matrix(dy, "dy");
  need_own_rows(out, "out");
  TORCH_CHECK(mean.dim() == 1 && rstd.dim() == 1 && mean.numel() == dy.size(0) && rstd.numel() == dy.size(0),
              "mean and rstd must hold one value a row");
  need_like(mean, dy, at::kFloat, "mean"); need_like(rstd, dy, at::kFloat, "rstd");
  Spare spare(dy, false, workspace);
  at::Tensor dx = out ? *out : rows_like(dy);
  c10::optional<at::Tensor> y, none;
  if (b) y = rows_like(dy);
  run_join_bwd(dy, dres, x, none, RowStats{mean.data_ptr<float>(), rstd.data_ptr<float>(), nullptr, nullptr}, none,
               none, none, w, b, dx, none, y, spare.grads, spare.workspace, 1.0);
  const int64_t cols = dy.size(1);
  return {dx, part(spare.grads, {cols}, 0), part(spare.grads, {cols}, cols), y};
}
}  // namespace

// Launch entry points touch no Python object: the GIL is released while they
// run, so other Python threads (e.g. a stall watchdog) keep running.
using nogil = pybind11::call_guard<pybind11::gil_scoped_release>;

void register_kernels(pybind11::module& m) {
  m.def("taco_encode", &taco_encode, nogil());
  m.def("taco_decode", &taco_decode, nogil());
  m.def("taco_decode_reduce", &taco_decode_reduce, nogil());
  m.def("ordered_reduce", &ordered_reduce, nogil());
  m.def("diagnostic_delay", &diagnostic_delay, nogil());
  m.def("layernorm_fwd", &layernorm_fwd, nogil());
  m.def("layernorm_bwd_workspace", &layernorm_bwd_workspace, nogil());
  m.def("layernorm_bwd", &layernorm_bwd, nogil());
  m.def("column_sum", &column_sum, nogil());
  m.def("gelu_bwd", &gelu_bwd, nogil());
  m.def("ce_stats", &ce_stats, nogil());
  m.def("ce_sumexp", &ce_sumexp, nogil());
  m.def("ce_loss", &ce_loss, nogil());
  m.def("ce_bwd", &ce_bwd, nogil());
  m.def("score_fwd", &score_fwd, nogil());
  m.def("score_merge", &score_merge, nogil());
  m.def("token_logprobs", &token_logprobs, nogil());
  m.def("token_logprobs_backward", &token_logprobs_backward, nogil());
  m.def("pack", &pack, nogil());
  m.def("unpack", &unpack, nogil());
  m.def("block_join_fwd", &block_join_fwd, nogil());
  m.def("block_join_bwd", &block_join_bwd, nogil());
  m.def("layer_norm_bwd_packed", &layer_norm_bwd_packed, nogil());
  m.def("act_pack", &act_pack, nogil());
  m.def("act_unpack", &act_unpack, nogil());
  m.def("join_bwd", &join_bwd, nogil());
  m.def("grad_sqsum_parts", &grad_sqsum_parts, nogil());
  m.def("grad_sqsum", &grad_sqsum, nogil());
  m.def("adamw_step", &adamw_step, nogil());
  m.def("embed_fwd", &embed_fwd, nogil());
  m.def("add_position", &add_position, nogil());
  m.def("position_bwd", &position_bwd, nogil());
  m.def("embed_bwd_workspace", &embed_bwd_workspace, nogil());
  m.def("embed_bwd", &embed_bwd, nogil());
  m.def("attention_fwd_tc", &attention_fwd_tc, pybind11::arg("qkv"), pybind11::arg("out"), pybind11::arg("lse"),
        pybind11::arg("B"), pybind11::arg("S"), pybind11::arg("H"), pybind11::arg("scale"), pybind11::arg("status"),
        pybind11::arg("timeout_ns"), pybind11::arg("trace") = 0, nogil());
  m.def("attention_bwd_tc", &attention_bwd_tc, nogil());
}
