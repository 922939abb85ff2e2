// Python bindings for the MI355X kernel suite (torch extension).
// Thin layer: dtype/contiguity checks, output allocation, stream plumbing.
#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>

#include <hip/hip_runtime.h>

#include <algorithm>

extern "C" {
void lah_batched_gemm_nt(const void*, const void*, void*, const void*, void*, int, int,
                         int, int, int, hipStream_t);
void lah_batched_gemm_tn(const void*, const void*, void*, int, int, int, int, int,
                         hipStream_t);
void lah_batched_gemm_tn_sgd_sr(const void*, const void*, void*, void*, int, int, int,
                                int, float, float, unsigned, hipStream_t);
void lah_flash_attn_fwd(const void*, const void*, const void*, void*, void*, void*, int, int,
                        hipStream_t);
void lah_flash_attn_bwd(const void*, const void*, const void*, const void*, const void*,
                        const void*, void*, void*, void*, void*, void*, void*, int, int,
                        hipStream_t);
void lah_gating_topk_fwd(const void*, void*, void*, void*, int, int, int, hipStream_t);
void lah_gating_topk_bwd(const void*, const void*, const void*, const void*, const void*,
                         void*, int, int, int, hipStream_t);
void lah_assign_slots(const void*, void*, void*, void*, int, int, int, int, hipStream_t);
void lah_dispatch_gather(const void*, const void*, void*, int, int, int, int, hipStream_t);
void lah_dispatch_bwd(const void*, const void*, const void*, void*, int, int, int, int,
                      hipStream_t);
void lah_combine_fwd(const void*, const void*, const void*, const void*, void*, int, int,
                     int, int, float, hipStream_t);
void lah_combine_bwd(const void*, const void*, const void*, const void*, const void*,
                     const void*, void*, void*, int, int, int, int, float, hipStream_t);
void lah_zero_padding(const void*, void*, int, int, int, hipStream_t);
void lah_sgd_step(void*, const void*, void*, void*, long, float, float, float,
                  const void*, hipStream_t);
void lah_sgd_step_t(void*, const void*, void*, void*, int, int, int, float, float,
                    const void*, hipStream_t);
void lah_sgd_step_sr_t(void*, const void*, void*, int, int, int, float, float,
                       unsigned, const void*, hipStream_t);
void lah_transpose_bf16(const void*, void*, int, int, int, hipStream_t);
void lah_ce_rowstats(const void*, const void*, void*, void*, int, long, int, int,
                     hipStream_t);
void lah_ce_bwd(const void*, const void*, const void*, void*, float, int, long, int,
                int, hipStream_t);
void lah_colsum(const void*, void*, int, int, int, hipStream_t);
long lah_ragged_layout_table(long, int);
void lah_ragged_layout(const void*, int, long, int, void*, void*, void*, void*, hipStream_t);
long lah_ragged_tiles_room(long, int);
void lah_ragged_nt(const void*, const void*, void*, const void*, const void*, int, void*,
                   long, int, int, int, int, void*, int, void*, hipStream_t);
void lah_ragged_nn(const void*, const void*, void*, const void*, void*, long, int, int, int,
                   void*, int, void*, hipStream_t);
int lah_ragged_parts(long, int, int, int, bool);
long lah_ragged_tn_work(long, int, int, int);
void lah_ragged_tn(const void*, const void*, void*, void*, int, const void*, long, int, int,
                   int, int, void*, hipStream_t);
long lah_ragged_slope_work(long, int, int);
void lah_ragged_slope(const void*, const void*, void*, void*, int, const void*, long, int, int, void*,
                      hipStream_t);
long lah_clip_partials(int);
void lah_grad_norm(void* const*, const long*, const int*, int, void*, float, float, void*,
                   void*, hipStream_t);
void lah_grad_scale(void* const*, const long*, const int*, int, const void*, hipStream_t);
void lah_master_sgd(void* const*, void* const*, void* const*, void* const*, const long*,
                    const int*, int, const void*, float, float, float, hipStream_t);
}

namespace {

hipStream_t cur_stream() { return at::hip::getCurrentHIPStream().stream(); }

#define CHECK_BF16(t) TORCH_CHECK((t).scalar_type() == at::kBFloat16, #t " must be bf16")
#define CHECK_F32(t) TORCH_CHECK((t).scalar_type() == at::kFloat, #t " must be fp32")
#define CHECK_I32(t) TORCH_CHECK((t).scalar_type() == at::kInt, #t " must be int32")
#define CHECK_CONTIG(t) TORCH_CHECK((t).is_contiguous(), #t " must be contiguous")
#define CHECK_CUDA(t) TORCH_CHECK((t).is_cuda(), #t " must be on GPU")
// Work goes to the tensors' own device, on its current stream.
#define ON_DEVICE_OF(t) const c10::OptionalDeviceGuard device_guard(at::device_of(t))
#define CHECK_LAUNCH()                                                      \
  do {                                                                      \
    const hipError_t err = hipGetLastError();                               \
    TORCH_CHECK(err == hipSuccess, "launch: ", hipGetErrorString(err));     \
  } while (0)

// The kernels have no forward-mode derivative: a tangent would be lost without a word.
bool has_tangent(const torch::Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
#define CHECK_NO_TANGENT(t, name) \
  TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(t), name " has no forward-mode derivative on the GPU")

// contiguous, from a multiple of 16 bytes on: what the kernels load
torch::Tensor ready(const torch::Tensor& t) {
  const auto c = t.contiguous();
  return ((uintptr_t)c.data_ptr() & 15) == 0 ? c : c.clone();
}

// C[e] = A[e] @ B[e]^T with fused epilogue; see ffn_gemm.hip
torch::Tensor batched_gemm_nt(torch::Tensor A, torch::Tensor B,
                              c10::optional<torch::Tensor> bias,
                              c10::optional<torch::Tensor> pre, int64_t epi) {
  CHECK_CUDA(A); CHECK_BF16(A); CHECK_CONTIG(A);
  CHECK_BF16(B); CHECK_CONTIG(B);
  int E = A.size(0), M = A.size(1), K = A.size(2);
  int N = B.size(1);
  TORCH_CHECK(B.size(0) == E && B.size(2) == K, "A/B shape mismatch");
  TORCH_CHECK(N % 128 == 0, "N must be a multiple of 128");
  TORCH_CHECK(K % 64 == 0, "K must be a multiple of 64");
  auto C = torch::empty({E, M, N}, A.options());
  const void* bias_p = nullptr;
  void* pre_p = nullptr;
  if (bias.has_value()) { CHECK_F32(*bias); CHECK_CONTIG(*bias); bias_p = bias->data_ptr(); }
  if (epi == 2) {  // BIAS_GELU stores pre-activation
    TORCH_CHECK(pre.has_value(), "epi=2 requires a pre-activation output tensor");
  }
  if (pre.has_value()) { CHECK_BF16(*pre); CHECK_CONTIG(*pre); pre_p = pre->data_ptr(); }
  lah_batched_gemm_nt(A.data_ptr(), B.data_ptr(), C.data_ptr(), bias_p, pre_p, E, M, N, K,
                      (int)epi, cur_stream());
  return C;
}

// C[e,i,j] (fp32, written in place) = sum_m A[e,m,i] * B[e,m,j]
void batched_gemm_tn(torch::Tensor A, torch::Tensor B, torch::Tensor C,
                     bool accumulate) {
  CHECK_CUDA(A); CHECK_BF16(A); CHECK_CONTIG(A);
  CHECK_BF16(B); CHECK_CONTIG(B); CHECK_F32(C); CHECK_CONTIG(C);
  int E = A.size(0), M = A.size(1), I = A.size(2), J = B.size(2);
  TORCH_CHECK(B.size(0) == E && B.size(1) == M, "A/B shape mismatch");
  TORCH_CHECK(C.size(0) == E && C.size(1) == I && C.size(2) == J, "C shape mismatch");
  TORCH_CHECK(M % 64 == 0, "M must be a multiple of 64");
  TORCH_CHECK(I % 128 == 0 && J % 128 == 0, "I/J must be multiples of 128");
  lah_batched_gemm_tn(A.data_ptr(), B.data_ptr(), C.data_ptr(), E, M, I, J,
                      accumulate ? 1 : 0, cur_stream());
}

// fused dW + stochastic-rounding SGD: W[e] -= lr * (A[e]^T @ B[e] + wd*W[e]),
// SR-rounded in place, with the transposed bf16 copy refreshed in the same
// pass — replaces batched_gemm_tn + sgd_step_sr_t for the single-backward-
// per-step regime (see ffn_gemm_tn.hip)
void fused_dw_sgd_sr(torch::Tensor A, torch::Tensor B, torch::Tensor W,
                     torch::Tensor WT, double lr, double weight_decay,
                     int64_t seed) {
  CHECK_CUDA(A); CHECK_BF16(A); CHECK_CONTIG(A);
  CHECK_BF16(B); CHECK_CONTIG(B);
  CHECK_BF16(W); CHECK_CONTIG(W); CHECK_BF16(WT); CHECK_CONTIG(WT);
  int E = A.size(0), M = A.size(1), I = A.size(2), J = B.size(2);
  TORCH_CHECK(B.size(0) == E && B.size(1) == M, "A/B shape mismatch");
  TORCH_CHECK(W.size(0) == E && W.size(1) == I && W.size(2) == J, "W shape mismatch");
  TORCH_CHECK(WT.size(0) == E && WT.size(1) == J && WT.size(2) == I, "WT shape mismatch");
  TORCH_CHECK(M % 64 == 0, "M must be a multiple of 64");
  TORCH_CHECK(I % 256 == 0 && J % 256 == 0,
              "fused dW+SGD needs I/J multiples of 256 (use the unfused path)");
  lah_batched_gemm_tn_sgd_sr(A.data_ptr(), B.data_ptr(), W.data_ptr(), WT.data_ptr(),
                             E, M, I, J, (float)lr, (float)weight_decay,
                             (unsigned)seed, cur_stream());
}

// chunked lm_head CE row stats: (lse, picked) per row, one logits read
std::vector<torch::Tensor> ce_rowstats(torch::Tensor logits, torch::Tensor labels,
                                       int64_t ignore_index) {
  CHECK_CUDA(logits); CHECK_CONTIG(logits);
  bool bf16 = logits.scalar_type() == at::kBFloat16;
  TORCH_CHECK(bf16 || logits.scalar_type() == at::kFloat, "logits must be bf16 or fp32");
  CHECK_I32(labels); CHECK_CONTIG(labels);
  int T = logits.size(0);
  long V = logits.size(1);
  TORCH_CHECK(labels.size(0) == T, "labels/logits mismatch");
  TORCH_CHECK(V % 4 == 0, "V must be a multiple of 4");
  auto lse = torch::empty({T}, logits.options().dtype(at::kFloat));
  auto picked = torch::empty({T}, logits.options().dtype(at::kFloat));
  lah_ce_rowstats(logits.data_ptr(), labels.data_ptr(), lse.data_ptr(),
                  picked.data_ptr(), T, V, (int)ignore_index, (int)bf16,
                  cur_stream());
  return {lse, picked};
}

torch::Tensor ce_bwd(torch::Tensor logits, torch::Tensor labels, torch::Tensor lse,
                     double gscale, int64_t ignore_index) {
  CHECK_CUDA(logits); CHECK_CONTIG(logits);
  bool bf16 = logits.scalar_type() == at::kBFloat16;
  TORCH_CHECK(bf16 || logits.scalar_type() == at::kFloat, "logits must be bf16 or fp32");
  CHECK_I32(labels); CHECK_CONTIG(labels); CHECK_F32(lse); CHECK_CONTIG(lse);
  int T = logits.size(0);
  long V = logits.size(1);
  TORCH_CHECK(V % 4 == 0, "V must be a multiple of 4");
  auto d = torch::empty({T, V}, logits.options().dtype(at::kBFloat16));
  lah_ce_bwd(logits.data_ptr(), labels.data_ptr(), lse.data_ptr(), d.data_ptr(),
             (float)gscale, T, V, (int)ignore_index, (int)bf16, cur_stream());
  return d;
}

std::vector<torch::Tensor> gating_topk_fwd(torch::Tensor logits, int64_t k) {
  CHECK_CUDA(logits); CHECK_F32(logits); CHECK_CONTIG(logits);
  int T = logits.size(0), E = logits.size(1);
  TORCH_CHECK(E <= 4096, "gating kernel supports up to 4096 experts, got ", E);
  TORCH_CHECK(k == 1 || k == 2 || k == 4 || k == 8,
              "gating kernel supports k in {1,2,4,8}, got ", k);
  ON_DEVICE_OF(logits);
  auto probs = torch::empty({T, E}, logits.options().dtype(at::kBFloat16));
  auto topk_idx = torch::empty({T, k}, logits.options().dtype(at::kInt));
  auto topk_w = torch::empty({T, k}, logits.options());
  lah_gating_topk_fwd(logits.data_ptr(), probs.data_ptr(), topk_idx.data_ptr(),
                      topk_w.data_ptr(), T, E, (int)k, cur_stream());
  CHECK_LAUNCH();
  return {probs, topk_idx, topk_w};
}

torch::Tensor gating_topk_bwd(torch::Tensor probs, torch::Tensor topk_idx,
                              torch::Tensor topk_w, torch::Tensor d_topk_w,
                              c10::optional<torch::Tensor> aux_g) {
  CHECK_BF16(probs); CHECK_I32(topk_idx); CHECK_F32(topk_w); CHECK_F32(d_topk_w);
  int T = probs.size(0), E = probs.size(1), k = topk_idx.size(1);
  TORCH_CHECK(E <= 4096, "gating kernel supports up to 4096 experts, got ", E);
  auto d_logits = torch::empty({T, E}, topk_w.options());
  const void* aux_p = nullptr;
  if (aux_g.has_value()) { CHECK_F32(*aux_g); CHECK_CONTIG(*aux_g); aux_p = aux_g->data_ptr(); }
  lah_gating_topk_bwd(probs.data_ptr(), topk_idx.data_ptr(), topk_w.data_ptr(),
                      d_topk_w.contiguous().data_ptr(), aux_p, d_logits.data_ptr(), T, E, k,
                      cur_stream());
  CHECK_LAUNCH();
  return d_logits;
}

std::vector<torch::Tensor> assign_slots(torch::Tensor topk_idx, int64_t E, int64_t C) {
  CHECK_CUDA(topk_idx); CHECK_I32(topk_idx); CHECK_CONTIG(topk_idx);
  int T = topk_idx.size(0), k = topk_idx.size(1);
  auto pos = torch::empty({T, k}, topk_idx.options());
  auto counts = torch::zeros({E}, topk_idx.options());
  auto inv = torch::full({E, C}, -1, topk_idx.options());
  lah_assign_slots(topk_idx.data_ptr(), pos.data_ptr(), counts.data_ptr(), inv.data_ptr(),
                   T, k, (int)C, (int)E, cur_stream());
  CHECK_LAUNCH();
  return {pos, counts, inv};
}

// dispatch.hip has a wave for each row, and a launch below 2^32 threads
#define CHECK_WAVES(rows) TORCH_CHECK((rows) < (int64_t)1 << 26, "below 2^26 rows, got ", rows)

// What a kernel of dispatch.hip takes rows and slots from: [T, k] int32, on the rows' GPU
static void check_slots(const torch::Tensor& rows, const torch::Tensor& topk_idx, const torch::Tensor& pos) {
  CHECK_CUDA(rows);
  CHECK_I32(topk_idx); CHECK_I32(pos);
  TORCH_CHECK(topk_idx.dim() == 2 && topk_idx.sizes() == pos.sizes(), "topk_idx and pos must be [T, k]");
  CHECK_WAVES(topk_idx.size(0));
  TORCH_CHECK(topk_idx.device() == rows.device() && pos.device() == rows.device(),
              "all tensors must be on one GPU");
}

static void check_buffer(const torch::Tensor& buf) {
  CHECK_BF16(buf);
  TORCH_CHECK(buf.dim() == 3, "the buffer must be [E, C, D]");
  CHECK_WAVES(buf.size(0) * buf.size(1));
  TORCH_CHECK(buf.size(2) % 8 == 0, "D must be a multiple of 8");
}

torch::Tensor dispatch_gather(torch::Tensor x, torch::Tensor inv, int64_t k) {
  CHECK_CUDA(x); CHECK_BF16(x); CHECK_I32(inv);
  TORCH_CHECK(x.dim() == 2 && inv.dim() == 2 && x.device() == inv.device(),
              "x must be [T, D] and inv [E, C], on one GPU");
  int E = inv.size(0), C = inv.size(1), D = x.size(1);
  TORCH_CHECK(D % 8 == 0, "D must be a multiple of 8");
  TORCH_CHECK(k > 0 || inv.numel() == 0, "k must be positive");
  CHECK_WAVES(inv.numel());
  ON_DEVICE_OF(x);
  x = ready(x);
  inv = inv.contiguous();
  auto xbuf = torch::empty({E, C, D}, x.options());
  lah_dispatch_gather(x.data_ptr(), inv.data_ptr(), xbuf.data_ptr(), E, C, D, (int)k,
                      cur_stream());
  CHECK_LAUNCH();
  return xbuf;
}

torch::Tensor dispatch_bwd(torch::Tensor dxbuf, torch::Tensor topk_idx, torch::Tensor pos,
                           int64_t T) {
  check_buffer(dxbuf);
  check_slots(dxbuf, topk_idx, pos);
  TORCH_CHECK(topk_idx.size(0) == T, "topk_idx must be [T, k]");
  int C = dxbuf.size(1), D = dxbuf.size(2), k = topk_idx.size(1);
  ON_DEVICE_OF(dxbuf);
  dxbuf = ready(dxbuf);
  topk_idx = topk_idx.contiguous();
  pos = pos.contiguous();
  auto dx = torch::empty({T, D}, dxbuf.options());
  lah_dispatch_bwd(dxbuf.data_ptr(), topk_idx.data_ptr(), pos.data_ptr(), dx.data_ptr(),
                   (int)T, D, k, C, cur_stream());
  CHECK_LAUNCH();
  return dx;
}

torch::Tensor combine_fwd(torch::Tensor ybuf, torch::Tensor topk_idx, torch::Tensor pos,
                          torch::Tensor w, double least) {
  check_buffer(ybuf);
  check_slots(ybuf, topk_idx, pos);
  CHECK_F32(w);
  TORCH_CHECK(w.sizes() == pos.sizes() && w.device() == ybuf.device(), "w must be [T, k] on the GPU of ybuf");
  int C = ybuf.size(1), D = ybuf.size(2);
  int T = topk_idx.size(0), k = topk_idx.size(1);
  ON_DEVICE_OF(ybuf);
  ybuf = ready(ybuf);
  topk_idx = topk_idx.contiguous();
  pos = pos.contiguous();
  w = w.contiguous();
  auto y = torch::empty({T, D}, ybuf.options());
  lah_combine_fwd(ybuf.data_ptr(), topk_idx.data_ptr(), pos.data_ptr(), w.data_ptr(),
                  y.data_ptr(), T, D, k, C, (float)least, cur_stream());
  CHECK_LAUNCH();
  return y;
}

std::vector<torch::Tensor> combine_bwd(torch::Tensor dy, torch::Tensor ybuf,
                                       torch::Tensor y, torch::Tensor topk_idx,
                                       torch::Tensor pos, torch::Tensor w,
                                       torch::Tensor inv, double least) {
  CHECK_BF16(dy); CHECK_BF16(y); CHECK_F32(w); CHECK_I32(inv);
  check_buffer(ybuf);
  check_slots(ybuf, topk_idx, pos);
  int E = ybuf.size(0), C = ybuf.size(1), D = ybuf.size(2);
  int T = topk_idx.size(0), k = topk_idx.size(1);
  TORCH_CHECK(w.sizes() == pos.sizes() && inv.dim() == 2 && inv.size(0) == E && inv.size(1) == C,
              "w must be [T, k] and inv [E, C]");
  TORCH_CHECK(y.dim() == 2 && y.size(0) == T && y.size(1) == D && dy.sizes() == y.sizes(),
              "dy and y must be [T, D]");
  for (const auto* t : {&dy, &y, &w, &inv})
    TORCH_CHECK(t->device() == ybuf.device(), "all tensors must be on one GPU");
  ON_DEVICE_OF(ybuf);
  dy = ready(dy);
  ybuf = ready(ybuf);
  y = ready(y);
  topk_idx = topk_idx.contiguous();
  pos = pos.contiguous();
  w = w.contiguous();
  inv = inv.contiguous();
  auto dybuf = torch::empty({E, C, D}, ybuf.options());
  auto dw = torch::empty({T, k}, w.options());
  // padding rows (inv < 0) are zero-filled; surviving rows written by scatter
  lah_zero_padding(inv.data_ptr(), dybuf.data_ptr(), E, C, D, cur_stream());
  lah_combine_bwd(dy.data_ptr(), ybuf.data_ptr(), y.data_ptr(),
                  topk_idx.data_ptr(), pos.data_ptr(), w.data_ptr(), dybuf.data_ptr(),
                  dw.data_ptr(), T, D, k, C, (float)least, cur_stream());
  CHECK_LAUNCH();
  return {dybuf, dw};
}

// the clipping factor, one fp32 number on the GPU, or null
const void* scale_ptr(const c10::optional<torch::Tensor>& s, const torch::Tensor& like) {
  if (!s.has_value()) return nullptr;
  CHECK_F32(*s);
  TORCH_CHECK(s->numel() == 1 && s->device() == like.device(),
              "the gradients' scale must be one number on their GPU");
  return s->data_ptr();
}

void sgd_step(torch::Tensor master, torch::Tensor grad, c10::optional<torch::Tensor> momentum,
              torch::Tensor out_bf16, double lr, double mu, double weight_decay,
              c10::optional<torch::Tensor> gscale) {
  CHECK_F32(master); CHECK_F32(grad); CHECK_BF16(out_bf16);
  CHECK_CONTIG(master); CHECK_CONTIG(grad); CHECK_CONTIG(out_bf16);
  long n = master.numel();
  TORCH_CHECK(grad.numel() == n && out_bf16.numel() == n, "size mismatch");
  TORCH_CHECK(n % 4 == 0, "numel must be a multiple of 4");
  void* mom_p = nullptr;
  if (momentum.has_value()) { CHECK_F32(*momentum); mom_p = momentum->data_ptr(); }
  lah_sgd_step(master.data_ptr(), grad.data_ptr(), mom_p, out_bf16.data_ptr(), n, (float)lr,
               (float)mu, (float)weight_decay, scale_ptr(gscale, master), cur_stream());
}

void sgd_step_t(torch::Tensor master, torch::Tensor grad, torch::Tensor out,
                torch::Tensor outT, double lr, double weight_decay,
                c10::optional<torch::Tensor> gscale) {
  CHECK_F32(master); CHECK_F32(grad); CHECK_BF16(out); CHECK_BF16(outT);
  CHECK_CONTIG(master); CHECK_CONTIG(grad); CHECK_CONTIG(out); CHECK_CONTIG(outT);
  int E = master.size(0), R = master.size(1), C = master.size(2);
  TORCH_CHECK(R % 64 == 0 && C % 64 == 0, "dims must be multiples of 64");
  TORCH_CHECK(outT.size(1) == C && outT.size(2) == R, "outT must be [E, C, R]");
  lah_sgd_step_t(master.data_ptr(), grad.data_ptr(), out.data_ptr(), outT.data_ptr(),
                 E, R, C, (float)lr, (float)weight_decay, scale_ptr(gscale, master),
                 cur_stream());
}

void sgd_step_sr_t(torch::Tensor param, torch::Tensor grad, torch::Tensor paramT,
                   double lr, double weight_decay, int64_t seed,
                   c10::optional<torch::Tensor> gscale) {
  CHECK_BF16(param); CHECK_F32(grad); CHECK_BF16(paramT);
  CHECK_CONTIG(param); CHECK_CONTIG(grad); CHECK_CONTIG(paramT);
  int E = param.size(0), R = param.size(1), C = param.size(2);
  TORCH_CHECK(R % 64 == 0 && C % 64 == 0, "dims must be multiples of 64");
  lah_sgd_step_sr_t(param.data_ptr(), grad.data_ptr(), paramT.data_ptr(), E, R, C,
                    (float)lr, (float)weight_decay, (unsigned)seed,
                    scale_ptr(gscale, param), cur_stream());
}

torch::Tensor transpose_bf16(torch::Tensor in) {
  CHECK_BF16(in); CHECK_CONTIG(in); CHECK_CUDA(in);
  int E = in.size(0), R = in.size(1), C = in.size(2);
  TORCH_CHECK(R % 64 == 0 && C % 64 == 0, "transpose dims must be multiples of 64");
  auto out = torch::empty({E, C, R}, in.options());
  lah_transpose_bf16(in.data_ptr(), out.data_ptr(), E, R, C, cur_stream());
  return out;
}

torch::Tensor colsum(torch::Tensor d) {
  CHECK_BF16(d); CHECK_CONTIG(d);
  int E = d.size(0), M = d.size(1), C = d.size(2);
  auto db = torch::empty({E, C}, d.options().dtype(at::kFloat));
  lah_colsum(d.data_ptr(), db.data_ptr(), E, M, C, cur_stream());
  return db;
}

}  // namespace


// causal flash-attention forward (experimental): q,k,v [B,H,S,64] bf16
static void check_attn_args(const torch::Tensor& q, const torch::Tensor& k,
                            const torch::Tensor& v) {
  CHECK_CUDA(q); CHECK_BF16(q); CHECK_CONTIG(q);
  CHECK_BF16(k); CHECK_CONTIG(k); CHECK_BF16(v); CHECK_CONTIG(v);
  TORCH_CHECK(q.dim() == 4 && q.size(3) == 64, "q must be [B, H, S, 64]");
  TORCH_CHECK(q.sizes() == k.sizes() && q.sizes() == v.sizes(), "q/k/v shape mismatch");
  TORCH_CHECK(q.size(2) % 128 == 0, "seq_len must be a multiple of 128");
}

torch::Tensor flash_attn_fwd(torch::Tensor q, torch::Tensor k, torch::Tensor v) {
  check_attn_args(q, k, v);
  auto o = torch::empty_like(q);
  auto vt = torch::empty_like(v);  // [BH, 64, S] scratch via torch allocator
  lah_flash_attn_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), vt.data_ptr(),
                     o.data_ptr(), nullptr, q.size(0) * q.size(1), q.size(2),
                     cur_stream());
  return o;
}

// (o, lse) — the training entry point; lse feeds the recompute-based backward
std::vector<torch::Tensor> flash_attn_fwd_lse(torch::Tensor q, torch::Tensor k,
                                              torch::Tensor v) {
  check_attn_args(q, k, v);
  auto o = torch::empty_like(q);
  auto vt = torch::empty_like(v);
  auto lse = torch::empty({q.size(0), q.size(1), q.size(2)},
                          q.options().dtype(at::kFloat));
  lah_flash_attn_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), vt.data_ptr(),
                     o.data_ptr(), lse.data_ptr(), q.size(0) * q.size(1), q.size(2),
                     cur_stream());
  return {o, lse};
}

std::vector<torch::Tensor> flash_attn_bwd(torch::Tensor q, torch::Tensor k,
                                          torch::Tensor v, torch::Tensor dout,
                                          torch::Tensor lse, torch::Tensor d) {
  check_attn_args(q, k, v);
  CHECK_BF16(dout); CHECK_CONTIG(dout);
  CHECK_F32(lse); CHECK_CONTIG(lse); CHECK_F32(d); CHECK_CONTIG(d);
  auto dq = torch::empty_like(q);
  auto dk = torch::empty_like(k);
  auto dv = torch::empty_like(v);
  auto qt = torch::empty_like(q);   // transposed-operand scratch
  auto kt = torch::empty_like(k);
  auto dot = torch::empty_like(dout);
  lah_flash_attn_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), dout.data_ptr(),
                     lse.data_ptr(), d.data_ptr(), qt.data_ptr(), kt.data_ptr(),
                     dot.data_ptr(), dq.data_ptr(), dk.data_ptr(),
                     dv.data_ptr(), q.size(0) * q.size(1), q.size(2), cur_stream());
  return {dq, dk, dv};
}

// ---- products grouped by expert, ragged sizes (ragged_gemm.hip, ragged_layout.hip) ----

#define CHECK_ALIGNED(t) \
  TORCH_CHECK(((uintptr_t)(t).data_ptr() & 15) == 0, #t " must start at a multiple of 16 bytes")

static void check_ragged(const torch::Tensor& a, const torch::Tensor& b,
                         const torch::Tensor& offsets) {
  CHECK_NO_TANGENT(a, "a product by groups");  // ragged_ffn's
  for (const auto* t : {&a, &b}) {
    CHECK_CUDA(*t); CHECK_BF16(*t); CHECK_CONTIG(*t); CHECK_ALIGNED(*t);
  }
  CHECK_I32(offsets); CHECK_CONTIG(offsets);
  TORCH_CHECK(offsets.dim() == 1 && offsets.numel() >= 2, "offsets must be [E + 1], E >= 1");
  TORCH_CHECK(a.device() == b.device() && a.device() == offsets.device(),
              "all tensors must be on one GPU");
  TORCH_CHECK(a.dim() == 2 && a.size(0) < (int64_t)1 << 31, "rows must be [R, K], R < 2^31");
}

static void check_slope(const torch::Tensor& der) {
  TORCH_CHECK(der.scalar_type() == at::kHalf, "der must be fp16");
  CHECK_CONTIG(der); CHECK_ALIGNED(der);
}

static void check_weight(const torch::Tensor& w, const torch::Tensor& offsets) {
  TORCH_CHECK(w.dim() == 3 && w.size(0) == offsets.numel() - 1, "weight must be [E, N, K]");
  TORCH_CHECK_VALUE(w.size(0) <= 4096, "at most 4096 experts, got ", w.size(0));  // the table of tiles
  TORCH_CHECK(w.size(1) > 0 && w.size(2) > 0 && w.size(1) % 8 == 0 && w.size(2) % 8 == 0,
              "N and K must be multiples of 8");
  TORCH_CHECK(w.size(1) * w.size(2) < (int64_t)1 << 30 && w.size(1) < 1 << 21 &&
              w.size(2) < 1 << 21, "N * K must be below 2^30, N and K below 2^21");
}

std::vector<torch::Tensor> ragged_layout(torch::Tensor ids, int64_t E) {
  CHECK_CUDA(ids);
  const bool wide = ids.scalar_type() == at::kLong;
  TORCH_CHECK_VALUE(ids.dim() == 2 && (wide || ids.scalar_type() == at::kInt),
                    "topk_idx must be [T, k] int32 or int64, got ", ids.sizes(), " ", ids.scalar_type());
  TORCH_CHECK_VALUE(E >= 1 && E <= 4096, "1 to 4096 experts, got ", E);
  ids = ids.contiguous();
  const int64_t n = ids.numel();
  TORCH_CHECK(n < ((int64_t)1 << 31) - 65536, "too many slots");
  ON_DEVICE_OF(ids);
  const auto opt = ids.options().dtype(at::kInt);
  auto offsets = torch::empty({E + 1}, opt), order = torch::empty({n}, opt);
  auto rows = torch::empty(ids.sizes(), opt);
  torch::Tensor table;
  if (const long room = lah_ragged_layout_table(n, (int)E)) table = torch::empty({room}, opt);
  lah_ragged_layout(ids.data_ptr(), wide, n, (int)E, table.defined() ? table.data_ptr() : nullptr,
                    offsets.data_ptr(), order.data_ptr(), rows.data_ptr(), cur_stream());
  CHECK_LAUNCH();
  return {offsets, order, rows};
}

// Tiles of 256 x 256 (one block a CU, a list of tiles) or 128 x 256: the large ones where
// there are some for half the CUs and experts have rows for them. Large against small, us:
// 8 experts of 512 rows, 1024 -> 1024 (64 tiles) 29 and 25, of 1024 rows (128) 31 and 38;
// 256 experts, 1024 -> 4096, of 64 rows 422 and 508; 4096 -> 1024, of 64 rows 537 and 458, of
// 96 rows 522 and 550, of 256 rows 633 and 1071. At 32 rows neither has all: 1024 -> 4096, even
// rows 383 and 419, uneven ones with gelu 459 and 435; 4096 -> 1024, 470 and 380.
static bool large_tiles(int64_t R, int64_t E, int64_t N) {
  const int64_t tiles = R / 256 * ((N + 255) / 256);
  return (R >= 96 * E && tiles >= 128) || (R >= 64 * E && tiles >= 512);
}

static torch::Tensor tile_table(const torch::Tensor& rows, int64_t E, int64_t N) {
  const int64_t R = rows.size(0);
  if (!large_tiles(R, E, N)) return {};
  return torch::empty({lah_ragged_tiles_room(R, (int)E) * 4}, rows.options().dtype(at::kInt));
}
static torch::Tensor part_sums(const torch::Tensor& rows, int parts, int64_t N) {
  return parts > 1 ? torch::empty({parts * rows.size(0) * N}, rows.options().dtype(at::kFloat)) : torch::Tensor();
}
static void* ptr_or_null(const torch::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// y[r] = act(W[e] x[r] + b[e]); epi 0 plain, 1 gelu, 2 gelu and its slope into der
torch::Tensor ragged_nt(torch::Tensor x, torch::Tensor w, torch::Tensor offsets,
                        c10::optional<torch::Tensor> bias, c10::optional<torch::Tensor> der,
                        int64_t epi) {
  check_ragged(x, w, offsets);
  check_weight(w, offsets);
  const int64_t R = x.size(0), E = w.size(0), N = w.size(1), K = w.size(2);
  TORCH_CHECK(x.size(1) == K, "x must be [R, ", K, "], got [", R, ", ", x.size(1), "]");
  TORCH_CHECK(epi >= 0 && epi <= 2 && (epi == 2) == der.has_value(), "epi 2 goes with der");
  const void* bias_p = nullptr;
  int bias_bf16 = 0;
  if (bias.has_value()) {
    CHECK_CONTIG(*bias); CHECK_ALIGNED(*bias);
    bias_bf16 = bias->scalar_type() == at::kBFloat16;
    TORCH_CHECK(bias_bf16 || bias->scalar_type() == at::kFloat, "bias must be bf16 or fp32");
    TORCH_CHECK(bias->dim() == 2 && bias->size(0) == E && bias->size(1) == N &&
                bias->device() == x.device(), "bias must be [E, N] on the GPU of x");
    bias_p = bias->data_ptr();
  }
  void* der_p = nullptr;
  if (der.has_value()) {
    check_slope(*der);
    TORCH_CHECK(der->dim() == 2 && der->size(0) == R && der->size(1) == N &&
                der->device() == x.device(), "der must be [R, N] on the GPU of x");
    der_p = der->data_ptr();
  }
  ON_DEVICE_OF(x);
  auto y = torch::empty({R, N}, x.options());
  if (R == 0) return y;
  const auto table = tile_table(x, E, N);
  const int parts = table.defined() ? 1 : lah_ragged_parts(R, (int)E, (int)N, (int)K, true);
  const auto work = part_sums(x, parts, N);
  lah_ragged_nt(x.data_ptr(), w.data_ptr(), y.data_ptr(), offsets.data_ptr(), bias_p, bias_bf16,
                der_p, R, (int)E, (int)N, (int)K, (int)epi, ptr_or_null(table), parts,
                ptr_or_null(work), cur_stream());
  CHECK_LAUNCH();
  return y;
}

// out[r] = W[e]^T d[r], times der[r] if given
torch::Tensor ragged_nn(torch::Tensor d, torch::Tensor w, torch::Tensor offsets,
                        c10::optional<torch::Tensor> der) {
  check_ragged(d, w, offsets);
  check_weight(w, offsets);
  const int64_t R = d.size(0), E = w.size(0), K = w.size(1), N = w.size(2);
  TORCH_CHECK(d.size(1) == K, "d must be [R, ", K, "], got [", R, ", ", d.size(1), "]");
  void* der_p = nullptr;
  if (der.has_value()) {
    check_slope(*der);
    TORCH_CHECK(der->dim() == 2 && der->size(0) == R && der->size(1) == N &&
                der->device() == d.device(), "der must be [R, N] on the GPU of d");
    der_p = der->data_ptr();
  }
  ON_DEVICE_OF(d);
  auto out = torch::empty({R, N}, d.options());
  if (R == 0) return out;
  const auto table = tile_table(d, E, N);
  const int parts = table.defined() ? 1 : lah_ragged_parts(R, (int)E, (int)N, (int)K, false);
  const auto work = part_sums(d, parts, N);
  lah_ragged_nn(d.data_ptr(), w.data_ptr(), out.data_ptr(), offsets.data_ptr(), der_p, R, (int)E,
                (int)N, (int)K, ptr_or_null(table), parts, ptr_or_null(work), cur_stream());
  CHECK_LAUNCH();
  return out;
}

// dw[e] = sum_r d[r] x[r]^T (added to what is there if accumulate), db[e] = sum_r d[r]
void ragged_tn(torch::Tensor d, torch::Tensor x, torch::Tensor offsets, torch::Tensor dw,
               c10::optional<torch::Tensor> db, bool accumulate) {
  check_ragged(d, x, offsets);
  const int64_t R = d.size(0), M = d.size(1), E = offsets.numel() - 1;
  TORCH_CHECK(x.dim() == 2 && x.size(0) == R, "d and x must have the same rows");
  const int64_t N = x.size(1);
  CHECK_CONTIG(dw); CHECK_ALIGNED(dw);
  const bool bf16 = dw.scalar_type() == at::kBFloat16;
  TORCH_CHECK(bf16 || dw.scalar_type() == at::kFloat, "dw must be bf16 or fp32");
  TORCH_CHECK(!(bf16 && accumulate), "sums over several calls are held in fp32");
  TORCH_CHECK(dw.dim() == 3 && dw.size(1) == M && dw.size(2) == N && dw.device() == d.device(),
              "dw must be [E, M, N] on the GPU of d");
  check_weight(dw, offsets);
  void* db_p = nullptr;
  int db_bf16 = 0;
  if (db.has_value()) {
    CHECK_CONTIG(*db);
    db_bf16 = db->scalar_type() == at::kBFloat16;
    TORCH_CHECK(db_bf16 || db->scalar_type() == at::kFloat, "db must be bf16 or fp32");
    TORCH_CHECK(!(db_bf16 && accumulate), "sums over several calls are held in fp32");
    TORCH_CHECK(db->dim() == 2 && db->size(0) == E && db->size(1) == M &&
                db->device() == d.device(), "db must be [E, M] on the GPU of d");
    db_p = db->data_ptr();
  }
  ON_DEVICE_OF(d);
  const long bytes = lah_ragged_tn_work(R, (int)E, (int)N, (int)M);
  torch::Tensor work;
  if (bytes > 0) work = torch::empty({bytes / 4}, d.options().dtype(at::kInt));
  lah_ragged_tn(d.data_ptr(), x.data_ptr(), dw.data_ptr(), db_p, db_bf16, offsets.data_ptr(), R,
                (int)E, (int)N, (int)M, bf16 ? 2 : accumulate ? 1 : 0, ptr_or_null(work),
                cur_stream());
  CHECK_LAUNCH();
}

// dP = dy * der in bf16 (if `write`; rows of nobody are left as they are), and db[e], if given,
// its sums over the rows of e before the rounding
torch::Tensor ragged_slope(torch::Tensor dy, torch::Tensor der, torch::Tensor offsets,
                           c10::optional<torch::Tensor> db, bool write) {
  check_ragged(dy, dy, offsets);
  check_slope(der);
  TORCH_CHECK(dy.sizes() == der.sizes() && dy.device() == der.device() && dy.size(1) % 8 == 0 &&
              dy.size(1) < 1 << 21, "dy and der must be [R, N], N a multiple of 8");
  TORCH_CHECK(write || db.has_value(), "nothing is asked for");
  const int64_t R = dy.size(0), N = dy.size(1), E = offsets.numel() - 1;
  TORCH_CHECK(E <= 4096, "at most 4096 groups, got ", E);
  void* db_p = nullptr;
  int db_bf16 = 0;
  if (db.has_value()) {
    CHECK_CONTIG(*db);
    db_bf16 = db->scalar_type() == at::kBFloat16;
    TORCH_CHECK(db_bf16 || db->scalar_type() == at::kFloat, "db must be bf16 or fp32");
    TORCH_CHECK(db->dim() == 2 && db->size(0) == E && db->size(1) == N && db->device() == dy.device(),
                "db must be [E, N] on the GPU of dy");
    db_p = db->data_ptr();
  }
  ON_DEVICE_OF(dy);
  torch::Tensor dp, work;
  if (write) dp = torch::empty_like(dy);
  if (N == 0) return dp;
  const long room = db.has_value() ? lah_ragged_slope_work(R, (int)E, (int)N) : 0;
  if (room > 0) work = torch::empty({room}, dy.options().dtype(at::kFloat));
  lah_ragged_slope(dy.data_ptr(), der.data_ptr(), ptr_or_null(dp), db_p, db_bf16, offsets.data_ptr(), R, (int)E,
                   (int)N, ptr_or_null(work), cur_stream());
  CHECK_LAUNCH();
  return dp;
}

// ---- the differentiable product ----

struct GroupedLinear : public torch::autograd::Function<GroupedLinear> {
  static torch::Tensor forward(torch::autograd::AutogradContext* ctx, const torch::Tensor& x_in,
                               const torch::Tensor& w_in, const c10::optional<torch::Tensor>& bias,
                               const torch::Tensor& offsets, bool gelu) {
    const auto x = ready(x_in), w = ready(w_in);
    c10::optional<torch::Tensor> b, der;
    if (bias.has_value()) b = ready(*bias);
    if (gelu) der = torch::empty({x.size(0), w.size(1)}, x.options().dtype(at::kHalf));
    ctx->save_for_backward({x, w, offsets, der.value_or(torch::Tensor())});
    ctx->saved_data["bias"] = b.has_value() ? (int64_t)b->scalar_type() : (int64_t)-1;
    return ragged_nt(x, w, offsets, b, der, gelu ? 2 : 0);
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "grouped_linear is differentiable once");
    const auto saved = ctx->get_saved_variables();
    const auto &x = saved[0], &w = saved[1], &offsets = saved[2], &der = saved[3];
    const int64_t bias = ctx->saved_data["bias"].toInt();
    if (!grads[0].defined()) return {{}, {}, {}, {}, {}};
    auto d = ready(grads[0]);
    torch::Tensor dx, dw, db;
    const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1);
    c10::optional<torch::Tensor> b;
    if (bias >= 0 && ctx->needs_input_grad(2))
      b = db = torch::empty({w.size(0), w.size(1)}, w.options().dtype((at::ScalarType)bias));
    if (der.defined()) {
      if (want_x || want_w || db.defined()) d = ragged_slope(d, der, offsets, b, want_x || want_w);
      b.reset();
    }
    if (want_x) dx = ragged_nn(d, w, offsets, c10::nullopt);
    if (want_w || b.has_value()) {
      dw = torch::empty_like(w);
      ragged_tn(d, x, offsets, dw, b, false);
      if (!want_w) dw = torch::Tensor();
    }
    return {dx, dw, db, {}, {}};
  }
};

torch::Tensor grouped_linear(torch::Tensor x, torch::Tensor w, torch::Tensor offsets,
                             c10::optional<torch::Tensor> bias, c10::optional<std::string> activation) {
  for (const auto* t : {&x, &w}) CHECK_NO_TANGENT(*t, "grouped_linear");
  if (bias.has_value()) CHECK_NO_TANGENT(*bias, "grouped_linear");
  TORCH_CHECK_VALUE(x.dim() == 2 && w.dim() == 3 && x.size(1) == w.size(2),
                    "x must be [R, K] and weight [E, N, K], got ", x.sizes(), " and ", w.sizes());
  TORCH_CHECK_VALUE(offsets.scalar_type() == at::kInt && offsets.dim() == 1 &&
                    offsets.size(0) == w.size(0) + 1,
                    "offsets must be [E + 1] int32, got ", offsets.sizes(), " ", offsets.scalar_type());
  TORCH_CHECK_VALUE(!activation.has_value() || *activation == "gelu",
                    "activation must be None or 'gelu', got ", activation.value_or(""));
  TORCH_CHECK_VALUE(x.scalar_type() == at::kBFloat16 && w.scalar_type() == at::kBFloat16,
                    "the GPU kernels take bf16, got ", x.scalar_type(), " and ", w.scalar_type());
  TORCH_CHECK_VALUE(w.numel() > 0, "weight must not be empty, got ", w.sizes());
  TORCH_CHECK_VALUE(w.size(1) % 8 == 0 && w.size(2) % 8 == 0,
                    "N and K must be multiples of 8 (16-byte rows), got ", w.sizes());
  TORCH_CHECK_VALUE(w.device() == x.device() && offsets.device() == x.device() &&
                    (!bias.has_value() || bias->device() == x.device()),
                    "x, weight, offsets and bias must be on one device");
  if (bias.has_value()) {
    TORCH_CHECK_VALUE(bias->dim() == 2 && bias->size(0) == w.size(0) && bias->size(1) == w.size(1),
                      "bias must be [E, N], got ", bias->sizes());
    TORCH_CHECK_VALUE(bias->scalar_type() == at::kBFloat16 || bias->scalar_type() == at::kFloat,
                      "bias must be bf16 or fp32, got ", bias->scalar_type());
  }
  const bool gelu = activation.has_value();
  const auto at = offsets.contiguous();
  if (at::GradMode::is_enabled() &&
      (x.requires_grad() || w.requires_grad() || (bias.has_value() && bias->requires_grad())))
    return GroupedLinear::apply(x, w, bias, at, gelu);
  c10::optional<torch::Tensor> b;
  if (bias.has_value()) b = ready(*bias);
  return ragged_nt(ready(x), ready(w), at, b, c10::nullopt, gelu ? 1 : 0);
}

// ---- gradient norm, clipping, clipped step of fp32 masters (clip.hip) ----

// kinds of clip.hip; -1: not the kernels'
static int clip_kind(const torch::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return 0;
    case at::kHalf: return 1;
    case at::kFloat: return 2;
    default: return -1;
  }
}

struct ClipList {
  std::vector<void*> p;
  std::vector<long> n;
  std::vector<int> kind;
  bool taken = true;  // all on one GPU, of kinds and layouts that the kernels take
  bool tangent = false;
  explicit ClipList(const std::vector<torch::Tensor>& ts) {
    TORCH_CHECK_VALUE(!ts.empty(), "no tensors");
    p.reserve(ts.size()); n.reserve(ts.size()); kind.reserve(ts.size());
    for (const auto& t : ts) {
      const int k = clip_kind(t);
      taken = taken && t.is_cuda() && t.device() == ts[0].device() && k >= 0 && t.is_contiguous();
      tangent = tangent || has_tangent(t);
      p.push_back(t.data_ptr());
      n.push_back(t.numel());
      kind.push_back(k);
    }
    TORCH_CHECK_NOT_IMPLEMENTED(!(taken && tangent), "gradient norms, clipping and steps have no forward-mode "
                                                     "derivative on the GPU");
  }
};

// One launch writes them all: a tensor that is there twice would be written by two blocks at once.
static void check_distinct(const ClipList& l, const char* name) {
  std::vector<void*> p;
  p.reserve(l.p.size());
  for (size_t i = 0; i < l.p.size(); ++i)
    if (l.n[i] > 0) p.push_back(l.p[i]);
  std::sort(p.begin(), p.end());
  TORCH_CHECK_VALUE(std::adjacent_find(p.begin(), p.end()) == p.end(), "the same tensor twice among the ", name);
}

// (norm, scale); nothing where a tensor is not the kernels'
std::vector<torch::Tensor> grad_norm(const std::vector<torch::Tensor>& grads, double max_norm, double eps) {
  const ClipList l(grads);
  if (!l.taken) return {};
  ON_DEVICE_OF(grads[0]);
  const auto opt = grads[0].options();
  auto partial = torch::empty({lah_clip_partials((int)l.p.size())}, opt.dtype(at::kDouble));
  auto norm = torch::empty({}, opt.dtype(at::kFloat)), scale = torch::empty({}, opt.dtype(at::kFloat));
  lah_grad_norm(l.p.data(), l.n.data(), l.kind.data(), (int)l.p.size(), partial.data_ptr(),
                (float)max_norm, (float)eps, norm.data_ptr(), scale.data_ptr(), cur_stream());
  CHECK_LAUNCH();
  return {norm, scale};
}

// whether it was done
bool grad_scale_(const std::vector<torch::Tensor>& grads, const torch::Tensor& scale) {
  const ClipList l(grads);
  if (!l.taken) return false;
  check_distinct(l, "tensors");
  const void* s = scale_ptr(scale, grads[0]);
  ON_DEVICE_OF(grads[0]);
  lah_grad_scale(l.p.data(), l.n.data(), l.kind.data(), (int)l.p.size(), s, cur_stream());
  CHECK_LAUNCH();
  return true;
}

// whether it was done: bf16 params with fp32 masters and buffers, all contiguous
bool master_sgd_(const std::vector<torch::Tensor>& params, const std::vector<torch::Tensor>& masters,
                 const std::vector<torch::Tensor>& grads, const std::vector<torch::Tensor>& bufs,
                 const c10::optional<torch::Tensor>& scale, double lr, double mu, double weight_decay) {
  const size_t count = params.size();
  TORCH_CHECK_VALUE(masters.size() == count && grads.size() == count && (bufs.empty() || bufs.size() == count),
                    "params, masters, grads and momentum_bufs must go together");
  for (size_t i = 0; i < count; ++i) {
    TORCH_CHECK_VALUE(masters[i].scalar_type() == at::kFloat &&
                      (bufs.empty() || bufs[i].scalar_type() == at::kFloat),
                      "masters and momentum_bufs must be fp32");
    TORCH_CHECK_VALUE(params[i].sizes() == masters[i].sizes() && params[i].sizes() == grads[i].sizes(),
                      "params, masters and grads must have the same shapes");
    TORCH_CHECK_VALUE(bufs.empty() || bufs[i].sizes() == params[i].sizes(),
                      "momentum_bufs must have the shapes of the params");
  }
  const ClipList p(params), m(masters), g(grads);
  bool taken = p.taken && m.taken && g.taken && masters[0].device() == params[0].device() &&
               grads[0].device() == params[0].device();
  std::vector<void*> b;
  if (!bufs.empty()) {
    const ClipList l(bufs);
    taken = taken && l.taken && bufs[0].device() == params[0].device();
    if (taken) check_distinct(l, "momentum_bufs");
    b = l.p;
  }
  for (const int k : p.kind) taken = taken && k == 0;
  if (!taken) return false;
  check_distinct(p, "params");
  check_distinct(m, "masters");
  const void* s = scale_ptr(scale, params[0]);
  ON_DEVICE_OF(params[0]);
  lah_master_sgd(p.p.data(), m.p.data(), g.p.data(), b.empty() ? nullptr : b.data(), p.n.data(),
                 g.kind.data(), (int)p.p.size(), s, (float)lr, (float)mu, (float)weight_decay,
                 cur_stream());
  CHECK_LAUNCH();
  return true;
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("batched_gemm_nt", &batched_gemm_nt, "batched NT GEMM with fused epilogue",
        py::arg("A"), py::arg("B"), py::arg("bias") = py::none(),
        py::arg("pre") = py::none(), py::arg("epi") = 0);
  m.def("batched_gemm_tn", &batched_gemm_tn, py::arg("A"), py::arg("B"), py::arg("C"),
        py::arg("accumulate") = false);
  m.def("fused_dw_sgd_sr", &fused_dw_sgd_sr, py::arg("A"), py::arg("B"), py::arg("W"),
        py::arg("WT"), py::arg("lr"), py::arg("weight_decay") = 0.0,
        py::arg("seed") = 0);
  m.def("ce_rowstats", &ce_rowstats, py::arg("logits"), py::arg("labels"),
        py::arg("ignore_index") = -100);
  m.def("ce_bwd", &ce_bwd, py::arg("logits"), py::arg("labels"), py::arg("lse"),
        py::arg("gscale"), py::arg("ignore_index") = -100);
  m.def("flash_attn_fwd", &flash_attn_fwd);
  m.def("flash_attn_fwd_lse", &flash_attn_fwd_lse);
  m.def("flash_attn_bwd", &flash_attn_bwd);
  m.def("gating_topk_fwd", &gating_topk_fwd);
  m.def("gating_topk_bwd", &gating_topk_bwd, py::arg("probs"), py::arg("topk_idx"),
        py::arg("topk_w"), py::arg("d_topk_w"), py::arg("aux_g") = py::none());
  m.def("assign_slots", &assign_slots);
  m.def("dispatch_gather", &dispatch_gather);
  m.def("dispatch_bwd", &dispatch_bwd);
  m.def("combine_fwd", &combine_fwd, py::arg("ybuf"), py::arg("topk_idx"), py::arg("pos"),
        py::arg("w"), py::arg("least") = 0.2);
  m.def("combine_bwd", &combine_bwd, py::arg("dy"), py::arg("ybuf"), py::arg("y"),
        py::arg("topk_idx"), py::arg("pos"), py::arg("w"), py::arg("inv"), py::arg("least") = 0.2);
  m.def("sgd_step", &sgd_step, py::arg("master"), py::arg("grad"),
        py::arg("momentum"), py::arg("out_bf16"),
        py::arg("lr") = 0.01, py::arg("mu") = 0.0, py::arg("weight_decay") = 0.0,
        py::arg("gscale") = py::none());
  m.def("sgd_step_t", &sgd_step_t, py::arg("master"), py::arg("grad"), py::arg("out"),
        py::arg("outT"), py::arg("lr") = 0.01, py::arg("weight_decay") = 0.0,
        py::arg("gscale") = py::none());
  m.def("sgd_step_sr_t", &sgd_step_sr_t, py::arg("param"), py::arg("grad"),
        py::arg("paramT"), py::arg("lr") = 0.01, py::arg("weight_decay") = 0.0,
        py::arg("seed") = 0, py::arg("gscale") = py::none());
  m.def("transpose_bf16", &transpose_bf16);
  m.def("colsum", &colsum);
  m.def("ragged_layout", &ragged_layout, py::arg("ids"), py::arg("num_experts"));
  m.def("ragged_nt", &ragged_nt, py::arg("x"), py::arg("w"), py::arg("offsets"),
        py::arg("bias") = py::none(), py::arg("der") = py::none(), py::arg("epi") = 0);
  m.def("ragged_nn", &ragged_nn, py::arg("d"), py::arg("w"), py::arg("offsets"),
        py::arg("der") = py::none());
  m.def("ragged_tn", &ragged_tn, py::arg("d"), py::arg("x"), py::arg("offsets"), py::arg("dw"),
        py::arg("db") = py::none(), py::arg("accumulate") = false);
  m.def("grouped_linear", &grouped_linear, py::arg("x"), py::arg("weight"), py::arg("offsets"),
        py::arg("bias") = py::none(), py::arg("activation") = py::none());
  m.def("ragged_slope", &ragged_slope, py::arg("dy"), py::arg("der"), py::arg("offsets"),
        py::arg("db") = py::none(), py::arg("write") = true);
  m.def("grad_norm", &grad_norm, py::arg("grads"), py::arg("max_norm"), py::arg("eps") = 1e-6);
  m.def("grad_scale_", &grad_scale_, py::arg("grads"), py::arg("scale"));
  m.def("master_sgd_", &master_sgd_, py::arg("params"), py::arg("masters"), py::arg("grads"),
        py::arg("bufs"), py::arg("scale"), py::arg("lr"), py::arg("mu"), py::arg("weight_decay"));
}
