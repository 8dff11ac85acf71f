// PyTorch bindings for the learningorchestra_amd gfx950 kernel library.
// Thin argument-checking wrappers; all compute is in the .hip translation
// units. Built in-tree (build_ext.py) as learningorchestra_amd/_lo_C.so.
#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/impl/VirtualGuardImpl.h>

#include <hip/hip_runtime.h>

#include <algorithm>
#include <array>
#include <climits>
#include <cmath>
#include <cstring>

#include "newton_schulz_plan.h"

namespace lo {
struct ConvGeom {
  int B, H, W, C;
  int KH, KW, SH, SW, PH, PW;
  int OH, OW;
  unsigned mgOW = 0, mgOH = 0;
  int sOW = 0, sOH = 0;
};

// magic-division constants (see gemm.hip fdiv): exact for n < 2^31
static inline void fill_fastdiv(lo::ConvGeom& g) {
  auto mk = [](unsigned d, unsigned& mg, int& s) {
    if (d <= 1) { mg = 0; s = 0; return; }
    s = 0;
    while ((1u << s) < d) ++s;
    if ((1u << s) == d) { mg = 1; return; }          // power of two: q = n>>s
    // mg = ceil(2^(31+s)/d) fits u32 (2^s/d in (1,2)); device computes
    // q = mulhi(n, mg) >> (s-1) == (n*mg) >> (31+s), exact for n < 2^31
    const unsigned long long L = 1ull << (31 + s);
    mg = (unsigned)((L + d - 1) / d);
    s = s - 1;
  };
  mk((unsigned)g.OW, g.mgOW, g.sOW);
  mk((unsigned)g.OH, g.mgOH, g.sOH);
}
struct GemmArgs {
  const void *A, *B;
  void* C;
  const float* bias;
  long lda, ldb, ldc;
  int M, N, K;
  bool ta, tb;
  int epi;
  bool out_f32;
  int splits;
  int gather;
  ConvGeom geom;
  float* stats_sum = nullptr;
  float* stats_sumsq = nullptr;
  const void* addend = nullptr;
};
bool gemm_dispatch(const GemmArgs& g, hipStream_t s);
void launch_mfma_probe(const void* A, const void* B, float* D, hipStream_t s);
void launch_im2col(const void* in, void* col, int B, int H, int W, int C,
                   int KH, int KW, int SH, int SW, int PH, int PW,
                   int OH, int OW, int Kpad, hipStream_t s);
bool launch_conv_fwd_small(const void* x, const void* w, long ldw,
                           const void* bias, void* y, long ldy, int B, int H,
                           int W, int C, int KH, int KW, int SH, int SW,
                           int PH, int PW, int OH, int OW, int outC, int relu,
                           hipStream_t s);
bool launch_conv1d_fwd(const void* x, const void* w, long ldw,
                       const void* bias, void* y, long ldy, int B, int H,
                       int C, int KH, int PH, int OH, int outC, int relu,
                       hipStream_t s);
bool launch_conv1d_dx(const void* dy2, long ldy, const void* wt, long ldw,
                      void* dx, int B, int H, int C, int KH, int PH, int OH,
                      int outC, int accumulate, hipStream_t s);
bool launch_conv_dw_c1(const void* dy2, long ldy, const void* x, void* dw,
                       long ldw, int B, int H, int W, int KH, int KW, int SH,
                       int SW, int PH, int PW, int OH, int OW, int outC,
                       hipStream_t s);
bool launch_conv_dw_smallc(const void* dy2, long ldy, const void* x, void* dw,
                           long ldw, int B, int H, int W, int C, int KH,
                           int KW, int SH, int SW, int PH, int PW, int OH,
                           int OW, int outC, hipStream_t s);
bool launch_conv_dx(const void* dy2, long ldy, const void* wt, long ldw,
                    void* dx, int B, int H, int W, int C, int KH, int KW,
                    int SH, int SW, int PH, int PW, int OH, int OW, int outC,
                    hipStream_t s);
void launch_col2im(const void* dcol, void* dx, int B, int H, int W, int C,
                   int KH, int KW, int SH, int SW, int PH, int PW, int OH,
                   int OW, int Kpad, hipStream_t s);
void launch_maxpool_fwd(const void* in, void* out, void* idx, int B, int H, int W,
                        int C, int KH, int KW, int SH, int SW, int PH, int PW,
                        int OH, int OW, int relu_sentinel, hipStream_t s);
void launch_maxpool_bwd(const void* dy, const void* idx, void* dx,
                        const void* relu_y, int B, int H,
                        int W, int C, int KH, int KW, int SH, int SW, int PH,
                        int PW, int OH, int OW, hipStream_t s);
void launch_bn_stats(const void* x, void* sum, void* sumsq, long M, int C,
                     hipStream_t s);
void launch_bn_fwd(const void* x, void* y, const void* mean, const void* invstd,
                   const void* gamma, const void* beta, const void* residual,
                   long M, int C, int relu, hipStream_t s);
void launch_bn_bwd_reduce(const void* dy, const void* y, const void* x,
                          const void* mean, const void* invstd, void* dbeta,
                          void* dgamma, long M, int C, int relu, hipStream_t s);
void launch_bn_finalize_stats(const void* scratch, void* mean, void* invstd,
                              void* rmean, void* rvar, float invM,
                              float momentum, float eps, int C,
                              hipStream_t s);
void launch_bn_bwd_dx(const void* dy, const void* y, const void* x, void* dx,
                      const void* mean, const void* invstd, const void* gamma,
                      const void* dbeta, const void* dgamma, long M, int C,
                      int relu, hipStream_t s);
void launch_add_relu(const void* a, const void* b, void* z, long n, int relu,
                     hipStream_t s);
void launch_avgpool_global(const void* x, void* out, int B, int HW, int C,
                           hipStream_t s);
void launch_avgpool_global_bwd(const void* dy, void* dx, int B, int HW, int C,
                               hipStream_t s);
void launch_relu_bwd(const void* dy, const void* y, void* dx, long n, hipStream_t s);
void launch_sgd(void* master, const void* grad, void* mom, void* mirror, long n,
                float lr, float mu, float wd, float gscale, hipStream_t s);
void launch_adam(void* master, const void* grad, void* m1, void* m2, void* mirror,
                 const void* step_dev, const void* ranges, int n_ranges,
                 long longest, long n, float lr, float b1, float b2,
                 float eps, float wd, float gscale, hipStream_t s);
void launch_colsum(const void* dy, void* out, long M, int N, long ldy, hipStream_t s);
void launch_colsum_masked(const void* dy, const void* mask, void* out, long M,
                          int N, long ldy, hipStream_t s);
void launch_argmax_rows(const void* x, void* out, long M, int C, int Cvalid,
                        long ldx, hipStream_t s);
void launch_accuracy_count(const void* pred, const void* label, void* out, long M,
                           hipStream_t s);
void launch_softmax_ce(const void* logits, const void* labels, void* dlogits,
                       void* loss_sum, void* correct, long M, int C, int Cvalid,
                       float gscale, hipStream_t s);
void launch_tree_hist(const void* binned, const void* node_of, const void* grad,
                      const void* hess, void* hist, long N, int F, int n_nodes,
                      int B, double gbound, double hbound, hipStream_t s);
void launch_embedding_fwd(const void* ids, const void* table, void* out,
                          long n, int dim, hipStream_t s);
void launch_embedding_bwd(const void* ids, const void* dy, void* gtable,
                          long n, int dim, hipStream_t s);
void launch_layernorm_fwd(int dtype, const void* x, long ldx, const void* res,
                          long ldr, const float* gamma, const float* beta,
                          void* y, long ldy, void* sum, long lds, float* mean,
                          float* invstd, long rows, int cols, float eps,
                          hipStream_t s);
int layernorm_bwd_parts(int dtype, long rows, int cols);
void launch_layernorm_bwd(int dtype, const void* dy, long ldy, const void* x,
                          long ldx, const void* skip, long ldk,
                          const float* mean, const float* invstd,
                          const float* gamma, void* dx, long ldd, float* part,
                          float* dgamma, float* dbeta, long rows, int cols,
                          hipStream_t s);
}  // namespace lo

namespace {

hipStream_t stream() { return at::hip::getCurrentHIPStream().stream(); }

void check_bf16(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be on GPU");
  TORCH_CHECK(t.scalar_type() == at::kBFloat16, name, " must be bf16");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

void check_f32(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be on GPU");
  TORCH_CHECK(t.scalar_type() == at::kFloat, name, " must be fp32");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

// gemm: C = op_ta(A) @ op_tb(B) (+bias)(+relu). Returns false if no native
// config covers the shape (python falls back to a library GEMM).
bool gemm(at::Tensor A, at::Tensor B, at::Tensor C,
          c10::optional<at::Tensor> bias, bool ta, bool tb, int64_t epi,
          int64_t splits, c10::optional<at::Tensor> stats = c10::nullopt,
          c10::optional<at::Tensor> addend = c10::nullopt) {
  check_bf16(A, "A");
  check_bf16(B, "B");
  TORCH_CHECK(C.is_cuda() && C.is_contiguous(), "C must be contiguous GPU");
  const bool out_f32 = C.scalar_type() == at::kFloat;
  TORCH_CHECK(out_f32 || C.scalar_type() == at::kBFloat16, "C must be bf16 or fp32");
  const int M = (int)C.size(0), N = (int)C.size(1);
  const int K = (int)(ta ? A.size(0) : A.size(1));
  TORCH_CHECK((int)(ta ? A.size(1) : A.size(0)) == M, "A/M mismatch");
  TORCH_CHECK((int)(tb ? B.size(1) : B.size(0)) == K, "B/K mismatch");
  TORCH_CHECK((int)(tb ? B.size(0) : B.size(1)) == N, "B/N mismatch");
  const float* bias_p = nullptr;
  if (bias.has_value()) {
    check_f32(*bias, "bias");
    TORCH_CHECK(bias->numel() == N, "bias/N mismatch");
    bias_p = bias->data_ptr<float>();
  }
  lo::GemmArgs g{A.data_ptr(), B.data_ptr(), C.data_ptr(), bias_p,
                 A.size(1), B.size(1), C.size(1), M, N, K, ta, tb,
                 (int)epi, out_f32, (int)splits, 0, {}};
  if (addend.has_value()) {
    check_bf16(*addend, "addend");
    TORCH_CHECK(!out_f32 && splits == 1, "addend needs bf16 non-split-K out");
    TORCH_CHECK(addend->sizes() == C.sizes(), "addend/C shape mismatch");
    g.addend = addend->data_ptr();
  }
  if (stats.has_value()) {
    check_f32(*stats, "stats");
    TORCH_CHECK(stats->numel() == 2 * N, "stats must be [2, N]");
    g.stats_sum = stats->data_ptr<float>();
    g.stats_sumsq = g.stats_sum + N;
  }
  return lo::gemm_dispatch(g, stream());
}

// implicit-GEMM conv forward: y2d[B*OH*OW, outC] = im2col(x) @ W^T (+bias,
// +relu) without materializing col. W is [outC, kpad].
bool gemm_conv_fwd(at::Tensor x, at::Tensor Wt, at::Tensor C,
                   c10::optional<at::Tensor> bias, bool relu,
                   int64_t KH, int64_t KW, int64_t SH, int64_t SW,
                   int64_t PH, int64_t PW) {
  check_bf16(x, "x");
  check_bf16(Wt, "W");
  check_bf16(C, "C");
  const int B = (int)x.size(0), H = (int)x.size(1), W = (int)x.size(2),
            Ci = (int)x.size(3);
  const int OH = (int)((H + 2 * PH - KH) / SH) + 1;
  const int OW = (int)((W + 2 * PW - KW) / SW) + 1;
  const int M = (int)C.size(0), N = (int)C.size(1);
  const int K = (int)Wt.size(1);  // kpad
  TORCH_CHECK(M == (long)B * OH * OW && N == Wt.size(0), "conv shapes");
  const float* bias_p = nullptr;
  if (bias.has_value()) { check_f32(*bias, "bias"); bias_p = bias->data_ptr<float>(); }
  lo::ConvGeom geom{B, H, W, Ci, (int)KH, (int)KW, (int)SH, (int)SW,
                    (int)PH, (int)PW, OH, OW};
  fill_fastdiv(geom);
  lo::GemmArgs g{x.data_ptr(), Wt.data_ptr(), C.data_ptr(), bias_p,
                 K, Wt.size(1), C.size(1), M, N, K, false, true,
                 relu ? 1 : 0, false, 1, 1, geom};
  return lo::gemm_dispatch(g, stream());
}

// implicit-GEMM conv dW: gw[outC, kpad] = dY^T @ im2col(x), fp32 split-K
bool gemm_conv_dw(at::Tensor dy2, at::Tensor x, at::Tensor gw, int64_t splits,
                  int64_t KH, int64_t KW, int64_t SH, int64_t SW,
                  int64_t PH, int64_t PW) {
  check_bf16(dy2, "dy2");
  check_bf16(x, "x");
  check_f32(gw, "gw");
  const int B = (int)x.size(0), H = (int)x.size(1), W = (int)x.size(2),
            Ci = (int)x.size(3);
  const int OH = (int)((H + 2 * PH - KH) / SH) + 1;
  const int OW = (int)((W + 2 * PW - KW) / SW) + 1;
  const int M = (int)gw.size(0), N = (int)gw.size(1);   // outC, kpad
  const long K = dy2.size(0);                           // B*OH*OW
  TORCH_CHECK(K == (long)B * OH * OW && M == dy2.size(1), "conv dW shapes");
  lo::ConvGeom geom{B, H, W, Ci, (int)KH, (int)KW, (int)SH, (int)SW,
                    (int)PH, (int)PW, OH, OW};
  fill_fastdiv(geom);
  lo::GemmArgs g{dy2.data_ptr(), x.data_ptr(), gw.data_ptr(), nullptr,
                 dy2.size(1), N, gw.size(1), M, N, (int)K, true, false,
                 0, true, (int)std::max<int64_t>(splits, 2), 2, geom};
  return lo::gemm_dispatch(g, stream());
}

at::Tensor mfma_probe(at::Tensor A, at::Tensor B) {
  check_bf16(A, "A");
  check_bf16(B, "B");
  TORCH_CHECK(A.size(0) == 16 && A.size(1) == 32 && B.size(0) == 32 && B.size(1) == 16);
  auto D = at::zeros({16, 16}, A.options().dtype(at::kFloat));
  lo::launch_mfma_probe(A.data_ptr(), B.data_ptr(), D.data_ptr<float>(), stream());
  return D;
}

at::Tensor im2col(at::Tensor in, int64_t KH, int64_t KW, int64_t SH, int64_t SW,
                  int64_t PH, int64_t PW, int64_t Kpad, at::Tensor col) {
  check_bf16(in, "in");
  check_bf16(col, "col");
  const int B = (int)in.size(0), H = (int)in.size(1), W = (int)in.size(2),
            C = (int)in.size(3);
  const int OH = (H + 2 * (int)PH - (int)KH) / (int)SH + 1;
  const int OW = (W + 2 * (int)PW - (int)KW) / (int)SW + 1;
  TORCH_CHECK(col.size(0) == (long)B * OH * OW && col.size(1) == Kpad, "col shape");
  TORCH_CHECK(Kpad >= KH * KW * C && Kpad % 8 == 0, "Kpad");
  lo::launch_im2col(in.data_ptr(), col.data_ptr(), B, H, W, C, (int)KH, (int)KW,
                    (int)SH, (int)SW, (int)PH, (int)PW, OH, OW, (int)Kpad, stream());
  return col;
}

at::Tensor col2im(at::Tensor dcol, int64_t B, int64_t H, int64_t W, int64_t C,
                  int64_t KH, int64_t KW, int64_t SH, int64_t SW, int64_t PH,
                  int64_t PW, at::Tensor dx) {
  check_bf16(dcol, "dcol");
  check_bf16(dx, "dx");
  const int OH = (int)((H + 2 * PH - KH) / SH) + 1;
  const int OW = (int)((W + 2 * PW - KW) / SW) + 1;
  TORCH_CHECK(dcol.size(0) == B * OH * OW, "dcol rows");
  lo::launch_col2im(dcol.data_ptr(), dx.data_ptr(), (int)B, (int)H, (int)W, (int)C,
                    (int)KH, (int)KW, (int)SH, (int)SW, (int)PH, (int)PW, OH, OW,
                    (int)dcol.size(1), stream());
  return dx;
}

// small-image fused conv forward: x image staged in LDS, w tiles
// double-buffered, y written once.  Returns false if shape not eligible.
bool conv_fwd_small(at::Tensor x, at::Tensor w,
                    c10::optional<at::Tensor> bias, at::Tensor y, int64_t KH,
                    int64_t KW, int64_t SH, int64_t SW, int64_t PH,
                    int64_t PW, bool relu) {
  check_bf16(x, "x");
  check_bf16(w, "w");
  check_bf16(y, "y");
  const int B = (int)x.size(0), H = (int)x.size(1), W = (int)x.size(2),
            C = (int)x.size(3);
  const int OH = (H + 2 * (int)PH - (int)KH) / (int)SH + 1;
  const int OW = (W + 2 * (int)PW - (int)KW) / (int)SW + 1;
  const int outC = (int)y.size(1);
  TORCH_CHECK(y.size(0) == (long)B * OH * OW, "y rows");
  TORCH_CHECK(w.size(0) == outC && w.size(1) >= (long)KH * KW * C, "w shape");
  const void* bp = nullptr;
  if (bias) {
    TORCH_CHECK(bias->scalar_type() == at::kFloat && bias->numel() >= outC);
    bp = bias->data_ptr();
  }
  return lo::launch_conv_fwd_small(
      x.data_ptr(), w.data_ptr(), w.stride(0), bp, y.data_ptr(), y.stride(0),
      B, H, W, C, (int)KH, (int)KW, (int)SH, (int)SW, (int)PH, (int)PW, OH,
      OW, outC, relu ? 1 : 0, stream());
}

// 1-D (sequence) conv forward: W==1, KW==1, stride 1 — h-tiled x window
// in LDS, outC in 64-wide slices.
bool conv1d_fwd(at::Tensor x, at::Tensor w, c10::optional<at::Tensor> bias,
                at::Tensor y, int64_t KH, int64_t PH, bool relu) {
  check_bf16(x, "x");
  check_bf16(w, "w");
  check_bf16(y, "y");
  const int B = (int)x.size(0), H = (int)x.size(1), C = (int)x.size(3);
  TORCH_CHECK(x.size(2) == 1, "conv1d needs W==1");
  const int OH = H + 2 * (int)PH - (int)KH + 1;
  const int outC = (int)y.size(1);
  TORCH_CHECK(y.size(0) == (long)B * OH, "y rows");
  const void* bp = nullptr;
  if (bias) bp = bias->data_ptr();
  return lo::launch_conv1d_fwd(x.data_ptr(), w.data_ptr(), w.stride(0), bp,
                               y.data_ptr(), y.stride(0), B, H, C, (int)KH,
                               (int)PH, OH, outC, relu ? 1 : 0, stream());
}

// 1-D conv dX: h-tiled LDS fp32 accumulator, non-atomic RMW scatter.
bool conv1d_dx(at::Tensor dy2, at::Tensor wt, at::Tensor dx, int64_t KH,
               int64_t PH, bool accumulate) {
  check_bf16(dy2, "dy2");
  check_bf16(wt, "wt");
  check_bf16(dx, "dx");
  const int B = (int)dx.size(0), H = (int)dx.size(1), C = (int)dx.size(3);
  TORCH_CHECK(dx.size(2) == 1, "conv1d needs W==1");
  const int OH = H + 2 * (int)PH - (int)KH + 1;
  const int outC = (int)dy2.size(1);
  TORCH_CHECK(dy2.size(0) == (long)B * OH, "dy2 rows");
  return lo::launch_conv1d_dx(dy2.data_ptr(), dy2.stride(0), wt.data_ptr(),
                              wt.stride(0), dx.data_ptr(), B, H, C, (int)KH,
                              (int)PH, OH, outC, accumulate ? 1 : 0,
                              stream());
}

// C=1 conv dW: dY^T @ im2col(x) with x images LDS-resident; dw fp32
// accumulated with one atomicAdd per element per block (dw zeroed here).
bool conv_dw_small(at::Tensor dy2, at::Tensor x, at::Tensor dw, int64_t KH,
                   int64_t KW, int64_t SH, int64_t SW, int64_t PH, int64_t PW) {
  check_bf16(dy2, "dy2");
  check_bf16(x, "x");
  TORCH_CHECK(dw.scalar_type() == at::kFloat, "dw must be fp32");
  const int B = (int)x.size(0), H = (int)x.size(1), W = (int)x.size(2),
            C = (int)x.size(3);
  const int OH = (H + 2 * (int)PH - (int)KH) / (int)SH + 1;
  const int OW = (W + 2 * (int)PW - (int)KW) / (int)SW + 1;
  const int outC = (int)dy2.size(1);
  TORCH_CHECK(dy2.size(0) == (long)B * OH * OW, "dy2 rows");
  TORCH_CHECK(dw.size(0) == outC && dw.size(1) >= KH * KW * C, "dw shape");
  dw.zero_();  // harmless extra zero when ineligible (fallback re-zeroes)
  return lo::launch_conv_dw_smallc(dy2.data_ptr(), dy2.stride(0), x.data_ptr(),
                                   dw.data_ptr(), dw.stride(0), B, H, W, C,
                                   (int)KH, (int)KW, (int)SH, (int)SW,
                                   (int)PH, (int)PW, OH, OW, outC, stream());
}

bool conv_dw_c1(at::Tensor dy2, at::Tensor x, at::Tensor dw, int64_t KH,
                int64_t KW, int64_t SH, int64_t SW, int64_t PH, int64_t PW) {
  check_bf16(dy2, "dy2");
  check_bf16(x, "x");
  TORCH_CHECK(dw.scalar_type() == at::kFloat, "dw must be fp32");
  const int B = (int)x.size(0), H = (int)x.size(1), W = (int)x.size(2);
  TORCH_CHECK(x.size(3) == 1, "conv_dw_c1 needs C=1");
  const int OH = (H + 2 * (int)PH - (int)KH) / (int)SH + 1;
  const int OW = (W + 2 * (int)PW - (int)KW) / (int)SW + 1;
  const int outC = (int)dy2.size(1);
  TORCH_CHECK(dy2.size(0) == (long)B * OH * OW, "dy2 rows");
  TORCH_CHECK(dw.size(0) == outC && dw.size(1) >= KH * KW, "dw shape");
  dw.zero_();
  return lo::launch_conv_dw_c1(dy2.data_ptr(), dy2.stride(0), x.data_ptr(),
                               dw.data_ptr(), dw.stride(0), B, H, W, (int)KH,
                               (int)KW, (int)SH, (int)SW, (int)PH, (int)PW,
                               OH, OW, outC, stream());
}

// fused conv dX: dy2 [B*OH*OW, outC] @ wt[kpad, outC]^T scattered into
// dx [B,H,W,C] through an LDS fp32 accumulator (no dcol matrix).
// Returns false when the shape is not eligible (caller falls back).
bool conv_dx(at::Tensor dy2, at::Tensor wt, at::Tensor dx, int64_t KH,
             int64_t KW, int64_t SH, int64_t SW, int64_t PH, int64_t PW) {
  check_bf16(dy2, "dy2");
  check_bf16(wt, "wt");
  check_bf16(dx, "dx");
  const int B = (int)dx.size(0), H = (int)dx.size(1), W = (int)dx.size(2),
            C = (int)dx.size(3);
  const int OH = (H + 2 * (int)PH - (int)KH) / (int)SH + 1;
  const int OW = (W + 2 * (int)PW - (int)KW) / (int)SW + 1;
  const int outC = (int)dy2.size(1);
  TORCH_CHECK(dy2.size(0) == (long)B * OH * OW, "dy2 rows");
  TORCH_CHECK(wt.size(0) >= (long)KH * KW * C && wt.size(1) == outC, "wt shape");
  return lo::launch_conv_dx(dy2.data_ptr(), dy2.stride(0), wt.data_ptr(),
                            wt.stride(0), dx.data_ptr(), B, H, W, C, (int)KH,
                            (int)KW, (int)SH, (int)SW, (int)PH, (int)PW, OH,
                            OW, outC, stream());
}

std::vector<at::Tensor> maxpool_fwd(at::Tensor in, int64_t KH, int64_t KW,
                                    int64_t SH, int64_t SW, int64_t PH, int64_t PW,
                                    bool relu_sentinel = false) {
  check_bf16(in, "in");
  const int B = (int)in.size(0), H = (int)in.size(1), W = (int)in.size(2),
            C = (int)in.size(3);
  const int OH = (H + 2 * (int)PH - (int)KH) / (int)SH + 1;
  const int OW = (W + 2 * (int)PW - (int)KW) / (int)SW + 1;
  auto out = at::empty({B, OH, OW, C}, in.options());
  auto idx = at::empty({B, OH, OW, C}, in.options().dtype(at::kByte));
  lo::launch_maxpool_fwd(in.data_ptr(), out.data_ptr(), idx.data_ptr(), B, H, W, C,
                         (int)KH, (int)KW, (int)SH, (int)SW, (int)PH, (int)PW,
                         OH, OW, relu_sentinel ? 1 : 0, stream());
  return {out, idx};
}

at::Tensor maxpool_bwd(at::Tensor dy, at::Tensor idx, int64_t H, int64_t W,
                       int64_t KH, int64_t KW, int64_t SH, int64_t SW,
                       int64_t PH, int64_t PW, at::Tensor dx,
                       c10::optional<at::Tensor> relu_y) {
  check_bf16(dy, "dy");
  check_bf16(dx, "dx");
  const int B = (int)dy.size(0), OH = (int)dy.size(1), OW = (int)dy.size(2),
            C = (int)dy.size(3);
  const void* yp = nullptr;
  if (relu_y) {
    check_bf16(*relu_y, "relu_y");
    TORCH_CHECK(relu_y->numel() == dx.numel(), "relu_y shape");
    yp = relu_y->data_ptr();
  }
  lo::launch_maxpool_bwd(dy.data_ptr(), idx.data_ptr(), dx.data_ptr(), yp, B, (int)H,
                         (int)W, C, (int)KH, (int)KW, (int)SH, (int)SW,
                         (int)PH, (int)PW, OH, OW, stream());
  return dx;
}

// ----------------------------------------------------------- batchnorm ----
void bn_stats(at::Tensor x, at::Tensor sum, at::Tensor sumsq) {
  check_bf16(x, "x");
  check_f32(sum, "sum");
  check_f32(sumsq, "sumsq");
  const int C = (int)x.size(-1);
  TORCH_CHECK(C % 8 == 0 && sum.numel() == C && sumsq.numel() == C);
  lo::launch_bn_stats(x.data_ptr(), sum.data_ptr(), sumsq.data_ptr(),
                      x.numel() / C, C, stream());
}

void bn_fwd(at::Tensor x, at::Tensor y, at::Tensor mean, at::Tensor invstd,
            at::Tensor gamma, at::Tensor beta, bool relu,
            c10::optional<at::Tensor> residual = c10::nullopt) {
  check_bf16(x, "x");
  check_bf16(y, "y");
  const int C = (int)x.size(-1);
  const void* res = nullptr;
  if (residual.has_value()) {
    check_bf16(*residual, "residual");
    TORCH_CHECK(residual->numel() == x.numel(), "residual shape");
    res = residual->data_ptr();
  }
  lo::launch_bn_fwd(x.data_ptr(), y.data_ptr(), mean.data_ptr(),
                    invstd.data_ptr(), gamma.data_ptr(), beta.data_ptr(),
                    res, x.numel() / C, C, relu ? 1 : 0, stream());
}

void bn_bwd_reduce(at::Tensor dy, at::Tensor y, at::Tensor x, at::Tensor mean,
                   at::Tensor invstd, at::Tensor dbeta, at::Tensor dgamma,
                   bool relu) {
  check_bf16(dy, "dy");
  const int C = (int)x.size(-1);
  lo::launch_bn_bwd_reduce(dy.data_ptr(), y.data_ptr(), x.data_ptr(),
                           mean.data_ptr(), invstd.data_ptr(), dbeta.data_ptr(),
                           dgamma.data_ptr(), x.numel() / C, C, relu ? 1 : 0,
                           stream());
}

void bn_bwd_dx(at::Tensor dy, at::Tensor y, at::Tensor x, at::Tensor dx,
               at::Tensor mean, at::Tensor invstd, at::Tensor gamma,
               at::Tensor dbeta, at::Tensor dgamma, bool relu) {
  check_bf16(dx, "dx");
  const int C = (int)x.size(-1);
  lo::launch_bn_bwd_dx(dy.data_ptr(), y.data_ptr(), x.data_ptr(), dx.data_ptr(),
                       mean.data_ptr(), invstd.data_ptr(), gamma.data_ptr(),
                       dbeta.data_ptr(), dgamma.data_ptr(), x.numel() / C, C,
                       relu ? 1 : 0, stream());
}

void bn_finalize_stats(at::Tensor scratch, at::Tensor mean, at::Tensor invstd,
                       int64_t M,
                       c10::optional<at::Tensor> rmean,
                       c10::optional<at::Tensor> rvar,
                       double momentum, double eps) {
  check_f32(scratch, "scratch");
  check_f32(mean, "mean");
  lo::launch_bn_finalize_stats(
      scratch.data_ptr(), mean.data_ptr(), invstd.data_ptr(),
      rmean ? rmean->data_ptr() : nullptr,
      rvar ? rvar->data_ptr() : nullptr,
      1.f / (float)M, (float)momentum, (float)eps,
      (int)mean.numel(), stream());
}

void add_relu(at::Tensor a, at::Tensor b, at::Tensor z, bool relu) {
  check_bf16(a, "a");
  check_bf16(b, "b");
  check_bf16(z, "z");
  TORCH_CHECK(a.numel() == b.numel() && a.numel() == z.numel() &&
              a.numel() % 8 == 0);
  lo::launch_add_relu(a.data_ptr(), b.data_ptr(), z.data_ptr(), a.numel(),
                      relu ? 1 : 0, stream());
}

at::Tensor avgpool_global(at::Tensor x, at::Tensor out) {
  check_bf16(x, "x");
  check_bf16(out, "out");
  const int B = (int)x.size(0);
  const int C = (int)x.size(-1);
  const int HW = (int)(x.numel() / ((long)B * C));
  lo::launch_avgpool_global(x.data_ptr(), out.data_ptr(), B, HW, C, stream());
  return out;
}

at::Tensor avgpool_global_bwd(at::Tensor dy, at::Tensor dx) {
  check_bf16(dy, "dy");
  check_bf16(dx, "dx");
  const int B = (int)dy.size(0);
  const int C = (int)dy.size(-1);
  const int HW = (int)(dx.numel() / ((long)B * C));
  lo::launch_avgpool_global_bwd(dy.data_ptr(), dx.data_ptr(), B, HW, C, stream());
  return dx;
}

at::Tensor relu_bwd(at::Tensor dy, at::Tensor y, at::Tensor dx) {
  check_bf16(dy, "dy");
  check_bf16(y, "y");
  check_bf16(dx, "dx");
  TORCH_CHECK(dy.numel() == y.numel() && dy.numel() == dx.numel());
  TORCH_CHECK(dy.numel() % 8 == 0, "relu_bwd needs 8-aligned numel");
  lo::launch_relu_bwd(dy.data_ptr(), y.data_ptr(), dx.data_ptr(), dy.numel(),
                      stream());
  return dx;
}

void sgd_step(at::Tensor master, at::Tensor grad, at::Tensor mom, at::Tensor mirror,
              double lr, double mu, double wd, double gscale) {
  check_f32(master, "master");
  check_f32(grad, "grad");
  check_f32(mom, "mom");
  check_bf16(mirror, "mirror");
  TORCH_CHECK(master.numel() == grad.numel() && master.numel() == mom.numel() &&
              master.numel() == mirror.numel());
  TORCH_CHECK(master.numel() % 4 == 0, "arena must be 4-aligned");
  lo::launch_sgd(master.data_ptr(), grad.data_ptr(), mom.data_ptr(),
                 mirror.data_ptr(), master.numel(), (float)lr, (float)mu,
                 (float)wd, (float)gscale, stream());
}

void adam_step(at::Tensor master, at::Tensor grad, at::Tensor m1, at::Tensor m2,
               at::Tensor mirror, at::Tensor step_dev, double lr, double b1,
               double b2, double eps, double wd, double gscale) {
  check_f32(master, "master");
  check_f32(grad, "grad");
  check_f32(m1, "m1");
  check_f32(m2, "m2");
  check_bf16(mirror, "mirror");
  TORCH_CHECK(step_dev.scalar_type() == at::kInt && step_dev.is_cuda(),
              "step_dev must be int32 on GPU");
  TORCH_CHECK(master.numel() % 4 == 0, "arena must be 4-aligned");
  lo::launch_adam(master.data_ptr(), grad.data_ptr(), m1.data_ptr(), m2.data_ptr(),
                  mirror.data_ptr(), step_dev.data_ptr(), nullptr, 0, 0,
                  master.numel(), (float)lr, (float)b1, (float)b2, (float)eps,
                  (float)wd, (float)gscale, stream());
}

// where a tensor's rows (one, if it is flat) lie, in bytes; none: no rows
struct Span {
  int64_t at = 0, width = 0, row = 0, rows = 0, end = 0;
  const char* name = "";
  Span() = default;
  Span(const at::Tensor& t, const char* name_) : name(name_) {
    if (t.numel() == 0) return;
    const auto sizes = t.sizes();
    const int64_t size = t.itemsize();
    const bool flat = sizes.size() != 2;  // and contiguous
    at = (int64_t)t.const_data_ptr();
    width = (flat ? t.numel() : sizes[1]) * size;
    row = flat || sizes[0] < 2 ? 0 : t.strides()[0] * size;
    rows = row ? sizes[0] : 1;
    end = at + (rows - 1) * row + width;
  }
  Span(const c10::optional<at::Tensor>& t, const char* name_) {
    if (t) *this = Span(*t, name_);
  }
};

// whether some row of a shares memory with v, which has one row
bool touches(const Span& a, const Span& v) {
  if (a.rows == 0 || v.rows == 0 || a.end <= v.at || v.end <= a.at) return false;
  // the first row that ends behind v's start
  const int64_t gap = v.at - a.at - a.width;
  const int64_t r = a.row && gap >= 0 ? gap / a.row + 1 : 0;
  return a.at + r * a.row < v.end;
}

// an arena's tensors, all contiguous
void check_arena(std::initializer_list<Span> ts) {
  for (auto a = ts.begin(); a != ts.end(); ++a)
    for (auto b = ts.begin(); b != a; ++b)
      TORCH_CHECK(!touches(*a, *b), "the arena's ", b->name, " and ", a->name,
                  " must not share memory");
}

// what an object keeps may be used on another stream than it was made on: its
// memory is not given to others before this stream is done with it
void used_here(std::initializer_list<at::Tensor> kept) {
  for (const at::Tensor& t : kept) {
    const c10::impl::VirtualGuardImpl impl(t.device().type());
    if (t.numel()) t.record_stream(impl.getStream(t.device()));
  }
}

// the same step on parts of the arena only: ranges [k, 2] (start, end), int64
// on the GPU, the longest of them long
void adam_ranges(at::Tensor master, at::Tensor grad, at::Tensor m1,
                 at::Tensor m2, at::Tensor mirror, at::Tensor step_dev,
                 at::Tensor ranges, int64_t longest, double lr, double b1,
                 double b2, double eps, double wd, double gscale) {
  check_f32(master, "master");
  check_f32(grad, "grad");
  check_f32(m1, "m1");
  check_f32(m2, "m2");
  check_bf16(mirror, "mirror");
  for (const auto& t : {grad, m1, m2, mirror})
    TORCH_CHECK(t.numel() == master.numel() && t.device() == master.device(),
                "the arena's tensors must match");
  TORCH_CHECK(master.numel() % 4 == 0, "arena must be 4-aligned");
  TORCH_CHECK(step_dev.scalar_type() == at::kInt &&
                  step_dev.device() == master.device(),
              "step_dev must be int32 on the arena's GPU");
  TORCH_CHECK(ranges.scalar_type() == at::kLong && ranges.is_contiguous() &&
                  ranges.dim() == 2 && ranges.size(1) == 2 &&
                  ranges.device() == master.device() &&
                  ranges.size(0) <= 65535,
              "ranges must be int64 [k, 2] on the arena's GPU");
  TORCH_CHECK(step_dev.numel() == 1, "step_dev must hold one value");
  check_arena({{master, "master"}, {grad, "grad"}, {m1, "m1"}, {m2, "m2"},
               {mirror, "mirror"}});
  if (ranges.size(0) == 0 || longest <= 0) return;
  const c10::DeviceGuard guard(master.device());
  used_here({ranges});
  lo::launch_adam(master.data_ptr(), grad.data_ptr(), m1.data_ptr(), m2.data_ptr(),
                  mirror.data_ptr(), step_dev.data_ptr(), ranges.data_ptr(),
                  (int)ranges.size(0), longest, master.numel(), (float)lr,
                  (float)b1, (float)b2, (float)eps, (float)wd, (float)gscale,
                  stream());
}

at::Tensor colsum(at::Tensor dy, at::Tensor out,
                  c10::optional<at::Tensor> mask = c10::nullopt) {
  check_bf16(dy, "dy");
  check_f32(out, "out");
  TORCH_CHECK(dy.dim() == 2 && out.numel() == dy.size(1));
  if (mask) {
    TORCH_CHECK(mask->scalar_type() == at::kByte && mask->is_contiguous() &&
                mask->numel() == dy.numel(), "mask: u8, same shape");
    TORCH_CHECK(dy.size(1) <= 256, "masked colsum: N <= 256");
    lo::launch_colsum_masked(dy.data_ptr(), mask->data_ptr(), out.data_ptr(),
                             dy.size(0), (int)dy.size(1), dy.size(1),
                             stream());
    return out;
  }
  lo::launch_colsum(dy.data_ptr(), out.data_ptr(), dy.size(0), (int)dy.size(1),
                    dy.size(1), stream());
  return out;
}

at::Tensor argmax_rows(at::Tensor x, int64_t cvalid) {
  check_bf16(x, "x");
  TORCH_CHECK(x.dim() == 2);
  auto out = at::empty({x.size(0)}, x.options().dtype(at::kInt));
  lo::launch_argmax_rows(x.data_ptr(), out.data_ptr(), x.size(0), (int)x.size(1),
                         (int)cvalid, x.size(1), stream());
  return out;
}

at::Tensor accuracy_count(at::Tensor pred, at::Tensor label) {
  TORCH_CHECK(pred.scalar_type() == at::kInt && label.scalar_type() == at::kLong);
  auto out = at::zeros({1}, pred.options());
  lo::launch_accuracy_count(pred.data_ptr(), label.data_ptr(), out.data_ptr(),
                            pred.numel(), stream());
  return out;
}

// fused softmax-CE: writes dlogits; returns nothing (loss_sum/correct are
// caller-provided accumulators so one graph-captured step reuses them)
void softmax_ce(at::Tensor logits, at::Tensor labels, at::Tensor dlogits,
                c10::optional<at::Tensor> loss_sum, c10::optional<at::Tensor> correct,
                int64_t cvalid, double gscale) {
  check_bf16(logits, "logits");
  check_bf16(dlogits, "dlogits");
  TORCH_CHECK(labels.scalar_type() == at::kLong && labels.is_cuda());
  TORCH_CHECK(logits.dim() == 2 && logits.sizes() == dlogits.sizes());
  TORCH_CHECK(cvalid <= logits.size(1));
  TORCH_CHECK(cvalid <= 32 || logits.size(1) % 8 == 0,
              "wave path needs 8-aligned C");
  void* lp = nullptr;
  void* cp = nullptr;
  if (loss_sum.has_value()) { check_f32(*loss_sum, "loss_sum"); lp = loss_sum->data_ptr(); }
  if (correct.has_value()) { cp = correct->data_ptr(); }
  lo::launch_softmax_ce(logits.data_ptr(), labels.data_ptr(), dlogits.data_ptr(),
                        lp, cp, logits.size(0), (int)logits.size(1), (int)cvalid,
                        (float)gscale, stream());
}

void tree_hist(at::Tensor binned, at::Tensor node_of, at::Tensor grad,
               at::Tensor hess, at::Tensor hist, int64_t n_nodes, int64_t n_bins,
               double gbound = 0.0, double hbound = 0.0) {
  TORCH_CHECK(binned.is_cuda() && binned.scalar_type() == at::kByte &&
              binned.is_contiguous(), "binned must be contiguous u8 GPU");
  TORCH_CHECK(node_of.scalar_type() == at::kInt && node_of.is_contiguous());
  check_f32(grad, "grad");
  check_f32(hess, "hess");
  check_f32(hist, "hist");
  const long N = binned.size(0);
  const int F = (int)binned.size(1);
  TORCH_CHECK(node_of.numel() == N && grad.numel() == N && hess.numel() == N);
  TORCH_CHECK(hist.numel() == n_nodes * F * n_bins * 2, "hist size");
  lo::launch_tree_hist(binned.data_ptr(), node_of.data_ptr(), grad.data_ptr(),
                       hess.data_ptr(), hist.data_ptr(), N, F, (int)n_nodes,
                       (int)n_bins, gbound, hbound, stream());
}

at::Tensor embedding_fwd(at::Tensor ids, at::Tensor table, at::Tensor out) {
  TORCH_CHECK(ids.scalar_type() == at::kLong && ids.is_cuda() && ids.is_contiguous());
  check_bf16(table, "table");
  check_bf16(out, "out");
  const int dim = (int)table.size(1);
  TORCH_CHECK(dim % 8 == 0, "embedding dim must be 8-aligned");
  TORCH_CHECK(out.numel() == ids.numel() * dim, "out shape");
  lo::launch_embedding_fwd(ids.data_ptr(), table.data_ptr(), out.data_ptr(),
                           ids.numel(), dim, stream());
  return out;
}

void embedding_bwd(at::Tensor ids, at::Tensor dy, at::Tensor gtable) {
  TORCH_CHECK(ids.scalar_type() == at::kLong && ids.is_cuda() && ids.is_contiguous());
  check_bf16(dy, "dy");
  check_f32(gtable, "gtable");
  const int dim = (int)gtable.size(1);
  TORCH_CHECK(dy.numel() == ids.numel() * dim, "dy shape");
  lo::launch_embedding_bwd(ids.data_ptr(), dy.data_ptr(), gtable.data_ptr(),
                           ids.numel(), dim, stream());
}

// ----------------------------------------------------------- layernorm ----
int float_code(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be on GPU");
  switch (t.scalar_type()) {
    case at::kBFloat16: return 0;
    case at::kHalf: return 1;
    case at::kFloat: return 2;
    default: TORCH_CHECK(false, name, " must be bf16, fp16 or fp32");
  }
}

void check_launch(const char* name) {
  const hipError_t e = hipGetLastError();
  TORCH_CHECK(e == hipSuccess, name, ": ", hipGetErrorString(e));
}

// rows of like's shape, type and device; the row stride is free. out: written
// to, so its rows may not overlap
void check_rows(const at::Tensor& t, const at::Tensor& like, const char* name,
                bool out) {
  TORCH_CHECK(t.dim() == 2 && t.sizes() == like.sizes(), name,
              " must have the input's shape");
  TORCH_CHECK(t.scalar_type() == like.scalar_type(), name,
              " must have the input's type");
  TORCH_CHECK(t.device() == like.device(), name,
              " must be on the input's device");
  TORCH_CHECK(t.size(1) <= 1 || t.stride(1) == 1, name,
              " must be contiguous along its columns");
  TORCH_CHECK(t.size(0) <= 1 || t.stride(0) >= (out ? t.size(1) : 0), name,
              out ? " must not overlap itself" : " has a negative row stride");
}

// out may be an input, or lie beside it (columns of one wider buffer, say), but
// not be a part of it: other blocks would read rows that are written already
void check_apart(const at::Tensor& out, const at::Tensor& in,
                 const char* name) {
  if (out.numel() == 0) return;
  const int64_t rows = out.size(0), cols = out.size(1), size = out.itemsize();
  const int64_t ldo = rows > 1 ? out.stride(0) : cols;
  const int64_t ldi = rows > 1 ? in.stride(0) : cols;
  const auto a = (int64_t)out.data_ptr(), b = (int64_t)in.data_ptr();
  if (a == b && ldo == ldi) return;
  const int64_t end_a = a + ((rows - 1) * ldo + cols) * size;
  const int64_t end_b = b + ((rows - 1) * ldi + cols) * size;
  if (end_a <= b || end_b <= a) return;
  const int64_t row = ldo * size, off = ((a - b) % row + row) % row;
  TORCH_CHECK(ldo == ldi && off >= cols * size && off <= row - cols * size,
              name, " may be an input, but not overlap one in part");
}

void check_vec(const at::Tensor& t, const at::Tensor& like, int64_t n,
               const char* name) {
  check_f32(t, name);
  TORCH_CHECK(t.device() == like.device(), name,
              " must be on the input's device");
  TORCH_CHECK(t.numel() == n, name, " must hold ", n, " values");
}

// statistics and parameters' gradients share no memory with anything else, nor
// do the activations' outputs with statistics and parameters
void check_own(const Span& vec_out0, const Span& vec_out1,
               std::initializer_list<Span> vecs,
               std::initializer_list<Span> outs,
               std::initializer_list<Span> ins) {
  auto apart = [](const Span& a, const Span& b) {
    TORCH_CHECK(!touches(a, b), a.name, " and ", b.name,
                " must not share memory");
  };
  apart(vec_out0, vec_out1);
  for (const auto* others : {&vecs, &outs, &ins})
    for (const Span& o : *others) apart(o, vec_out0), apart(o, vec_out1);
  for (const Span& o : outs)
    for (const Span& v : vecs) apart(o, v);
}

constexpr int64_t kLayerNormCols = 32768;  // a row fits one block's registers

void check_layernorm(const at::Tensor& x) {
  TORCH_CHECK(x.dim() == 2, "x must be [rows, cols]");
  TORCH_CHECK(x.size(1) >= 1 && x.size(1) <= kLayerNormCols,
              "layer norm takes 1 to ", kLayerNormCols, " columns");
}

void layernorm_fwd(at::Tensor x, at::Tensor gamma, at::Tensor beta, double eps,
                   at::Tensor out, c10::optional<at::Tensor> mean,
                   c10::optional<at::Tensor> invstd,
                   c10::optional<at::Tensor> residual,
                   c10::optional<at::Tensor> sum_out) {
  const int code = float_code(x, "x");
  check_layernorm(x);
  const int64_t rows = x.size(0), cols = x.size(1);
  check_rows(x, x, "x", false);
  check_rows(out, x, "out", true);
  check_vec(gamma, x, cols, "gamma");
  check_vec(beta, x, cols, "beta");
  TORCH_CHECK(mean.has_value() == invstd.has_value(),
              "mean and invstd come together");
  if (mean) {
    check_vec(*mean, x, rows, "mean");
    check_vec(*invstd, x, rows, "invstd");
  }
  TORCH_CHECK(!sum_out || residual, "sum_out needs a residual");
  if (residual) check_rows(*residual, x, "residual", false);
  check_apart(out, x, "out");
  if (residual) check_apart(out, *residual, "out");
  if (sum_out) {
    check_rows(*sum_out, x, "sum_out", true);
    TORCH_CHECK(rows == 0 || sum_out->data_ptr() != out.data_ptr(),
                "out and sum_out must be two tensors");
    check_apart(*sum_out, x, "sum_out");
    check_apart(*sum_out, *residual, "sum_out");
    check_apart(*sum_out, out, "sum_out");
  }
  check_own({mean, "mean"}, {invstd, "invstd"},
            {{gamma, "gamma"}, {beta, "beta"}},
            {{out, "out"}, {sum_out, "sum_out"}},
            {{x, "x"}, {residual, "residual"}});
  if (rows == 0) return;
  const c10::DeviceGuard guard(x.device());
  lo::launch_layernorm_fwd(
      code, x.data_ptr(), x.stride(0), residual ? residual->data_ptr() : nullptr,
      residual ? residual->stride(0) : 0, gamma.data_ptr<float>(),
      beta.data_ptr<float>(), out.data_ptr(), out.stride(0),
      sum_out ? sum_out->data_ptr() : nullptr, sum_out ? sum_out->stride(0) : 0,
      mean ? mean->data_ptr<float>() : nullptr,
      invstd ? invstd->data_ptr<float>() : nullptr, rows, (int)cols,
      (float)eps, stream());
  check_launch("layernorm_fwd");
}

void layernorm_bwd(at::Tensor dy, at::Tensor x, at::Tensor mean,
                   at::Tensor invstd, at::Tensor gamma, at::Tensor dgamma,
                   at::Tensor dbeta, at::Tensor dx,
                   c10::optional<at::Tensor> dskip) {
  const int code = float_code(x, "x");
  check_layernorm(x);
  const int64_t rows = x.size(0), cols = x.size(1);
  check_rows(x, x, "x", false);
  check_rows(dy, x, "dy", false);
  check_rows(dx, x, "dx", true);
  if (dskip) check_rows(*dskip, x, "dskip", false);
  check_apart(dx, x, "dx");
  check_apart(dx, dy, "dx");
  if (dskip) check_apart(dx, *dskip, "dx");
  check_vec(mean, x, rows, "mean");
  check_vec(invstd, x, rows, "invstd");
  check_vec(gamma, x, cols, "gamma");
  check_vec(dgamma, x, cols, "dgamma");
  check_vec(dbeta, x, cols, "dbeta");
  check_own({dgamma, "dgamma"}, {dbeta, "dbeta"},
            {{gamma, "gamma"}, {mean, "mean"}, {invstd, "invstd"}},
            {{dx, "dx"}}, {{dy, "dy"}, {x, "x"}, {dskip, "dskip"}});
  const c10::DeviceGuard guard(x.device());
  if (rows == 0) {
    dgamma.zero_();
    dbeta.zero_();
    return;
  }
  at::Tensor part;
  const int n = lo::layernorm_bwd_parts(code, rows, (int)cols);
  if (n) part = at::empty({n, 2, cols}, gamma.options());
  lo::launch_layernorm_bwd(
      code, dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0),
      dskip ? dskip->data_ptr() : nullptr, dskip ? dskip->stride(0) : 0,
      mean.data_ptr<float>(), invstd.data_ptr<float>(),
      gamma.data_ptr<float>(), dx.data_ptr(), dx.stride(0),
      n ? part.data_ptr<float>() : nullptr, dgamma.data_ptr<float>(),
      dbeta.data_ptr<float>(), rows, (int)cols, stream());
  check_launch("layernorm_bwd");
}

// -------------------------------------------- Newton-Schulz and Muon ----
// G [batch, rows, cols] -> out
void orthogonalize(at::Tensor g, at::Tensor out, std::vector<double> coeffs,
                   double eps) {
  const int code = float_code(g, "g");
  TORCH_CHECK(g.dim() == 3 && g.is_contiguous(),
              "g must be contiguous [batch, rows, cols]");
  TORCH_CHECK(out.sizes() == g.sizes() && out.is_contiguous() &&
                  out.scalar_type() == g.scalar_type() &&
                  out.device() == g.device(),
              "out must be contiguous and of g's shape, type and device");
  const int64_t rows = g.size(1), cols = g.size(2);
  TORCH_CHECK(rows <= lo::kNsSide && cols <= lo::kNsSide, "sides end at ", lo::kNsSide);
  TORCH_CHECK(eps >= 0, "eps must not be negative");
  const auto st = lo::ns_steps(coeffs);
  if (g.numel() == 0) return;
  check_apart(out.view({1, -1}), g.view({1, -1}), "out");
  const c10::DeviceGuard guard(g.device());
  auto mats = lo::ns_plan({{rows, cols}}, g.size(0));
  const lo::NsInput in{g.data_ptr(), nullptr, 1.f, 0.f, 0};
  const lo::NsOutput o{out.data_ptr(), nullptr, nullptr, 0.f, 0.f};
  const int shortest = (int)std::min(rows, cols);
  const int longest = (int)std::max(rows, cols);
  if (lo::ns_fit_block(shortest, longest) &&
      (int)st.size() <= lo::kNsSmallSteps) {
    lo::NsGroup ng{};
    ng.one = mats[0];
    ng.src_step = rows * cols;
    const int64_t most = 1 << 22;  // blocks of 512 threads in one launch
    for (int64_t b0 = 0; b0 < g.size(0); b0 += most) {
      ng.count = (int)std::min(most, g.size(0) - b0);
      ng.one.src = b0 * rows * cols;
      lo::launch_newton_schulz_small(ng, shortest, longest, code, in, st.data(),
                                     (int)st.size(), (float)eps, o, stream());
      check_launch("orthogonalize");
    }
    return;
  }
  lo::NsNeeds n;
  lo::ns_place(mats, n);
  // at most 4 GiB of workspace beyond one matrix's own
  const int64_t most = std::max<int64_t>(1, (int64_t(1) << 31) / n.halfs);
  const int64_t group = std::min(g.size(0), most);
  auto bytes = g.options().dtype(at::kByte);
  auto ws = at::empty({group * n.halfs * 2}, bytes);
  auto sums = at::empty({group * n.chunks * 8}, bytes);
  auto parts = at::empty({group * n.parts * 4}, bytes);
  auto slots = at::empty({group * n.slots * 4}, bytes);
  lo::NsGroup ng{};
  ng.one = mats[0];
  ng.src_step = rows * cols;
  ng.ws_step = n.halfs;
  ng.sum_step = (int)n.chunks;
  ng.chunks = (int)n.chunks;
  ng.splits = (int)n.splits;
  ng.ws = ws.data_ptr();
  ng.sums = (double*)sums.data_ptr();
  ng.parts = (float*)parts.data_ptr();
  ng.slots = (unsigned*)slots.data_ptr();
  ng.slot_step = (int)n.slots;
  ng.part_step = n.parts;
  for (int k = 0; k < lo::NS_KINDS; ++k) {
    ng.kinds[k] = (int)n.kinds[k];
    ng.tile[k] = lo::ns_tile(mats, k);
  }
  for (int64_t b0 = 0; b0 < g.size(0); b0 += group) {
    const int64_t count = std::min(group, g.size(0) - b0);
    ng.count = (int)count;
    ng.all_chunks = n.chunks * count;
    ng.all_splits = n.splits * count;
    ng.all_slots = (int)(n.slots * count);
    for (int k = 0; k < lo::NS_KINDS; ++k) ng.all_kinds[k] = n.kinds[k] * count;
    ng.one.src = b0 * rows * cols;
    lo::launch_newton_schulz(ng, code, in, st.data(), (int)st.size(),
                             (float)eps, o, stream());
    check_launch("orthogonalize");
  }
}

// tables and workspace of the Muon steps over one arena's matrices
struct MuonPlan {
  at::Tensor table, ws, sums, parts, slots;
  lo::NsGroup g{};
  int64_t numel;
  int shortest = 0, longest = 0;  // the largest short and long sides

  // views: (offset, rows, cols) in ascending order; gains: the factors on the
  // learning rate
  MuonPlan(std::vector<std::array<int64_t, 3>> views, std::vector<double> gains,
           int64_t numel_, at::Device device)
      : numel(numel_) {
    TORCH_CHECK(device.is_cuda(), "the plan's device must be a GPU");
    TORCH_CHECK(!views.empty(), "a Muon plan needs a matrix");
    TORCH_CHECK(gains.size() == views.size(), "a gain for each matrix");
    int64_t end = 0;
    std::vector<std::pair<int64_t, int64_t>> sides;
    for (const auto& v : views) {
      TORCH_CHECK(v[0] >= end && v[0] % 8 == 0, "matrices must start on a "
                  "multiple of 8 elements and not overlap");
      TORCH_CHECK(v[1] >= 1 && v[2] >= 1 && v[1] <= lo::kNsSide &&
                      v[2] <= lo::kNsSide,
                  "matrix sides must be 1 to ", lo::kNsSide);
      end = v[0] + v[1] * v[2];
      sides.emplace_back(v[1], v[2]);
    }
    TORCH_CHECK(end <= numel, "a matrix ends outside the arena");
    const c10::DeviceGuard guard(device);
    auto mats = lo::ns_plan(sides, 1);
    lo::NsNeeds n;
    lo::ns_place(mats, n);
    for (size_t i = 0; i < mats.size(); ++i) {
      mats[i].src = views[i][0];
      mats[i].gain = (float)gains[i];
    }
    for (const lo::NsMat& m : mats) {
      shortest = std::max(shortest, std::min(m.rows, m.cols));
      longest = std::max(longest, std::max(m.rows, m.cols));
    }
    std::vector<lo::NsBlock> chunks, splits;
    for (int i = 0; i < (int)mats.size(); ++i) {
      const lo::NsMat& m = mats[i];
      for (int at = 0; at < m.chunks; ++at) chunks.push_back({i, at});
      for (int at = 0; at < m.mp / 64 * (m.np / 64); ++at)
        splits.push_back({i, at});
    }
    // one table of them all, each part on a line of its own
    std::vector<uint8_t> host;
    auto put = [&](const auto& v) {
      const size_t at = host.size(), bytes = v.size() * sizeof(v[0]);
      host.resize(at + (bytes + 63) / 64 * 64);
      std::memcpy(host.data() + at, v.data(), bytes);
      return at;
    };
    const size_t at_mats = put(mats), at_chunks = put(chunks),
                 at_splits = put(splits);
    size_t at_tasks[lo::NS_KINDS];
    for (int k = 0; k < lo::NS_KINDS; ++k) at_tasks[k] = put(lo::ns_tasks(mats, k));
    table = at::empty({(int64_t)host.size()},
                      at::TensorOptions(at::kByte).device(device));
    table.copy_(at::from_blob(host.data(), {(int64_t)host.size()}, at::kByte));
    auto* d = table.data_ptr<uint8_t>();
    g.mats = (const lo::NsMat*)(d + at_mats);
    g.chunk_blocks = (const lo::NsBlock*)(d + at_chunks);
    g.split_blocks = (const lo::NsBlock*)(d + at_splits);
    for (int k = 0; k < lo::NS_KINDS; ++k)
      g.tasks[k] = (const lo::NsTask*)(d + at_tasks[k]);
    ws = at::empty({n.halfs * 2}, table.options());
    sums = at::empty({n.chunks * 8}, table.options());
    parts = at::empty({n.parts * 4}, table.options());
    slots = at::empty({n.slots * 4}, table.options());
    g.count = (int)mats.size();
    g.all_chunks = n.chunks;
    g.all_splits = n.splits;
    g.all_slots = (int)n.slots;
    for (int k = 0; k < lo::NS_KINDS; ++k) {
      g.all_kinds[k] = n.kinds[k];
      g.tile[k] = lo::ns_tile(mats, k);
    }
    g.ws = ws.data_ptr();
    g.sums = (double*)sums.data_ptr();
    g.parts = (float*)parts.data_ptr();
    g.slots = (unsigned*)slots.data_ptr();
  }

  void step(at::Tensor master, at::Tensor grad, at::Tensor mom,
            at::Tensor mirror, double lr, double mu, double wd, double gscale,
            bool nesterov, std::vector<double> coeffs, double eps) {
    check_f32(master, "master");
    check_f32(grad, "grad");
    check_f32(mom, "mom");
    check_bf16(mirror, "mirror");
    for (const auto& t : {master, grad, mom, mirror}) {
      TORCH_CHECK(t.numel() == numel, "the plan is for ", numel, " elements");
      TORCH_CHECK(t.device() == table.device(), "the plan is on ",
                  table.device());
    }
    check_arena({{master, "master"}, {grad, "grad"}, {mom, "mom"},
                 {mirror, "mirror"}});
    TORCH_CHECK(eps >= 0, "eps must not be negative");
    const auto st = lo::ns_steps(coeffs);
    const c10::DeviceGuard guard(table.device());
    used_here({table, ws, sums, parts, slots});
    const lo::NsInput in{grad.data_ptr(), mom.data_ptr<float>(), (float)gscale,
                         (float)mu, nesterov ? 1 : 0};
    const lo::NsOutput out{nullptr, master.data_ptr<float>(),
                           mirror.data_ptr(), (float)lr,
                           (float)(1.0 - lr * wd)};
    if (lo::ns_fit_block(shortest, longest) &&
        (int)st.size() <= lo::kNsSmallSteps)
      lo::launch_newton_schulz_small(g, shortest, longest, 2, in, st.data(),
                                     (int)st.size(), (float)eps, out, stream());
    else
      lo::launch_newton_schulz(g, 2, in, st.data(), (int)st.size(), (float)eps,
                               out, stream());
    check_launch("muon_step");
  }
};

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("gemm", &gemm, "bf16 MFMA GEMM (gfx950)",
        py::arg("A"), py::arg("B"), py::arg("C"), py::arg("bias") = py::none(),
        py::arg("ta") = false, py::arg("tb") = false, py::arg("epi") = 0,
        py::arg("splits") = 1, py::arg("stats") = py::none(),
        py::arg("addend") = py::none());
  m.def("gemm_conv_fwd", &gemm_conv_fwd);
  m.def("gemm_conv_dw", &gemm_conv_dw);
  m.def("mfma_probe", &mfma_probe);
  m.def("im2col", &im2col);
  m.def("conv_fwd_small", &conv_fwd_small, "small-image fused conv fwd");
  m.def("conv1d_fwd", &conv1d_fwd, "1-D conv fwd (h-tiled LDS window)");
  m.def("conv1d_dx", &conv1d_dx, "1-D conv dX (h-tiled LDS RMW)");
  m.def("conv_dw_c1", &conv_dw_c1, "C=1 conv dW (x LDS-resident)");
  m.def("conv_dw_small", &conv_dw_small,
        "small-image C%8==0 conv dW (x+dyT LDS-resident per image)");
  m.def("conv_dx", &conv_dx, "fused conv dX (LDS-accumulated scatter)");
  m.def("col2im", &col2im);
  m.def("maxpool_fwd", &maxpool_fwd, py::arg("in"), py::arg("KH"),
        py::arg("KW"), py::arg("SH"), py::arg("SW"), py::arg("PH"),
        py::arg("PW"), py::arg("relu_sentinel") = false);
  m.def("maxpool_bwd", &maxpool_bwd);
  m.def("relu_bwd", &relu_bwd);
  m.def("sgd_step", &sgd_step);
  m.def("adam_step", &adam_step);
  m.def("adam_ranges", &adam_ranges);
  m.def("colsum", &colsum, py::arg("dy"), py::arg("out"),
        py::arg("mask") = py::none());
  m.def("argmax_rows", &argmax_rows);
  m.def("accuracy_count", &accuracy_count);
  m.def("tree_hist", &tree_hist, py::arg("binned"), py::arg("node_of"),
        py::arg("grad"), py::arg("hess"), py::arg("hist"),
        py::arg("n_nodes"), py::arg("n_bins"),
        py::arg("gbound") = 0.0, py::arg("hbound") = 0.0);
  m.def("embedding_fwd", &embedding_fwd);
  m.def("bn_stats", &bn_stats);
  m.def("bn_fwd", &bn_fwd, py::arg("x"), py::arg("y"), py::arg("mean"),
        py::arg("invstd"), py::arg("gamma"), py::arg("beta"),
        py::arg("relu"), py::arg("residual") = py::none());
  m.def("bn_bwd_reduce", &bn_bwd_reduce);
  m.def("bn_bwd_dx", &bn_bwd_dx);
  m.def("bn_finalize_stats", &bn_finalize_stats, py::arg("scratch"),
        py::arg("mean"), py::arg("invstd"), py::arg("M"),
        py::arg("rmean") = py::none(), py::arg("rvar") = py::none(),
        py::arg("momentum") = 0.0, py::arg("eps") = 1e-5);
  m.def("layernorm_fwd", &layernorm_fwd, py::arg("x"), py::arg("gamma"),
        py::arg("beta"), py::arg("eps"), py::arg("out"),
        py::arg("mean") = py::none(), py::arg("invstd") = py::none(),
        py::arg("residual") = py::none(), py::arg("sum_out") = py::none());
  m.def("layernorm_bwd", &layernorm_bwd, py::arg("dy"), py::arg("x"),
        py::arg("mean"), py::arg("invstd"), py::arg("gamma"),
        py::arg("dgamma"), py::arg("dbeta"), py::arg("dx"),
        py::arg("dskip") = py::none());
  m.def("orthogonalize", &orthogonalize);
  py::class_<MuonPlan>(m, "MuonPlan")
      .def(py::init([](std::vector<std::array<int64_t, 3>> views,
                       std::vector<double> gains, int64_t numel,
                       const std::string& device) {
        return new MuonPlan(std::move(views), std::move(gains), numel,
                            at::Device(device));
      }))
      .def("step", &MuonPlan::step);
  m.def("add_relu", &add_relu);
  m.def("avgpool_global", &avgpool_global);
  m.def("avgpool_global_bwd", &avgpool_global_bwd);
  m.def("embedding_bwd", &embedding_bwd);
  m.def("softmax_ce", &softmax_ce,
        py::arg("logits"), py::arg("labels"), py::arg("dlogits"),
        py::arg("loss_sum") = py::none(), py::arg("correct") = py::none(),
        py::arg("cvalid") = 0, py::arg("gscale") = 1.0);
}
