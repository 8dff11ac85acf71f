// Layer norm over the last axis, forward and backward, for gfx950.
//
//   s  = x, or round_T(x + residual)
//   y  = (s - mean) * invstd * gamma + beta,  invstd = (var + eps)^-1/2
//   dx = invstd * (h - avg(h) - xhat * avg(h * xhat)) (+ dskip),  h = dy * gamma
//   dgamma = sum_rows dy * xhat,  dbeta = sum_rows dy
//
// Activations are bf16, fp16 or fp32 (T) with any row stride; statistics,
// parameters and their gradients are fp32.
//
// The bound is HBM traffic, so each array is touched once: a row lives in the
// registers of TPR threads (NV vectors of VE elements each, 16 bytes a load),
// mean and variance come from two reductions over those registers (the second
// over squared differences, so a large mean costs no digits), and the backward
// pass forms dx and its share of dgamma/dbeta from the same loads. A block
// walks rows blockIdx, blockIdx + grid, ... with gamma, beta and the two
// gradient sums in registers; the blocks' sums go to a [blocks, 2, cols]
// workspace that a second small kernel adds in a fixed order, so results do
// not depend on timing. With one block the sums are written directly.
//
// Columns need not be a multiple of VE: the vector that would cross the row's
// end is moved back to end with it, and the elements it shares with its
// neighbour (skip of them) count only there. gfx950 loads 16 bytes from any
// element-aligned address, so odd strides take the same path. A row's reads
// all come before its writes, so an output may be one of the inputs.

#include "lo_common.h"

namespace lo {

namespace {

template <typename T, int VE>
struct RowVec {
  typedef T type __attribute__((ext_vector_type(VE), aligned(sizeof(T))));
};
template <typename T>
struct RowVec<T, 1> {
  typedef T type;
};

template <int VE, typename V>
LO_DEVICE float elem(const V& v, int j) {
  if constexpr (VE == 1) return (float)v;
  else return (float)v[j];
}

template <int VE>
LO_DEVICE void load_f32(const float* __restrict__ p, float (&o)[VE]) {
  #pragma unroll
  for (int j = 0; j < VE; ++j) o[j] = p[j];
}

// sums over the TPR threads that share a row; every one of them gets both.
// For TPR > 64 the LDS slots alternate between calls, so one barrier per call
// is enough: a slot is rewritten two calls later, past the barrier that its
// last readers reach before the next call's.
template <int TPR>
LO_DEVICE void row_sum2(float& a, float& b, float* red, int& turn) {
  #pragma unroll
  for (int off = (TPR < 64 ? TPR : 64) / 2; off > 0; off >>= 1) {
    a += __shfl_xor(a, off);
    b += __shfl_xor(b, off);
  }
  if constexpr (TPR > 64) {
    constexpr int W = TPR / 64;
    float* slot = red + (turn & 1) * 2 * W;
    ++turn;
    if ((threadIdx.x & 63) == 0) {
      slot[threadIdx.x >> 6] = a;
      slot[W + (threadIdx.x >> 6)] = b;
    }
    __syncthreads();
    a = 0.f;
    b = 0.f;
    #pragma unroll
    for (int w = 0; w < W; ++w) {
      a += slot[w];
      b += slot[W + w];
    }
  }
}

constexpr int ln_block(int tpr) { return tpr > 256 ? tpr : 256; }

template <typename T, int VE, int TPR, int NV>
__global__ __launch_bounds__(ln_block(TPR)) void layernorm_fwd_kernel(
    const T* x, long ldx, const T* res, long ldr,
    const float* __restrict__ gamma, const float* __restrict__ beta,
    T* y, long ldy, T* sum, long lds, float* __restrict__ mean,
    float* __restrict__ invstd, long rows, int cols, float eps) {
  typedef typename RowVec<T, VE>::type V;
  constexpr int RPB = ln_block(TPR) / TPR;
  __shared__ float red[TPR > 64 ? 4 * (TPR / 64) : 1];
  const int t = threadIdx.x % TPR;
  const float n = (float)cols;
  int base[NV], skip[NV];
  float gm[NV][VE], bt[NV][VE];
  #pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c0 = (i * TPR + t) * VE;
    base[i] = min(c0, cols - VE);
    skip[i] = min(c0 - base[i], VE);
    load_f32<VE>(gamma + base[i], gm[i]);
    load_f32<VE>(beta + base[i], bt[i]);
  }
  int turn = 0;
  for (long r = (long)blockIdx.x * RPB + threadIdx.x / TPR; r < rows;
       r += (long)gridDim.x * RPB) {
    V xv[NV];
    #pragma unroll
    for (int i = 0; i < NV; ++i) xv[i] = *(const V*)(x + r * ldx + base[i]);
    if (res) {
      #pragma unroll
      for (int i = 0; i < NV; ++i) {
        const V rv = *(const V*)(res + r * ldr + base[i]);
        if constexpr (VE == 1) {
          xv[i] = (T)((float)xv[i] + (float)rv);
        } else {
          #pragma unroll
          for (int j = 0; j < VE; ++j)
            xv[i][j] = (T)((float)xv[i][j] + (float)rv[j]);
        }
      }
    }
    float s1 = 0.f, s2 = 0.f;
    #pragma unroll
    for (int i = 0; i < NV; ++i)
      #pragma unroll
      for (int j = 0; j < VE; ++j)
        s1 += j >= skip[i] ? elem<VE>(xv[i], j) : 0.f;
    row_sum2<TPR>(s1, s2, red, turn);
    const float mu = s1 / n;
    s1 = 0.f;
    s2 = 0.f;
    #pragma unroll
    for (int i = 0; i < NV; ++i)
      #pragma unroll
      for (int j = 0; j < VE; ++j) {
        const float d = elem<VE>(xv[i], j) - mu;
        s1 += j >= skip[i] ? d * d : 0.f;
      }
    row_sum2<TPR>(s1, s2, red, turn);
    const float is = 1.f / sqrtf(s1 / n + eps);
    #pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (skip[i] >= VE) continue;
      V o;
      if constexpr (VE == 1) {
        o = (T)(((float)xv[i] - mu) * is * gm[i][0] + bt[i][0]);
      } else {
        #pragma unroll
        for (int j = 0; j < VE; ++j)
          o[j] = (T)(((float)xv[i][j] - mu) * is * gm[i][j] + bt[i][j]);
      }
      *(V*)(y + r * ldy + base[i]) = o;
      if (sum) *(V*)(sum + r * lds + base[i]) = xv[i];
    }
    if (t == 0 && mean) {
      mean[r] = mu;
      invstd[r] = is;
    }
  }
}

// part: [gridDim.x, 2, cols] sums of dy * xhat and of dy, or null with one
// block, which then writes dgamma/dbeta itself
template <typename T, int VE, int TPR, int NV>
__global__ __launch_bounds__(ln_block(TPR)) void layernorm_bwd_kernel(
    const T* dy, long ldy, const T* x, long ldx,
    const T* skipg, long ldk, const float* __restrict__ mean,
    const float* __restrict__ invstd, const float* __restrict__ gamma,
    T* dx, long ldd, float* __restrict__ part, float* __restrict__ dgamma,
    float* __restrict__ dbeta, long rows, int cols) {
  typedef typename RowVec<T, VE>::type V;
  constexpr int RPB = ln_block(TPR) / TPR;
  __shared__ float red[TPR > 64 ? 4 * (TPR / 64) : 1];
  extern __shared__ __attribute__((aligned(16))) float acc[];  // [2][cols]
  const int t = threadIdx.x % TPR;
  const float n = (float)cols;
  int base[NV], skip[NV];
  float gm[NV][VE], dg[NV][VE] = {}, db[NV][VE] = {};
  #pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c0 = (i * TPR + t) * VE;
    base[i] = min(c0, cols - VE);
    skip[i] = min(c0 - base[i], VE);
    load_f32<VE>(gamma + base[i], gm[i]);
  }
  int turn = 0;
  for (long r = (long)blockIdx.x * RPB + threadIdx.x / TPR; r < rows;
       r += (long)gridDim.x * RPB) {
    V xv[NV], gv[NV], kv[NV];
    #pragma unroll
    for (int i = 0; i < NV; ++i) {
      xv[i] = *(const V*)(x + r * ldx + base[i]);
      gv[i] = *(const V*)(dy + r * ldy + base[i]);
      if (skipg) kv[i] = *(const V*)(skipg + r * ldk + base[i]);
    }
    const float mu = mean[r], is = invstd[r];
    float s1 = 0.f, s2 = 0.f;
    #pragma unroll
    for (int i = 0; i < NV; ++i)
      #pragma unroll
      for (int j = 0; j < VE; ++j) {
        const float g = j >= skip[i] ? elem<VE>(gv[i], j) : 0.f;
        const float xh = (elem<VE>(xv[i], j) - mu) * is;
        const float h = g * gm[i][j];
        s1 += h;
        s2 += j >= skip[i] ? h * xh : 0.f;
        db[i][j] += g;
        dg[i][j] += j >= skip[i] ? g * xh : 0.f;
      }
    row_sum2<TPR>(s1, s2, red, turn);
    const float c1 = s1 / n, c2 = s2 / n;
    #pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (skip[i] >= VE) continue;
      V o;
      #pragma unroll
      for (int j = 0; j < VE; ++j) {
        const float xh = (elem<VE>(xv[i], j) - mu) * is;
        float d = is * (elem<VE>(gv[i], j) * gm[i][j] - c1 - xh * c2);
        if (skipg) d += elem<VE>(kv[i], j);
        if constexpr (VE == 1) o = (T)d;
        else o[j] = (T)d;
      }
      *(V*)(dx + r * ldd + base[i]) = o;
    }
  }
  float* og = part ? part + (long)blockIdx.x * 2 * cols : dgamma;
  float* ob = part ? og + cols : dbeta;
  if constexpr (TPR >= ln_block(TPR)) {
    // one row group per block: each column has one owner
    #pragma unroll
    for (int i = 0; i < NV; ++i)
      #pragma unroll
      for (int j = 0; j < VE; ++j)
        if (j >= skip[i]) {
          og[base[i] + j] = dg[i][j];
          ob[base[i] + j] = db[i][j];
        }
  } else {
    // the wave's row groups join by shuffles, the waves one after the other
    #pragma unroll
    for (int off = 32; off >= TPR; off >>= 1)
      #pragma unroll
      for (int i = 0; i < NV; ++i)
        #pragma unroll
        for (int j = 0; j < VE; ++j) {
          dg[i][j] += __shfl_xor(dg[i][j], off);
          db[i][j] += __shfl_xor(db[i][j], off);
        }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int w = 0; w < (int)blockDim.x / 64; ++w) {
      if (w == wave && lane < TPR) {
        #pragma unroll
        for (int i = 0; i < NV; ++i)
          #pragma unroll
          for (int j = 0; j < VE; ++j)
            if (j >= skip[i]) {
              const int c = base[i] + j;
              acc[c] = (w ? acc[c] : 0.f) + dg[i][j];
              acc[cols + c] = (w ? acc[cols + c] : 0.f) + db[i][j];
            }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < cols; c += blockDim.x) {
      og[c] = acc[c];
      ob[c] = acc[cols + c];
    }
  }
}

// column sums of part [n, width]: 32 columns a block, 32 threads to a column
__global__ __launch_bounds__(1024) void layernorm_join_kernel(
    const float* __restrict__ part, float* __restrict__ dgamma,
    float* __restrict__ dbeta, int n, int cols) {
  __shared__ float s[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int width = 2 * cols;
  const int c = blockIdx.x * 32 + tx;
  float a = 0.f;
  if (c < width) {
    // eight loads on their way at a time
    for (int r0 = ty; r0 < n; r0 += 256) {
      float v[8];
      #pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = r0 + 32 * i;
        v[i] = r < n ? part[(long)r * width + c] : 0.f;
      }
      #pragma unroll
      for (int i = 0; i < 8; ++i) a += v[i];
    }
  }
  s[ty][tx] = a;
  __syncthreads();
  if (ty == 0 && c < width) {
    a = 0.f;
    #pragma unroll
    for (int i = 0; i < 32; ++i) a += s[i][tx];
    if (c < cols) dgamma[c] = a;
    else dbeta[c - cols] = a;
  }
}

template <typename T, int VE, int TPR, int NV>
struct LnConfig {
  static constexpr int rpb = ln_block(TPR) / TPR;
  static void fwd(const void* x, long ldx, const void* res, long ldr,
                  const float* gamma, const float* beta, void* y, long ldy,
                  void* sum, long lds, float* mean, float* invstd, long rows,
                  int cols, float eps, hipStream_t s) {
    const long grid = min((rows + rpb - 1) / rpb, 2048L);
    hipLaunchKernelGGL((layernorm_fwd_kernel<T, VE, TPR, NV>), dim3(grid),
                       dim3(ln_block(TPR)), 0, s, (const T*)x, ldx,
                       (const T*)res, ldr, gamma, beta, (T*)y, ldy, (T*)sum,
                       lds, mean, invstd, rows, cols, eps);
  }
  static int blocks(long rows) {
    const long most = TPR > 256 ? 512 : 1024;
    return (int)min((rows + rpb - 1) / rpb, most);
  }
  static void bwd(const void* dy, long ldy, const void* x, long ldx,
                  const void* skip, long ldk, const float* mean,
                  const float* invstd, const float* gamma, void* dx, long ldd,
                  float* part, float* dgamma, float* dbeta, long rows,
                  int cols, hipStream_t s) {
    const int grid = blocks(rows);
    const size_t lds = TPR < ln_block(TPR) ? 8ul * cols : 0;
    hipLaunchKernelGGL((layernorm_bwd_kernel<T, VE, TPR, NV>), dim3(grid),
                       dim3(ln_block(TPR)), lds, s, (const T*)dy, ldy,
                       (const T*)x, ldx, (const T*)skip, ldk, mean, invstd,
                       gamma, (T*)dx, ldd, grid > 1 ? part : nullptr, dgamma,
                       dbeta, rows, cols);
    if (grid > 1)
      hipLaunchKernelGGL(layernorm_join_kernel, dim3((2 * cols + 31) / 32),
                         dim3(1024), 0, s, part, dgamma, dbeta, grid, cols);
  }
};

// calls f(LnConfig<...>{}) with the threads and vectors a row of cols takes
template <typename T, typename F>
auto ln_pick(int cols, F f) {
  constexpr int VE = 16 / sizeof(T);
  if (cols < VE) return f(LnConfig<T, 1, 8, 1>{});
  const int nv = (cols + VE - 1) / VE;
  if (nv <= 1) return f(LnConfig<T, VE, 1, 1>{});
  if (nv <= 2) return f(LnConfig<T, VE, 2, 1>{});
  if (nv <= 4) return f(LnConfig<T, VE, 4, 1>{});
  if (nv <= 8) return f(LnConfig<T, VE, 8, 1>{});
  if (nv <= 16) return f(LnConfig<T, VE, 16, 1>{});
  if (nv <= 32) return f(LnConfig<T, VE, 32, 1>{});
  if (nv <= 64) return f(LnConfig<T, VE, 64, 1>{});
  if (nv <= 128) return f(LnConfig<T, VE, 64, 2>{});
  if (nv <= 256) return f(LnConfig<T, VE, 256, 1>{});
  if (nv <= 512) return f(LnConfig<T, VE, 256, 2>{});
  if (nv <= 1024) return f(LnConfig<T, VE, 1024, 1>{});
  if (nv <= 2048) return f(LnConfig<T, VE, 1024, 2>{});
  if constexpr (VE == 8) {
    return f(LnConfig<T, VE, 1024, 4>{});
  } else {
    if (nv <= 4096) return f(LnConfig<T, VE, 1024, 4>{});
    return f(LnConfig<T, VE, 1024, 8>{});
  }
}

template <typename F>
auto ln_typed(int dtype, int cols, F f) {
  if (dtype == 0) return ln_pick<bf16>(cols, f);
  if (dtype == 1) return ln_pick<_Float16>(cols, f);
  return ln_pick<float>(cols, f);
}

}  // namespace

// dtype: 0 bf16, 1 fp16, 2 fp32; 1 <= cols <= 32768, rows >= 1
void launch_layernorm_fwd(int dtype, const void* x, long ldx, const void* res,
                          long ldr, const float* gamma, const float* beta,
                          void* y, long ldy, void* sum, long lds, float* mean,
                          float* invstd, long rows, int cols, float eps,
                          hipStream_t s) {
  ln_typed(dtype, cols, [&](auto cfg) {
    cfg.fwd(x, ldx, res, ldr, gamma, beta, y, ldy, sum, lds, mean, invstd,
            rows, cols, eps, s);
  });
}

// rows of the [n, 2, cols] workspace that the backward pass wants (0: none)
int layernorm_bwd_parts(int dtype, long rows, int cols) {
  const int n = ln_typed(dtype, cols,
                         [&](auto cfg) { return cfg.blocks(rows); });
  return n > 1 ? n : 0;
}

void launch_layernorm_bwd(int dtype, const void* dy, long ldy, const void* x,
                          long ldx, const void* skip, long ldk,
                          const float* mean, const float* invstd,
                          const float* gamma, void* dx, long ldd, float* part,
                          float* dgamma, float* dbeta, long rows, int cols,
                          hipStream_t s) {
  ln_typed(dtype, cols, [&](auto cfg) {
    cfg.bwd(dy, ldy, x, ldx, skip, ldk, mean, invstd, gamma, dx, ldd, part,
            dgamma, dbeta, rows, cols, s);
  });
}

}  // namespace lo
