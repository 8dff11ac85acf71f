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
// walks rows blockIdx, blockIdx + grid, ..., backwards with the next row's
// loads on their way; its gradient sums stay in registers and go to a
// [blocks, 2, cols] workspace that a second small kernel adds in a fixed
// order, so results do not depend on timing. With one block the sums are
// written directly. Where a block has few rows, its sums are more to write
// than the rows were to read, and rows of more than 16 elements a thread
// (16384 columns) have no registers left for them: there a kernel of its own
// takes the sums down the columns, at the price of a second reading.
//
// Columns need not be a multiple of VE: the vector that would cross the row's
// end is moved back to end with it, and the elements it shares with its
// neighbour (skip of them) count only there. gfx950 loads 16 bytes from any
// element-aligned address, so odd strides take the same path. What a row's
// results need is read before it is written, so an output may be one of the
// inputs.
//
// Measured on one MI355X, where a 1 GiB copy moves 5.0 TB/s:
//   1048576 x 128 bf16           forward 102 us, 5.2 TB/s; backward 171 us,
//                                4.7 TB/s, and 5 us to join 1024 sums
//   8192 x 8192 bf16 + residual  forward 98 us, 5.5 TB/s; backward with dskip
//                                126 us, 4.3 TB/s, and 5 us
//   4099 x 1001 fp32             forward 8.5 us, backward 12.6 us, 3.9 TB/s
//                                both; 4.4 us to join; 23 us with the launches
//   1 x 384 bf16                 forward 1.8 us, a launch each 4.5 us

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

// v + the value of the lane that a DPP pattern names
template <int CTRL>
LO_DEVICE float add_dpp(float v) {
  const int o = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL,
                                            0xf, 0xf, false);
  return v + __builtin_bit_cast(float, o);
}

// The sum over aligned groups of N lanes, in every lane. Within 16 lanes by
// DPP (1, 2 apart, then the mirror images of 8 and of 16), then by swapping
// rows of 16 and halves: a tenth of the way through LDS that shuffles take.
template <int N>
LO_DEVICE float lane_sum(float v) {
  if constexpr (N >= 2) v = add_dpp<0xb1>(v);    // quad_perm 1 0 3 2
  if constexpr (N >= 4) v = add_dpp<0x4e>(v);    // quad_perm 2 3 0 1
  if constexpr (N >= 8) v = add_dpp<0x141>(v);   // row_half_mirror
  if constexpr (N >= 16) v = add_dpp<0x140>(v);  // row_mirror
  if constexpr (N >= 32) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    const auto p = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const unsigned a = p[0], b = p[1];
    v = __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
  }
  if constexpr (N >= 64) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    const auto p = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const unsigned a = p[0], b = p[1];
    v = __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
  }
  return v;
}

// K sums over the TPR threads that share a row; every one of them gets all.
// For TPR > 64 the LDS slots alternate between calls, so one barrier per call
// is enough: a slot is rewritten two calls later, past the barrier that its
// last readers reach before the next call's.
template <int TPR, int K>
LO_DEVICE void row_sum(float (&v)[K], float* red, int& turn) {
  #pragma unroll
  for (int k = 0; k < K; ++k) v[k] = lane_sum<(TPR < 64 ? TPR : 64)>(v[k]);
  if constexpr (TPR > 64) {
    constexpr int W = TPR / 64;
    float* slot = red + (turn & 1) * 2 * W;
    ++turn;
    if ((threadIdx.x & 63) == 0) {
      #pragma unroll
      for (int k = 0; k < K; ++k) slot[k * W + (threadIdx.x >> 6)] = v[k];
    }
    __syncthreads();
    #pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = 0.f;
      #pragma unroll
      for (int w = 0; w < W; ++w) v[k] += slot[k * W + w];
    }
  }
}

// a * b, rounded: fused into the sum that follows, dy * gamma would not be the
// value that its mean was taken of, and what is left of it, times invstd, would
// stand where dx is zero (rows of one column)
LO_DEVICE float rounded_product(float a, float b) {
  return __builtin_fmaf(a, b, 0.f);
}

constexpr int ln_block(int tpr) { return tpr > 256 ? tpr : 256; }

// gamma and beta stay in registers for all of a block's rows, but where a row
// fills those: then they come from the cache each time, and the backward pass
// does without the next row's loads
template <int VE, int TPR, int NV>
constexpr bool ln_hoist() { return TPR < 1024 || NV * VE <= 8; }

template <typename T, int VE, int TPR, int NV>
__global__ __launch_bounds__(ln_block(TPR)) void layernorm_fwd_kernel(
    const T* x, long ldx, const T* res, long ldr,
    const float* __restrict__ gamma, const float* __restrict__ beta,
    T* y, long ldy, T* sum, long lds, float* __restrict__ mean,
    float* __restrict__ invstd, long rows, int cols, float eps) {
  typedef typename RowVec<T, VE>::type V;
  constexpr int RPB = ln_block(TPR) / TPR;
  constexpr bool HOIST = ln_hoist<VE, TPR, NV>();
  __shared__ float red[TPR > 64 ? 4 * (TPR / 64) : 1];
  const int t = threadIdx.x % TPR;
  const float n = (float)cols;
  int base[NV], skip[NV];
  float gm[HOIST ? NV : 1][VE], bt[HOIST ? NV : 1][VE];
  #pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c0 = (i * TPR + t) * VE;
    base[i] = min(c0, cols - VE);
    skip[i] = min(c0 - base[i], VE);
    if constexpr (HOIST) {
      load_f32<VE>(gamma + base[i], gm[i]);
      load_f32<VE>(beta + base[i], bt[i]);
    }
  }
  int turn = 0;
  const long step = (long)gridDim.x * RPB;
  long r = (long)blockIdx.x * RPB + threadIdx.x / TPR;
  for (; r < rows; r += step) {
    V s[NV];
    #pragma unroll
    for (int i = 0; i < NV; ++i) s[i] = *(const V*)(x + r * ldx + base[i]);
    if (res) {
      #pragma unroll
      for (int i = 0; i < NV; ++i) {
        const V rv = *(const V*)(res + r * ldr + base[i]);
        if constexpr (VE == 1) {
          s[i] = (T)((float)s[i] + (float)rv);
        } else {
          #pragma unroll
          for (int j = 0; j < VE; ++j)
            s[i][j] = (T)((float)s[i][j] + (float)rv[j]);
        }
      }
    }
    float acc[1] = {0.f};
    #pragma unroll
    for (int i = 0; i < NV; ++i)
      #pragma unroll
      for (int j = 0; j < VE; ++j)
        acc[0] += j >= skip[i] ? elem<VE>(s[i], j) : 0.f;
    row_sum<TPR>(acc, red, turn);
    const float mu = acc[0] / n;
    acc[0] = 0.f;
    #pragma unroll
    for (int i = 0; i < NV; ++i)
      #pragma unroll
      for (int j = 0; j < VE; ++j) {
        const float d = elem<VE>(s[i], j) - mu;
        acc[0] += j >= skip[i] ? d * d : 0.f;
      }
    row_sum<TPR>(acc, red, turn);
    const float is = 1.f / sqrtf(acc[0] / n + eps);
    #pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (skip[i] >= VE) continue;
      float g[VE], b[VE];
      if constexpr (HOIST) {
        #pragma unroll
        for (int j = 0; j < VE; ++j) g[j] = gm[i][j], b[j] = bt[i][j];
      } else {
        load_f32<VE>(gamma + base[i], g);
        load_f32<VE>(beta + base[i], b);
      }
      V o;
      #pragma unroll
      for (int j = 0; j < VE; ++j) {
        const float v = (elem<VE>(s[i], j) - mu) * is * g[j] + b[j];
        if constexpr (VE == 1) o = (T)v;
        else o[j] = (T)v;
      }
      *(V*)(y + r * ldy + base[i]) = o;
      if (sum) *(V*)(sum + r * lds + base[i]) = s[i];
    }
    if (t == 0 && mean) {
      mean[r] = mu;
      invstd[r] = is;
    }
  }
}

// part: [gridDim.x, 2, cols] sums of dy * xhat and of dy, or null with one
// block, which then writes dgamma/dbeta itself. SUMS: whether they are taken
// here at all.
template <typename T, int VE, int TPR, int NV, bool SUMS>
__global__ __launch_bounds__(ln_block(TPR)) void layernorm_bwd_kernel(
    const T* dy, long ldy, const T* x, long ldx,
    const T* skipg, long ldk, const float* __restrict__ mean,
    const float* __restrict__ invstd, const float* __restrict__ gamma,
    T* dx, long ldd, float* __restrict__ part, float* __restrict__ dgamma,
    float* __restrict__ dbeta, long rows, int cols) {
  typedef typename RowVec<T, VE>::type V;
  constexpr int RPB = ln_block(TPR) / TPR;
  constexpr bool HOIST = ln_hoist<VE, TPR, NV>();
  __shared__ float red[TPR > 64 ? 4 * (TPR / 64) : 1];
  extern __shared__ __attribute__((aligned(16))) float acc[];  // [2][cols]
  const int t = threadIdx.x % TPR;
  const float n = (float)cols;
  int base[NV], skip[NV];
  float gm[HOIST ? NV : 1][VE];
  float dg[SUMS ? NV : 1][VE] = {}, db[SUMS ? NV : 1][VE] = {};
  #pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c0 = (i * TPR + t) * VE;
    base[i] = min(c0, cols - VE);
    skip[i] = min(c0 - base[i], VE);
    if constexpr (HOIST) load_f32<VE>(gamma + base[i], gm[i]);
  }
  int turn = 0;
  const long step = (long)gridDim.x * RPB;
  long r = (long)blockIdx.x * RPB + threadIdx.x / TPR;
  V nx[NV], ng[NV];
  float nmu = 0.f, nis = 0.f;
  auto load = [&](long at) {
    #pragma unroll
    for (int i = 0; i < NV; ++i) {
      nx[i] = *(const V*)(x + at * ldx + base[i]);
      ng[i] = *(const V*)(dy + at * ldy + base[i]);
    }
    nmu = mean[at];
    nis = invstd[at];
  };
  auto gammas = [&](int i, float (&ga)[VE]) {
    if constexpr (HOIST) {
      #pragma unroll
      for (int j = 0; j < VE; ++j) ga[j] = gm[i][j];
    } else {
      // an address that is new to the compiler: it would keep both readings
      const float* p = gamma + base[i];
      asm volatile("" : "+v"(p));
      load_f32<VE>(p, ga);
    }
  };
  if (HOIST && r < rows) load(r);
  for (; r < rows; r += step) {
    if (!HOIST) load(r);
    V xv[NV], gv[NV], kv[NV];
    #pragma unroll
    for (int i = 0; i < NV; ++i) xv[i] = nx[i], gv[i] = ng[i];
    const float mu = nmu, is = nis;
    if (HOIST && r + step < rows) load(r + step);
    if (skipg) {
      #pragma unroll
      for (int i = 0; i < NV; ++i)
        kv[i] = *(const V*)(skipg + r * ldk + base[i]);
    }
    float s[2] = {0.f, 0.f};
    #pragma unroll
    for (int i = 0; i < NV; ++i) {
      float ga[VE];
      gammas(i, ga);
      #pragma unroll
      for (int j = 0; j < VE; ++j) {
        const float g = j >= skip[i] ? elem<VE>(gv[i], j) : 0.f;
        const float xh = (elem<VE>(xv[i], j) - mu) * is;
        const float h = rounded_product(g, ga[j]);
        s[0] += h;
        s[1] += j >= skip[i] ? h * xh : 0.f;
        if constexpr (SUMS) {
          db[i][j] += g;
          dg[i][j] += j >= skip[i] ? g * xh : 0.f;
        }
      }
    }
    row_sum<TPR>(s, red, turn);
    const float c1 = s[0] / n, c2 = s[1] / n;
    #pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (skip[i] >= VE) continue;
      float ga[VE];
      gammas(i, ga);
      V o;
      #pragma unroll
      for (int j = 0; j < VE; ++j) {
        const float xh = (elem<VE>(xv[i], j) - mu) * is;
        const float h = rounded_product(elem<VE>(gv[i], j), ga[j]);
        float d = is * (h - c1 - xh * c2);
        if (skipg) d += elem<VE>(kv[i], j);
        if constexpr (VE == 1) o = (T)d;
        else o[j] = (T)d;
      }
      T* to = dx + r * ldd + base[i];
      if constexpr (VE > 1) {
        // dx may lie where dskip does: another wave may have written the
        // elements that a moved vector shares with its neighbour before this
        // one's of dskip were read
        if (skipg && skip[i] > 0) {
          #pragma unroll
          for (int j = 0; j < VE; ++j)
            if (j >= skip[i]) to[j] = o[j];
          continue;
        }
      }
      *(V*)to = o;
    }
  }
  float* og = part ? part + (long)blockIdx.x * 2 * cols : dgamma;
  float* ob = part ? og + cols : dbeta;
  if constexpr (!SUMS) {
  } else if constexpr (TPR >= ln_block(TPR)) {
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

// The gradient sums alone, down the columns: a block takes 64 vectors of VE
// columns and every gridDim.y-th group of four rows, a wave a row at a time.
// The sums go to part [gridDim.y, 2, cols].
template <typename T, int VE>
__global__ __launch_bounds__(256) void layernorm_sums_kernel(
    const T* __restrict__ dy, long ldy, const T* __restrict__ x, long ldx,
    const float* __restrict__ mean, const float* __restrict__ invstd,
    float* __restrict__ part, long rows, int cols) {
  typedef typename RowVec<T, VE>::type V;
  __shared__ float join[4][2][64 * VE];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c0 = (blockIdx.x * 64 + lane) * VE;
  const int base = min(c0, cols - VE);
  float dg[VE] = {}, db[VE] = {};
  #pragma unroll 2
  for (long r = blockIdx.y * 4 + wave; r < rows; r += gridDim.y * 4) {
    const V xv = *(const V*)(x + r * ldx + base);
    const V gv = *(const V*)(dy + r * ldy + base);
    const float mu = mean[r], is = invstd[r];
    #pragma unroll
    for (int j = 0; j < VE; ++j) {
      const float g = elem<VE>(gv, j);
      db[j] += g;
      dg[j] += g * ((elem<VE>(xv, j) - mu) * is);
    }
  }
  #pragma unroll
  for (int j = 0; j < VE; ++j) {
    join[wave][0][lane * VE + j] = dg[j];
    join[wave][1][lane * VE + j] = db[j];
  }
  __syncthreads();
  // a vector moved back at the row's end writes the columns that are its own
  if (wave < 2 && c0 < cols) {
    float* to = part + ((long)blockIdx.y * 2 + wave) * cols;
    #pragma unroll
    for (int j = 0; j < VE; ++j) {
      float v = 0.f;
      #pragma unroll
      for (int w = 0; w < 4; ++w) v += join[w][wave][lane * VE + j];
      if (base + j >= c0) to[base + j] = v;
    }
  }
}

// column sums of part [n, 2 cols]: 32 columns a block, 32 threads to a column
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
    for (int r0 = ty; r0 < n; r0 += 8 * 32) {
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
  // blocks that run at once: one more round would wait for a whole one, and
  // each has a set of sums to hand over
  static int blocks(long rows) {
    const long most = TPR > 256 ? 256 : TPR < 64 ? 1024 : 768;
    return (int)min((rows + rpb - 1) / rpb, most);
  }
  // Whether the gradient sums are taken along with dx: then 16 bytes a column
  // and block are written and read, otherwise the two arrays are read again.
  // Along / apart, us: bf16 8192 x 768 19 / 27, 4096 x 2048 22 / 23, 2048 x 2048
  // 21 / 14, 1024 x 8192 38 / 23; fp32 1024 x 4096 16 / 19, 512 x 4096 14 / 12.
  // Rows of 1024 threads' 2-byte values have the fewest registers for the sums:
  // 2048 x 8192 45 / 35, 4096 x 8192 58 / 58, 8192 x 8192 96 / 123.
  static bool along(long rows) {
    if (TPR < 64) return true;
    if (TPR == 1024 && NV * VE > 16) return false;
    const long apart = TPR == 1024 && sizeof(T) == 2 ? 16 : 8;
    return blocks(rows) == 1 || rows * sizeof(T) > apart * blocks(rows);
  }
  static int parts(long rows) {
    if (!along(rows)) return (int)min((rows + 15) / 16, 64L);
    const int n = blocks(rows);
    return n > 1 ? n : 0;
  }
  template <bool SUMS>
  static void dx_pass(const void* dy, long ldy, const void* x, long ldx,
                      const void* skip, long ldk, const float* mean,
                      const float* invstd, const float* gamma, void* dx,
                      long ldd, float* part, float* dgamma, float* dbeta,
                      long rows, int cols, hipStream_t s) {
    const size_t lds = SUMS && TPR < ln_block(TPR) ? 8ul * cols : 0;
    hipLaunchKernelGGL((layernorm_bwd_kernel<T, VE, TPR, NV, SUMS>),
                       dim3(blocks(rows)), dim3(ln_block(TPR)), lds, s,
                       (const T*)dy, ldy, (const T*)x, ldx, (const T*)skip, ldk,
                       mean, invstd, gamma, (T*)dx, ldd, part, dgamma, dbeta,
                       rows, cols);
  }
  static void bwd(const void* dy, long ldy, const void* x, long ldx,
                  const void* skip, long ldk, const float* mean,
                  const float* invstd, const float* gamma, void* dx, long ldd,
                  float* part, float* dgamma, float* dbeta, long rows,
                  int cols, hipStream_t s) {
    const int n = parts(rows);
    bool done = false;
    if constexpr (TPR >= 64) {
      if (!along(rows)) {
        // the sums first: dx may be written where dy or x lie
        hipLaunchKernelGGL((layernorm_sums_kernel<T, VE>),
                           dim3((cols + 64 * VE - 1) / (64 * VE), n), dim3(256),
                           0, s, (const T*)dy, ldy, (const T*)x, ldx, mean,
                           invstd, part, rows, cols);
        dx_pass<false>(dy, ldy, x, ldx, skip, ldk, mean, invstd, gamma, dx, ldd,
                       nullptr, nullptr, nullptr, rows, cols, s);
        done = true;
      }
    }
    if constexpr (TPR < 1024 || NV * VE <= 16) {
      if (!done)
        dx_pass<true>(dy, ldy, x, ldx, skip, ldk, mean, invstd, gamma, dx, ldd,
                      n ? part : nullptr, dgamma, dbeta, rows, cols, s);
    }
    if (n)
      hipLaunchKernelGGL(layernorm_join_kernel, dim3((2 * cols + 31) / 32),
                         dim3(1024), 0, s, part, dgamma, dbeta, n, cols);
  }
};

// calls f(LnConfig<...>{}) with the threads and vectors a row of cols takes
template <typename T, typename F>
auto ln_pick(int cols, F f) {
  constexpr int VE = 16 / sizeof(T);
  if (cols < VE) return f(LnConfig<T, 1, 1, VE - 1>{});
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
  return ln_typed(dtype, cols, [&](auto cfg) { return cfg.parts(rows); });
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
