// Orthogonalisation by Newton-Schulz steps, and the Muon update around it.
//
//   X = G / (|G|_F + eps)
//   A = X X^T;  B = b A + c A A^T;  X <- a X + B X        (each step)
//
// drives the singular values of G towards one and keeps its singular vectors.
// X has the short side m as rows (G is taken transposed where it is tall).
//
// Precision. A step multiplies small singular values by a (3.4445), so what is
// rounded off X early returns up to a^4 times larger: products of bf16 values
// end 1.5e-2 off in the mean (512 x 512 noise), of fp16 values 1.8e-3. Here a
// matrix is kept as two fp16 halves, hi = fp16(v S) and lo = fp16(v S - hi)
// (22 bits, S a power of two that keeps v S below 2^15), and a product is
// hi hi + hi lo + lo hi in fp32 accumulators: 1.9e-6 off where fp32 arithmetic
// ends at 1.8e-6, at three fp16 matrix instructions instead of fp32's sixteen.
//
// Layout. A row holds 32 hi, then 32 lo values in turn, so that one 128-byte
// line of a row feeds one 16x16x32 instruction of each kind. X is kept by rows
// and, as Y, by columns: then every product is rows times rows,
//   A = X X^T,  A A^T (A is symmetric),  X' = a X + B Y^T,
// and A and B, being symmetric, are computed on one triangle of tiles and
// written to both. Sides are padded with zeros to whole tiles.
//
// A call works on a group of matrices at once; a block finds its matrix in a
// table of tile counts (a batch of equal matrices needs no table).

#include "lo_common.h"
#include "newton_schulz.h"

namespace lo {

namespace {

typedef _Float16 f16;
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// element (row, k) of a split matrix with ld values a row; its lo half is 32
// further
LO_DEVICE long split_at(long row, int k, int ld) {
  return row * 2 * ld + (k >> 5) * 64 + (k & 31);
}

LO_DEVICE void split(float v, f16& hi, f16& lo) {
  hi = (f16)v;
  lo = (f16)(v - (float)hi);
}

// the block's matrix, and its place within it in t
LO_DEVICE NsMat find(const NsGroup& g, const int* __restrict__ starts, long per,
                     long& t) {
  if (!g.mats) {
    const long i = t / per;
    t -= i * per;
    NsMat m = g.one;
    m.src += i * g.src_step;
    m.ws += i * g.ws_step;
    m.part += (int)(i * g.part_step);
    return m;
  }
  int lo = 0, hi = g.count;  // starts[lo] <= t < starts[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (starts[mid] <= t) lo = mid;
    else hi = mid;
  }
  t -= starts[lo];
  return g.mats[lo];
}

// a matrix's workspace: X and Y, twice (a step reads one pair and writes the
// other), A, B
struct Planes {
  f16* w;
  long n, a_;
  LO_DEVICE f16* x(int i) const { return w + 2 * i * n; }
  LO_DEVICE f16* y(int i) const { return w + (2 * i + 1) * n; }
  LO_DEVICE f16* a() const { return w + 4 * n; }
  LO_DEVICE f16* b() const { return w + 4 * n + a_; }
};

LO_DEVICE Planes planes(const NsMat& m, void* ws) {
  return {(f16*)ws + m.ws, 2l * m.mp * m.np, 2l * m.mp * m.mp};
}

template <typename T>
LO_DEVICE float grad_at(const NsInput& in, long i) {
  const float g = (float)((const T*)in.grad)[i] * in.gscale;
  return in.mom && in.nesterov ? g + in.mu * in.mom[i]
                               : (in.mom ? in.mom[i] : g);
}

// momentum (where there is one) and the squares' sums of the update's
// elements, one per kNsChunk of them
template <typename T>
__global__ __launch_bounds__(256) void ns_momentum_kernel(NsGroup g,
                                                          NsInput in) {
  long t = blockIdx.x;
  const NsMat m = find(g, g.chunk_starts, g.chunks, t);
  const long size = (long)m.rows * m.cols;
  const long e0 = t * kNsChunk;
  const long e1 = min(size, e0 + kNsChunk);
  double acc = 0.0;
  for (long e = e0 + threadIdx.x; e < e1; e += 256) {
    const long i = m.src + e;
    if (in.mom)
      in.mom[i] = in.mu * in.mom[i] + (float)((const T*)in.grad)[i] * in.gscale;
    const float u = grad_at<T>(in, i);
    acc += (double)u * (double)u;
  }
  for (int off = 32; off > 0; off >>= 1) acc += __shfl_xor(acc, off);
  __shared__ double red[4];
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
  __syncthreads();
  if (threadIdx.x == 0)
    g.parts[m.part + t] = red[0] + red[1] + red[2] + red[3];
}

// X and Y from the update: 64 x 64 elements a block
template <typename T>
__global__ __launch_bounds__(256) void ns_split_kernel(NsGroup g, NsInput in,
                                                       float scale, float eps) {
  __shared__ float tile[64][65];
  __shared__ double red[4];
  long t = blockIdx.x;
  const NsMat m = find(g, g.split_starts, g.splits, t);
  const Planes p = planes(m, g.ws);
  const int tn = m.np / 64;
  const int r0 = (int)(t / tn) * 64, c0 = (int)(t % tn) * 64;

  double acc = 0.0;
  for (int i = threadIdx.x; i < m.chunks; i += 256) acc += g.parts[m.part + i];
  for (int off = 32; off > 0; off >>= 1) acc += __shfl_xor(acc, off);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
  __syncthreads();
  const float norm = (float)sqrt(red[0] + red[1] + red[2] + red[3]);
  const float f = scale / (norm + eps);

  const bool tall = m.rows > m.cols;
  for (int i = threadIdx.x; i < 64 * 64; i += 256) {
    // consecutive threads along the input's rows
    const int a = i >> 6, b = i & 63;
    const int row = tall ? c0 + a : r0 + a;
    const int col = tall ? r0 + b : c0 + b;
    float v = 0.f;
    if (row < m.rows && col < m.cols)
      v = grad_at<T>(in, m.src + (long)row * m.cols + col) * f;
    if (tall) tile[b][a] = v;
    else tile[a][b] = v;
  }
  __syncthreads();
  const int r = threadIdx.x >> 2, k = (threadIdx.x & 3) * 16;
  f16* ox = p.x(0) + split_at(r0 + r, c0 + k, m.np);
  f16* oy = p.y(0) + split_at(c0 + r, r0 + k, m.mp);
  #pragma unroll
  for (int h = 0; h < 2; ++h) {
    f16x8 xh, xl, yh, yl;
    #pragma unroll
    for (int j = 0; j < 8; ++j) {
      f16 hi, lo;
      split(tile[r][k + h * 8 + j], hi, lo);
      xh[j] = hi;
      xl[j] = lo;
      split(tile[k + h * 8 + j][r], hi, lo);
      yh[j] = hi;
      yl[j] = lo;
    }
    *(f16x8*)(ox + h * 8) = xh;
    *(f16x8*)(ox + h * 8 + 32) = xl;
    *(f16x8*)(oy + h * 8) = yh;
    *(f16x8*)(oy + h * 8 + 32) = yl;
  }
}

// One product of a step on T x T tiles, four waves:
//   GRAM   A  = X X^T             one triangle, written to both
//   POLY   B  = b A + c A A^T     one triangle, written to both
//   APPLY  X' = a X + B Y^T       written as X' and Y'
// out = alpha * sum + beta * source, all of them carrying their scales.
enum { GRAM, POLY, APPLY };

template <int T, int KIND, int S>
__global__ __launch_bounds__(256) void ns_product_kernel(NsGroup g, int from,
                                                         float alpha,
                                                         float beta) {
  constexpr int W = T / 2;      // a wave's square
  constexpr int F = W / 16;     // its 16 x 16 fragments a side
  constexpr int IMG = T * 128;  // bytes of one operand's tile: T rows, 32 k
  constexpr int LOADS = T / 32; // a wave's loads of one operand's tile
  extern __shared__ __attribute__((aligned(1024))) char lds[];  // [S][2][IMG]
  long t = xcd_swizzle(blockIdx.x, gridDim.x);
  const NsMat m = find(g, KIND == APPLY ? g.rect_starts : g.tri_starts,
                       KIND == APPLY ? g.rects : g.tris, t);
  const Planes pl = planes(m, g.ws);
  int ti, tj;
  if (KIND == APPLY) {
    const int tm = m.mp / T;
    ti = (int)(t % tm);
    tj = (int)(t / tm);
  } else {
    ti = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
    while ((long)ti * (ti + 1) / 2 > t) --ti;
    while ((long)(ti + 1) * (ti + 2) / 2 <= t) ++ti;
    tj = (int)(t - (long)ti * (ti + 1) / 2);
  }
  const int ld = KIND == GRAM ? m.np : m.mp;  // values a row of both operands
  const f16* P = KIND == GRAM ? pl.x(from) : KIND == POLY ? pl.a() : pl.b();
  const f16* Q = KIND == GRAM ? pl.x(from) : KIND == POLY ? pl.a() : pl.y(from);
  P += (long)ti * T * 2 * ld;
  Q += (long)tj * T * 2 * ld;

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wr = wave >> 1, wc = wave & 1;

  // 1 KiB (8 rows of 128 bytes) an instruction; the 16-byte piece that lands
  // at place p of a row is piece p ^ (row & 7), which spreads a column of
  // pieces over the banks
  auto stage = [&](int kt) {
    char* buf = lds + (kt % S) * 2 * IMG;
    #pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int seg = wave * LOADS + i;
      const int row = seg * 8 + lane / 8;
      const long off = (long)row * 2 * ld + kt * 64 + ((lane % 8) ^ (row & 7)) * 8;
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) unsigned int*)(P + off),
          (__attribute__((address_space(3))) unsigned int*)(buf + seg * 1024),
          16, 0, 0);
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) unsigned int*)(Q + off),
          (__attribute__((address_space(3))) unsigned int*)(buf + IMG +
                                                            seg * 1024),
          16, 0, 0);
    }
  };
  auto frag = [&](const char* img, int row, int half) {
    return *(const f16x8*)(img + row * 128 +
                           ((half * 64 + (lane >> 4) * 16) ^ ((row & 7) << 4)));
  };

  f32x4 acc[F][F] = {};
  const int nk = ld / 32;
  for (int kt = 0; kt < S - 1; ++kt)
    if (kt < nk) stage(kt);
  for (int kt = 0; kt < nk; ++kt) {
    // tile kt has landed (the S - 2 after it may be on their way), and every
    // wave is done with the buffer that the next one goes to
    if (kt + S - 2 < nk)
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(
                       (S - 2) * 2 * LOADS)
                   : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const char* img = lds + (kt % S) * 2 * IMG;
    f16x8 ph[F], pw[F], qh[F], ql[F];
    #pragma unroll
    for (int i = 0; i < F; ++i) {
      const int row = i * 16 + (lane & 15);
      ph[i] = frag(img, wr * W + row, 0);
      qh[i] = frag(img + IMG, wc * W + row, 0);
    }
    #pragma unroll
    for (int i = 0; i < F; ++i) {
      const int row = i * 16 + (lane & 15);
      pw[i] = frag(img, wr * W + row, 1);
      ql[i] = frag(img + IMG, wc * W + row, 1);
    }
    if (kt + S - 1 < nk) stage(kt + S - 1);
    // kind by kind: an accumulator's next use is F * F instructions away
    auto products = [&](const f16x8 (&p)[F], const f16x8 (&q)[F]) {
      #pragma unroll
      for (int i = 0; i < F; ++i)
        #pragma unroll
        for (int j = 0; j < F; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(p[i], q[j],
                                                             acc[i][j], 0, 0, 0);
    };
    products(ph, qh);
    products(ph, ql);
    products(pw, qh);
  }

  // a lane holds rows r..r+3 of column c
  f16* rowsOut = KIND == GRAM ? pl.a() : KIND == POLY ? pl.b() : pl.x(from ^ 1);
  f16* colsOut = KIND == APPLY ? pl.y(from ^ 1) : rowsOut;
  const f16* source = KIND == POLY ? pl.a() : pl.y(from);
  const int ldr = KIND == APPLY ? m.np : m.mp;
  const bool both = KIND == APPLY || ti != tj;
  #pragma unroll
  for (int i = 0; i < F; ++i)
    #pragma unroll
    for (int j = 0; j < F; ++j) {
      const int r = ti * T + wr * W + i * 16 + (lane >> 4) * 4;
      const int c = tj * T + wc * W + j * 16 + (lane & 15);
      const long col = split_at(c, r, m.mp);
      f32x4 v = acc[i][j] * alpha;
      if (KIND != GRAM) {
        const f16x4 sh = *(const f16x4*)(source + col);
        const f16x4 sl = *(const f16x4*)(source + col + 32);
        #pragma unroll
        for (int e = 0; e < 4; ++e)
          v[e] += beta * ((float)sh[e] + (float)sl[e]);
      }
      f16x4 hi, lo;
      #pragma unroll
      for (int e = 0; e < 4; ++e) {
        f16 h, l;
        split(v[e], h, l);
        hi[e] = h;
        lo[e] = l;
        const long at = split_at(r + e, c, ldr);
        rowsOut[at] = h;
        rowsOut[at + 32] = l;
      }
      if (both) {
        *(f16x4*)(colsOut + col) = hi;
        *(f16x4*)(colsOut + col + 32) = lo;
      }
    }
}

// the result in the input's own layout, 32 columns of a row per 8 threads
template <typename T>
__global__ __launch_bounds__(256) void ns_store_kernel(NsGroup g, int from,
                                                       float unscale,
                                                       NsOutput out) {
  long t = blockIdx.x;
  const NsMat m = find(g, g.chunk_starts, g.chunks, t);
  const Planes p = planes(m, g.ws);
  const bool tall = m.rows > m.cols;
  const f16* src = tall ? p.y(from) : p.x(from);
  const int ld = tall ? m.mp : m.np;
  const long size = (long)m.rows * m.cols;
  const long e1 = min(size, (t + 1) * kNsChunk);
  const float step = out.lr * m.gain;
  for (long e = t * kNsChunk + threadIdx.x; e < e1; e += 256) {
    const long row = e / m.cols;
    const long at = split_at(row, (int)(e - row * m.cols), ld);
    const float o = ((float)src[at] + (float)src[at + 32]) * unscale;
    const long i = m.src + e;
    if (out.master) {
      const float w = out.master[i] * out.keep - step * o;
      out.master[i] = w;
      ((bf16*)out.mirror)[i] = tobf16(w);
    } else {
      ((T*)out.out)[i] = (T)o;
    }
  }
}

template <int T, int KIND>
void product(const NsGroup& g, int from, float alpha, float beta,
             hipStream_t s) {
  const long blocks = KIND == APPLY ? g.all_rects : g.all_tris;
  constexpr int S = T == 64 ? 4 : 2;
  hipLaunchKernelGGL((ns_product_kernel<T, KIND, S>), dim3(blocks), dim3(256),
                     S * 2 * T * 128, s, g, from, alpha, beta);
}

template <int T>
int steps(const NsGroup& g, const NsStep* st, int n, hipStream_t s) {
  int from = 0;
  for (int i = 0; i < n; ++i, from ^= 1) {
    const NsStep& k = st[i];
    product<T, GRAM>(g, from, k.sa / (k.sx * k.sx), 0.f, s);
    product<T, POLY>(g, from, k.c * k.sb / (k.sa * k.sa), k.b * k.sb / k.sa, s);
    product<T, APPLY>(g, from, k.sn / (k.sb * k.sx), k.a * k.sn / k.sx, s);
  }
  return from;
}

template <typename T>
void run(const NsGroup& g, const NsInput& in, const NsStep* st, int n,
         float eps, const NsOutput& out, hipStream_t s) {
  hipLaunchKernelGGL(ns_momentum_kernel<T>, dim3(g.all_chunks), dim3(256), 0, s,
                     g, in);
  hipLaunchKernelGGL(ns_split_kernel<T>, dim3(g.all_splits), dim3(256), 0, s, g,
                     in, st[0].sx, eps);
  const int from = g.tile == 128 ? steps<128>(g, st, n, s)
                                 : steps<64>(g, st, n, s);
  hipLaunchKernelGGL(ns_store_kernel<T>, dim3(g.all_chunks), dim3(256), 0, s, g,
                     from, 1.f / st[n - 1].sn, out);
}

}  // namespace

void launch_newton_schulz(const NsGroup& g, int dtype, const NsInput& in,
                          const NsStep* st, int n, float eps,
                          const NsOutput& out, hipStream_t s) {
  if (dtype == 0) run<bf16>(g, in, st, n, eps, out, s);
  else if (dtype == 1) run<f16>(g, in, st, n, eps, out, s);
  else run<float>(g, in, st, n, eps, out, s);
}

}  // namespace lo
