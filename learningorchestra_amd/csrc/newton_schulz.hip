// Orthogonalisation by Newton-Schulz steps, and the Muon update around it.
//
//   X = G / (|G|_F + eps)
//   A = X X^T;  C = a + b A + c A A^T;  X <- C X          (each step)
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
// That holds in the norm of the whole matrix. S is one for all rows, and the
// lower half ends at 2^-24 / S: 2^-38 of X and A, 2^-37 of C, absolute, where
// fp32 keeps 24 bits of a row however small it is. After five steps a row is
// off by some 1e-8 beside rows of length one. Small rows of 128 x 640, scaled
// down against the others by 1e-2, 1e-4, 1e-6, 1e-8, end 5e-7, 2.4e-6, 2.4e-4,
// 2.4e-2 off relative to themselves (fp32: 4e-7), which a bf16 result shows
// below 1e-6. A scale for each row would have to be carried through both sides
// of A and C.
//
// Layout. 32 columns of a row are a 128-byte line, 32 hi values, then 32 lo
// ones, which feeds one 16x16x32 instruction of each kind; the lines of 32
// columns lie together, row after row, so that all that a tile takes for a
// step of its sum is one piece of memory (4096 x 4096 took 3 % longer with a
// row's lines together). A = X X^T and A A^T (A is symmetric) are rows times
// rows; X' = C X takes columns of X, which LDS turns as they are read
// (ds_read_b64_tr_b16). With a second copy of X, by columns, to write and read
// instead, 16 x 512 x 2048 took 742 us in place of 644, ResNet-50's matrices
// 1290 in place of 1126. A and C, being symmetric, are computed on one
// triangle of tiles and written to both. Sides are padded with zeros to whole
// tiles.
//
// Sharing out. A call works on a group of matrices at once: a block finds its
// matrix and tile in a table made with the plan, or by arithmetic for a batch
// of equal ones. Where tiles are few, or few are left over after full rounds
// of the chip, several blocks sum a part of a tile each; the last to arrive
// adds the parts, in their order, so that results do not depend on timing. No
// block waits for another.
//
// Measured on one MI355X, where 8192^3 library products reach 1.2 PFLOP/s in
// fp16 and 0.154 in fp32 (five steps; rates count all three fp16 products):
//   4096 x 4096        3.3 to 3.5 ms between cards; C X 309 us, 1.33 PFLOP/s,
//                      matrix pipes busy 88 % of a CU's cycles; X X^T 185 us,
//                      1.15 PFLOP/s, 68 %. The clock falls to 1.7 GHz: power
//                      bounds it.
//   16 x 512 x 2048    566 to 620 us; C X 56 us, 0.92 PFLOP/s; X X^T 44 us,
//                      0.66; A A^T 21 us. The ends of rounds and the traffic
//                      between the dies (X is 67 MB) bound it.
//   ResNet-50's matrices, a whole step: 929 to 1006 us, of which 118 move the
//                      momentum, the update and X's first form at 5 TB/s
//   256 x 3136 bf16    108 us for 17 launches of 4 to 9 us, of which some 3.5
//                      are the launch, the first loads and the end

#include <type_traits>

#include "lo_common.h"
#include "newton_schulz_plan.h"

namespace lo {

namespace {

typedef _Float16 f16;
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef __fp16 h16x4 __attribute__((ext_vector_type(4)));  // the builtin's
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// four elements at any element-aligned address
template <typename T>
struct Quad {
  typedef T type __attribute__((ext_vector_type(4), aligned(sizeof(T))));
};

// element (row, k) of a split matrix of so many rows; its lo half is 32 further
LO_DEVICE long split_at(int row, int k, int rows) {
  return ((long)(k >> 5) * rows + row) * 64 + (k & 31);
}

LO_DEVICE void split(float v, f16& hi, f16& lo) {
  hi = (f16)v;
  lo = (f16)(v - (float)hi);
}

LO_DEVICE unsigned pack(float v) {
  f16 hi, lo;
  split(v, hi, lo);
  return (unsigned)__builtin_bit_cast(unsigned short, hi) |
         (unsigned)__builtin_bit_cast(unsigned short, lo) << 16;
}

LO_DEVICE void unpack8(const u32x4& a, const u32x4& b, f16x8& hi, f16x8& lo) {
  #pragma unroll
  for (int j = 0; j < 8; ++j) {
    const unsigned v = j < 4 ? a[j] : b[j - 4];
    hi[j] = __builtin_bit_cast(f16, (unsigned short)v);
    lo[j] = __builtin_bit_cast(f16, (unsigned short)(v >> 16));
  }
}

// the block's matrix, and its place within it
LO_DEVICE NsMat find(const NsGroup& g, const NsBlock* __restrict__ table,
                     int per, int id, int& at) {
  if (g.mats) {
    const NsBlock b = table[id];
    at = b.at;
    return g.mats[b.mat];
  }
  const int i = id / per;
  at = id - i * per;
  NsMat m = g.one;
  m.src += i * g.src_step;
  m.ws += i * g.ws_step;
  m.sum += i * g.sum_step;
  return m;
}

// a matrix's workspace: X twice (a step reads one and writes the other), A, C
struct Planes {
  f16* w;
  long n, a_;
  LO_DEVICE f16* x(int i) const { return w + i * n; }
  LO_DEVICE f16* a() const { return w + 2 * n; }
  LO_DEVICE f16* c() const { return w + 2 * n + a_; }
};

template <typename M>  // NsMat or NsTask
LO_DEVICE Planes planes(const M& m, void* ws) {
  return {(f16*)ws + m.ws, 2l * m.mp * m.np, 2l * m.mp * m.mp};
}

// n (at most 4) elements from i on; the rest are zero
template <typename T>
LO_DEVICE f32x4 load4(const T* p, long i, int n) {
  f32x4 v = {};
  if (n >= 4) {
    const typename Quad<T>::type q = *(const typename Quad<T>::type*)(p + i);
    #pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = (float)q[j];
  } else {
    #pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) v[j] = (float)p[i + j];
  }
  return v;
}

template <typename T>
LO_DEVICE void store4(T* p, long i, int n, const f32x4& v) {
  if (n >= 4) {
    typename Quad<T>::type q;
    #pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = (T)v[j];
    *(typename Quad<T>::type*)(p + i) = q;
  } else {
    #pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) p[i + j] = (T)v[j];
  }
}

// X = U f 2^-e from the sum of U's squares: 1 / (norm + eps), so that neither
// tiny nor huge updates leave fp32's range on the way; zeros stay zero without
// an eps, too
struct NsNorm {
  float f;
  int e;
  LO_DEVICE NsNorm(double squares, float eps) {
    const double m = frexp(sqrt(squares) + (double)eps, &e);
    f = m == 0.0 ? 0.f : (float)(1.0 / m);
  }
  LO_DEVICE f32x4 operator()(f32x4 u) const {
    #pragma unroll
    for (int j = 0; j < 4; ++j) u[j] = ldexpf(u[j], -e) * f;
    return u;
  }
};

// the update's elements, from the momentum that the step has brought forward
template <typename T>
LO_DEVICE f32x4 update4(const NsInput& in, long i, int n) {
  if (!in.mom) return load4((const T*)in.grad, i, n) * in.gscale;
  const f32x4 m = load4(in.mom, i, n);
  if (!in.nesterov) return m;
  return load4((const T*)in.grad, i, n) * in.gscale + in.mu * m;
}

// momentum (where there is one) and the squares' sums of the update's
// elements, one per kNsChunk of them, in 64 bits: no norm overflows
template <typename T>
__global__ __launch_bounds__(256) void ns_momentum_kernel(NsGroup g,
                                                          NsInput in) {
  int at;
  const NsMat m = find(g, g.chunk_blocks, g.chunks, blockIdx.x, at);
  const long size = (long)m.rows * m.cols;
  const long e0 = (long)at * kNsChunk;
  double acc = 0.0;
  #pragma unroll
  for (int k = 0; k < kNsChunk / 1024; ++k) {
    const long e = e0 + k * 1024 + threadIdx.x * 4;
    const int n = (int)min(size - e, 4l);
    if (n <= 0) continue;
    const long i = m.src + e;
    f32x4 u = load4((const T*)in.grad, i, n) * in.gscale;
    if (in.mom) {
      const f32x4 v = in.mu * load4(in.mom, i, n) + u;
      store4(in.mom, i, n, v);
      u = in.nesterov ? u + in.mu * v : v;
    }
    #pragma unroll
    for (int j = 0; j < 4; ++j) acc += (double)u[j] * (double)u[j];
  }
  for (int off = 32; off > 0; off >>= 1) acc += __shfl_xor(acc, off);
  __shared__ double red[4];
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
  __syncthreads();
  if (threadIdx.x == 0)
    g.sums[m.sum + at] = red[0] + red[1] + red[2] + red[3];
  // the products' counters start a call at zero
  const int stride = gridDim.x * 256;
  for (int i = blockIdx.x * 256 + threadIdx.x; i < g.all_slots; i += stride)
    g.slots[i] = 0;
}

// X from the update: 64 x 64 elements a block
template <typename T>
__global__ __launch_bounds__(256) void ns_split_kernel(NsGroup g, NsInput in,
                                                       float scale, float eps) {
  __shared__ float tile[64][65];
  __shared__ double red[4];
  int at;
  const NsMat m = find(g, g.split_blocks, g.splits, blockIdx.x, at);
  const Planes p = planes(m, g.ws);
  const int tn = m.np / 64;
  const int r0 = at / tn * 64, c0 = at % tn * 64;
  const bool tall = m.rows > m.cols;

  // four elements along the input's rows a load
  f32x4 v[4];
  const int b = threadIdx.x % 16 * 4;
  #pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int a = i * 16 + threadIdx.x / 16;
    const int row = (tall ? c0 : r0) + a, col = (tall ? r0 : c0) + b;
    v[i] = f32x4{};
    if (row < m.rows && col < m.cols)
      v[i] = update4<T>(in, m.src + (long)row * m.cols + col, m.cols - col);
  }
  double acc = 0.0;
  for (int i = threadIdx.x; i < m.chunks; i += 256) acc += g.sums[m.sum + i];
  for (int off = 32; off > 0; off >>= 1) acc += __shfl_xor(acc, off);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
  __syncthreads();
  const NsNorm norm(red[0] + red[1] + red[2] + red[3], eps);
  #pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int a = i * 16 + threadIdx.x / 16;
    v[i] = norm(v[i]);
    #pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float x = v[i][j] * scale;
      if (tall) tile[b + j][a] = x;
      else tile[a][b + j] = x;
    }
  }
  __syncthreads();
  const int r = threadIdx.x >> 2, k = (threadIdx.x & 3) * 16;
  f16* ox = p.x(0) + split_at(r0 + r, c0 + k, m.mp);
  #pragma unroll
  for (int h = 0; h < 2; ++h) {
    f16x8 xh, xl;
    #pragma unroll
    for (int j = 0; j < 8; ++j) {
      f16 hi, lo;
      split(tile[r][k + h * 8 + j], hi, lo);
      xh[j] = hi;
      xl[j] = lo;
    }
    *(f16x8*)(ox + h * 8) = xh;
    *(f16x8*)(ox + h * 8 + 32) = xl;
  }
}

// What a product's launch hands its blocks. The first lines are what each
// block reads before it can start.
struct NsProduct {
  const NsTask* tasks;  // or null: equal matrices
  void* ws;
  int from;                 // the X that the step reads
  int mp, np, tile;         // equal matrices: their shape,
  int blocks, whole, splits, count;  // blocks of one, and how shared out,
  long ws_step, part_step;  // and their spacing
  int slot_step;
  float alpha, beta, diag;  // out = alpha * sum + beta * A (+ diag where i = j)
  float* parts;
  unsigned* slots;
};

// the last step's output
struct NsFinal {
  NsOutput out;
  const NsMat* mats;
  NsMat one;
  long src_step;
};

template <int KIND>
LO_DEVICE NsTask task_of(const NsProduct& pr) {
  int id = blockIdx.x;
  if (pr.tasks) return pr.tasks[id];
  // neighbouring tiles on one die, for its cache (the split tiles of a single
  // matrix are spread over all dies)
  const int whole = pr.count == 1 ? pr.whole : (int)gridDim.x;
  if (id < whole) id = xcd_swizzle(id, whole);
  NsTask t;
  t.mat = 0;
  if (pr.count > 1) {
    t.mat = id / pr.blocks;
    id -= t.mat * pr.blocks;
  }
  t.ws = t.mat * pr.ws_step;
  t.part = t.mat * pr.part_step;
  t.slot = t.mat * pr.slot_step;
  t.mp = pr.mp;
  t.np = pr.np;
  t.tile = pr.tile;
  t.slice = 0;
  t.splits = 1;
  if (id >= pr.whole) {
    t.splits = pr.splits;
    const int cut = (id - pr.whole) / t.splits;
    t.slice = id - pr.whole - cut * t.splits;
    t.part += (long)cut * t.splits * t.tile * t.tile;
    t.slot += cut;
    id = pr.whole + cut;
  }
  const int shift = t.tile == 128 ? 7 : t.tile == 64 ? 6 : 5;
  ns_tile_at(KIND, id, t.mp >> shift, t.np >> shift, t.ti, t.tj);
  const int depth = (KIND == NS_GRAM ? t.np : t.mp) / 32;
  t.k0 = 0;
  t.k1 = depth;
  if (t.splits > 1) {
    t.k0 = depth / 2 * t.slice / t.splits * 2;
    t.k1 = depth / 2 * (t.slice + 1) / t.splits * 2;
  }
  return t;
}

// One product on T x T tiles, four waves, S staged tiles of both operands (32
// values of the sum each) in LDS. FINAL: the last step's X' goes to the output
// in place of the workspace.
template <int T, int KIND, int S, int KB, typename O, bool FINAL>
LO_DEVICE void product_tile(const NsTask& t, const NsProduct& pr,
                            const NsFinal& fin, char* lds) {
  constexpr int W = T / 2;      // a wave's square
  constexpr int F = W / 16;     // its 16 x 16 fragments a side
  constexpr int IMG = T * 128;  // bytes of one operand's tile: T rows, 32 k
  constexpr int LOADS = T / 32; // a wave's loads of one operand's tile
  const Planes pl = planes(t, pr.ws);
  const int ti = t.ti, tj = t.tj, splits = t.splits, slice = t.slice;
  const int k0 = t.k0, k1 = t.k1;
  const f16* P = KIND == NS_GRAM   ? pl.x(pr.from)
                 : KIND == NS_POLY ? pl.a()
                                   : pl.c();
  const f16* Q = KIND == NS_POLY ? pl.a() : pl.x(pr.from);

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wave >> 1, wc = wave & 1;

  // 1 KiB (8 lines) an instruction; the 16-byte piece that lands at place p of
  // line l is piece p ^ (l & 7), which spreads a column of pieces over the
  // banks. Addresses are a scalar base and a lane's offset, and the loop below
  // is unrolled over the S buffers: with one wave a SIMD, what is computed
  // between the loads would be waited for.
  // APPLY's Q is 32 rows of X and T of its columns, an image of 32 lines for
  // each 32 columns. There 4 lanes read 32 bytes of a line, 8 lines (0..3 and
  // 8..11, say) at once: piece p lands at p ^ 2 ((l / 2 & 1) + 2 (l / 8 & 1)).
  const unsigned lane_p = lane / 8 * 128 + ((lane % 8) ^ (lane / 8)) * 16;
  const unsigned lane_q =
      KIND != NS_APPLY
          ? lane_p
          : lane / 8 * 128 + ((lane % 8) ^ (lane / 8 & 2) ^ (wave & 1) * 4) * 16;
  const long panel = (long)t.mp * 128;  // bytes of 32 columns
  const char* Pb = (const char*)P + (ti * T + wave * LOADS * 8) * 128l;
  const char* Qb = KIND != NS_APPLY
                       ? (const char*)Q + (tj * T + wave * LOADS * 8) * 128l
                       : (const char*)Q + tj * (T / 32) * panel + wave * 1024;
  const unsigned lds_at =
      (unsigned)(size_t)(__attribute__((address_space(3))) char*)lds;
  auto stage = [&](int buf, int kt) {
    const unsigned to = lds_at + buf * (2 * KB * IMG);
    // Written out, since before a ds_read_b64_tr_b16 the compiler waits for
    // all loads to LDS that it knows of. These have no result in registers;
    // `ready` waits for them.
    auto load = [&](const char* from, unsigned lane_at, unsigned at) {
      asm volatile(
          "s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(at),
          "v"(lane_at), "s"(from)
          : "m0", "memory");
    };
    #pragma unroll
    for (int h = 0; h < KB; ++h)
      #pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const unsigned p = to + h * 2 * IMG;
        load(Pb + (kt + h) * panel + i * 1024, lane_p,
             p + (wave * LOADS + i) * 1024);
        if constexpr (KIND == NS_APPLY)
          load(Qb + (kt + h) * 4096l + i * panel, lane_q,
               p + IMG + (i * 4 + wave) * 1024);
        else
          load(Qb + (kt + h) * panel + i * 1024, lane_q,
               p + IMG + (wave * LOADS + i) * 1024);
      }
  };
  struct Frags {
    f16x8 ph[F], pw[F], qh[F], ql[F];
  };
  auto frag = [&](const char* img, int row, int half) {
    return *(const f16x8*)(img + row * 128 +
                           ((half * 64 + (lane >> 4) * 16) ^ ((row & 7) << 4)));
  };
  // columns i*16.. of APPLY's Q: of 16 lanes, lane l names four columns of row
  // l / 4, and gets column l of the four rows
  const int q_row = (lane >> 4) * 8 + (lane >> 2 & 3);
  const int q_at = q_row * 128 + (lane & 3) * 8 +
                   ((lane >> 3 & 1) + (lane >> 4 & 1) * 2) * 32;
  auto turned = [&](const char* img, int i, int half) {
    const int col = wc * W + i * 16;
    const char* at = img + (col >> 5) * 4096 +
                     (q_at ^ ((half * 2 + (col >> 4 & 1)) * 32));
    f16x8 v;
    #pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f16x4 four = __builtin_bit_cast(
          f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16(
                     (__attribute__((address_space(3))) h16x4*)(at + h * 512)));
      #pragma unroll
      for (int j = 0; j < 4; ++j) v[h * 4 + j] = four[j];
    }
    return v;
  };
  auto frag_q = [&](const char* img, int i, int half) {
    if constexpr (KIND == NS_APPLY) return turned(img, i, half);
    else return frag(img, wc * W + i * 16 + (lane & 15), half);
  };
  auto read = [&](int buf, int h, Frags& s) {
    const char* img = lds + (buf * KB + h) * 2 * IMG;
    #pragma unroll
    for (int i = 0; i < F; ++i) {
      s.ph[i] = frag(img, wr * W + i * 16 + (lane & 15), 0);
      s.qh[i] = frag_q(img + IMG, i, 0);
    }
    #pragma unroll
    for (int i = 0; i < F; ++i) {
      s.ql[i] = frag_q(img + IMG, i, 1);
      s.pw[i] = frag(img, wr * W + i * 16 + (lane & 15), 1);
    }
  };
  f32x4 acc[F][F] = {};
  // kind by kind: an accumulator's next use is F * F instructions away
  auto products = [&](const f16x8 (&p)[F], const f16x8 (&q)[F]) {
    #pragma unroll
    for (int i = 0; i < F; ++i)
      #pragma unroll
      for (int j = 0; j < F; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(p[i], q[j],
                                                           acc[i][j], 0, 0, 0);
  };
  auto add = [&](const Frags& s) {
    products(s.ph, s.qh);
    products(s.ph, s.ql);
    products(s.pw, s.qh);
  };

  // A's part of C: A is symmetric, so its row c holds a lane's four values in
  // a line. Small tiles fetch it while the sum is taken (large ones have no
  // registers to spare, and more to do meanwhile).
  constexpr bool EARLY = KIND == NS_POLY && T < 128;
  f16x4 ah[EARLY ? F * F : 1], al[EARLY ? F * F : 1];
  auto fetch = [&](int i, int j, f16x4& hi, f16x4& lo) {
    const int r = ti * T + wr * W + i * 16 + (lane >> 4) * 4;
    const int c = tj * T + wc * W + j * 16 + (lane & 15);
    const f16* s = pl.a() + split_at(c, r, t.mp);
    hi = *(const f16x4*)s;
    lo = *(const f16x4*)(s + 32);
  };
  if constexpr (EARLY) {
    #pragma unroll
    for (int i = 0; i < F * F; ++i) fetch(i / F, i % F, ah[i], al[i]);
  }

  // KB steps a stage and barrier. The loop adds a step's fragments while the
  // next one's are read from LDS and S - 1 stages are on their way. `ready`
  // waits until the stage at kt has landed and every wave has read the one
  // before, whose buffer is then free.
  auto ready = [&](int newest) {
    if (newest < k1)
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(
                       (S - 2) * 2 * LOADS * KB)
                   : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  };
  #pragma unroll
  for (int s = 0; s < S - 1; ++s)
    if (k0 + s * KB < k1) stage(s, k0 + s * KB);
  Frags even, odd;
  ready(k0 + (S - 2) * KB);
  read(0, 0, even);
  if (k0 + (S - 1) * KB < k1) stage(S - 1, k0 + (S - 1) * KB);
  [&] {
    constexpr int ROUND = S * KB * (S * KB % 2 + 1);  // even
    for (int k = k0;; k += ROUND) {
      #pragma unroll
      for (int n = 0; n < ROUND; ++n) {
        const int kt = k + n, s = n / KB % S, next = (n + 1) % (S * KB);
        if (kt + 1 < k1) {
          const bool fresh = next % KB == 0;
          if (fresh) ready(kt + 1 + (S - 2) * KB);
          read(next / KB, next % KB, n % 2 ? even : odd);
          // k1 - k0 is a multiple of KB
          if (fresh && kt + 1 + (S - 1) * KB < k1)
            stage(s, kt + 1 + (S - 1) * KB);
        }
        add(n % 2 ? odd : even);
        if (kt + 1 >= k1) return;
      }
    }
  }();
  __syncthreads();  // the staging buffers are free from here on

  if (splits > 1) {
    // Parts are written through to where all dies see them (agent-scope
    // stores), and have arrived there before the counter goes up, so that no
    // cache needs writing back. Nor has any cache an older copy to drop: the
    // last block is the first of this launch to read these lines, and what
    // earlier launches left went where this one began. (A release and an
    // acquire cost 8 us a launch instead, at 36 tiles.)
    typedef unsigned long long u64;
    u64* part = (u64*)(pr.parts + t.part);
    const int mine = wave * F * F * 128 + lane;
    #pragma unroll
    for (int i = 0; i < F * F; ++i) {
      const f32x4& v = acc[i / F][i % F];
      u64* to = part + (long)slice * (T * T / 2) + mine + i * 128;
      __hip_atomic_store(to, __builtin_bit_cast(u64, f32x2{v[0], v[1]}),
                         __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(to + 64, __builtin_bit_cast(u64, f32x2{v[2], v[3]}),
                         __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    unsigned* last = (unsigned*)lds;
    if (threadIdx.x == 0)
      *last = __hip_atomic_fetch_add(pr.slots + t.slot, 1u,
                                     __ATOMIC_RELAXED,
                                     __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    const bool join = *last == (unsigned)splits - 1;
    if (!join) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
    __syncthreads();  // all have read it
    if (threadIdx.x == 0)
      __hip_atomic_store(pr.slots + t.slot, 0u, __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_AGENT);
    f32x4 own[F * F];
    #pragma unroll
    for (int i = 0; i < F * F; ++i) {
      own[i] = acc[i / F][i % F];
      acc[i / F][i % F] = f32x4{};
    }
    for (int q = 0; q < splits; ++q) {
      u64* from = part + (long)q * (T * T / 2) + mine;
      #pragma unroll
      for (int i = 0; i < F * F; ++i) {
        f32x4 v = own[i];
        if (q != slice) {
          const f32x2 a = __builtin_bit_cast(
              f32x2, __hip_atomic_load(from + i * 128, __ATOMIC_RELAXED,
                                        __HIP_MEMORY_SCOPE_AGENT));
          const f32x2 b = __builtin_bit_cast(
              f32x2, __hip_atomic_load(from + i * 128 + 64, __ATOMIC_RELAXED,
                                        __HIP_MEMORY_SCOPE_AGENT));
          v = f32x4{a.x, a.y, b.x, b.y};
        }
        acc[i / F][i % F] += v;
      }
    }
  }

  // a lane holds rows r..r+3 of column c of each fragment; each wave turns its
  // square in its own part of LDS, so that it can write whole lines by rows
  // and by columns
  constexpr int PITCH = W + 4;
  unsigned* sq = (unsigned*)lds + wave * W * PITCH;
  const int rw = ti * T + wr * W, cw = tj * T + wc * W;
  #pragma unroll
  for (int i = 0; i < F; ++i)
    #pragma unroll
    for (int j = 0; j < F; ++j) {
      const int r = i * 16 + (lane >> 4) * 4, c = j * 16 + (lane & 15);
      f32x4 v = acc[i][j] * pr.alpha;
      if constexpr (KIND == NS_POLY) {
        f16x4 hi, lo;
        if constexpr (EARLY) hi = ah[i * F + j], lo = al[i * F + j];
        else fetch(i, j, hi, lo);
        #pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] += pr.beta * ((float)hi[e] + (float)lo[e]);
          if (rw + r + e == cw + c) v[e] += pr.diag;
        }
      }
      #pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = v[e];
        sq[(r + e) * PITCH + c] = FINAL ? __builtin_bit_cast(unsigned, x)
                                        : pack(x);
      }
    }
  // only this wave reads its square, after its own writes
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  // 8 values by rows: (r, c) .. (r, c + 7); by columns: (r, c) .. (r + 7, c)
  auto along_row = [&](int idx, int& r, int& c, u32x4& a, u32x4& b) {
    r = idx / (W / 8);
    c = idx % (W / 8) * 8;
    a = *(const u32x4*)(sq + r * PITCH + c);
    b = *(const u32x4*)(sq + r * PITCH + c + 4);
  };
  auto along_col = [&](int idx, int& r, int& c, u32x4& a, u32x4& b) {
    r = (idx >> 4) % (W / 8) * 8;
    c = (idx >> 4) / (W / 8) * 16 + (idx & 15);
    #pragma unroll
    for (int j = 0; j < 4; ++j) {
      a[j] = sq[(r + j) * PITCH + c];
      b[j] = sq[(r + 4 + j) * PITCH + c];
    }
  };
  if constexpr (FINAL) {
    const NsOutput& out = fin.out;
    const NsMat* m = fin.mats ? fin.mats + t.mat : &fin.one;
    const int nrows = m->rows, ncols = m->cols;
    const long src = m->src + (fin.mats ? 0 : t.mat * fin.src_step);
    const bool tall = nrows > ncols;
    const float step = out.lr * m->gain;
    // where a lane's eight values of piece idx go, and how many are left there
    auto place = [&](int idx, long& at) {
      const int r = tall ? (idx >> 4) % (W / 8) * 8 : idx / (W / 8);
      const int c = tall ? (idx >> 4) / (W / 8) * 16 + (idx & 15)
                         : idx % (W / 8) * 8;
      const int row = tall ? cw + c : rw + r, col = tall ? rw + r : cw + c;
      at = src + (long)row * ncols + col;
      return row < nrows ? ncols - col : 0;
    };
    constexpr int N = W * W < 512 ? 1 : W * W / 512;  // pieces a lane
    constexpr int CH = N < 4 ? N : 4;  // whose weights are read at a time
    for (int i0 = 0; i0 < N; i0 += CH) {
      f32x4 w[CH][2] = {};
      if (out.master) {
        #pragma unroll
        for (int i = 0; i < CH; ++i) {
          long at;
          const int idx = lane + (i0 + i) * 64;
          const int n = idx < W * W / 8 ? place(idx, at) : 0;
          #pragma unroll
          for (int h = 0; h < 2; ++h)
            if (n > h * 4) w[i][h] = load4(out.master, at + h * 4, n - h * 4);
        }
      }
      #pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int idx = lane + (i0 + i) * 64;
        if (idx >= W * W / 8) continue;
        long at;
        const int n = place(idx, at);
        int r, c;
        u32x4 a, b;
        if (tall) along_col(idx, r, c, a, b);
        else along_row(idx, r, c, a, b);
        #pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (n <= h * 4) continue;
          const f32x4 o = __builtin_bit_cast(f32x4, h ? b : a);
          if (out.master) {
            const f32x4 v = w[i][h] * out.keep - step * o;
            store4(out.master, at + h * 4, n - h * 4, v);
            store4((bf16*)out.mirror, at + h * 4, n - h * 4, v);
          } else {
            store4((O*)out.out, at + h * 4, n - h * 4, o);
          }
        }
      }
    }
  } else {
    f16* rows = KIND == NS_GRAM   ? pl.a()
                : KIND == NS_POLY ? pl.c()
                                  : pl.x(pr.from ^ 1);
    #pragma unroll 4
    for (int idx = lane; idx < W * W / 8; idx += 64) {
      int r, c;
      u32x4 a, b;
      f16x8 hi, lo;
      along_row(idx, r, c, a, b);
      unpack8(a, b, hi, lo);
      f16* to = rows + split_at(rw + r, cw + c, t.mp);
      *(f16x8*)to = hi;
      *(f16x8*)(to + 32) = lo;
      if (KIND != NS_APPLY && ti != tj) {  // the other triangle
        along_col(idx, r, c, a, b);
        unpack8(a, b, hi, lo);
        to = rows + split_at(cw + c, rw + r, t.mp);
        *(f16x8*)to = hi;
        *(f16x8*)(to + 32) = lo;
      }
    }
  }
}

// MANY: only 64 x 64 tiles, more than fit the chip at two blocks a CU. With
// three staged tiles there is room for three: 16 x 512 x 2048 (576 tiles) takes
// 603 us in place of 629.
template <int KIND, typename O, bool FINAL, bool MANY>
__global__ __launch_bounds__(256, MANY ? 3 : 2) void ns_product_kernel(
    NsProduct pr, NsFinal fin) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const NsTask t = task_of<KIND>(pr);
  if constexpr (MANY) product_tile<64, KIND, 3, 1, O, FINAL>(t, pr, fin, lds);
  else if (t.tile == 128) product_tile<128, KIND, 2, 1, O, FINAL>(t, pr, fin, lds);
  else if (t.tile == 64) product_tile<64, KIND, 4, 1, O, FINAL>(t, pr, fin, lds);
  else product_tile<32, KIND, 4, 2, O, FINAL>(t, pr, fin, lds);
}

// ------------------------------------------- matrices that fit one block ----
// Up to 64 x 1024 or 32 x 2048: one block does the whole call, momentum and
// norm included, with X in the registers of its eight waves.
//
// A wave owns groups of 32 columns. A lane's share of X' = C X serves as it is
// as an operand of the next product, because the order in which a sum is taken
// is free as long as both operands follow it: the accumulator gives lane
// (g, c) = (lane / 16, lane % 16) rows 16 b + 4 g + e of column c, and so the
// sum over rows runs, in steps f of 32, over rows 32 f + 4 g + (0..3) and
// 32 f + 16 + 4 g + (0..3); C is laid out in that order in LDS. For X' X'^T a
// group is turned in LDS, each wave in its own part, where the waves' shares
// of A then meet and C is made from them.
struct NsSmallSteps {
  NsStep st[kNsSmallSteps];
  int n;
};

// eight values as packed halves (kept as words: a vector of f16 that lives
// across a loop is given a register an element)
struct Halves {
  u32x4 hi, lo;
};

// scale is a power of two, so either is one rounding of v * scale
LO_DEVICE void split_scaled(float v, float scale, f16& hi, f16& lo) {
  hi = (f16)__builtin_fmaf(v, scale, 0.f);
  lo = (f16)__builtin_fmaf(v, scale, -(float)hi);
}

LO_DEVICE Halves halves(const f32x4& a, const f32x4& b, float scale) {
  Halves h;
  #pragma unroll
  for (int j = 0; j < 4; ++j) {
    f16x2 hi, lo;
    #pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = (j & 1) * 2 + e;
      f16 vh, vl;
      split_scaled(j < 2 ? a[i] : b[i], scale, vh, vl);
      hi[e] = vh;
      lo[e] = vl;
    }
    h.hi[j] = __builtin_bit_cast(unsigned, hi);
    h.lo[j] = __builtin_bit_cast(unsigned, lo);
  }
  return h;
}

LO_DEVICE f32x4 mma(const u32x4& p, const u32x4& q, const f32x4& acc) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, p),
                                                __builtin_bit_cast(f16x8, q),
                                                acc, 0, 0, 0);
}

LO_DEVICE void mma3(f32x4& acc, const Halves& p, const Halves& q) {
  acc = mma(p.lo, q.hi, acc);
  acc = mma(p.hi, q.lo, acc);
  acc = mma(p.hi, q.hi, acc);
}

// a square image of 16 MB rows in LDS; its 16-byte pieces hold eight values in
// the sum's order, and an exclusive or spreads a column of them over the banks
template <int MB>
struct Image {
  static constexpr int UNITS = MB * 4;  // pieces a row
  static constexpr int BYTES = MB * 16 * UNITS * 16;
  char* p;
  LO_DEVICE char* piece(int row, int f, int half, int g) const {
    return p + row * UNITS * 16 +
           (((f * 8 + half * 4 + g) ^ (row & (UNITS - 1))) << 4);
  }
  LO_DEVICE Halves get(int row, int f, int g) const {
    return {*(const u32x4*)piece(row, f, 0, g),
            *(const u32x4*)piece(row, f, 1, g)};
  }
  // rows 16 b + 4 g + (0..3) of column c, as row c of the symmetric matrix
  LO_DEVICE void put4(int c, int b, int g, const f32x4& v) const {
    f16x4 hi, lo;
    #pragma unroll
    for (int e = 0; e < 4; ++e) {
      f16 h, l;
      split(v[e], h, l);
      hi[e] = h;
      lo[e] = l;
    }
    *(f16x4*)(piece(c, b >> 1, 0, g) + (b & 1) * 8) = hi;
    *(f16x4*)(piece(c, b >> 1, 1, g) + (b & 1) * 8) = lo;
  }
  LO_DEVICE void get4(int c, int b, int g, f32x4& v) const {
    const f16x4 hi = *(const f16x4*)(piece(c, b >> 1, 0, g) + (b & 1) * 8);
    const f16x4 lo = *(const f16x4*)(piece(c, b >> 1, 1, g) + (b & 1) * 8);
    #pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (float)hi[e] + (float)lo[e];
  }
  LO_DEVICE void put1(int row, int k, float v) const {
    f16 hi, lo;
    split(v, hi, lo);
    const int b = k >> 4, g = (k >> 2) & 3;
    const int at = (b & 1) * 8 + (k & 3) * 2;
    *(f16*)(piece(row, b >> 1, 0, g) + at) = hi;
    *(f16*)(piece(row, b >> 1, 1, g) + at) = lo;
  }
};

// keeps what is read from LDS on its side: a group of columns re-reads C
// rather than hold all of it in registers
LO_DEVICE void keep_apart() { asm volatile("" ::: "memory"); }

// a wave's part of LDS: its blocks of A (16 x 16 of the lower triangle, 1 KiB
// each), or before those the group of X that it turns (16 MB rows of 36 words)
template <int MB>
constexpr int ns_small_part() {
  return MB == 2 ? 32 * 36 * 4 : MB * (MB + 1) / 2 * 1024;
}
template <int MB>
constexpr int ns_small_lds() {
  return 2 * Image<MB>::BYTES + 8 * ns_small_part<MB>();
}

// 16 MB rows, NG groups of 32 columns a wave
template <typename T, int MB, int NG>
__global__ __launch_bounds__(512, 2) void ns_small_kernel(NsGroup gr, NsInput in,
                                                          NsSmallSteps steps,
                                                          float eps,
                                                          NsOutput out) {
  constexpr int FB = MB / 2, TRI = MB * (MB + 1) / 2;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const Image<MB> imgA{lds}, imgC{lds + Image<MB>::BYTES};
  constexpr int PART = ns_small_part<MB>() / 16;
  f32x4* parts = (f32x4*)(lds + 2 * Image<MB>::BYTES);  // [8][PART]
  __shared__ double red[8];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int g = lane >> 4, cl = lane & 15;
  NsMat m = gr.mats ? gr.mats[blockIdx.x] : gr.one;
  if (!gr.mats) m.src += blockIdx.x * gr.src_step;
  const bool tall = m.rows > m.cols;
  const int short_ = min(m.rows, m.cols), long_ = max(m.rows, m.cols);
  const int groups = (long_ + 31) / 32;

  // Rows r..r+3 of column c of X lie together in a tall input, a row apart in
  // a wide one. Places outside the matrix read its first element and count as
  // zero, which keeps the loads free of branches.
  const long stride_r = tall ? 1 : m.cols, stride_c = tall ? m.cols : 1;
  auto place = [&](int r, int c) {
    const bool ok = r < short_ && c < long_;
    return m.src + (ok ? r * stride_r + c * stride_c : 0);
  };
  auto inside = [&](int r, int c) { return r < short_ && c < long_; };
  // four at once where all four are there and lie together
  auto read4 = [&](const auto* p, int r, int c) {
    f32x4 v;
    if (tall && (short_ & 3) == 0) {
      v = load4(p, place(r, c), 4);
      if (!inside(r, c)) v = f32x4{};
    } else {
      #pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (float)p[place(r + e, c)];
      #pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = inside(r + e, c) ? v[e] : 0.f;
    }
    return v;
  };
  auto write4 = [&](auto* p, int r, int c, const f32x4& v) {
    typedef std::remove_reference_t<decltype(*p)> P;
    if (tall && (short_ & 3) == 0) {
      if (inside(r, c)) store4(p, place(r, c), 4, v);
    } else {
      #pragma unroll
      for (int e = 0; e < 4; ++e)
        if (inside(r + e, c)) p[place(r + e, c)] = (P)v[e];
    }
  };

  f32x4 u[NG][2][MB];
  double acc2 = 0.0;
  #pragma unroll
  for (int i = 0; i < NG; ++i) {
    #pragma unroll
    for (int h = 0; h < 2; ++h)
      #pragma unroll
      for (int b = 0; b < MB; ++b) u[i][h][b] = f32x4{};
    if (w + 8 * i >= groups) continue;
    #pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = (w + 8 * i) * 32 + h * 16 + cl;
      #pragma unroll
      for (int b = 0; b < MB; ++b)
        u[i][h][b] = read4((const T*)in.grad, b * 16 + g * 4, c) * in.gscale;
      if (in.mom) {
        f32x4 mo[MB];
        #pragma unroll
        for (int b = 0; b < MB; ++b) mo[b] = read4(in.mom, b * 16 + g * 4, c);
        #pragma unroll
        for (int b = 0; b < MB; ++b) {
          mo[b] = in.mu * mo[b] + u[i][h][b];
          write4(in.mom, b * 16 + g * 4, c, mo[b]);
          u[i][h][b] = in.nesterov ? u[i][h][b] + in.mu * mo[b] : mo[b];
        }
      }
      #pragma unroll
      for (int b = 0; b < MB; ++b)
        #pragma unroll
        for (int e = 0; e < 4; ++e)
          acc2 += (double)u[i][h][b][e] * (double)u[i][h][b][e];
    }
  }
  for (int off = 32; off > 0; off >>= 1) acc2 += __shfl_xor(acc2, off);
  if (lane == 0) red[w] = acc2;
  __syncthreads();
  double total = 0.0;
  for (int i = 0; i < 8; ++i) total += red[i];
  const NsNorm norm(total, eps);
  const float sx = steps.st[0].sx;
  Halves x[NG][2][FB];  // [group][16 columns][32 rows]
  #pragma unroll
  for (int i = 0; i < NG; ++i)
    #pragma unroll
    for (int h = 0; h < 2; ++h)
      #pragma unroll
      for (int f = 0; f < FB; ++f)
        x[i][h][f] = halves(norm(u[i][h][2 * f]), norm(u[i][h][2 * f + 1]), sx);

  // C X of a group's columns
  auto apply = [&](const Halves (&xi)[2][FB], f32x4 (&d)[2][MB]) {
    #pragma unroll
    for (int b = 0; b < MB; ++b) {
      keep_apart();
      d[0][b] = d[1][b] = f32x4{};
      #pragma unroll
      for (int f = 0; f < FB; ++f) {
        const Halves c = imgC.get(b * 16 + cl, f, g);
        #pragma unroll
        for (int h = 0; h < 2; ++h) mma3(d[h][b], c, xi[h][f]);
      }
    }
  };
  // a group of X as [rows][32 columns] words (hi below lo), 4 words between
  // rows: no two lanes of a write meet in a bank
  constexpr int PITCH = 36;
  unsigned* turn = (unsigned*)(parts + w * PART);
  static_assert(16 * MB * PITCH <= PART * 4 && TRI * 64 <= PART);

  for (int s = 0; s < steps.n; ++s) {
    const NsStep& k = steps.st[s];
    // X <- C X (but before the first C), its scale from the last step's
    // sc * sx to sx, and A = X X^T of it
    f32x4 gram[MB][MB];
    #pragma unroll
    for (int a = 0; a < MB; ++a)
      #pragma unroll
      for (int b = 0; b <= a; ++b) gram[a][b] = f32x4{};
    #pragma unroll
    for (int i = 0; i < NG; ++i) {
      if (w + 8 * i >= groups) continue;
      if (s > 0) {
        const NsStep& last = steps.st[s - 1];
        const float scale = last.sn / (last.sc * last.sx);
        f32x4 d[2][MB];
        apply(x[i], d);
        #pragma unroll
        for (int h = 0; h < 2; ++h)
          #pragma unroll
          for (int f = 0; f < FB; ++f)
            x[i][h][f] = halves(d[h][2 * f], d[h][2 * f + 1], scale);
      }
      // only this wave's lanes meet here; LDS serves them in order
      keep_apart();
      #pragma unroll
      for (int h = 0; h < 2; ++h)
        #pragma unroll
        for (int f = 0; f < FB; ++f)
          #pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int row = f * 32 + (j >> 1) * 16 + g * 4 + (j & 1) * 2;
            const unsigned hi = x[i][h][f].hi[j], lo = x[i][h][f].lo[j];
            turn[row * PITCH + h * 16 + cl] =
                __builtin_amdgcn_perm(lo, hi, 0x05040100);
            turn[(row + 1) * PITCH + h * 16 + cl] =
                __builtin_amdgcn_perm(lo, hi, 0x07060302);
          }
      keep_apart();
      Halves q[MB];  // rows of X, 32 columns
      #pragma unroll
      for (int a = 0; a < MB; ++a) {
        const unsigned* row = turn + (a * 16 + cl) * PITCH + g * 4;
        const u32x4 u0 = *(const u32x4*)row, u1 = *(const u32x4*)(row + 16);
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
          const unsigned even = j < 2 ? u0[2 * j] : u1[2 * j - 4];
          const unsigned odd = j < 2 ? u0[2 * j + 1] : u1[2 * j - 3];
          q[a].hi[j] = __builtin_amdgcn_perm(odd, even, 0x05040100);
          q[a].lo[j] = __builtin_amdgcn_perm(odd, even, 0x07060302);
        }
      }
      #pragma unroll
      for (int a = 0; a < MB; ++a)
        #pragma unroll
        for (int b = 0; b <= a; ++b) mma3(gram[a][b], q[a], q[b]);
    }
    keep_apart();
    #pragma unroll
    for (int a = 0; a < MB; ++a)
      #pragma unroll
      for (int b = 0; b <= a; ++b)
        parts[w * PART + (a * (a + 1) / 2 + b) * 64 + lane] = gram[a][b];
    __syncthreads();
    // the waves' sums in their order
    const int used = min(groups, 8);
    for (int t = w; t < TRI; t += 8) {
      f32x4 v = {};
      #pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < used) v += parts[i * PART + t * 64 + lane];
      int a = 0;
      while ((a + 1) * (a + 2) / 2 <= t) ++a;
      const int b = t - a * (a + 1) / 2;
      v *= k.sa / (k.sx * k.sx);
      // v: rows 16 a + 4 g + e of column 16 b + cl
      imgA.put4(b * 16 + cl, a, g, v);
      if (a != b) {
        #pragma unroll
        for (int e = 0; e < 4; ++e)
          imgA.put1(a * 16 + g * 4 + e, b * 16 + cl, v[e]);
      }
    }
    __syncthreads();
    const float alpha = k.c * k.sc / (k.sa * k.sa), beta = k.b * k.sc / k.sa;
    for (int t = w; t < MB * MB; t += 8) {
      const int a = t / MB, b = t % MB;
      f32x4 d = {}, av;
      #pragma unroll
      for (int f = 0; f < FB; ++f)
        mma3(d, imgA.get(a * 16 + cl, f, g), imgA.get(b * 16 + cl, f, g));
      imgA.get4(b * 16 + cl, a, g, av);
      #pragma unroll
      for (int e = 0; e < 4; ++e) {
        d[e] = d[e] * alpha + beta * av[e];
        if (a == b && g * 4 + e == cl) d[e] += k.a * k.sc;
      }
      imgC.put4(b * 16 + cl, a, g, d);
    }
    __syncthreads();
  }

  // the last X' = C X goes out
  const NsStep& last = steps.st[steps.n - 1];
  const float scale = 1.f / (last.sc * last.sx), step = out.lr * m.gain;
  #pragma unroll
  for (int i = 0; i < NG; ++i) {
    if (w + 8 * i >= groups) continue;
    f32x4 d[2][MB];
    apply(x[i], d);
    #pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = (w + 8 * i) * 32 + h * 16 + cl;
      if (out.master) {
        f32x4 v[MB];
        #pragma unroll
        for (int b = 0; b < MB; ++b)
          v[b] = read4(out.master, b * 16 + g * 4, c) * out.keep -
                 d[h][b] * (scale * step);
        #pragma unroll
        for (int b = 0; b < MB; ++b) {
          write4(out.master, b * 16 + g * 4, c, v[b]);
          write4((bf16*)out.mirror, b * 16 + g * 4, c, v[b]);
        }
      } else {
        #pragma unroll
        for (int b = 0; b < MB; ++b)
          write4((T*)out.out, b * 16 + g * 4, c, d[h][b] * scale);
      }
    }
  }
}

template <typename T, int MB, int NG>
void run_small(const NsGroup& g, const NsInput& in, const NsSmallSteps& st,
               float eps, const NsOutput& out, hipStream_t s) {
  hipLaunchKernelGGL((ns_small_kernel<T, MB, NG>), dim3(g.count), dim3(512),
                     ns_small_lds<MB>(), s, g, in, st, eps, out);
}

template <typename T>
void pick_small(const NsGroup& g, int shortest, int longest, const NsInput& in,
                const NsSmallSteps& st, float eps, const NsOutput& out,
                hipStream_t s) {
  if (shortest <= 32) {
    if (longest <= 256) run_small<T, 2, 1>(g, in, st, eps, out, s);
    else if (longest <= 512) run_small<T, 2, 2>(g, in, st, eps, out, s);
    else if (longest <= 1024) run_small<T, 2, 4>(g, in, st, eps, out, s);
    else run_small<T, 2, 8>(g, in, st, eps, out, s);
  } else if (longest <= 256) {
    run_small<T, 4, 1>(g, in, st, eps, out, s);
  } else if (longest <= 512) {
    run_small<T, 4, 2>(g, in, st, eps, out, s);
  } else {
    run_small<T, 4, 4>(g, in, st, eps, out, s);
  }
}

// every tile size's staging buffers take 64 KiB; 128's squares need 4 KiB more
constexpr int kNsLds = 4 * 64 * (64 + 4) * 4;
constexpr int kNsLdsMany = 3 * 2 * 64 * 128;

template <int KIND, typename O, bool FINAL>
void product(const NsGroup& g, int from, float alpha, float beta, float diag,
             const NsFinal& fin, hipStream_t s) {
  const NsMat& m = g.one;
  const NsProduct pr{g.tasks[KIND],     g.ws,
                     from,              m.mp,
                     m.np,              m.kind[KIND].tile,
                     g.kinds[KIND],     m.kind[KIND].whole,
                     m.kind[KIND].splits, g.count,
                     g.ws_step,         g.part_step,
                     g.slot_step,       alpha,
                     beta,              diag,
                     g.parts,           g.slots};
  const long blocks = g.all_kinds[KIND];
  if (g.tile[KIND] == 64 && blocks > kNsSlots)
    hipLaunchKernelGGL((ns_product_kernel<KIND, O, FINAL, true>), dim3(blocks),
                       dim3(256), kNsLdsMany, s, pr, fin);
  else
    hipLaunchKernelGGL((ns_product_kernel<KIND, O, FINAL, false>), dim3(blocks),
                       dim3(256), kNsLds, s, pr, fin);
}

template <typename T>
void run(const NsGroup& g, const NsInput& in, const NsStep* st, int n,
         float eps, const NsOutput& out, hipStream_t s) {
  hipLaunchKernelGGL(ns_momentum_kernel<T>, dim3(g.all_chunks), dim3(256), 0, s,
                     g, in);
  hipLaunchKernelGGL(ns_split_kernel<T>, dim3(g.all_splits), dim3(256), 0, s, g,
                     in, st[0].sx, eps);
  const NsFinal fin{out, g.mats, g.one, g.src_step};
  for (int i = 0; i < n; ++i) {
    const NsStep& k = st[i];
    const int from = i & 1;
    product<NS_GRAM, float, false>(g, from, k.sa / (k.sx * k.sx), 0.f, 0.f,
                                   fin, s);
    product<NS_POLY, float, false>(g, from, k.c * k.sc / (k.sa * k.sa),
                                   k.b * k.sc / k.sa, k.a * k.sc, fin, s);
    if (i + 1 < n)
      product<NS_APPLY, float, false>(g, from, k.sn / (k.sc * k.sx), 0.f, 0.f,
                                      fin, s);
    else
      product<NS_APPLY, T, true>(g, from, 1.f / (k.sc * k.sx), 0.f, 0.f, fin,
                                 s);
  }
}

}  // namespace

void launch_newton_schulz_small(const NsGroup& g, int shortest, int longest,
                                int dtype, const NsInput& in, const NsStep* st,
                                int n, float eps, const NsOutput& out,
                                hipStream_t s) {
  NsSmallSteps all{};
  all.n = n;
  for (int i = 0; i < n; ++i) all.st[i] = st[i];
  if (dtype == 0) pick_small<bf16>(g, shortest, longest, in, all, eps, out, s);
  else if (dtype == 1) pick_small<f16>(g, shortest, longest, in, all, eps, out, s);
  else pick_small<float>(g, shortest, longest, in, all, eps, out, s);
}

void launch_newton_schulz(const NsGroup& g, int dtype, const NsInput& in,
                          const NsStep* st, int n, float eps,
                          const NsOutput& out, hipStream_t s) {
  if (dtype == 0) run<bf16>(g, in, st, n, eps, out, s);
  else if (dtype == 1) run<f16>(g, in, st, n, eps, out, s);
  else run<float>(g, in, st, n, eps, out, s);
}

}  // namespace lo
