// Layer normalisation, dropout and the two fused behind a residual connection, on column-major
// matrices (a column = one token's features).  All of it is bound by HBM bandwidth: each kernel
// reads its operands once and keeps a column in registers between the reduction and the result.
//
//   norm forward  : h = residual + drop(x)  (plain normalisation: h = x)
//                   mu = mean(h), r = 1 / sqrt(mean((h - mu)^2) + eps), y = gain (h - mu) r + bias
//   norm backward : xh = (h - mu) r, G = gain dy
//                   dh' = r (G - mean(G) - xh mean(G xh)) + dh,   dres (+)= dh',  dx (+)= drop'(dh')
//                   dgain (+)= sum over columns of dy xh,  dbias (+)= sum over columns of dy
//   dropout       : y = residual + drop(x),  dx (+)= drop'(dy)
//
// Statistics, sums and weight gradients are fp32 whatever the storage type; each result is rounded
// once.  Weight gradients: every CTA adds its columns in registers and leaves one vector of
// partial sums; a second small kernel adds those in a fixed order, so a call's result does not
// depend on which CTA finishes first.
//
// Measured, device time of a call in a loop (a plain copy of this size moves 6.5 TB/s):
//   forward           1024 x 16384 Half 14.5 us, 4.6 TB/s;  4096 x 8192 fp32 50 us, 5.4 TB/s
//   with the residual 1024 x 16384 Half 28 us, 4.8 TB/s;    4096 x 8192 fp32 86 us, 6.2 TB/s
//   backward          384 x 16384 fp32 20 us, 3.8 TB/s;     8192 x 4096 fp32 80 us, 5.0 TB/s;
//                     8192 x 8192 Half 98 us, 4.1 TB/s
//   dropout           4096 x 16384 Half with a residual 70 us, 5.7 TB/s
// The Half backward pass is bound by the instructions of its 16 warps, not by memory: with copies of 16
// bytes instead of whole columns it takes 95 us of the 98.
#include <cuda_fp16.h>
#include "math.cuh"
#include "ptx.cuh"
#include "launch.h"

namespace gb {

namespace {

constexpr int kEl = 8;  // elements a thread handles together: one generator block

__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void load8(const __half* p, float (&x)[8]) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(__half* p, const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) *reinterpret_cast<__half2*>(&w[i]) = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// Rows of a column that a thread of a group of G threads handles.  VEC: eight consecutive rows
// (16-byte accesses).  Otherwise a warp covers 256 consecutive rows, its lanes side by side, so
// that accesses of any alignment coalesce.  `piece` counts the group's sweeps of 8 G rows.
template <bool VEC>
__device__ __forceinline__ long long first_row(long long piece, int G, int t) {
  if (VEC) return (piece * G + t) * kEl;
  return (piece * G + (t & ~31)) * kEl + (t & 31);
}
template <bool VEC>
__device__ __forceinline__ constexpr int row_step() { return VEC ? 1 : 32; }

// The thread's eight elements of one column, zero behind the last row.
template <bool VEC, typename T>
__device__ __forceinline__ void load_piece(const T* col, long long r0, long long rows, float (&x)[8]) {
  if (VEC) {
    if (r0 < rows) {
      load8(col + r0, x);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = 0.f;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const long long r = r0 + 32 * e;
      x[e] = r < rows ? to_f(col[r]) : 0.f;
    }
  }
}
template <bool VEC, typename T>
__device__ __forceinline__ void store_piece(T* col, long long r0, long long rows, const float (&x)[8]) {
  if (VEC) {
    if (r0 < rows) store8(col + r0, x);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const long long r = r0 + 32 * e;
      if (r < rows) col[r] = from_f<T>(x[e]);
    }
  }
}
// Dropout of those eight elements (the whole warp calls it).
template <bool VEC>
__device__ __forceinline__ void drop_piece(const Philox& gen, float factor, long long col, long long rows, long long r0,
                                           int lane, float (&x)[8]) {
  const unsigned long long e0 = static_cast<unsigned long long>(col) * rows;
  if (VEC) {  // rows % 8 == 0: r0 starts a block
    gen.drop8((e0 + r0) >> 3, factor, x);
    return;
  }
  const uint32_t keep = gen.keep_strided(e0 + (r0 - lane), lane);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = (keep >> e) & 1u ? x[e] * factor : 0.f;
}

// Eight elements as they lie in memory: what a prefetch keeps of a column.
template <typename T>
struct Raw8;
template <>
struct Raw8<__half> {
  uint4 w;
  __device__ __forceinline__ void load(const __half* p) { w = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void zero() { w = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
};
template <>
struct Raw8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = *reinterpret_cast<const float4*>(p);
    b = *reinterpret_cast<const float4*>(p + 4);
  }
  __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  }
};

// Sum over the G threads (a power of two, at least 32) that share a column; `slot` holds one value per warp
// of the CTA and alternates between two buffers, so one barrier per reduction is enough.
__device__ __forceinline__ float group_sum(float v, int G, int t, float* slot) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (G == 32) return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = G >> 5;
  if (lane == 0) slot[warp] = v;
  asm volatile("bar.sync %0, %1;" ::"r"(1 + static_cast<int>(threadIdx.x) / G), "r"(G) : "memory");
  v = lane < n ? slot[warp - (t >> 5) + lane] : 0.f;
  for (int o = n >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return __shfl_sync(0xffffffffu, v, 0);
}
// Two sums at once: half of a warp's lanes reduce the one, half the other, within the warp and, behind the
// barrier, over the warps' values (a float2 per warp in `slot`).  The kernels that need it for every column
// are bound by what they issue, so it is held to eleven shuffles; every thread adding up the sixteen
// values itself takes fewer steps one after the other, but a quarter more instructions in all.
__device__ __forceinline__ float2 group_sum2(float2 v, int G, int t, float2* slot) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool upper = lane >= 16;
  float a = (upper ? v.y : v.x) + __shfl_xor_sync(0xffffffffu, upper ? v.x : v.y, 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  if (G > 32) {
    float* s = reinterpret_cast<float*>(slot + (warp - (t >> 5))) + (upper ? 1 : 0);
    const int n = G >> 5, k = lane & 15;
    if (k == 0) s[2 * (t >> 5)] = a;
    asm volatile("bar.sync %0, %1;" ::"r"(1 + static_cast<int>(threadIdx.x) / G), "r"(G) : "memory");
    a = k < n ? s[2 * k] : 0.f;
    if (n > 8) a += __shfl_xor_sync(0xffffffffu, a, 8);
    if (n > 4) a += __shfl_xor_sync(0xffffffffu, a, 4);
    if (n > 2) a += __shfl_xor_sync(0xffffffffu, a, 2);
    a += __shfl_xor_sync(0xffffffffu, a, 1);
  }
  return make_float2(__shfl_sync(0xffffffffu, a, 0), __shfl_sync(0xffffffffu, a, 16));
}

template <typename T>
struct NormFwd {
  const T* x;
  const T* res;   // may be null
  const T* gain;  // may be null: 1
  const T* bias;  // may be null: 0
  T* h;           // null: plain normalisation of x
  T* y;
  float* mean;    // may be null
  float* rstd;    // may be null
  long long ldx, ldres, ldh, ldy, rows, cols;
  float eps;
  Dropout drop;
};

// h of the thread's eight elements: the residual sum as it is stored.
template <bool VEC, typename T>
__device__ __forceinline__ void form_h(const NormFwd<T>& p, const Philox& gen, long long col,
                                       long long r0, int lane, float (&v)[8]) {
  load_piece<VEC>(p.x + col * p.ldx, r0, p.rows, v);
  if (p.h == nullptr) return;
  if (p.drop.threshold != 0) drop_piece<VEC>(gen, p.drop.factor, col, p.rows, r0, lane, v);
  if (p.res != nullptr) {
    float q[8];
    load_piece<VEC>(p.res + col * p.ldres, r0, p.rows, q);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += q[e];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = to_f(from_f<T>(v[e]));
  store_piece<VEC>(p.h + col * p.ldh, r0, p.rows, v);
}

// y = ((h - mean) rstd) gain + bias, two values at a time.  The mean is subtracted first: a constant
// column gives exactly the bias.
template <bool VEC, typename T>
__device__ __forceinline__ void write_y(const NormFwd<T>& p, long long col, long long r0, float mean,
                                        float rstd, float (&v)[8]) {
  const F2 rs(rstd), shift(-mean);
  F2 x[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = mul2(add2(F2(v[2 * e], v[2 * e + 1]), shift), rs);
  float g[8];
  if (p.gain != nullptr) {
    load_piece<VEC>(p.gain, r0, p.rows, g);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = mul2(x[e], F2(g[2 * e], g[2 * e + 1]));
  }
  if (p.bias != nullptr) {
    load_piece<VEC>(p.bias, r0, p.rows, g);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = add2(x[e], F2(g[2 * e], g[2 * e + 1]));
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e].get(v[2 * e], v[2 * e + 1]);
  store_piece<VEC>(p.y + col * p.ldy, r0, p.rows, v);
}

// Eight elements on their way from memory, in either order of rows.
template <typename T, bool VEC>
struct Piece {
  Raw8<T> x;
  __device__ __forceinline__ void load(const T* col, long long r0, long long rows) {
    if (r0 < rows) x.load(col + r0);
    else x.zero();
  }
  __device__ __forceinline__ void get(float (&v)[8]) const { x.get(v); }
};
template <typename T>
struct Piece<T, false> {
  T x[8];
  __device__ __forceinline__ void load(const T* col, long long r0, long long rows) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = r0 + 32 * e < rows ? col[r0 + 32 * e] : from_f<T>(0.f);
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = to_f(x[e]);
  }
};

// One group of G threads per column, the column in registers (8 NV elements per thread): the
// variance is formed from the differences to the mean, not from a difference of squares.  RES: behind
// dropout and a residual connection.  The column's loads are all issued before its first store (which
// might overwrite what they read, as far as the compiler knows), and the random numbers, which need
// nothing, are formed while they are on their way.
template <typename T, bool VEC, int NV, bool RES>
__global__ void __launch_bounds__(512)
norm_forward_kernel(const NormFwd<T> p, int G) {
  __shared__ float slot[2][16];
  pdl_wait();
  pdl_launch_dependents();
  const int t = threadIdx.x % G, lane = threadIdx.x & 31;
  const long long col = static_cast<long long>(blockIdx.x) * (blockDim.x / G) + threadIdx.x / G;
  if (col >= p.cols) return;  // uniform over the group
  float v[NV][8];
  float s = 0.f;
  Piece<T, VEC> x[NV], q8[RES ? NV : 1];
#pragma unroll
  for (int i = 0; i < NV; ++i) x[i].load(p.x + col * p.ldx, first_row<VEC>(i, G, t), p.rows);
  if (RES && p.res != nullptr) {
#pragma unroll
    for (int i = 0; i < NV; ++i) q8[RES ? i : 0].load(p.res + col * p.ldres, first_row<VEC>(i, G, t), p.rows);
  }
  uint4 words[RES && VEC ? NV : 1];
  uint32_t keep[RES && !VEC ? NV : 1];
  const Philox gen(p.drop);
  if (RES && p.drop.threshold != 0) {
    const unsigned long long e0 = static_cast<unsigned long long>(col) * p.rows;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const long long r0 = first_row<VEC>(i, G, t);
      if (VEC) words[RES && VEC ? i : 0] = gen.words((e0 + r0) >> 3);
      else keep[RES && !VEC ? i : 0] = gen.keep_strided(e0 + (r0 - lane), lane);
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    x[i].get(v[i]);
    if (RES) {
      if (p.drop.threshold != 0) {
        if (VEC) {
          gen.apply(words[RES && VEC ? i : 0], p.drop.factor, v[i]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[i][e] = (keep[RES && !VEC ? i : 0] >> e) & 1u ? v[i][e] * p.drop.factor : 0.f;
        }
      }
      if (p.res != nullptr) {
        float q[8];
        q8[RES ? i : 0].get(q);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] += q[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = to_f(from_f<T>(v[i][e]));  // as it is stored
      store_piece<VEC>(p.h + col * p.ldh, first_row<VEC>(i, G, t), p.rows, v[i]);
    }
    s += ((v[i][0] + v[i][1]) + (v[i][2] + v[i][3])) + ((v[i][4] + v[i][5]) + (v[i][6] + v[i][7]));
  }
  const float mean = group_sum(s, G, t, slot[0]) / static_cast<float>(p.rows);
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const long long r0 = first_row<VEC>(i, G, t);
    if (VEC) {
      F2 a(0.f);
      const F2 m2(-mean);
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const F2 d = add2(F2(v[i][e], v[i][e + 1]), m2);
        a = fma2(d, d, a);
      }
      if (r0 < p.rows) q += a.sum();
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = v[i][e] - mean;
        if (r0 + 32 * e < p.rows) q += d * d;
      }
    }
  }
  const float rstd = 1.f / sqrtf(group_sum(q, G, t, slot[1]) / static_cast<float>(p.rows) + p.eps);
  if (t == 0) {
    if (p.mean != nullptr) p.mean[col] = mean;
    if (p.rstd != nullptr) p.rstd[col] = rstd;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) write_y<VEC>(p, col, first_row<VEC>(i, G, t), mean, rstd, v[i]);
}

// Columns too long for the registers of one CTA: three sweeps over the column, the later ones
// from cache.
template <typename T, bool VEC>
__global__ void __launch_bounds__(512)
norm_forward_long_kernel(const NormFwd<T> p) {
  __shared__ float slot[2][16];
  pdl_wait();
  pdl_launch_dependents();
  const int G = blockDim.x, t = threadIdx.x, lane = t & 31;
  const long long col = blockIdx.x, pieces = (p.rows + 8LL * G - 1) / (8LL * G);
  const Philox gen(p.drop);
  // the second and third sweep read what the first one wrote, each thread its own elements
  const T* src = p.h != nullptr ? p.h + col * p.ldh : p.x + col * p.ldx;
  float s = 0.f;
  for (long long i = 0; i < pieces; ++i) {
    float v[8];
    form_h<VEC>(p, gen, col, first_row<VEC>(i, G, t), lane, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) s += v[e];
  }
  const float mean = group_sum(s, G, t, slot[0]) / static_cast<float>(p.rows);
  float q = 0.f;
  for (long long i = 0; i < pieces; ++i) {
    const long long r0 = first_row<VEC>(i, G, t);
    float v[8];
    load_piece<VEC>(src, r0, p.rows, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = v[e] - mean;
      if (VEC ? r0 < p.rows : r0 + 32 * e < p.rows) q += d * d;
    }
  }
  const float rstd = 1.f / sqrtf(group_sum(q, G, t, slot[1]) / static_cast<float>(p.rows) + p.eps);
  if (t == 0) {
    if (p.mean != nullptr) p.mean[col] = mean;
    if (p.rstd != nullptr) p.rstd[col] = rstd;
  }
  for (long long i = 0; i < pieces; ++i) {
    const long long r0 = first_row<VEC>(i, G, t);
    float v[8];
    load_piece<VEC>(src, r0, p.rows, v);
    write_y<VEC>(p, col, r0, mean, rstd, v);
  }
}

template <typename T>
struct NormBwd {
  const T* h;
  const T* gain;  // may be null: 1
  const float* mean;
  const float* rstd;
  const T* dy;
  const T* dh;    // gradient that reaches h from elsewhere; may be null
  T* dres;        // may be null
  T* dx;          // may be null
  float* partial; // gridDim.x x 2 x rows sums (dgain, dbias); null when neither is wanted
  long long ldh, lddy, lddh, lddres, lddx, rows, cols;
  int accumulate;
  Dropout drop;
};

// The gradient of h to its two destinations.
template <bool VEC, typename T>
__device__ __forceinline__ void write_out(const NormBwd<T>& p, const Philox& gen, long long col, long long r0, int lane,
                                          float (&d)[8]) {
  float o[8];
  if (p.dres != nullptr) {
    T* c = p.dres + col * p.lddres;
    if (p.accumulate) {
      load_piece<VEC>(c, r0, p.rows, o);
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] += d[e];
      store_piece<VEC>(c, r0, p.rows, o);
    } else {
      store_piece<VEC>(c, r0, p.rows, d);
    }
  }
  if (p.dx != nullptr) {
    T* c = p.dx + col * p.lddx;
    if (p.drop.threshold != 0) drop_piece<VEC>(gen, p.drop.factor, col, p.rows, r0, lane, d);
    if (p.accumulate) {
      load_piece<VEC>(c, r0, p.rows, o);
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] += o[e];
    }
    store_piece<VEC>(c, r0, p.rows, d);
  }
}
// Gradient of the normalisation's input from the column sums, added to d.
__device__ __forceinline__ void add_input_grad(float rstd, float2 m, const float (&xh)[8], const float (&g)[8], float (&d)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) d[e] += rstd * (g[e] - m.x - xh[e] * m.y);
}

// A CTA's weight gradients: the groups add theirs through shared memory, in order, and the sums go to
// this CTA's partial vector.
template <bool VEC, int NV, typename T>
__device__ __forceinline__ void leave_partial(const NormBwd<T>& p, int G, int t, int group, int groups, float* sums,
                                              const float (&dg)[NV][8], const float (&db)[NV][8]) {
  if (p.partial == nullptr) return;
  for (int k = 0; k < groups; ++k) {
    __syncthreads();
    if (group != k) continue;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const long long r0 = first_row<VEC>(i, G, t);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const long long r = r0 + row_step<VEC>() * e;
        if (r < p.rows) {
          sums[r] = (k ? sums[r] : 0.f) + dg[i][e];
          sums[p.rows + r] = (k ? sums[p.rows + r] : 0.f) + db[i][e];
        }
      }
    }
  }
  __syncthreads();
  float* out = p.partial + static_cast<long long>(blockIdx.x) * 2 * p.rows;
  for (long long r = threadIdx.x; r < 2 * p.rows; r += blockDim.x) out[r] = sums[r];
}

// Groups of G threads walk the columns; a thread meets the same rows in every column, so the
// weight gradients stay in its registers until the end, where the groups of the CTA add theirs
// through shared memory (2 x rows floats).
// Columns off the 16-byte grid take it; they are loaded when their turn comes.
template <typename T, int NV>
__global__ void __launch_bounds__(512, 1)
norm_backward_kernel(const NormBwd<T> p, int G) {
  constexpr bool VEC = false;
  __shared__ __align__(16) float2 slot[2][16];
  extern __shared__ float sums[];
  pdl_wait();
  pdl_launch_dependents();
  const int groups = blockDim.x / G, group = threadIdx.x / G;
  const int t = threadIdx.x % G, lane = threadIdx.x & 31;
  const Philox gen(p.drop);
  float dg[NV][8], db[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) dg[i][e] = db[i][e] = 0.f;
  const float inv = 1.f / static_cast<float>(p.rows);
  int turn = 0;
  for (long long col = static_cast<long long>(blockIdx.x) * groups + group; col < p.cols;
       col += static_cast<long long>(gridDim.x) * groups, turn ^= 1) {
    float xh[NV][8], g[NV][8];
    const float mean = p.mean[col], rstd = p.rstd[col];
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const long long r0 = first_row<VEC>(i, G, t);
      load_piece<VEC>(p.h + col * p.ldh, r0, p.rows, xh[i]);
      load_piece<VEC>(p.dy + col * p.lddy, r0, p.rows, g[i]);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const long long r0 = first_row<VEC>(i, G, t);
      float w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = 1.f;
      if (p.gain != nullptr) load_piece<VEC>(p.gain, r0, p.rows, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        xh[i][e] = (xh[i][e] - mean) * rstd;
        dg[i][e] += g[i][e] * xh[i][e];  // dy is zero behind the last row
        db[i][e] += g[i][e];
        g[i][e] *= w[e];
        s.x += g[i][e];
        s.y += g[i][e] * xh[i][e];
      }
    }
    s = group_sum2(s, G, t, slot[turn]);
    s.x *= inv;
    s.y *= inv;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const long long r0 = first_row<VEC>(i, G, t);
      float d[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = 0.f;
      if (p.dh != nullptr) load_piece<VEC>(p.dh + col * p.lddh, r0, p.rows, d);
      add_input_grad(rstd, s, xh[i], g[i], d);
      write_out<VEC>(p, gen, col, r0, lane, d);
    }
  }
  leave_partial<VEC, NV>(p, G, t, group, groups, sums, dg, db);
}

// The same for columns on the 16-byte grid, through a ring in shared memory: a column's reduction (a barrier
// behind two shuffle trees) waits for all of its loads, so without the next columns on their way the memory
// idles between two.  Every group has a ring of its own, filled by its first thread with one bulk copy per
// operand; a stage is free once the group is through the barrier behind the reduction, since what it holds is
// in registers by then.  No registers are spent on what is still to come, and the bytes in flight are what
// shared memory holds (two to eight columns).
// Columns longer than 512 threads hold are shared by the CTAs of a cluster, each with a run of rows; they
// exchange their column sums through each other's shared memory.
// The gain lies in shared memory as fp32.  Places behind the last row are zeros that no copy overwrites, so
// that reading takes no bounds.  DH: there is a gradient from elsewhere.
// Shared memory serves a 16-byte access eight lanes at a time, and eight lanes 32 bytes apart meet in the same
// banks.  fp32 pieces are therefore read with the two halves exchanged in every second four lanes, and stay in
// that order in the registers; the gain lies as two arrays, the first and the second halves of the pieces.
template <typename T>
struct Order {  // Half: eight elements are one access
  __device__ __forceinline__ explicit Order(int) {}
  __device__ __forceinline__ int gain_part() const { return 0; }
  template <typename P>
  __device__ __forceinline__ void load(const P* p, float (&x)[8]) const { load8(p, x); }
  template <typename P>
  __device__ __forceinline__ void store(P* p, const float (&x)[8]) const { store8(p, x); }
  __device__ __forceinline__ void read(const T* p, Raw8<T>& x) const { x.load(p); }
  __device__ __forceinline__ uint4 words(const uint4 w) const { return w; }
};
template <>
struct Order<float> {
  int a;  // the half this lane holds first: offset 0 or 4
  __device__ __forceinline__ explicit Order(int lane) : a(lane & 4) {}
  __device__ __forceinline__ int gain_part() const { return a >> 2; }
  __device__ __forceinline__ void load(const float* p, float (&x)[8]) const {
    const float4 u = *reinterpret_cast<const float4*>(p + a), v = *reinterpret_cast<const float4*>(p + (a ^ 4));
    x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
    x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
  }
  __device__ __forceinline__ void store(float* p, const float (&x)[8]) const {
    *reinterpret_cast<float4*>(p + a) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(p + (a ^ 4)) = make_float4(x[4], x[5], x[6], x[7]);
  }
  __device__ __forceinline__ void read(const float* p, Raw8<float>& x) const {
    x.a = *reinterpret_cast<const float4*>(p + a);
    x.b = *reinterpret_cast<const float4*>(p + (a ^ 4));
  }
  __device__ __forceinline__ uint4 words(const uint4 w) const { return a ? make_uint4(w.z, w.w, w.x, w.y) : w; }
};
constexpr int kMaxBars = 64;
struct NormRing {
  int G, stages, cluster, run;  // run: rows per CTA of a cluster
};
template <typename T, int NV, bool DH>
__global__ void __launch_bounds__(512, 1)
norm_backward_ring_kernel(const NormBwd<T> p, const NormRing ring, int* __restrict__ status) {
  __shared__ __align__(16) float2 slot[2][16], peers[2][8];
  __shared__ __align__(8) uint64_t full[kMaxBars];
  extern __shared__ __align__(16) float gain[];  // then the groups' rings, in the end the weight sums of several groups
  constexpr int OPS = DH ? 3 : 2;
  const int G = ring.G, groups = blockDim.x / G, group = threadIdx.x / G;
  const int t = threadIdx.x % G, lane = threadIdx.x & 31;
  const int rank = ring.cluster > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int row0 = rank * ring.run, left = static_cast<int>(p.rows) - row0, rows = left < ring.run ? left : ring.run;
  const int places = NV * kEl * G;  // rows a group holds
  const uint32_t bytes = rows * static_cast<uint32_t>(sizeof(T)), pitch = places * static_cast<uint32_t>(sizeof(T));
  T* mine = reinterpret_cast<T*>(gain + places) + static_cast<size_t>(group) * ring.stages * OPS * places;
  uint64_t* bars = full + group * ring.stages;
  if (threadIdx.x == 0) {
    for (int i = 0; i < groups * ring.stages; ++i) mbar_init(smem_u32(&full[i]), 1);
    fence_mbar_init();
  }
  for (int k = 0; k < ring.stages * OPS; ++k)
    for (int r = rows + t; r < places; r += G) mine[static_cast<size_t>(k) * places + r] = from_f<T>(0.f);
  pdl_wait();
  pdl_launch_dependents();
  for (int r = threadIdx.x; r < places; r += blockDim.x)
    gain[(r >> 3) * 4 + (r & 3) + ((r >> 2) & 1) * (places / 2)] = r < rows ? (p.gain != nullptr ? to_f(p.gain[row0 + r]) : 1.f) : 0.f;
  __syncthreads();
  if (ring.cluster > 1) cluster_sync_all();  // every CTA of the cluster is there before one writes to it
  const Philox gen(p.drop);
  const Order<T> order(lane);
  const long long first = static_cast<long long>(blockIdx.x / ring.cluster) * groups + group;
  const long long step = static_cast<long long>(gridDim.x / ring.cluster) * groups;
  auto issue = [&](long long col, int s) {
    const uint32_t bar = smem_u32(&bars[s]), dst = smem_u32(mine + static_cast<size_t>(s) * OPS * places);
    mbar_arrive_expect_tx(bar, OPS * bytes);
    bulk_load(dst, p.h + col * p.ldh + row0, bytes, bar);
    bulk_load(dst + pitch, p.dy + col * p.lddy + row0, bytes, bar);
    if (DH) bulk_load(dst + 2 * pitch, p.dh + col * p.lddh + row0, bytes, bar);
  };
  if (t == 0)
    for (int s = 0; s < ring.stages; ++s)
      if (first + s * step < p.cols) issue(first + s * step, s);
  // this thread's places in the results, moving on with the columns
  T* dres = p.dres != nullptr ? p.dres + first * p.lddres + row0 + t * kEl : nullptr;
  T* dx = p.dx != nullptr ? p.dx + first * p.lddx + row0 + t * kEl : nullptr;
  const long long dres_step = p.dres != nullptr ? step * p.lddres : 0, dx_step = p.dx != nullptr ? step * p.lddx : 0;
  F2 dg[NV][4], db[NV][4];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) dg[i][e] = db[i][e] = F2(0.f);
  const float inv = 1.f / static_cast<float>(p.rows);
  float mean = 0.f, rstd = 0.f;
  if (first < p.cols) {
    mean = p.mean[first];
    rstd = p.rstd[first];
  }
  bool ok = true;
  int s = 0, phase = 0, turn = 0;
  for (long long col = first; col < p.cols; col += step, turn ^= 1) {
    const float mean1 = mean, rstd1 = rstd;
    if (col + step < p.cols) {
      mean = p.mean[col + step];
      rstd = p.rstd[col + step];
    }
    uint4 words[NV];
    if (p.dx != nullptr && p.drop.threshold != 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        words[i] = order.words(gen.words((static_cast<unsigned long long>(col) * p.rows + row0 + (i * G + t) * kEl) >> 3));
    }
    // the kernel's waits have an end: a group that gave up goes on without its data
    ok = ok && mbar_wait(smem_u32(&bars[s]), phase, status, DEV_TIMEOUT_FULL, 0x100);
    const T* stage = mine + static_cast<size_t>(s) * OPS * places;
    const F2 rs(rstd1), shift(-mean1);
    F2 xh[NV][4], g[NV][4], sx(0.f), sy(0.f);
    Raw8<T> z[DH ? NV : 1];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int r0 = (i * G + t) * kEl;
      Raw8<T> x, y;
      order.read(stage + r0, x);
      order.read(stage + places + r0, y);
      if (DH) order.read(stage + 2 * places + r0, z[i]);
      float a[8], b[8];
      x.get(a);
      y.get(b);
      const float4* w = reinterpret_cast<const float4*>(gain) + (i * G + t);
      const int half = places / 8, part = order.gain_part();
      const float4 k[2] = {w[part * half], w[(part ^ 1) * half]};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // the mean is subtracted first, as in the forward pass: the difference of close values is exact, where
        // x rstd - mean rstd is off by 2^-24 of |mean| rstd (a constant column would not give zero)
        xh[i][e] = mul2(add2(F2(a[2 * e], a[2 * e + 1]), shift), rs);
        const F2 d(b[2 * e], b[2 * e + 1]);  // zero behind the last row
        dg[i][e] = fma2(d, xh[i][e], dg[i][e]);
        db[i][e] = add2(db[i][e], d);
        g[i][e] = mul2(d, e & 1 ? F2(k[e >> 1].z, k[e >> 1].w) : F2(k[e >> 1].x, k[e >> 1].y));
        sx = add2(sx, g[i][e]);
        sy = fma2(g[i][e], xh[i][e], sy);
      }
    }
    float2 sum = group_sum2(make_float2(sx.sum(), sy.sum()), G, t, slot[turn]);
    __syncwarp();  // groups of one warp meet no barrier in the reduction: their reads of the stage end here
    if (t == 0 && ok && col + ring.stages * step < p.cols) issue(col + ring.stages * step, s);
    if (++s == ring.stages) {
      s = 0;
      phase ^= 1;
    }
    if (ring.cluster > 1) {
      if (threadIdx.x < ring.cluster) {
        const uint32_t to = mapa_shared(smem_u32(&peers[turn][rank]), threadIdx.x);
        st_shared_remote(to, __float_as_uint(sum.x));
        st_shared_remote(to + 4, __float_as_uint(sum.y));
      }
      __syncwarp();
      cluster_sync_all();
      sum = make_float2(0.f, 0.f);
      for (int k = 0; k < ring.cluster; ++k) {
        sum.x += peers[turn][k].x;
        sum.y += peers[turn][k].y;
      }
    }
    // rstd (g - sum.x / rows - xh sum.y / rows)
    const F2 c0(-rstd1 * sum.x * inv), c1(-rstd1 * sum.y * inv);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int r0 = (i * G + t) * kEl;
      float d[8], q[8];
      if (DH) z[i].get(q);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        F2 v = fma2(g[i][e], rs, fma2(xh[i][e], c1, c0));
        if (DH) v = add2(v, F2(q[2 * e], q[2 * e + 1]));
        v.get(d[2 * e], d[2 * e + 1]);
      }
      if (r0 >= rows) continue;
      if (dres != nullptr) {
        T* to = dres + i * G * kEl;
        if (p.accumulate) {
          order.load(to, q);
#pragma unroll
          for (int e = 0; e < 8; ++e) q[e] += d[e];
          order.store(to, q);
        } else {
          order.store(to, d);
        }
      }
      if (dx != nullptr) {
        T* to = dx + i * G * kEl;
        if (p.drop.threshold != 0) gen.apply(words[i], p.drop.factor, d);
        if (p.accumulate) {
          order.load(to, q);
#pragma unroll
          for (int e = 0; e < 8; ++e) d[e] += q[e];
        }
        order.store(to, d);
      }
    }
    dres += dres_step;
    dx += dx_step;
  }
  if (p.partial == nullptr) return;
  float* out = p.partial + static_cast<long long>(blockIdx.x / ring.cluster) * 2 * p.rows;
  float* sums = gain + places;
  // one group leaves its weight gradients directly, several add theirs in order first
  for (int k = 0; k < groups; ++k) {
    if (groups > 1) __syncthreads();  // the first time: the rings are done with
    if (group != k) continue;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int r0 = (i * G + t) * kEl;
      if (r0 >= rows) continue;
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        float v[8], q[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) (part ? db : dg)[i][e].get(v[2 * e], v[2 * e + 1]);
        if (k > 0) {
          order.load(sums + part * rows + r0, q);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] += q[e];
        }
        order.store(k + 1 == groups ? out + part * p.rows + row0 + r0 : sums + part * rows + r0, v);
      }
    }
  }
}

// Long columns: the column sums and the input's gradient in two sweeps, one CTA per column.
template <typename T>
__global__ void __launch_bounds__(512)
norm_backward_long_kernel(const NormBwd<T> p) {
  constexpr bool VEC = false;
  __shared__ __align__(16) float2 slot[16];
  pdl_wait();
  pdl_launch_dependents();
  const int G = blockDim.x, t = threadIdx.x, lane = t & 31;
  const long long col = blockIdx.x, pieces = (p.rows + 8LL * G - 1) / (8LL * G);
  const Philox gen(p.drop);
  const float mean = p.mean[col], rstd = p.rstd[col];
  float2 s = make_float2(0.f, 0.f);
  auto fetch = [&](long long r0, float (&xh)[8], float (&g)[8]) {
    load_piece<VEC>(p.h + col * p.ldh, r0, p.rows, xh);
    load_piece<VEC>(p.dy + col * p.lddy, r0, p.rows, g);
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = 1.f;
    if (p.gain != nullptr) load_piece<VEC>(p.gain, r0, p.rows, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      xh[e] = (xh[e] - mean) * rstd;
      g[e] *= w[e];
    }
  };
  for (long long i = 0; i < pieces; ++i) {
    float xh[8], g[8];
    fetch(first_row<VEC>(i, G, t), xh, g);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      s.x += g[e];
      s.y += g[e] * xh[e];
    }
  }
  s = group_sum2(s, G, t, slot);
  s.x /= static_cast<float>(p.rows);
  s.y /= static_cast<float>(p.rows);
  for (long long i = 0; i < pieces; ++i) {
    const long long r0 = first_row<VEC>(i, G, t);
    float xh[8], g[8], d[8];
    fetch(r0, xh, g);
#pragma unroll
    for (int e = 0; e < 8; ++e) d[e] = 0.f;
    if (p.dh != nullptr) load_piece<VEC>(p.dh + col * p.lddh, r0, p.rows, d);
    add_input_grad(rstd, s, xh, g, d);
    write_out<VEC>(p, gen, col, r0, lane, d);
  }
}

// Weight gradients of long columns: a thread owns a row, a CTA a range of columns.
template <typename T>
__global__ void __launch_bounds__(256)
norm_weight_grad_kernel(const NormBwd<T> p, long long cols_per_part) {
  pdl_wait();
  pdl_launch_dependents();
  const long long r = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (r >= p.rows) return;
  const long long c0 = blockIdx.y * cols_per_part;
  const long long c1 = c0 + cols_per_part < p.cols ? c0 + cols_per_part : p.cols;
  float dg = 0.f, db = 0.f;
  for (long long c = c0; c < c1; ++c) {
    const float d = to_f(p.dy[c * p.lddy + r]);
    dg += d * ((to_f(p.h[c * p.ldh + r]) - p.mean[c]) * p.rstd[c]);
    db += d;
  }
  float* out = p.partial + static_cast<long long>(blockIdx.y) * 2 * p.rows;
  out[r] = dg;
  out[p.rows + r] = db;
}

// dgain / dbias (+)= the sum over `parts` partial vectors, always in the same order.  A CTA serves
// 32 rows; its 32 warps take every 32nd vector.
template <typename T>
__global__ void __launch_bounds__(1024)
norm_weight_sum_kernel(const float* __restrict__ partial, int parts, long long rows,
                       T* __restrict__ dgain, T* __restrict__ dbias, int accumulate) {
  __shared__ float red[32][32];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long r = static_cast<long long>(blockIdx.x) * 32 + lane;
  T* out = blockIdx.y ? dbias : dgain;
  if (out == nullptr) return;
  float s = 0.f;
  if (r < rows)
    for (int k = warp; k < parts; k += 32) s += partial[(2LL * k + blockIdx.y) * rows + r];
  red[warp][lane] = s;
  __syncthreads();
  if (warp != 0 || r >= rows) return;
  float a = accumulate ? to_f(out[r]) : 0.f;
#pragma unroll
  for (int w = 0; w < 32; ++w) a += red[w][lane];
  out[r] = from_f<T>(a);
}

// y = (add) + drop(x) on runs of `len` elements, eight per thread and pass, the next eight on their way
// meanwhile.  `add` is the residual forward and the gradient itself when it accumulates.  COLS: one warp
// per column of a matrix with gaps between its columns (rows % 8 == 0); otherwise the whole matrix is
// one run.  Runs start on 16-byte boundaries.
template <typename T, bool COLS>
__global__ void __launch_bounds__(256)
dropout_kernel(const T* x, long long ldx, const T* add, long long lda, T* y, long long ldy, long long len,
               long long cols, Dropout drop) {
  pdl_wait();
  pdl_launch_dependents();
  const Philox gen(drop);
  const int lane = threadIdx.x & 31;
  long long col = COLS ? static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5) : 0;
  const long long col_step = COLS ? static_cast<long long>(gridDim.x) * 8 : 1;
  const long long first = COLS ? lane : static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  const long long step = COLS ? 32 : static_cast<long long>(gridDim.x) * 256;
  const long long blocks = len >> 3;  // whole ones
  for (; col < cols; col += col_step) {
    const T* xp = x + col * ldx + first * 8;
    const T* ap = add + col * lda + first * 8;
    T* yp = y + col * ldy + first * 8;
    const unsigned long long b0 = static_cast<unsigned long long>(col) * blocks;
    Raw8<T> xr, ar;
    ar.zero();
    if (first < blocks) {
      xr.load(xp);
      if (add != nullptr) ar.load(ap);
    }
    for (long long q = first; q < blocks; q += step) {
      float v[8], a[8];
      xr.get(v);
      ar.get(a);
      xp += step * 8;
      ap += step * 8;
      if (q + step < blocks) {
        xr.load(xp);
        if (add != nullptr) ar.load(ap);
      }
      if (drop.threshold != 0) gen.drop8(b0 + q, drop.factor, v);
      if (add != nullptr)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += a[e];
      store8(yp, v);
      yp += step * 8;
    }
    // the elements behind the last whole block of a flat matrix
    if (!COLS && first == 0 && (len & 7) != 0) {
      const uint32_t keep = drop.threshold != 0 ? gen.keep8(blocks) : 0xffu;
      for (int e = 0; e < (len & 7); ++e) {
        float v = (keep >> e) & 1u ? to_f(x[blocks * 8 + e]) * drop.factor : 0.f;
        if (add != nullptr) v += to_f(add[blocks * 8 + e]);
        y[blocks * 8 + e] = from_f<T>(v);
      }
    }
  }
}

// The same for any alignment, element by element.
template <typename T>
__global__ void __launch_bounds__(256)
dropout_any_kernel(const T* x, long long ldx, const T* add, long long lda, T* y, long long ldy, long long rows,
                   long long cols, Dropout drop) {
  pdl_wait();
  pdl_launch_dependents();
  const Philox gen(drop);
  for (long long q = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; q < rows * cols;
       q += static_cast<long long>(gridDim.x) * 256) {
    const long long col = q / rows, r = q - col * rows;
    float v = to_f(x[col * ldx + r]);
    if (drop.threshold != 0)
      v = (gen.keep8(static_cast<unsigned long long>(q) >> 3) >> (q & 7)) & 1u ? v * drop.factor : 0.f;
    if (add != nullptr) v += to_f(add[col * lda + r]);
    y[col * ldy + r] = from_f<T>(v);
  }
}

// Every column of a matrix starts on a 16-byte boundary.
bool cols16(const void* p, long long ld, int es, long long cols) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (cols <= 1 || (ld * es) % 16 == 0);
}

// Threads per column (32 at least) such that 8 * nv elements per thread cover it; 0 = too long.
int group_size(long long rows, int nv) {
  for (int g = 32; g <= 512; g *= 2)
    if (rows <= 8LL * nv * g) return g;
  return 0;
}

// How a backward pass is laid out.  Columns on the 16-byte grid go through the ring kernel, those longer
// than 512 threads hold (16 rows each) on clusters of two to eight CTAs; other columns are loaded when their
// turn comes, and longer ones take the kernels of two sweeps.
struct NormPlan {
  bool ring = false, two_sweeps = false;
  int nv = 1, G = 0, cluster = 1, run = 0, stages = 0, parts = 0, smem = 0;
};
constexpr int kNormSmem = 225 * 1024;
NormPlan plan_backward(const NormGradArgs& a, int es, int num_sms) {
  NormPlan w;
  if (a.cols == 0) return w;  // no columns, no parts: weight gradients are sums of nothing
  const bool vec = a.rows % 8 == 0 && cols16(a.h, a.ldh, es, a.cols) && cols16(a.dy, a.lddy, es, a.cols) &&
                   cols16(a.dh, a.lddh, es, a.cols) && cols16(a.dres, a.lddres, es, a.cols) &&
                   cols16(a.dx, a.lddx, es, a.cols);
  constexpr long long kHeld = 8192;  // rows that 512 threads hold, 16 each
  while (vec && w.cluster < 8 && a.rows > kHeld * w.cluster) w.cluster *= 2;
  if (a.rows > kHeld * w.cluster) {
    w.two_sweeps = true;
    // weight gradients: enough CTAs to fill the device with 256 rows each, at most 64 partial vectors
    const long long row_blocks = (a.rows + 255) / 256;
    long long parts = (4LL * num_sms + row_blocks - 1) / row_blocks;
    parts = parts > 64 ? 64 : parts;
    parts = parts > a.cols ? a.cols : parts;
    const long long per = (a.cols + parts - 1) / parts;
    w.parts = static_cast<int>((a.cols + per - 1) / per);
    return w;
  }
  w.ring = vec;
  w.run = static_cast<int>((a.rows / 8 + w.cluster - 1) / w.cluster * 8);
  w.nv = a.rows <= (es == 2 ? 256 : 512) ? 1 : 2;
  w.G = group_size(vec ? w.run : a.rows, w.nv);
  const int groups = 512 / w.G;
  const long long want = (a.cols + groups - 1) / groups, most = num_sms / w.cluster;
  w.parts = static_cast<int>(want < most ? want : most);
  if (!vec) {
    w.smem = a.dgain != nullptr || a.dbias != nullptr ? static_cast<int>(2 * a.rows * sizeof(float)) : 0;
    return w;
  }
  const int places = 8 * w.nv * w.G, stage = (a.dh != nullptr ? 3 : 2) * places * es * groups;
  const int fixed = places * static_cast<int>(sizeof(float));
  w.stages = (kNormSmem - fixed) / stage;
  w.stages = w.stages > 8 ? 8 : w.stages;
  w.stages = w.stages * groups > kMaxBars ? kMaxBars / groups : w.stages;
  w.smem = fixed + w.stages * stage;
  return w;
}

template <typename T, bool VEC>
cudaError_t forward_tv(const NormFwd<T>& p, int num_sms, cudaStream_t stream) {
  // Rows per thread: 32 as long as one CTA covers the column that way; 16 off the 16-byte grid (1001 x 5003
  // fp32: 28 us with 32) and for fp32 behind a residual connection (4096 x 8192: 95 us with 32, 86 with 16),
  // where 32 hold too many registers.  Fewer where the columns alone would leave SMs idle: then a column's
  // latency counts.
  const bool many = !VEC || (sizeof(T) == 4 && p.h != nullptr);
  int nv = p.rows <= 256 ? 1 : p.rows <= 512 || (many && p.rows <= 8192) ? 2 : 4;
  while (nv > 1 && p.rows <= 2048 * nv && p.cols * group_size(p.rows, nv) < 256LL * num_sms) nv /= 2;
  const int G = group_size(p.rows, nv);
  if (G == 0) {
    if (p.cols > 0x7fffffffLL) return cudaErrorInvalidValue;
    return launch_kernel(norm_forward_long_kernel<T, VEC>, dim3(static_cast<unsigned>(p.cols)), dim3(512), 0,
                         stream, pdl_enabled(), p);
  }
  const int threads = G > 256 ? G : 256;
  const long long per = threads / G, grid = (p.cols + per - 1) / per;
  if (grid > 0x7fffffffLL) return cudaErrorInvalidValue;
  auto kern = nv == 1 ? norm_forward_kernel<T, VEC, 1, false> : nv == 2 ? norm_forward_kernel<T, VEC, 2, false> : norm_forward_kernel<T, VEC, 4, false>;
  if (p.h != nullptr) kern = nv == 1 ? norm_forward_kernel<T, VEC, 1, true> : nv == 2 ? norm_forward_kernel<T, VEC, 2, true> : norm_forward_kernel<T, VEC, 4, true>;
  return launch_kernel(kern, dim3(static_cast<unsigned>(grid)), dim3(threads), 0, stream, pdl_enabled(), p, G);
}

template <typename T>
cudaError_t forward_t(const NormArgs& a, int num_sms, cudaStream_t stream) {
  NormFwd<T> p;
  p.x = static_cast<const T*>(a.x);
  p.res = static_cast<const T*>(a.res);
  p.gain = static_cast<const T*>(a.gain);
  p.bias = static_cast<const T*>(a.bias);
  p.h = static_cast<T*>(a.h);
  p.y = static_cast<T*>(a.y);
  p.mean = a.mean;
  p.rstd = a.rstd;
  p.ldx = a.ldx; p.ldres = a.ldres; p.ldh = a.ldh; p.ldy = a.ldy;
  p.rows = a.rows; p.cols = a.cols;
  p.eps = a.eps;
  p.drop = a.drop;
  const int es = sizeof(T);
  const bool vec = a.rows % 8 == 0 && cols16(a.x, a.ldx, es, a.cols) && cols16(a.y, a.ldy, es, a.cols) &&
                   cols16(a.res, a.ldres, es, a.cols) && cols16(a.h, a.ldh, es, a.cols) &&
                   cols16(a.gain, 0, es, 1) && cols16(a.bias, 0, es, 1);
  return vec ? forward_tv<T, true>(p, num_sms, stream) : forward_tv<T, false>(p, num_sms, stream);
}

template <typename T>
cudaError_t backward_t(const NormGradArgs& a, float* partial, int num_sms, cudaStream_t stream, int* status) {
  NormBwd<T> p;
  p.h = static_cast<const T*>(a.h);
  p.gain = static_cast<const T*>(a.gain);
  p.mean = a.mean;
  p.rstd = a.rstd;
  p.dy = static_cast<const T*>(a.dy);
  p.dh = static_cast<const T*>(a.dh);
  p.dres = static_cast<T*>(a.dres);
  p.dx = static_cast<T*>(a.dx);
  p.partial = partial;
  p.ldh = a.ldh; p.lddy = a.lddy; p.lddh = a.lddh; p.lddres = a.lddres; p.lddx = a.lddx;
  p.rows = a.rows; p.cols = a.cols;
  p.accumulate = a.accumulate;
  p.drop = a.drop;
  const NormPlan w = plan_backward(a, sizeof(T), num_sms);
  const bool weights = a.dgain != nullptr || a.dbias != nullptr;
  cudaError_t e = cudaSuccess;
  if (p.cols == 0) {
    // weight gradients that are sums of nothing
  } else if (w.two_sweeps) {
    if (p.cols > 0x7fffffffLL) return cudaErrorInvalidValue;
    if (weights)  // first: dx or dres may be written over dy
      e = launch_kernel(norm_weight_grad_kernel<T>, dim3(static_cast<unsigned>((p.rows + 255) / 256), static_cast<unsigned>(w.parts)),
                        dim3(256), 0, stream, pdl_enabled(), p, (p.cols + w.parts - 1) / w.parts);
    if (e == cudaSuccess && (p.dres != nullptr || p.dx != nullptr))
      e = launch_kernel(norm_backward_long_kernel<T>, dim3(static_cast<unsigned>(p.cols)), dim3(512), 0, stream, pdl_enabled(), p);
  } else if (w.ring) {
    const bool dh = p.dh != nullptr;
    auto kern = w.nv == 1 ? (dh ? norm_backward_ring_kernel<T, 1, true> : norm_backward_ring_kernel<T, 1, false>)
                          : (dh ? norm_backward_ring_kernel<T, 2, true> : norm_backward_ring_kernel<T, 2, false>);
    static unsigned long long smem_set[4] = {};  // one per kernel of this template instantiation
    e = set_smem_limit_once(reinterpret_cast<const void*>(kern), kNormSmem, &smem_set[(w.nv - 1) * 2 + dh]);
    if (e != cudaSuccess) return e;
    const NormRing ring = {w.G, w.stages, w.cluster, w.run};
    e = launch_cluster_kernel(kern, dim3(static_cast<unsigned>(w.parts * w.cluster)), dim3(512), static_cast<unsigned>(w.cluster), w.smem,
                              stream, pdl_enabled(), p, ring, status);
  } else {
    auto kern = w.nv == 1 ? norm_backward_kernel<T, 1> : norm_backward_kernel<T, 2>;
    static unsigned long long smem_set[2] = {};
    e = set_smem_limit_once(reinterpret_cast<const void*>(kern), 2 * 8192 * static_cast<int>(sizeof(float)), &smem_set[w.nv - 1]);
    if (e != cudaSuccess) return e;
    e = launch_kernel(kern, dim3(static_cast<unsigned>(w.parts)), dim3(512), w.smem, stream, pdl_enabled(), p, w.G);
  }
  if (e != cudaSuccess || !weights) return e;
  return launch_kernel(norm_weight_sum_kernel<T>, dim3(static_cast<unsigned>((a.rows + 31) / 32), 2), dim3(1024), 0, stream,
                       pdl_enabled(), static_cast<const float*>(partial), w.parts, a.rows, static_cast<T*>(a.dgain),
                       static_cast<T*>(a.dbias), a.accumulate);
}

template <typename T>
cudaError_t dropout_t(const void* x, long long ldx, const void* add, long long lda, void* y, long long ldy,
                      long long rows, long long cols, const Dropout& drop, int num_sms, cudaStream_t stream) {
  if (cols > 1 && ldx == rows && ldy == rows && (add == nullptr || lda == rows)) {
    rows *= cols;  // nothing between the columns: one run, whatever its length
    cols = 1;
  }
  const int es = sizeof(T);
  const bool vec = (cols == 1 || rows % 8 == 0) && cols16(x, ldx, es, cols) && cols16(y, ldy, es, cols) &&
                   cols16(add, lda, es, cols);
  const T* xp = static_cast<const T*>(x);
  const T* ap = static_cast<const T*>(add);
  T* yp = static_cast<T*>(y);
  const long long most = static_cast<long long>(num_sms) * 8;
  auto grid = [&](long long want) { return dim3(static_cast<unsigned>(want < 1 ? 1 : want < most ? want : most)); };
  if (!vec)
    return launch_kernel(dropout_any_kernel<T>, grid((rows * cols + 255) / 256), dim3(256), 0, stream, pdl_enabled(), xp, ldx, ap,
                         lda, yp, ldy, rows, cols, drop);
  if (cols > 1)
    return launch_kernel(dropout_kernel<T, true>, grid((cols + 7) / 8), dim3(256), 0, stream, pdl_enabled(), xp, ldx, ap, lda, yp,
                         ldy, rows, cols, drop);
  return launch_kernel(dropout_kernel<T, false>, grid((rows / 8 + 255) / 256), dim3(256), 0, stream, pdl_enabled(), xp, ldx, ap,
                       lda, yp, ldy, rows, cols, drop);
}

}  // namespace

int norm_backward_parts(int dtype, const NormGradArgs& a, int num_sms, int* launches) {
  const NormPlan w = plan_backward(a, dtype == 0 ? 4 : 2, num_sms);
  const bool weights = a.dgain != nullptr || a.dbias != nullptr;
  *launches = weights;
  if (a.cols > 0) *launches += w.two_sweeps ? weights + (a.dres != nullptr || a.dx != nullptr) : 1;
  return w.parts;
}

cudaError_t launch_norm_forward(int dtype, const NormArgs& a, int num_sms, cudaStream_t stream) {
  return dtype == 0 ? forward_t<float>(a, num_sms, stream) : forward_t<__half>(a, num_sms, stream);
}

cudaError_t launch_norm_backward(int dtype, const NormGradArgs& a, float* partial, int num_sms, cudaStream_t stream,
                                 int* status) {
  return dtype == 0 ? backward_t<float>(a, partial, num_sms, stream, status) : backward_t<__half>(a, partial, num_sms, stream, status);
}

cudaError_t launch_dropout(int dtype, const void* x, long long ldx, const void* add, long long lda, void* y,
                           long long ldy, long long rows, long long cols, const Dropout& drop, int num_sms,
                           cudaStream_t stream) {
  return dtype == 0 ? dropout_t<float>(x, ldx, add, lda, y, ldy, rows, cols, drop, num_sms, stream)
                    : dropout_t<__half>(x, ldx, add, lda, y, ldy, rows, cols, drop, num_sms, stream);
}

}  // namespace gb
