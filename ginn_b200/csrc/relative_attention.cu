// Attention with a learned relative position bias: the passes around the fp32 products of the
// composed path (api.cu puts them together).
//
//   s[j, i] = scale * k_j . q_i + bias[map[clamp(d)]],   d = j - (i + offset)
//   p = column softmax of s over the visible keys,  o_i = sum_j p[j, i] v_j,  lse_i = log sum exp s
//   dp[j, i] = v_j . do_i,  ds = p (dp - sum_j p dp),  dtable[bucket] = sum of ds over its pairs
//
// Scores lie key index first (a query's scores are contiguous), one matrix per (sequence, head),
// for as many heads at a time as keep them in the L2 cache.
#include <cuda_fp16.h>
#include "math.cuh"
#include "ptx.cuh"
#include "launch.h"
#include "relative_attention.cuh"

namespace gb {

namespace {

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Bias of every distance, head by head, in fp32: out[head][reach + d].
template <typename T>
__global__ void __launch_bounds__(256)
rel_bias_expand_kernel(const T* __restrict__ table, long long ldt, const int* __restrict__ map, int buckets,
                       long long reach, int heads, float factor, float* __restrict__ out) {
  pdl_wait();
  pdl_launch_dependents();
  const long long n = 2 * reach + 1, at = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (at >= n * heads) return;
  const long long head = at / n;
  const int b = map[at - head * n];
  out[at] = b >= 0 && b < buckets ? to_f(table[head * ldt + b]) * factor : 0.f;
}

// dst[b][head][t][hsp] (fp32, dense, rows hs..hsp zero) = src(h, t, head, b); positions behind the
// sequence's length become zero whatever they hold.
template <typename T>
__global__ void __launch_bounds__(256)
rel_pack_kernel(const T* __restrict__ src, long long ld, long long sh, long long sb, int hs, int hsp, int t_len,
                int heads, const int* __restrict__ lengths, long long total, float* __restrict__ dst) {
  pdl_wait();
  pdl_launch_dependents();
  for (long long at = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; at < total;
       at += static_cast<long long>(gridDim.x) * blockDim.x) {
    const int h = static_cast<int>(at % hsp);
    long long r = at / hsp;
    const int t = static_cast<int>(r % t_len);
    r /= t_len;
    const int head = static_cast<int>(r % heads), b = static_cast<int>(r / heads);
    const bool real = h < hs && t < rel_length(lengths, b, t_len);
    dst[at] = real ? to_f(src[h + t * ld + head * sh + b * sb]) : 0.f;
  }
}

// dst(h, t, head, b) (+)= src[b][head][t][hsp]; src null: zeros.
template <typename T>
__global__ void __launch_bounds__(256)
rel_unpack_kernel(const float* __restrict__ src, int hs, int hsp, int t_len, int heads, long long total,
                  int accumulate, T* __restrict__ dst, long long ld, long long sh, long long sb) {
  pdl_wait();
  pdl_launch_dependents();
  for (long long at = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; at < total;
       at += static_cast<long long>(gridDim.x) * blockDim.x) {
    const int h = static_cast<int>(at % hs);
    long long r = at / hs;
    const long long row = r;
    const int t = static_cast<int>(r % t_len);
    r /= t_len;
    const int head = static_cast<int>(r % heads), b = static_cast<int>(r / heads);
    T* d = dst + h + t * ld + head * sh + b * sb;
    const float v = src != nullptr ? src[row * hsp + h] : 0.f;
    *d = from_f<T>(accumulate ? to_f(*d) + v : v);
  }
}

// Sum or maximum over the G threads of a column: a warp, or the whole CTA.
template <bool BLOCK, bool MAX>
__device__ __forceinline__ float column_reduce(float v, float* red) {
  v = MAX ? warp_max(v) : warp_sum(v);
  if (!BLOCK) return v;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float r = red[0];
  for (int w = 1; w < static_cast<int>(blockDim.x >> 5); ++w) r = MAX ? fmaxf(r, red[w]) : r + red[w];
  return r;
}

// Scores -> probabilities in place, one warp per query up to 1024 keys and one CTA above.  With
// `lse_in` the row statistics are given (backward pass); otherwise they are formed and written.
// A query without visible keys gets zeros and lse = -inf.
template <bool BLOCK>
__global__ void __launch_bounds__(256)
rel_softmax_kernel(const RelScores s, const float* __restrict__ bias, const float* __restrict__ lse_in,
                   float* __restrict__ lse_out) {
  __shared__ float red[8];
  pdl_wait();
  pdl_launch_dependents();
  const int G = BLOCK ? blockDim.x : 32, g = BLOCK ? threadIdx.x : threadIdx.x & 31;
  const long long col = BLOCK ? blockIdx.x : static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (col >= s.matrices * s.nq) return;
  const RelQuery w(s, col);
  float* sc = s.s + (w.matrix * s.nq + w.local) * s.ld;
  const float* bh = bias != nullptr ? bias + w.head * (2 * s.reach + 1) + s.reach : nullptr;
  auto score = [&](int j) -> float {
    float b = 0.f;
    if (bh != nullptr) {
      long long d = j - w.pos;
      d = d > s.reach ? s.reach : d < -s.reach ? -s.reach : d;
      b = bh[d];
    }
    return fmaf(sc[j], s.scale, b);
  };
  const int last = w.visible;  // keys 0 .. last - 1 take part
  const long long stat = (static_cast<long long>(w.batch) * s.heads + w.head) * s.tq + w.query;
  float m = -INFINITY, inv = 0.f;
  if (lse_in != nullptr) {
    m = lse_in[stat];
    inv = 1.f;
  } else {
    for (int j = g; j < last; j += G) m = fmaxf(m, score(j));
    m = column_reduce<BLOCK, true>(m, red);
    const float base = m == -INFINITY ? 0.f : m;
    float sum = 0.f;
    for (int j = g; j < last; j += G) sum += expf(score(j) - base);
    sum = column_reduce<BLOCK, false>(sum, red);
    inv = sum > 0.f ? 1.f / sum : 0.f;
    if (g == 0) lse_out[stat] = logf(sum) + base;
    m = base;
  }
  const bool none = m == -INFINITY;
  for (int j = g; j < s.ld; j += G) sc[j] = j < last && !none ? expf(score(j) - m) * inv : 0.f;
}

// dS = factor * P (.) (dP - sum_j P dP), written over dP.
template <bool BLOCK>
__global__ void __launch_bounds__(256)
rel_softmax_grad_kernel(const RelScores s, const float* __restrict__ p, float* __restrict__ dp, float factor) {
  __shared__ float red[8];
  pdl_wait();
  pdl_launch_dependents();
  const int G = BLOCK ? blockDim.x : 32, g = BLOCK ? threadIdx.x : threadIdx.x & 31;
  const long long col = BLOCK ? blockIdx.x : static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (col >= s.matrices * s.nq) return;
  const RelQuery w(s, col);
  const float* pc = p + (w.matrix * s.nq + w.local) * s.ld;
  float* dc = dp + (w.matrix * s.nq + w.local) * s.ld;
  float sum = 0.f;
  for (int j = g; j < w.visible; j += G) sum += pc[j] * dc[j];
  sum = column_reduce<BLOCK, false>(sum, red);
  for (int j = g; j < s.ld; j += G) dc[j] = j < w.visible ? factor * (pc[j] * (dc[j] - sum)) : 0.f;
}

// Sums of dS along its diagonals (one distance each), for blocks of kRelDiagonal queries: thread by
// thread neighbouring distances, so the reads coalesce.  out[matrix][block][tq + tk - 1], distance
// j - i = index - (tq - 1).  Every element is met once, and left behind times `factor`.
__global__ void __launch_bounds__(256)
rel_diagonal_kernel(const RelScores s, float* __restrict__ ds, float factor, float* __restrict__ out, int blocks) {
  pdl_wait();
  pdl_launch_dependents();
  const long long width = static_cast<long long>(s.tq) + s.tk - 1;
  const long long at = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (at >= width) return;
  const long long d = at - (s.tq - 1);  // j - i
  const int block = blockIdx.y;         // within this call's queries
  const int i0 = block * kRelDiagonal, i1 = min(i0 + kRelDiagonal, s.nq);
  const long long matrix = blockIdx.z;
  float* m = ds + matrix * s.nq * s.ld;
  float sum = 0.f;
  for (int i = i0; i < i1; ++i) {
    const long long j = d + s.q0 + i;
    if (j >= 0 && j < s.tk) {
      const float v = m[i * s.ld + j];
      sum += v;
      m[i * s.ld + j] = v * factor;
    }
  }
  out[((s.matrix0 + matrix) * blocks + s.q0 / kRelDiagonal + block) * width + at] = sum;
}

// dtable[bucket, head] (+)= the diagonal sums of its distances over all sequences and query
// blocks, in a fixed order.  One CTA per (bucket, head).
template <typename T>
__global__ void __launch_bounds__(256)
rel_table_grad_kernel(const RelScores s, const float* __restrict__ diagonal, int blocks, long long matrices,
                      const int* __restrict__ map, int accumulate, T* __restrict__ dtable, long long lddt) {
  __shared__ float red[8];
  pdl_wait();
  pdl_launch_dependents();
  const int bucket = blockIdx.x, head = blockIdx.y;
  const long long width = static_cast<long long>(s.tq) + s.tk - 1;
  float sum = 0.f;
  for (long long m = head; m < matrices; m += s.heads) {
    const long long off = rel_offset(s.q_offset, s.q_offsets, static_cast<int>(m / s.heads));
    for (long long at = threadIdx.x; at < width; at += blockDim.x) {
      long long d = at - (s.tq - 1) - off;
      d = d > s.reach ? s.reach : d < -s.reach ? -s.reach : d;
      if (map[d + s.reach] != bucket) continue;
      for (int b = 0; b < blocks; ++b) sum += diagonal[(m * blocks + b) * width + at];
    }
  }
  sum = column_reduce<true, false>(sum, red);
  if (threadIdx.x != 0) return;
  T* d = dtable + head * lddt + bucket;
  *d = from_f<T>(accumulate ? to_f(*d) + sum : sum);
}

unsigned blocks_for(long long n) {
  const long long b = (n + 255) / 256;
  return static_cast<unsigned>(b < 16384 ? b : 16384);
}

}  // namespace

cudaError_t launch_rel_bias_expand(int dtype, const void* table, long long ldt, const int* map, int buckets,
                                   long long reach, int heads, float factor, float* out, cudaStream_t stream) {
  const long long n = (2 * reach + 1) * heads;
  const dim3 grid(static_cast<unsigned>((n + 255) / 256));
  if (dtype == 0)
    return launch_kernel(rel_bias_expand_kernel<float>, grid, dim3(256), 0, stream, pdl_enabled(),
                         static_cast<const float*>(table), ldt, map, buckets, reach, heads, factor, out);
  return launch_kernel(rel_bias_expand_kernel<__half>, grid, dim3(256), 0, stream, pdl_enabled(),
                       static_cast<const __half*>(table), ldt, map, buckets, reach, heads, factor, out);
}

cudaError_t launch_rel_pack(int dtype, const void* src, long long ld, long long sh, long long sb, int hs, int hsp,
                            int t_len, int heads, int batch, const int* lengths, float* dst, cudaStream_t stream) {
  const long long total = static_cast<long long>(hsp) * t_len * heads * batch;
  if (dtype == 0)
    return launch_kernel(rel_pack_kernel<float>, dim3(blocks_for(total)), dim3(256), 0, stream, pdl_enabled(),
                         static_cast<const float*>(src), ld, sh, sb, hs, hsp, t_len, heads, lengths, total, dst);
  return launch_kernel(rel_pack_kernel<__half>, dim3(blocks_for(total)), dim3(256), 0, stream, pdl_enabled(),
                       static_cast<const __half*>(src), ld, sh, sb, hs, hsp, t_len, heads, lengths, total, dst);
}

cudaError_t launch_rel_unpack(int dtype, const float* src, int hs, int hsp, int t_len, int heads, int batch,
                              int accumulate, void* dst, long long ld, long long sh, long long sb, cudaStream_t stream) {
  const long long total = static_cast<long long>(hs) * t_len * heads * batch;
  if (dtype == 0)
    return launch_kernel(rel_unpack_kernel<float>, dim3(blocks_for(total)), dim3(256), 0, stream, pdl_enabled(), src,
                         hs, hsp, t_len, heads, total, accumulate, static_cast<float*>(dst), ld, sh, sb);
  return launch_kernel(rel_unpack_kernel<__half>, dim3(blocks_for(total)), dim3(256), 0, stream, pdl_enabled(), src,
                       hs, hsp, t_len, heads, total, accumulate, static_cast<__half*>(dst), ld, sh, sb);
}

cudaError_t launch_rel_softmax(const RelScores& s, const float* bias, const float* lse_in, float* lse_out,
                               cudaStream_t stream) {
  const long long cols = s.matrices * s.nq;
  if (s.tk > 1024)
    return launch_kernel(rel_softmax_kernel<true>, dim3(static_cast<unsigned>(cols)), dim3(256), 0, stream,
                         pdl_enabled(), s, bias, lse_in, lse_out);
  return launch_kernel(rel_softmax_kernel<false>, dim3(static_cast<unsigned>((cols + 7) / 8)), dim3(256), 0, stream,
                       pdl_enabled(), s, bias, lse_in, lse_out);
}

cudaError_t launch_rel_softmax_grad(const RelScores& s, const float* p, float* dp, float factor, cudaStream_t stream) {
  const long long cols = s.matrices * s.nq;
  if (s.tk > 1024)
    return launch_kernel(rel_softmax_grad_kernel<true>, dim3(static_cast<unsigned>(cols)), dim3(256), 0, stream,
                         pdl_enabled(), s, p, dp, factor);
  return launch_kernel(rel_softmax_grad_kernel<false>, dim3(static_cast<unsigned>((cols + 7) / 8)), dim3(256), 0,
                       stream, pdl_enabled(), s, p, dp, factor);
}

cudaError_t launch_rel_diagonal(const RelScores& s, float* ds, float factor, float* out, int blocks,
                                cudaStream_t stream) {
  const long long width = static_cast<long long>(s.tq) + s.tk - 1;
  const dim3 grid(static_cast<unsigned>((width + 255) / 256), (s.nq + kRelDiagonal - 1) / kRelDiagonal,
                  static_cast<unsigned>(s.matrices));
  return launch_kernel(rel_diagonal_kernel, grid, dim3(256), 0, stream, pdl_enabled(), s, ds, factor, out,
                       blocks);
}

cudaError_t launch_rel_table_grad(int dtype, const RelScores& s, const float* diagonal, int blocks,
                                  long long matrices, const int* map, int buckets, int heads, int accumulate,
                                  void* dtable, long long lddt, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>(buckets), static_cast<unsigned>(heads));
  if (dtype == 0)
    return launch_kernel(rel_table_grad_kernel<float>, grid, dim3(256), 0, stream, pdl_enabled(), s, diagonal, blocks,
                         matrices, map, accumulate, static_cast<float*>(dtable), lddt);
  return launch_kernel(rel_table_grad_kernel<__half>, grid, dim3(256), 0, stream, pdl_enabled(), s, diagonal, blocks,
                       matrices, map, accumulate, static_cast<__half*>(dtable), lddt);
}

}  // namespace gb
