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

// Bias of every distance, head by head, in fp32: out[head][reach + d].  `clear`: words of the call's scratch that
// start as zero (a memset between two kernels would keep the second from being launched ahead).
template <typename T>
__global__ void __launch_bounds__(256)
rel_bias_expand_kernel(const T* __restrict__ table, long long ldt, const int* __restrict__ map, int buckets,
                       long long reach, int heads, float factor, float* __restrict__ out, float* __restrict__ clear,
                       long long nclear) {
  pdl_wait();
  pdl_launch_dependents();
  const long long n = 2 * reach + 1, at = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (at < nclear) clear[at] = 0.f;
  if (at >= n * heads) return;
  const long long head = at / n;
  const int b = map[at - head * n];
  out[at] = b >= 0 && b < buckets ? to_f(table[head * ldt + b]) * factor : 0.f;
}

// dst[b][head][t][hsp] (fp32, dense, rows hs..hsp zero) = src(h, t, head, b); queries behind the
// sequence's length and keys that no query sees become zero whatever they hold.
template <typename T>
__global__ void __launch_bounds__(256)
rel_pack_kernel(const T* __restrict__ src, long long ld, long long sh, long long sb, int hs, int hsp, int t_len,
                int heads, const RelExtent extent, bool query, long long total, float* __restrict__ dst) {
  pdl_wait();
  pdl_launch_dependents();
  for (long long at = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; at < total;
       at += static_cast<long long>(gridDim.x) * blockDim.x) {
    const int h = static_cast<int>(at % hsp);
    long long r = at / hsp;
    const int t = static_cast<int>(r % t_len);
    r /= t_len;
    const int head = static_cast<int>(r % heads), b = static_cast<int>(r / heads);
    const bool real = h < hs && t < rel_rows(extent, query, b);
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

__device__ __forceinline__ float exp_fast(float x) {  // relative error 2^-22 and 2^-24 |x|
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
  return y;
}

// Finished score of a query's key j from its raw product.
struct RelScore {
  const float* bias;  // of this head, at distance 0; may be null
  long long pos, reach;
  float scale, far;   // far: bias behind the reach
  __device__ __forceinline__ RelScore(const RelScores& s, const RelQuery& w, const float* b)
      : bias(b != nullptr ? b + w.head * (2 * s.reach + 1) + s.reach : nullptr), pos(w.pos), reach(s.reach), scale(s.scale),
        far(b != nullptr ? bias[-s.reach] : 0.f) {}
  __device__ __forceinline__ float operator()(float raw, int j) const {
    float b = far;
    const long long d = j - pos;
    if (bias != nullptr && d > -reach) b = bias[d > reach ? reach : d];
    return fmaf(raw, scale, b);
  }
};

// Column of a RelScores for this thread: a warp per query, or a CTA.
template <bool BLOCK>
__device__ __forceinline__ long long score_column() {
  return BLOCK ? blockIdx.x : static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
}

// Scores -> probabilities in place, statistics written: one warp per query up to 1024 keys and one CTA
// above, the query's scores in registers (NV per thread; NV = 0: read again for each of three sweeps).
// A query without visible keys gets zeros and lse = -inf.
template <int NV, bool BLOCK>
__global__ void __launch_bounds__(256)
rel_softmax_kernel(const RelScores s, const float* __restrict__ bias, float* __restrict__ lse) {
  __shared__ float red[8];
  pdl_wait();
  pdl_launch_dependents();
  const int G = BLOCK ? 256 : 32, g = BLOCK ? threadIdx.x : threadIdx.x & 31;
  const long long col = score_column<BLOCK>();
  if (col >= s.matrices * s.nq) return;
  const RelQuery w(s, col);
  float* sc = s.s + (w.matrix * s.nq + w.local) * s.ld;
  const RelScore score(s, w, bias);
  const int last = w.visible;  // keys 0 .. last - 1 take part
  float v[NV > 0 ? NV : 1];
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < NV; ++k) v[k] = g + G * k < last ? sc[g + G * k] : 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    v[k] = g + G * k < last ? score(v[k], g + G * k) : -INFINITY;
    m = fmaxf(m, v[k]);
  }
  if (NV == 0)
    for (int j = g; j < last; j += G) m = fmaxf(m, score(sc[j], j));
  m = column_reduce<BLOCK, true>(m, red);
  m = m == -INFINITY ? 0.f : m;
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    v[k] = exp_fast(v[k] - m);
    sum += v[k];
  }
  if (NV == 0)
    for (int j = g; j < last; j += G) sum += exp_fast(score(sc[j], j) - m);
  sum = column_reduce<BLOCK, false>(sum, red);
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
  if (g == 0) lse[(static_cast<long long>(w.batch) * s.heads + w.head) * s.tq + w.query] = logf(sum) + m;
#pragma unroll
  for (int k = 0; k < NV; ++k)
    if (g + G * k < s.ld) sc[g + G * k] = v[k] * inv;
  if (NV == 0)
    for (int j = g; j < s.ld; j += G) sc[j] = j < last ? exp_fast(score(sc[j], j) - m) * inv : 0.f;
}

// Backward: scores -> probabilities in place from the kept statistics, and over dp
// dS = factor * P (.) (dP - sum_j P dP).  One sweep with both in registers, NV = 0 two.  A query that sees
// one key gives it all its weight whatever the score: its dS is zero, not what is left of two roundings.
template <int NV, bool BLOCK>
__global__ void __launch_bounds__(256)
rel_softmax_grad_kernel(const RelScores s, const float* __restrict__ bias, const float* __restrict__ lse,
                        float* __restrict__ dp, float factor) {
  __shared__ float red[8];
  pdl_wait();
  pdl_launch_dependents();
  const int G = BLOCK ? 256 : 32, g = BLOCK ? threadIdx.x : threadIdx.x & 31;
  const long long col = score_column<BLOCK>();
  if (col >= s.matrices * s.nq) return;
  const RelQuery w(s, col);
  float* sc = s.s + (w.matrix * s.nq + w.local) * s.ld;
  float* dc = dp + (w.matrix * s.nq + w.local) * s.ld;
  const RelScore score(s, w, bias);
  const float m = lse[(static_cast<long long>(w.batch) * s.heads + w.head) * s.tq + w.query];
  const int last = m == -INFINITY ? 0 : w.visible;
  float v[NV > 0 ? NV : 1], d[NV > 0 ? NV : 1];
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int j = g + G * k;
    v[k] = j < last ? sc[j] : 0.f;
    d[k] = j < last ? dc[j] : 0.f;
  }
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int j = g + G * k;
    v[k] = j < last ? exp_fast(score(v[k], j) - m) : 0.f;
    sum += v[k] * d[k];
  }
  if (NV == 0)
    for (int j = g; j < last; j += G) {
      const float q = exp_fast(score(sc[j], j) - m);
      sc[j] = q;
      sum += q * dc[j];
    }
  sum = column_reduce<BLOCK, false>(sum, red);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int j = g + G * k;
    if (j < s.ld) {
      sc[j] = v[k];
      dc[j] = j < last && last > 1 ? factor * (v[k] * (d[k] - sum)) : 0.f;
    }
  }
  if (NV == 0)
    for (int j = g; j < s.ld; j += G) {
      dc[j] = j < last && last > 1 ? factor * (sc[j] * (dc[j] - sum)) : 0.f;
      if (j >= last) sc[j] = 0.f;
    }
}

// Sums of dS by distance for blocks of kRelDiagonal queries of one head: neighbouring threads take
// neighbouring distances, so the reads coalesce, and every element is met once; it is left behind
// times `factor`.  Distances at or behind the reach share an entry: those sums are collected per
// thread and joined at the end.  dist[head][block][width], layout as in rel_dist_sum_kernel.
__global__ void __launch_bounds__(256)
rel_diagonal_kernel(const RelScores s, float* __restrict__ ds, float factor, float* __restrict__ dist, int blocks, int width) {
  __shared__ float red[2][8];
  pdl_wait();
  pdl_launch_dependents();
  const int i0 = blockIdx.x * kRelDiagonal, n = min(kRelDiagonal, s.nq - i0);  // within this call's queries
  const long long matrix = blockIdx.y;
  const int batch = static_cast<int>((s.matrix0 + matrix) / s.heads);
  const long long first = s.q0 + i0 + rel_offset(s.q_offset, s.q_offsets, batch);  // position of the first query
  const long long low = rel_dist_low(s.reach, first + kRelDiagonal - 1);
  float* out = dist + ((s.matrix0 + matrix) * blocks + (s.q0 + i0) / kRelDiagonal) * width;
  for (int e = threadIdx.x; e < width; e += 256) out[e] = 0.f;
  __syncthreads();
  float* m = ds + (matrix * s.nq + i0) * s.ld;
  float lo = 0.f, hi = 0.f;
  for (int at = threadIdx.x; at < s.tk + n - 1; at += 256) {
    // keys at - (n - 1) + i of query i: one distance
    float sum = 0.f;
    for (int i0 = 0; i0 < n; i0 += 8) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {  // all loads before the first store
        const int j = at - (n - 1) + i0 + i;
        v[i] = i0 + i < n && j >= 0 && j < s.tk ? m[(i0 + i) * s.ld + j] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = at - (n - 1) + i0 + i;
        sum += v[i];
        if (i0 + i < n && j >= 0 && j < s.tk) m[(i0 + i) * s.ld + j] = v[i] * factor;
      }
    }
    const long long d = at - (n - 1) - first;
    if (d >= s.reach) hi += sum;
    else if (d <= -s.reach) lo += sum;
    else out[d - low] = sum;
  }
  lo = warp_sum(lo);
  hi = warp_sum(hi);
  if ((threadIdx.x & 31) == 0) {
    red[0][threadIdx.x >> 5] = lo;
    red[1][threadIdx.x >> 5] = hi;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  lo = hi = 0.f;
  for (int w = 0; w < 8; ++w) {
    lo += red[0][w];
    hi += red[1][w];
  }
  const long long elo = -s.reach - low, ehi = s.reach - low;
  if (elo >= 0 && elo < width) out[elo] += lo;
  if (ehi >= 0 && ehi < width) out[ehi] += hi;
}

// sums[head][reach + d] = the query tiles' sums of dS at distance d over all sequences, in order.
// dist[sequence][head][tile][slot][width]: entry e of a tile belongs to distance low + e, low the
// clamped smallest distance of its last query.  A CTA serves 32 distances, its 32 warps every
// 32nd (sequence, tile).
__global__ void __launch_bounds__(1024)
rel_dist_sum_kernel(const RelDist p, float* __restrict__ sums) {
  __shared__ float red[32][32];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, head = blockIdx.y;
  const long long at = static_cast<long long>(blockIdx.x) * 32 + lane, d = at - p.reach;
  float s = 0.f;
#pragma unroll 4
  for (int k = warp; k < p.batch * p.tiles; k += 32) {
    const int batch = k / p.tiles, tile = k - batch * p.tiles;
    const long long last = static_cast<long long>(tile + 1) * p.tile_rows - 1 + rel_offset(p.q_offset, p.q_offsets, batch);
    const long long e = d - rel_dist_low(p.reach, last);
    if (d > p.reach || e < 0 || e >= p.width) continue;
    const float* q = p.dist + ((static_cast<long long>(batch) * p.heads + head) * p.tiles + tile) * p.slots * p.width + e;
    s += p.slots == 2 ? q[0] + q[p.width] : q[0];
  }
  red[warp][lane] = s;
  __syncthreads();
  if (warp != 0 || d > p.reach) return;
  float a = 0.f;
#pragma unroll
  for (int w = 0; w < 32; ++w) a += red[w][lane];
  sums[head * (2 * p.reach + 1) + at] = a;
}

// dtable[bucket, head] (+)= the sums of the distances that map to it; one warp per (bucket, head).
// sums null: zeros.
template <typename T>
__global__ void __launch_bounds__(256)
rel_table_grad_kernel(const float* __restrict__ sums, const int* __restrict__ map, long long reach, int buckets, int heads,
                      int accumulate, T* __restrict__ dtable, long long lddt) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const long long at = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (at >= static_cast<long long>(buckets) * heads) return;
  const int head = static_cast<int>(at / buckets), bucket = static_cast<int>(at % buckets);
  float sum = 0.f;
  if (sums != nullptr)
    for (long long d = lane; d < 2 * reach + 1; d += 32)
      if (map[d] == bucket) sum += sums[head * (2 * reach + 1) + d];
  sum = warp_sum(sum);
  if (lane != 0) return;
  T* out = dtable + head * lddt + bucket;
  *out = from_f<T>(accumulate ? to_f(*out) + sum : sum);
}

// Kernel and grid for a sweep over the columns of `s`.
template <typename K>
K pick_columns(const RelScores& s, K w8, K w16, K w32, K b8, K b32, K any, dim3* grid) {
  const long long cols = s.matrices * s.nq;
  *grid = dim3(static_cast<unsigned>(s.tk > 1024 ? cols : (cols + 7) / 8));
  return s.tk <= 256 ? w8 : s.tk <= 512 ? w16 : s.tk <= 1024 ? w32 : s.tk <= 2048 ? b8 : s.tk <= 8192 ? b32 : any;
}

unsigned blocks_for(long long n) {
  const long long b = (n + 255) / 256;
  return static_cast<unsigned>(b < 16384 ? b : 16384);
}

}  // namespace

cudaError_t launch_rel_bias_expand(int dtype, const void* table, long long ldt, const int* map, int buckets,
                                   long long reach, int heads, float factor, float* out, float* clear, long long nclear,
                                   cudaStream_t stream) {
  const long long n = (2 * reach + 1) * heads, most = n > nclear ? n : nclear;
  const dim3 grid(static_cast<unsigned>((most + 255) / 256));
  if (dtype == 0)
    return launch_kernel(rel_bias_expand_kernel<float>, grid, dim3(256), 0, stream, pdl_enabled(),
                         static_cast<const float*>(table), ldt, map, buckets, reach, heads, factor, out, clear, nclear);
  return launch_kernel(rel_bias_expand_kernel<__half>, grid, dim3(256), 0, stream, pdl_enabled(),
                       static_cast<const __half*>(table), ldt, map, buckets, reach, heads, factor, out, clear, nclear);
}

cudaError_t launch_rel_pack(int dtype, const void* src, long long ld, long long sh, long long sb, int hs, int hsp,
                            int t_len, int heads, int batch, const RelExtent& extent, bool query, float* dst, cudaStream_t stream) {
  const long long total = static_cast<long long>(hsp) * t_len * heads * batch;
  if (dtype == 0)
    return launch_kernel(rel_pack_kernel<float>, dim3(blocks_for(total)), dim3(256), 0, stream, pdl_enabled(),
                         static_cast<const float*>(src), ld, sh, sb, hs, hsp, t_len, heads, extent, query, total, dst);
  return launch_kernel(rel_pack_kernel<__half>, dim3(blocks_for(total)), dim3(256), 0, stream, pdl_enabled(),
                       static_cast<const __half*>(src), ld, sh, sb, hs, hsp, t_len, heads, extent, query, total, dst);
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

cudaError_t launch_rel_softmax(const RelScores& s, const float* bias, float* lse, cudaStream_t stream) {
  dim3 grid;
  auto kern = pick_columns(s, rel_softmax_kernel<8, false>, rel_softmax_kernel<16, false>, rel_softmax_kernel<32, false>,
                           rel_softmax_kernel<8, true>, rel_softmax_kernel<32, true>, rel_softmax_kernel<0, true>, &grid);
  return launch_kernel(kern, grid, dim3(256), 0, stream, pdl_enabled(), s, bias, lse);
}

cudaError_t launch_rel_softmax_grad(const RelScores& s, const float* bias, const float* lse, float* dp, float factor,
                                    cudaStream_t stream) {
  dim3 grid;
  auto kern = pick_columns(s, rel_softmax_grad_kernel<8, false>, rel_softmax_grad_kernel<16, false>,
                           rel_softmax_grad_kernel<32, false>, rel_softmax_grad_kernel<8, true>,
                           rel_softmax_grad_kernel<32, true>, rel_softmax_grad_kernel<0, true>, &grid);
  return launch_kernel(kern, grid, dim3(256), 0, stream, pdl_enabled(), s, bias, lse, dp, factor);
}

cudaError_t launch_rel_diagonal(const RelScores& s, float* ds, float factor, float* dist, int blocks, int width,
                                cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>((s.nq + kRelDiagonal - 1) / kRelDiagonal), static_cast<unsigned>(s.matrices));
  return launch_kernel(rel_diagonal_kernel, grid, dim3(256), 0, stream, pdl_enabled(), s, ds, factor, dist, blocks, width);
}

cudaError_t launch_rel_table_grad(int dtype, const RelDist& d, float* sums, const int* map, int buckets, int accumulate,
                                  void* dtable, long long lddt, cudaStream_t stream) {
  if (d.dist != nullptr) {
    const long long n = 2 * d.reach + 1;
    const cudaError_t e = launch_kernel(rel_dist_sum_kernel,
                                        dim3(static_cast<unsigned>((n + 31) / 32), static_cast<unsigned>(d.heads)), dim3(1024), 0,
                                        stream, pdl_enabled(), d, sums);
    if (e != cudaSuccess) return e;
  }
  const dim3 grid(static_cast<unsigned>((static_cast<long long>(buckets) * d.heads + 7) / 8));
  const float* from = d.dist != nullptr ? sums : nullptr;
  if (dtype == 0)
    return launch_kernel(rel_table_grad_kernel<float>, grid, dim3(256), 0, stream, pdl_enabled(), from, map, d.reach, buckets,
                         d.heads, accumulate, static_cast<float*>(dtable), lddt);
  return launch_kernel(rel_table_grad_kernel<__half>, grid, dim3(256), 0, stream, pdl_enabled(), from, map, d.reach, buckets,
                       d.heads, accumulate, static_cast<__half*>(dtable), lddt);
}

}  // namespace gb
