// Half attention with a relative position bias whose scores never leave the SM.
//
// Forward: one CTA serves two tiles of 128 queries of one head and walks that head's keys in tiles
// of 128, once.  Query tile t has its scores S_t and its result O_t in tensor memory (128 lanes =
// queries; 4 x 128 columns of fp32 in all); a group of 128 threads, one per query, turns S_t into
// probabilities -- a row belongs to one thread, so the running maximum and sum need no exchange --
// and writes them over S_t as the fp16 left operand of O_t += P_t V.  While one tile's threads
// work, the tensor cores work on the other's products.
//   warp 0        TMA: Q once, K and V tiles through rings of NST stages
//   warp 1        tcgen05.mma: S_t = Q_t K^T (operands in shared memory), O_t += P_t V (P in tensor memory)
//   warps 4-7     softmax of query tile 0,  warps 8-11  of query tile 1
// Products issued by one thread run in order, so S_t of the next key tile may be issued right
// behind O_t += P_t V although it overwrites P_t.
//
// The running maximum lags: O_t is rescaled only when a row's maximum grew by more than 2^8
// (probabilities up to 256 lose nothing in fp16, and the sum is fp32), which after the first tiles
// is rare; a rescale costs a pass over O_t in tensor memory.
//
// Bias: within a tile of 128 x 128 pairs the distances fall in a window of 255; when the whole
// window lies beyond the reach (most tiles of a long sequence) its bias is one number, otherwise
// the threads lay the window out in shared memory, where neighbouring rows read neighbouring words.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cstring>
#include "ptx.cuh"
#include "math.cuh"
#include "launch.h"
#include "relative_attention.cuh"

namespace gb {

namespace {

constexpr int FT = 128;               // queries or keys per tile
constexpr int FCHUNK = FT * 128;      // bytes of 128 rows x 64 halves
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// A whole warp waits; its lanes agree on the outcome, so that none is left alone at a later barrier.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* status, int code, int detail) {
  return __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity, status, code, detail));
}
__device__ __forceinline__ void group_barrier(int id) { asm volatile("bar.sync %0, 128;" ::"r"(id) : "memory"); }

struct FlashParams {
  CUtensorMap tmQ, tmK, tmV;
  __half* O;
  long long ldo, sho, sbo;
  float* lse;
  const float* bias;
  int tq, tk, hs, heads, group, batch, qblocks;
  long long reach, q_offset;
  const int* q_offsets;
  const int* q_lengths;
  const int* k_lengths;
  float c1;  // scale * log2(e)
  int causal;
};

// What one (sequence, head) looks like to every role of a CTA.
struct FlashHead {
  int batch, head, kv, qlen, klen;
  long long off;
  __device__ __forceinline__ FlashHead(const FlashParams& p, int hb) {
    batch = hb / p.heads;
    head = hb - batch * p.heads;
    kv = head / p.group;
    qlen = rel_length(p.q_lengths, batch, p.tq);
    klen = rel_length(p.k_lengths, batch, p.tk);
    off = rel_offset(p.q_offset, p.q_offsets, batch);
  }
  __device__ __forceinline__ int visible(const FlashParams& p, int i) const {
    return i < qlen ? rel_visible(p.causal, i + off, klen) : 0;
  }
  // key tiles that the queries i0 .. i0 + 127 see
  __device__ __forceinline__ int tiles(const FlashParams& p, int i0) const {
    const int last = i0 + FT - 1 < qlen - 1 ? i0 + FT - 1 : qlen - 1;
    return i0 < qlen ? (visible(p, last) + FT - 1) / FT : 0;
  }
};

// Bias of a tile whose smallest distance is `dlo` (window dlo .. dlo + 254): one value for all of
// it, or window[c - r + 127] for column c of row r.  All 128 threads of a group call it.
struct TileBias {
  float value;         // when !near
  const float* row;    // when near: row[c] for this thread's row
  bool near;
  __device__ __forceinline__ TileBias(const float* bias, long long reach, long long dlo, int r, int slope,
                                      float* window, bool flat_ok) {
    value = 0.f;
    near = false;
    if (bias == nullptr) {
      near = !flat_ok;
      if (near) {
        window[r] = window[r + 128] = 0.f;
      }
    } else if (flat_ok && (dlo >= reach || dlo + 254 <= -reach)) {
      value = __ldg(bias + (dlo >= reach ? 2 * reach : 0));
    } else {
      near = true;
#pragma unroll
      for (int w = r; w < 256; w += 128) {
        long long d = dlo + w;
        d = d > reach ? reach : d < -reach ? -reach : d;
        window[w] = __ldg(bias + d + reach);
      }
    }
    row = window + 127 + slope * r;
  }
};

template <int HS, int NST>
__global__ void __launch_bounds__(384, 1)
flash_forward_kernel(const __grid_constant__ FlashParams p, int* __restrict__ status) {
  constexpr int TILE = FCHUNK * (HS / 64);  // bytes of one operand tile
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t q_full[2], k_full[NST], k_empty[NST], v_full[NST], v_empty[NST];
  __shared__ __align__(8) uint64_t s_full[2], p_full[2], o_full[2];
  __shared__ uint32_t tmem_slot;
  __shared__ float window[2][2][256];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* base_ptr = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t q_s = base, k_s = base + 2 * TILE, v_s = k_s + NST * TILE;

  if (warp == 0 && lane == 0) {
    prefetch_tmap(&p.tmQ);
    prefetch_tmap(&p.tmK);
    prefetch_tmap(&p.tmV);
  }
  if (warp == 1) {
    if (lane == 0) {
      for (int t = 0; t < 2; ++t) {
        mbar_init(smem_u32(&q_full[t]), 1);
        mbar_init(smem_u32(&s_full[t]), 1);
        mbar_init(smem_u32(&p_full[t]), 128);
        mbar_init(smem_u32(&o_full[t]), 1);
      }
      for (int s = 0; s < NST; ++s) {
        mbar_init(smem_u32(&k_full[s]), 1);
        mbar_init(smem_u32(&k_empty[s]), 1);
        mbar_init(smem_u32(&v_full[s]), 1);
        mbar_init(smem_u32(&v_empty[s]), 1);
      }
      fence_mbar_init();
    }
    __syncwarp();
    tmem_alloc(smem_u32(&tmem_slot), 512);
    tmem_relinquish();
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  pdl_wait();
  pdl_launch_dependents();

  // the last query blocks first: under a causal mask they have the most keys
  const int hbs = p.heads * p.batch;
  const int qb = p.qblocks - 1 - static_cast<int>(blockIdx.x) / hbs;
  const FlashHead hd(p, static_cast<int>(blockIdx.x) % hbs);
  const int i0 = qb * 2 * FT;
  const int n0 = hd.tiles(p, i0), n1 = hd.tiles(p, i0 + FT);
  const int n = n0 > n1 ? n0 : n1;

  if (warp == 0) {
    // ===================== TMA producer =====================
    if (elect_one()) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if ((t ? n1 : n0) == 0) continue;
        mbar_arrive_expect_tx(smem_u32(&q_full[t]), TILE);
        for (int c = 0; c < HS / 64; ++c)
          tma_load_4d(q_s + t * TILE + c * FCHUNK, &p.tmQ, smem_u32(&q_full[t]), 64 * c, i0 + t * FT, hd.head, hd.batch);
      }
      for (int j = 0; j < n; ++j) {
        const int s = j % NST;
        const uint32_t ph = (j / NST) & 1;
        if (!mbar_wait(smem_u32(&k_empty[s]), ph ^ 1u, status, DEV_TIMEOUT_EMPTY, 0xa00)) break;
        mbar_arrive_expect_tx(smem_u32(&k_full[s]), TILE);
        for (int c = 0; c < HS / 64; ++c)
          tma_load_4d(k_s + s * TILE + c * FCHUNK, &p.tmK, smem_u32(&k_full[s]), 64 * c, j * FT, hd.kv, hd.batch);
        if (!mbar_wait(smem_u32(&v_empty[s]), ph ^ 1u, status, DEV_TIMEOUT_EMPTY, 0xa01)) break;
        mbar_arrive_expect_tx(smem_u32(&v_full[s]), TILE);
        for (int c = 0; c < HS / 64; ++c)
          tma_load_4d(v_s + s * TILE + c * FCHUNK, &p.tmV, smem_u32(&v_full[s]), 64 * c, j * FT, hd.kv, hd.batch);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ===================== MMA issuer =====================
    constexpr uint32_t IDESC_S = make_idesc(0, 0, 0, FT, FT);
    constexpr uint32_t IDESC_O = make_idesc(0, 0, 1, FT, HS);
    const bool leader = elect_one();
    auto scores = [&](int t, int j) {
      if (leader) {
        const uint32_t a = q_s + t * TILE, b = k_s + (j % NST) * TILE;
#pragma unroll
        for (int ks = 0; ks < HS / 16; ++ks) {
          const uint32_t at = (ks / 4) * FCHUNK + (ks % 4) * 32;
          mma_f16(tmem + t * FT, make_smem_desc(a + at, 16, 1024), make_smem_desc(b + at, 16, 1024), IDESC_S, ks > 0);
        }
        tc_commit(smem_u32(&s_full[t]));
      }
    };
    bool ok = true;
    if (n > 0) ok = warp_wait(&k_full[0], 0, status, DEV_TIMEOUT_FULL, 0xb00);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if ((t ? n1 : n0) == 0 || !ok) continue;
      ok = warp_wait(&q_full[t], 0, status, DEV_TIMEOUT_FULL, 0xb01);
      tc_fence_after();
      if (ok) scores(t, 0);
    }
    if (leader && n > 0) tc_commit(smem_u32(&k_empty[0]));
    for (int j = 0; j < n && ok; ++j) {
      const int s = j % NST, s2 = (j + 1) % NST;
      ok = warp_wait(&v_full[s], (j / NST) & 1, status, DEV_TIMEOUT_FULL, 0xb02);
      if (ok && hd.klen < p.tk && (j + 1) * FT > hd.klen) {
        // rows behind the sequence's end may hold anything: their probabilities are zero, and so
        // must they be
        for (int at = lane * 16; at < ((j + 1) * FT - hd.klen) * 128; at += 512)
          for (int c = 0; c < HS / 64; ++c)
            *reinterpret_cast<uint4*>(base_ptr + (v_s - base) + s * TILE + c * FCHUNK + (hd.klen - j * FT) * 128 + at) =
                make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int nt = t ? n1 : n0;
        if (j >= nt || !ok) continue;
        ok = warp_wait(&p_full[t], j & 1, status, DEV_TIMEOUT_FULL, 0xb03 + t);
        if (!ok) break;
        tc_fence_after();
        if (leader) {
          const uint32_t b = v_s + s * TILE;
#pragma unroll
          for (int ks = 0; ks < FT / 16; ++ks)
            mma_f16_ts(tmem + 2 * FT + t * HS, tmem + t * FT + ks * 8, make_smem_desc(b + ks * 2048, FCHUNK, 1024),
                       IDESC_O, (j > 0 || ks > 0) ? 1u : 0u);
          if (j == nt - 1) tc_commit(smem_u32(&o_full[t]));
        }
        if (j + 1 < nt) {
          ok = warp_wait(&k_full[s2], ((j + 1) / NST) & 1, status, DEV_TIMEOUT_FULL, 0xb05);
          tc_fence_after();
          if (ok) scores(t, j + 1);
        }
      }
      if (leader) {
        tc_commit(smem_u32(&v_empty[s]));
        if (j + 1 < n) tc_commit(smem_u32(&k_empty[s2]));
      }
      __syncwarp();
    }
  } else if (warp >= 4) {
    // ===================== softmax =====================
    const int t = (warp - 4) >> 2, r = threadIdx.x & 127;
    const int nt = t ? n1 : n0;
    const int i = i0 + t * FT + r;
    const int vis = hd.visible(p, i);
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t s_col = lanes + t * FT, o_col = lanes + 2 * FT + t * HS;
    const float* bias = p.bias != nullptr ? p.bias + hd.head * (2 * p.reach + 1) : nullptr;
    const float c1 = p.c1;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < nt; ++j) {
      const TileBias tb(bias, p.reach, static_cast<long long>(j) * FT - (i0 + t * FT + FT - 1 + hd.off), r, -1,
                        window[t][j & 1], c1 >= 0.f);
      if (tb.near) group_barrier(1 + t);
      // a group that gave up still meets its barriers
      ok = ok && warp_wait(&s_full[t], j & 1, status, DEV_TIMEOUT_ACCUM, 0xc00 + t);
      if (!ok) continue;
      tc_fence_after();
      const int lim = vis - j * FT;  // columns below it are seen
      const bool masked = __any_sync(0xffffffffu, lim < FT);
      float top = -INFINITY;
      uint32_t v[32];
#pragma unroll
      for (int c = 0; c < FT; c += 32) {
        tmem_ld32(s_col + c, v);
        tmem_ld_wait();
        if (tb.near) {
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const float x = fmaf(__uint_as_float(v[e]), c1, tb.row[c + e]);
            top = fmaxf(top, !masked || c + e < lim ? x : -INFINITY);
          }
        } else {
          float raw = -INFINITY;
          if (masked) {
#pragma unroll
            for (int e = 0; e < 32; ++e) raw = fmaxf(raw, c + e < lim ? __uint_as_float(v[e]) : -INFINITY);
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) raw = fmaxf(raw, __uint_as_float(v[e]));
          }
          if (raw != -INFINITY) top = fmaxf(top, fmaf(raw, c1, tb.value));
        }
      }
      const bool grow = top > m + 8.f || (m == -INFINITY && top > m);
      if (__any_sync(0xffffffffu, grow)) {
        // O exists from the second tile on; what it holds for a row without keys so far is zero
        const float mn = fmaxf(m, top);
        const float a = mn == -INFINITY ? 1.f : ex2(m - mn);
        l *= a;
        m = mn;
        if (j > 0) {
#pragma unroll
          for (int c = 0; c < HS; c += 16) {
            uint32_t w[16];
            tmem_ld16(o_col + c, w);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(__uint_as_float(w[e]) * a);
            tmem_st16(o_col + c, w);
          }
        }
      }
      const float mu = m == -INFINITY ? 0.f : m;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < FT; c += 32) {
        tmem_ld32(s_col + c, v);
        tmem_ld_wait();
        float pr[32];
        const float shift = tb.value - mu;
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float x = tb.near ? fmaf(__uint_as_float(v[e]), c1, tb.row[c + e] - mu) : fmaf(__uint_as_float(v[e]), c1, shift);
          pr[e] = ex2(x);
        }
        if (masked) {
#pragma unroll
          for (int e = 0; e < 32; ++e) pr[e] = c + e < lim ? pr[e] : 0.f;
        }
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          sum[e & 3] += pr[2 * e] + pr[2 * e + 1];
          w[e] = pack_half2(pr[2 * e], pr[2 * e + 1]);
        }
        tmem_st16(s_col + c / 2, w);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(smem_u32(&p_full[t]));
    }
    // ---- result ----
    if (nt > 0 && ok) {
      ok = warp_wait(&o_full[t], 0, status, DEV_TIMEOUT_ACCUM, 0xc10 + t);
      tc_fence_after();
    }
    if (ok) {
      const bool real = i < p.tq;
      const float inv = l > 0.f ? 1.f / l : 0.f;
      __half* out = p.O + i * p.ldo + hd.head * p.sho + hd.batch * p.sbo;
#pragma unroll
      for (int c = 0; c < HS; c += 16) {
        uint32_t w[16];
        if (nt > 0) {
          tmem_ld16(o_col + c, w);
          tmem_ld_wait();
        }
        uint32_t h[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          h[e] = vis > 0 && nt > 0 && l > 0.f ? pack_half2(__uint_as_float(w[2 * e]) * inv, __uint_as_float(w[2 * e + 1]) * inv) : 0u;
        if (real && c < p.hs) *reinterpret_cast<uint4*>(out + c) = make_uint4(h[0], h[1], h[2], h[3]);
        if (real && c + 8 < p.hs) *reinterpret_cast<uint4*>(out + c + 8) = make_uint4(h[4], h[5], h[6], h[7]);
      }
      if (real)
        p.lse[(static_cast<long long>(hd.batch) * p.heads + hd.head) * p.tq + i] =
            l > 0.f ? (m + log2f(l)) * kLn2 : -INFINITY;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

bool heads_aligned(const FlashOperand& x, long long t, long long heads, long long batch) {
  if ((reinterpret_cast<uintptr_t>(x.p) & 15u) != 0) return false;
  const long long n[3] = {t, heads, batch}, s[3] = {x.ld, x.head, x.batch};
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && (s[i] % 8 != 0 || s[i] <= 0 || s[i] >= (1LL << 38))) return false;
  return true;
}

bool fill_params(const FlashArgs& a, FlashParams* p) {
  std::memset(p, 0, sizeof(*p));
  if (!encode_heads_tmap(&p->tmQ, a.q.p, a.hs, a.tq, a.heads, a.batch, a.q.ld, a.q.head, a.q.batch, FT) ||
      !encode_heads_tmap(&p->tmK, a.k.p, a.hs, a.tk, a.kv_heads, a.batch, a.k.ld, a.k.head, a.k.batch, FT) ||
      !encode_heads_tmap(&p->tmV, a.v.p, a.hs, a.tk, a.kv_heads, a.batch, a.v.ld, a.v.head, a.v.batch, FT))
    return false;
  p->O = static_cast<__half*>(const_cast<void*>(a.o.p));
  p->ldo = a.o.ld; p->sho = a.o.head; p->sbo = a.o.batch;
  p->lse = a.lse;
  p->bias = a.bias;
  p->tq = a.tq; p->tk = a.tk; p->hs = a.hs; p->heads = a.heads; p->group = a.heads / a.kv_heads; p->batch = a.batch;
  p->reach = a.reach; p->q_offset = a.q_offset;
  p->q_offsets = a.q_offsets; p->q_lengths = a.q_lengths; p->k_lengths = a.k_lengths;
  p->c1 = a.scale * kLog2e;
  p->causal = a.causal;
  return true;
}

template <int HS, int NST>
cudaError_t forward_hs(FlashParams& p, cudaStream_t stream, int* status) {
  const int smem = (2 + 2 * NST) * FCHUNK * (HS / 64) + 1024;
  static unsigned long long smem_set = 0;  // per template instantiation
  auto kern = flash_forward_kernel<HS, NST>;
  cudaError_t e = set_smem_limit_once(reinterpret_cast<const void*>(kern), smem, &smem_set);
  if (e != cudaSuccess) return e;
  p.qblocks = (p.tq + 2 * FT - 1) / (2 * FT);
  const long long grid = static_cast<long long>(p.qblocks) * p.heads * p.batch;
  if (grid > 0x7fffffffLL) return cudaErrorInvalidValue;
  return launch_kernel(kern, dim3(static_cast<unsigned>(grid)), dim3(384), smem, stream, pdl_enabled(), p, status);
}

}  // namespace

bool flash_supported(const FlashArgs& a) {
  return tmap_encoder_available() && a.hs % 8 == 0 && a.hs >= 8 && a.hs <= 128 && heads_aligned(a.q, a.tq, a.heads, a.batch) &&
         heads_aligned(a.k, a.tk, a.kv_heads, a.batch) && heads_aligned(a.v, a.tk, a.kv_heads, a.batch) &&
         heads_aligned(a.o, a.tq, a.heads, a.batch) &&
         static_cast<long long>((a.tq + 2 * FT - 1) / (2 * FT)) * a.heads * a.batch <= 0x7fffffffLL;
}

cudaError_t launch_flash_forward(const FlashArgs& a, cudaStream_t stream, int* status) {
  FlashParams p;
  if (!fill_params(a, &p)) return cudaErrorInvalidValue;
  return a.hs <= 64 ? forward_hs<64, 3>(p, stream, status) : forward_hs<128, 2>(p, stream, status);
}

}  // namespace gb
