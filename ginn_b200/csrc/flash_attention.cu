// Attention with a relative position bias whose scores never leave the SM: Half operands, and fp32 ones as
// two Half planes each.
//
// Forward: one CTA serves one or two tiles of 128 queries of one head and walks that head's keys in tiles
// of 128, once.  Query tile t has its scores S_t and its result O_t in tensor memory (128 lanes = queries,
// fp32); a group of 256 threads, two per query with half of the keys each, turns S_t into
// probabilities -- a row's maximum takes one exchange between two threads -- and writes them over S_t as the
// fp16 left operand of O_t += P_t V.  While one tile's (or another CTA's) threads work, the tensor cores
// work on the other's products.
//   warp 0        TMA: Q once, K and V tiles through rings of NST stages
//   warp 1        tcgen05.mma: S_t = Q_t K^T (operands in shared memory), O_t += P_t V (P in tensor memory)
//   warps 4-11    softmax of query tile 0,  warps 12-19  of query tile 1
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
//
// What bounds it: the threads between the two products (16 heads of 4096 x 4096 x 128, causal: 68.7 GFLOP in
// 90 us, 0.77 PFLOP/s, of 1.65 measured for a plain product), a row's exponentials, conversions and
// tensor-memory traffic against 2 x 128 x 128 x head size operations of the tensor core.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cstring>
#include <type_traits>
#include "ptx.cuh"
#include "math.cuh"
#include "launch.h"
#include "relative_attention.cuh"

namespace gb {

namespace {

constexpr int FT = 128;               // queries or keys per tile
constexpr int FTHREADS = 128 + 2 * 256;  // two working groups behind the warpgroup of TMA and MMA
constexpr int FCHUNK = FT * 128;      // bytes of 128 rows x 64 halves
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ uint32_t pack_half2(float a, float b);
// A pair of fp32 values as two Half pairs: what the first leaves, the second holds.
__device__ __forceinline__ void split_pair(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = pack_half2(a, b);
  const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  lo = pack_half2(a - h.x, b - h.y);
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Eight results of a row in the storage type, of which the first n exist: 16-byte stores where they are
// allowed (`vec`), element by element elsewhere and at the row's end.
__device__ __forceinline__ void store_row8(__half* to, int n, int vec, const float (&x)[8], bool add) {
  if (vec && n >= 8) {
    uint32_t w[4];
    uint4 old = make_uint4(0, 0, 0, 0);
    if (add) old = *reinterpret_cast<const uint4*>(to);
    const uint32_t o[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float2 q = make_float2(0.f, 0.f);
      if (add) q = __half22float2(*reinterpret_cast<const __half2*>(&o[e]));
      const __half2 h = __floats2half2_rn(x[2 * e] + q.x, x[2 * e + 1] + q.y);
      w[e] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) to[e] = __float2half_rn(add ? __half2float(to[e]) + x[e] : x[e]);
  }
}
__device__ __forceinline__ void store_row8(float* to, int n, int vec, const float (&x)[8], bool add) {
  if (vec && n >= 8) {
    float4 a = make_float4(x[0], x[1], x[2], x[3]), b = make_float4(x[4], x[5], x[6], x[7]);
    if (add) {
      const float4 c = *reinterpret_cast<const float4*>(to), d = *reinterpret_cast<const float4*>(to + 4);
      a.x += c.x; a.y += c.y; a.z += c.z; a.w += c.w;
      b.x += d.x; b.y += d.y; b.z += d.z; b.w += d.w;
    }
    *reinterpret_cast<float4*>(to) = a;
    *reinterpret_cast<float4*>(to + 4) = b;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) to[e] = add ? to[e] + x[e] : x[e];
  }
}
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// A whole warp waits; its lanes agree on the outcome, so that none is left alone at a later barrier.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* status, int code, int detail) {
  return __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity, status, code, detail));
}
__device__ __forceinline__ void group_barrier(int id) { asm volatile("bar.sync %0, 256;" ::"r"(id) : "memory"); }

struct FlashParams {
  CUtensorMap tmQ, tmK, tmV;
  void* O;
  long long ldo, sho, sbo;
  float* lse;
  const float* bias;
  const float *iq, *ik, *iv;  // split operands: inverse scales, [batch][kv heads]
  int tq, tk, hs, heads, kv_heads, group, batch, qblocks;
  int vec;                    // the result's rows allow 16-byte accesses
  int reach, q_offset;
  const int* q_offsets;
  const int* q_lengths;
  const int* k_lengths;
  float c1;  // scale * log2(e)
  int causal;
};

// What one (sequence, head) looks like to every role of a CTA.
struct FlashHead {
  int batch, head, kv, qlen, klen, off;
  __device__ __forceinline__ FlashHead(const FlashParams& p, int hb) {
    batch = hb / p.heads;
    head = hb - batch * p.heads;
    kv = head / p.group;
    qlen = rel_length(p.q_lengths, batch, p.tq);
    klen = rel_keys(p, batch);
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

// Bias of the 128 x 128 pairs of a tile whose smallest distance is `dlo`: one value for all of it
// (`flat`; a masked score is -inf before it is scaled, so that needs a positive scale), or
// window[c - r + 127] for column c of row r.  All 256 threads of a group call it.
struct TileBias {
  float value = 0.f;
  bool near = false;
  __device__ __forceinline__ TileBias(const float* bias, int reach, int dlo, int gt, float* window,
                                      bool flat_ok) {
    if (flat_ok && (bias == nullptr || dlo >= reach || dlo + 254 <= -reach)) {
      if (bias != nullptr) value = __ldg(bias + (dlo >= reach ? 2 * reach : 0));
    } else {
      near = true;
      int d = dlo + gt;
      d = d > reach ? reach : d < -reach ? -reach : d;
      window[gt] = bias != nullptr ? __ldg(bias + d + reach) : 0.f;
    }
  }
};

// The tensor core truncates each time it adds to an accumulator, once per 16 terms of a contraction.  Terms of one
// sign make that a bias that grows with the chain: fp32 results are off by 1.2e-6 of their size after 256 terms,
// 5.8e-6 after 1024, 2.5e-5 after 4096.  The kernels for fp32 operands therefore start a new chain every 512 terms
// and add the chains up with rounded additions: a result keeps 2^-17 of its terms' magnitudes (one sign 2.7e-6, the largest terms first 5.7e-6; chains of 1024 terms: 1.2e-5).  What ended lies
// in local memory, where a warp's accesses are neighbours: in the result's own place, rows apart, the end of a
// chain took 8 us of a CTA's time instead of 2.6 (4 heads of 4096 x 4096 x 64, seven of them: 126 us without, 144, and 180).
// Contractions of one chain have kernels without the code for its end (CHAINS), which they would pay registers for
// (256 heads of 256 x 256 x 64, a step: 255 us, and 247).
// Half results, which are rounded to 4.9e-4, take chains of 8192 terms (5.5e-5 of one sign; 131072 terms in one
// chain: 8.4e-4).
constexpr int kChain = 512, kChainHalf = 8192;

// SPLIT: fp32 operands as two Half planes each (see split_planes_kernel).  NQ: query tiles per CTA.  One tile
// of a 64-wide head leaves room for a second CTA on the SM (TWICE), whose start, loads and end then pass while
// the first computes; a thread has 80 registers there, so it reads its scores twice, 32 at a time, once
// for the maximum and once for the probabilities.  128-wide split operands (64 KB a tile) leave no room for
// two tiles either way: K and V have one stage each, which is loaded again while the other's product and the
// softmax run.
template <int HS, int NST, int NQ, bool SPLIT, bool CHAINS>
__global__ void __launch_bounds__(128 + 256 * NQ, NQ == 1 && HS == 64 ? 2 : 1)
flash_forward_kernel(const __grid_constant__ FlashParams p, int* __restrict__ status) {
  constexpr int WIDE = HS / 64;                  // 64-wide chunks of a plane
  constexpr int CHUNKS = (SPLIT ? 2 : 1) * WIDE;
  constexpr bool TWICE = NQ == 1 && HS == 64;
  constexpr int COLS = TWICE ? 256 : 512;
  constexpr int CROSS = NQ * HS;                 // tensor memory: from a tile's result to its cross terms
  constexpr int TILE = FCHUNK * CHUNKS;  // bytes of one operand tile
  constexpr float PSHIFT = SPLIT ? 7.f : 0.f;  // probabilities are formed times 2^PSHIFT: their low parts stay normal
  constexpr int CUT = (SPLIT ? kChain : kChainHalf) / FT;  // key tiles to a chain
  using Out = typename std::conditional<SPLIT, float, __half>::type;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t q_full[2], k_full[NST], k_empty[NST], v_full[NST], v_empty[NST];
  __shared__ __align__(8) uint64_t s_full[2], p_full[2], o_full[2];
  __shared__ uint32_t tmem_slot;
  __shared__ float window[2][2][256];
  __shared__ float exchange[2][2][2][FT];  // [tile][turn][half]: row maxima, at the end row sums

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* base_ptr = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t q_s = base, k_s = base + NQ * TILE, v_s = k_s + NST * TILE;

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
        mbar_init(smem_u32(&p_full[t]), 256);
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
    tmem_alloc(smem_u32(&tmem_slot), COLS);
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
  const int i0 = qb * NQ * FT;
  const int n0 = hd.tiles(p, i0), n1 = NQ > 1 ? hd.tiles(p, i0 + FT) : 0;
  const int n = n0 > n1 ? n0 : n1;

  if (warp == 0) {
    // ===================== TMA producer =====================
    auto load = [&](uint32_t dst, const CUtensorMap* map, uint64_t* bar, int at, int head) {
      mbar_arrive_expect_tx(smem_u32(bar), TILE);
      for (int c = 0; c < CHUNKS; ++c)
        tma_load_4d(dst + c * FCHUNK, map, smem_u32(bar), 64 * (c % WIDE), at, head, hd.batch + c / WIDE * p.batch);
    };
    if (elect_one()) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if ((t ? n1 : n0) > 0) load(q_s + t * TILE, &p.tmQ, &q_full[t], i0 + t * FT, hd.head);
      for (int j = 0; j < n; ++j) {
        const int s = j % NST;
        const uint32_t ph = (j / NST) & 1;
        if (!mbar_wait(smem_u32(&k_empty[s]), ph ^ 1u, status, DEV_TIMEOUT_EMPTY, 0xa00)) break;
        load(k_s + s * TILE, &p.tmK, &k_full[s], j * FT, hd.kv);
        if (!mbar_wait(smem_u32(&v_empty[s]), ph ^ 1u, status, DEV_TIMEOUT_EMPTY, 0xa01)) break;
        load(v_s + s * TILE, &p.tmV, &v_full[s], j * FT, hd.kv);
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
        // split operands: low x high and high x low first, while the accumulator is small
#pragma unroll
        for (int term = 0; term < (SPLIT ? 3 : 1); ++term)
#pragma unroll
          for (int ks = 0; ks < HS / 16; ++ks) {
            const uint32_t at = (ks / 4) * FCHUNK + (ks % 4) * 32;
            mma_f16(tmem + t * FT, make_smem_desc(a + at + (SPLIT && term == 0 ? WIDE * FCHUNK : 0), 16, 1024),
                    make_smem_desc(b + at + (SPLIT && term == 1 ? WIDE * FCHUNK : 0), 16, 1024), IDESC_S, term > 0 || ks > 0);
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
      if (!SPLIT && ok && hd.klen < p.tk && (j + 1) * FT > hd.klen) {
        // rows behind the sequence's end may hold anything: their probabilities are zero, and so
        // must they be
        for (int at = lane * 16; at < ((j + 1) * FT - hd.klen) * 128; at += 512)
          for (int c = 0; c < CHUNKS; ++c)
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
          for (int ks = 0; ks < FT / 16; ++ks) {
            const uint32_t o = tmem + NQ * FT + t * HS, a = tmem + t * FT + (ks / 2) * 32 + (ks % 2) * 8;
            const uint32_t add = ((CHAINS ? j % CUT : j) > 0 || ks > 0) ? 1u : 0u;
            mma_f16_ts(o, a, make_smem_desc(b + ks * 2048, FCHUNK, 1024), IDESC_O, add);
            if (SPLIT) {
              // The cross terms have an accumulator of their own: the tensor core truncates when it adds, so
              // the long chain of the main one should be as short as it can be.
              mma_f16_ts(o + CROSS, a, make_smem_desc(b + WIDE * FCHUNK + ks * 2048, FCHUNK, 1024), IDESC_O, add);
              mma_f16_ts(o + CROSS, a + 16, make_smem_desc(b + ks * 2048, FCHUNK, 1024), IDESC_O, 1u);
            }
          }
          if (j == nt - 1) tc_commit(smem_u32(&o_full[t]));
        }
        if (j + 1 < nt) {
          ok = warp_wait(&k_full[s2], ((j + 1) / NST) & 1, status, DEV_TIMEOUT_FULL, 0xb05);
          tc_fence_after();
          if (ok) scores(t, j + 1);
        }
      }
      if (leader) {
        // only where the producer waits for it: behind the last o_full nothing else keeps the CTA until it has arrived
        if (j + NST < n) tc_commit(smem_u32(&v_empty[s]));
        if (j + 1 + NST < n) tc_commit(smem_u32(&k_empty[s2]));
      }
      __syncwarp();
    }
  } else if (warp >= 4) {
    // ===================== softmax =====================
    // thread: query row r of tile t, keys 64 half .. 64 half + 63 of every key tile
    const int t = (warp - 4) >> 3, half = ((warp - 4) >> 2) & 1;
    const int r = threadIdx.x & 127, gt = (threadIdx.x - 128) & 255;
    const int nt = t ? n1 : n0;
    const int i = i0 + t * FT + r;
    const int vis = hd.visible(p, i);
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t s_col = lanes + t * FT + half * 64, o_col = lanes + NQ * FT + t * HS + half * (HS / 2);
    const float* bias = p.bias != nullptr ? p.bias + static_cast<long long>(hd.head) * (2 * p.reach + 1) : nullptr;
    const int unit = hd.batch * p.kv_heads + hd.kv;
    const float c1 = SPLIT ? p.c1 * p.iq[unit] * p.ik[unit] : p.c1;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    float md = -INFINITY;  // the maximum that the chains which ended are relative to
    // What they add up to.  Indexed in loops that stay loops, so that it lies in local memory and not among the
    // registers of every tile; a warp's accesses there are neighbours.
    float part[CHAINS ? HS / 2 : 1];
    // Elements c .. c + 7 of the chain in tensor memory and, where there are any, `old` times those before it.
    auto chain8 = [&](int c, bool before, float old, float (&x)[8]) {
      uint32_t w[8], cross[8];
      tmem_ld8(o_col + c, w);
      if (SPLIT) tmem_ld8(o_col + CROSS + c, cross);
      tmem_ld_wait();
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = SPLIT ? __uint_as_float(w[e]) + __uint_as_float(cross[e]) : __uint_as_float(w[e]);
      if (CHAINS && before) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = fmaf(part[CHAINS ? c + e : 0], old, x[e]);
      }
    };
    for (int j = 0; j < nt; ++j) {
      float* win = window[t][j & 1];
      const TileBias tb(bias, p.reach, j * FT - (i0 + t * FT + FT - 1 + hd.off), gt, win, c1 > 0.f);
      if (tb.near) group_barrier(1 + t);
      // a group that gave up still meets its barriers
      ok = ok && warp_wait(&s_full[t], j & 1, status, DEV_TIMEOUT_ACCUM, 0xc00 + t);
      float mn = -INFINITY;
      const float* row = win + (FT - 1) - r + 64 * half;
      const int lim = vis - j * FT - 64 * half;  // columns below it are seen
      // 32 scores from column `from` on: raw ones with a flat bias, finished ones with a window
      auto read = [&](int from, uint32_t* v) {
        tmem_ld32(s_col + from, *reinterpret_cast<uint32_t(*)[32]>(v));
        tmem_ld_wait();
        if (tb.near) {
#pragma unroll
          for (int c = 0; c < 32; ++c) v[c] = __float_as_uint(fmaf(__uint_as_float(v[c]), c1, row[from + c]));
        }
        if (__any_sync(0xffffffffu, lim < from + 32)) {
#pragma unroll
          for (int c = 0; c < 32; ++c) v[c] = from + c < lim ? v[c] : 0xff800000u;  // -inf
        }
      };
      uint32_t v[TWICE ? 32 : 64];
      if (ok) {
        tc_fence_after();
        if (CHAINS && j > 0 && j % CUT == 0) {  // a chain ends: the products of the tiles before it are done
          const float old = md == m ? 1.f : ex2(md - m);
#pragma unroll 1
          for (int c = 0; c < HS / 2; c += 8) {
            float x[8];
            chain8(c, j > CUT, old, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) part[CHAINS ? c + e : 0] = x[e];
          }
          md = m;
        }
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          uint32_t* x = v + (TWICE ? 0 : 32 * part);
          read(32 * part, x);
#pragma unroll
          for (int c = 0; c < 32; c += 8)
#pragma unroll
            for (int e = 0; e < 4; ++e) top[e] = fmaxf(top[e], fmaxf(__uint_as_float(x[c + 2 * e]), __uint_as_float(x[c + 2 * e + 1])));
        }
        mn = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        if (!tb.near && mn > -INFINITY) mn = fmaf(mn, c1, tb.value);
      }
      exchange[t][j & 1][half][r] = mn;
      group_barrier(1 + t);
      if (!ok) continue;
      mn = fmaxf(mn, exchange[t][j & 1][half ^ 1][r]);
      if (__any_sync(0xffffffffu, mn > m + 8.f)) {  // also a row's first visible key (m = -inf)
        mn = fmaxf(m, mn);
        const float a = mn == -INFINITY ? 1.f : ex2(m - mn);
        l *= a;
        m = mn;
        if ((CHAINS ? j % CUT : j) > 0) {  // O exists from the second tile of a chain on
#pragma unroll
          for (int c = 0; c < (SPLIT ? HS : HS / 2); c += 16) {
            const uint32_t col = o_col + c + (c >= HS / 2 ? CROSS - HS / 2 : 0);  // behind the main result: the cross terms
            uint32_t w[16];
            tmem_ld16(col, w);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(__uint_as_float(w[e]) * a);
            tmem_st16(col, w);
          }
        }
      }
      const float mu = m == -INFINITY ? 0.f : m;
      const float ca = tb.near ? 1.f : c1, cb = tb.value - mu + PSHIFT;
      const F2 ca2(ca, ca), cb2(cb, cb);
      F2 sum[2] = {F2(0.f, 0.f), F2(0.f, 0.f)};
#pragma unroll
      for (int c = 0; c < 64; c += 32) {
        uint32_t w[16], low[16];
        uint32_t* z = v + (TWICE ? 0 : c);
        if (TWICE) read(c, z);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float x, y;
          fma2(F2(__uint_as_float(z[2 * e]), __uint_as_float(z[2 * e + 1])), ca2, cb2).get(x, y);
          x = ex2(x);
          y = ex2(y);
          sum[e & 1] = add2(sum[e & 1], F2(x, y));
          if (SPLIT) split_pair(x, y, w[e], low[e]);
          else w[e] = pack_half2(x, y);
        }
        tmem_st16(s_col + c, w);  // over scores this thread is done with
        if (SPLIT) tmem_st16(s_col + c + 16, low);
      }
      float sa, sb;
      add2(sum[0], sum[1]).get(sa, sb);
      l += sa + sb;
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(smem_u32(&p_full[t]));
    }
    // ---- result ----
    // turn nt & 1 of the exchange was last read before the barrier of tile nt - 1
    exchange[t][nt & 1][half][r] = l;
    group_barrier(1 + t);
    l += exchange[t][nt & 1][half ^ 1][r];
    if (nt > 0 && ok) {
      ok = warp_wait(&o_full[t], 0, status, DEV_TIMEOUT_ACCUM, 0xc10 + t);
      tc_fence_after();
    }
    if (ok) {
      const bool real = i < p.tq, some = nt > 0 && vis > 0 && l != 0.f;  // (not a number stays one)
      const float inv = some ? (SPLIT ? p.iv[unit] : 1.f) / l : 0.f, old = md == m ? 1.f : ex2(md - m);
      Out* out = static_cast<Out*>(p.O) + i * p.ldo + hd.head * p.sho + hd.batch * p.sbo;
      auto eight = [&](int c) {
        float x[8];
        if (nt > 0) chain8(c, nt > CUT, old, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = some ? x[e] * inv : 0.f;
        const int at = half * (HS / 2) + c;
        if (real) store_row8(out + at, p.hs - at, p.vec, x, false);
      };
      if (CHAINS) {
#pragma unroll 1
        for (int c = 0; c < HS / 2; c += 8) eight(c);
      } else {
#pragma unroll
        for (int c = 0; c < HS / 2; c += 8) eight(c);
      }
      if (real && half == 0)
        p.lse[(static_cast<long long>(hd.batch) * p.heads + hd.head) * p.tq + i] = some ? (m + log2f(l) - PSHIFT) * kLn2 : -INFINITY;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, COLS);
  }
}

// ---- fp32 operands as Half planes -----------------------------------------------------------------
//
// An fp32 matrix times a power of two that brings its largest magnitude (per sequence and key head) to
// [2^14, 2^15) is written as the sum of two Half matrices, high = rn(x), low = rn(x - high): 22 bits of
// every element down to 2^-18 of the largest, and an absolute error of 2^-39 of the largest at most below
// that (half a step of a subnormal, 2^-25, against 2^14).  A product is then three Half products, high x high + high x low + low x high, at twice the
// rate of three TF32 products and with the same 2^-22 left out.  The planes are dense,
// [plane][sequence][head][t][64 or 128], zero behind the head size, in queries behind the
// lengths and in keys that no query sees.
struct SplitOperand {
  const float* x;
  long long ld, head, batch;
  __half* planes;
  int t, heads, per;      // heads per scale
  bool query;
  int vec;                // rows allow 16-byte accesses
  long long block0;       // first CTA of this operand
};
struct SplitParams {
  SplitOperand op[4];     // q, k, v and, for the backward pass, d_o
  RelExtent extent;
  int count, hs, batch, kv_heads;
  unsigned* most;         // [operand][batch][kv heads]: bits of the largest magnitude
  unsigned* norms;        // backward: [d_o, v][batch][kv heads]: bits of the largest row's squared norm
  float* inverse;         // [operand][batch][kv heads]: what a scaled value is multiplied by to get it back
  // backward: delta = sum d_o o and lse of every query
  const float* o;
  long long ldo, sho, sbo;
  int vec_o, tq_pad;
  const float* lse;
  float2* stats;
};
constexpr int kSplitRows = 128;  // per CTA: four elements of a row to a thread
// Rows row0 .. row0 + 127 of one head, by CTA; the operand's fields selected one by one (indexing the
// parameters would copy them to local memory).
struct SplitPart {
  const float* x = nullptr;
  __half* planes = nullptr;
  long long ld = 0, plane = 0;
  int which = 0, unit = 0, row0 = 0, rows = 0, real = 0, vec = 0, batch = 0, head = 0, heads = 1;
  __device__ __forceinline__ SplitPart(const SplitParams& p, int width) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i >= p.count || blockIdx.x < p.op[i].block0) continue;
      const long long at = blockIdx.x - p.op[i].block0;
      const int parts = (p.op[i].t + kSplitRows - 1) / kSplitRows, hb = static_cast<int>(at / parts);
      heads = p.op[i].heads;
      batch = hb / heads;
      head = hb - batch * heads;
      which = i;
      unit = batch * p.kv_heads + head / p.op[i].per;
      row0 = static_cast<int>(at % parts) * kSplitRows;
      rows = p.op[i].t;
      real = rel_rows(p.extent, p.op[i].query, batch);
      vec = p.op[i].vec;
      ld = p.op[i].ld;
      x = p.op[i].x + head * p.op[i].head + batch * p.op[i].batch;
      planes = p.op[i].planes + static_cast<long long>(hb) * rows * width;
      plane = static_cast<long long>(p.batch) * heads * rows * width;
    }
  }
};
// Elements col .. col + 3 of a row, zero from n on.
__device__ __forceinline__ float4 load_four(const float* x, int n, int vec) {
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (vec && n >= 4) return *reinterpret_cast<const float4*>(x);
  if (n > 0) v.x = x[0];
  if (n > 1) v.y = x[1];
  if (n > 2) v.z = x[2];
  if (n > 3) v.w = x[3];
  return v;
}

// Largest magnitude of every unit and, for the backward pass, the largest row norms of d_o and v.
template <int W>
__global__ void __launch_bounds__(256)
split_most_kernel(const __grid_constant__ SplitParams p) {
  __shared__ unsigned red[2][8];
  pdl_wait();
  pdl_launch_dependents();
  constexpr int LANES = W / 4, PER = 32 / LANES, SWEEPS = kSplitRows / (8 * PER);  // lanes to a row, rows to a warp
  const SplitPart part(p, W);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = 4 * (lane % LANES);
  const bool norm = p.norms != nullptr && part.which >= 2;
  float4 x[SWEEPS];
#pragma unroll
  for (int k = 0; k < SWEEPS; ++k) {
    const int row = part.row0 + (8 * k + warp) * PER + lane / LANES;
    x[k] = load_four(part.x + row * part.ld + col, row < part.real ? p.hs - col : 0, part.vec);
  }
  unsigned m = 0, q = 0;
#pragma unroll
  for (int k = 0; k < SWEEPS; ++k) {
    const float4 v = x[k];
    m = max(max(m, max(__float_as_uint(fabsf(v.x)), __float_as_uint(fabsf(v.y)))),
            max(__float_as_uint(fabsf(v.z)), __float_as_uint(fabsf(v.w))));
    if (norm) {
      float s = (v.x * v.x + v.y * v.y) + (v.z * v.z + v.w * v.w);
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      q = max(q, __float_as_uint(s));
    }
  }
  m = __reduce_max_sync(0xffffffffu, m);
  q = __reduce_max_sync(0xffffffffu, q);
  if (lane == 0) {
    red[0][warp] = m;
    red[1][warp] = q;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < 8; ++w) {
    m = max(m, red[0][w]);
    q = max(q, red[1][w]);
  }
  // maxima of non-negative values: the order of the updates does not matter
  const int units = p.batch * p.kv_heads;
  atomicMax(p.most + part.which * units + part.unit, m);
  if (norm) atomicMax(p.norms + (part.which == 3 ? 0 : units) + part.unit, q);
}

template <int W>
__global__ void __launch_bounds__(256)
split_planes_kernel(const __grid_constant__ SplitParams p) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int LANES = W / 4, PER = 32 / LANES, SWEEPS = kSplitRows / (8 * PER);  // lanes to a row, rows to a warp
  const SplitPart part(p, W);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = 4 * (lane % LANES);
  const int at = part.which * p.batch * p.kv_heads + part.unit;
  const unsigned most = p.most[at];
  // 2^(14 - exponent of the largest); not numbers and infinities go through as they are
  int e = 14 - (static_cast<int>(most >> 23) - 127);
  e = e > 126 ? 126 : e;
  if (most == 0 || most >= 0x7f800000u) e = 0;
  const float scale = __uint_as_float(static_cast<unsigned>(e + 127) << 23);
  if (part.row0 == 0 && threadIdx.x == 0) p.inverse[at] = 1.f / scale;
  const bool dot = p.stats != nullptr && part.which == 3;
  float4 x[SWEEPS];
#pragma unroll
  for (int k = 0; k < SWEEPS; ++k) {
    const int row = part.row0 + (8 * k + warp) * PER + lane / LANES;
    x[k] = load_four(part.x + row * part.ld + col, row < part.real ? p.hs - col : 0, part.vec);
  }
#pragma unroll
  for (int k = 0; k < SWEEPS; ++k) {
    const int row = part.row0 + (8 * k + warp) * PER + lane / LANES;
    if (row < part.rows) {
      uint2 hi, lo;
      split_pair(x[k].x * scale, x[k].y * scale, hi.x, lo.x);
      split_pair(x[k].z * scale, x[k].w * scale, hi.y, lo.y);
      __half* to = part.planes + static_cast<long long>(row) * W + col;
      *reinterpret_cast<uint2*>(to) = hi;
      *reinterpret_cast<uint2*>(to + part.plane) = lo;
    }
    if (!dot) continue;  // uniform over the CTA
    const float4 o = load_four(p.o + row * p.ldo + part.head * p.sho + part.batch * p.sbo + col, row < part.real ? p.hs - col : 0,
                               p.vec_o);
    float s = (x[k].x * o.x + x[k].y * o.y) + (x[k].z * o.z + x[k].w * o.w);
#pragma unroll
    for (int w = LANES / 2; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
    if (lane % LANES == 0 && row < p.tq_pad) {
      const long long hb = static_cast<long long>(part.batch) * part.heads + part.head;
      float2 st = make_float2(INFINITY, 0.f);
      if (row < part.real) {
        const float l = p.lse[hb * part.rows + row];
        if (l != -INFINITY) st = make_float2(l * kLog2e, s);
      }
      p.stats[hb * p.tq_pad + row] = st;
    }
  }
}

// Half operands off the 16-byte grid (head sizes that are no multiple of 8, odd strides): a dense copy,
// dst[sequence][head][t][W], zero behind the head size.  One warp per row and sweep.
template <int W>
__global__ void __launch_bounds__(256)
flash_pack_kernel(const __half* __restrict__ src, long long ld, long long sh, long long sb, int hs, int t, int heads,
                  long long rows, __half* __restrict__ dst) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  for (long long row = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5); row < rows; row += static_cast<long long>(gridDim.x) * 8) {
    const long long hb = row / t, b = hb / heads;
    const __half* x = src + (row - hb * t) * ld + (hb - b * heads) * sh + b * sb;
#pragma unroll
    for (int c = 0; c < W; c += 32) dst[row * W + c + lane] = c + lane < hs ? x[c + lane] : __float2half(0.f);
  }
}

// ---- a few queries against a long cache ---------------------------------------------------------
//
// A token's attention reads every cached key and value once and does little with them: it is bound by
// HBM, and what counts is many loads in flight and no work per byte beside them.  The queries that
// share a key head (heads of the group x positions, at most 16 rows) go together, so that the cache is
// read once.  The keys are split over CTAs, and over the four warps of a CTA in blocks of 16; a warp
// keeps its own running maximum, sum and result.  Operands go from global memory to registers in the
// layout of mma.m16n8k16 without a stop in shared memory: the order in which a contraction runs over
// the head elements is free, so a lane's 16 contiguous bytes of a key serve as its share of two
// fragments, and the values of two neighbouring keys, interleaved by byte permutes, as those of the second
// product.  (A tcgen05 tile would be 128 rows high for these 1 to 16, with the cache passing through
// shared memory.)  32 sequences of up to 8192 keys, four key heads of 128 with four queries each: 336 MB in
// 73 us, 4.6 TB/s of 6.5 copied; 370 us on the tiles above.
constexpr int kTokenRows = 16;
constexpr int kTokenWarps = 4;  // two CTAs on an SM: one loads while the other starts or joins its warps
// Most keys of a part of a cache.  The tensor core truncates each time it adds to an accumulator, eight keys of a warp at
// a time (Half: sixteen), and values of one sign make that a bias that grows with the chain: an fp32 part of 16384 keys is
// off by 4.8e-5 of the result, one of 2048 by 5.9e-6.  The parts' results are joined with rounded additions.
constexpr int kTokenChain = 1024, kTokenChainHalf = 32768;

struct TokenParams {
  const void *q, *k, *v;
  long long ldq, shq, sbq, ldk, shk, sbk, ldv, shv, sbv;
  void* o;
  long long ldo, sho, sbo;
  float* lse;
  float* part;    // [batch][kv][split][row][HS] results, then their (maximum, sum) pairs
  float2* stat;   // [batch][kv][split][row]
  const float* bias;
  int tq, tk, hs, heads, kv_heads, group, batch, rows, splits, chunk;
  int vec_k, vec_v;  // fp32: rows allow 16-byte accesses
  int reach, q_offset;
  const int* q_offsets;
  const int* q_lengths;
  const int* k_lengths;
  float c1;
  int causal;
};

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 load_stream(const __half* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// Final values of one row: o and lse.
template <typename T>
__device__ __forceinline__ void token_store(const TokenParams& p, int batch, int kv, int row, int h, float value, float m, float l) {
  const int head = kv * p.group + row / p.tq, i = row % p.tq;
  if (h < p.hs) static_cast<T*>(p.o)[h + i * p.ldo + head * p.sho + batch * p.sbo] = from_f<T>(l != 0.f ? value / l : 0.f);
  if (h == 0)
    p.lse[(static_cast<long long>(batch) * p.heads + head) * p.tq + i] = l != 0.f ? (m + log2f(l)) * kLn2 : -INFINITY;
}

// What a lane knows of its two rows of the scores, g and g + 8, and of its CTA's keys.
struct TokenLane {
  int warp, lane, g, c, split, batch, kv, begin, end;
  long long unit;
  int first_pos, vis[2], pos[2];
  const float* bias[2];
  float far_lo[2];
  float m[2], l[2];
  __device__ __forceinline__ explicit TokenLane(const TokenParams& p) {
    warp = threadIdx.x >> 5;
    lane = threadIdx.x & 31;
    g = lane >> 2;
    c = lane & 3;
    split = static_cast<int>(blockIdx.x) % p.splits;
    unit = blockIdx.x / p.splits;
    batch = static_cast<int>(unit / p.kv_heads);
    kv = static_cast<int>(unit % p.kv_heads);
    const int klen = rel_length(p.k_lengths, batch, p.tk), qlen = rel_length(p.q_lengths, batch, p.tq);
    first_pos = rel_offset(p.q_offset, p.q_offsets, batch);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int row = g + 8 * x, i = row % p.tq, head = kv * p.group + row / p.tq;
      const bool real = row < p.rows;
      pos[x] = i + first_pos;
      vis[x] = real && i < qlen ? rel_visible(p.causal, pos[x], klen) : 0;
      bias[x] = nullptr;
      far_lo[x] = 0.f;
      if (p.bias != nullptr && real) {
        bias[x] = p.bias + static_cast<long long>(head) * (2 * p.reach + 1) + p.reach;
        far_lo[x] = bias[x][-p.reach];
      }
      m[x] = -INFINITY;
      l[x] = 0.f;
    }
    const int last = qlen > 0 ? rel_visible(p.causal, qlen - 1 + first_pos, klen) : 0;  // the most any row sees
    begin = split * p.chunk;
    end = begin + p.chunk < last ? begin + p.chunk : last;
  }
  // A CTA without keys leaves what the join passes over.
  __device__ __forceinline__ bool nothing(const TokenParams& p) const {
    if (begin < end || p.splits == 1) return false;
    if (threadIdx.x < p.rows) p.stat[(unit * p.splits + split) * p.rows + threadIdx.x] = make_float2(-INFINITY, 0.f);
    return true;
  }
  // Raw scores of keys j .. j + 8 M - 1 (row g + 8 x at key j + 8 t + 2 c + y: sc[t][2 x + y]) become
  // probabilities; when a row's maximum grew, the result so far is rescaled.
  template <int N, int M>
  __device__ __forceinline__ void softmax(const TokenParams& p, int j, float (&sc)[M][4], float (&acc)[N][4]) {
    const bool flat = p.bias == nullptr || j + 8 * M - 1 - first_pos <= -p.reach;  // for every row: positions only grow
    const bool full = j + 8 * M <= vis[0] && j + 8 * M <= vis[1];
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int t = 0; t < M; ++t)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int key = j + 8 * t + 2 * c + y;
          float b = far_lo[x];
          if (!flat && bias[x] != nullptr) {
            int d = key - pos[x];
            d = d > p.reach ? p.reach : d < -p.reach ? -p.reach : d;
            b = bias[x][d];
          }
          float v = fmaf(sc[t][2 * x + y], p.c1, b);
          if (!full && key >= vis[x]) v = -INFINITY;
          sc[t][2 * x + y] = v;
          top[x] = fmaxf(top[x], v);
        }
    bool grow = false;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 1));
      top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 2));
      grow = grow || top[x] > m[x] + 8.f;
    }
    if (__any_sync(0xffffffffu, grow)) {
      float a[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float mn = fmaxf(m[x], top[x]);
        a[x] = mn == -INFINITY ? 1.f : ex2(m[x] - mn);
        m[x] = mn;
        l[x] *= a[x];
      }
#pragma unroll
      for (int e = 0; e < N; ++e) {
        acc[e][0] *= a[0];
        acc[e][1] *= a[0];
        acc[e][2] *= a[1];
        acc[e][3] *= a[1];
      }
    }
#pragma unroll
    for (int t = 0; t < M; ++t)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float mu = m[x] == -INFINITY ? 0.f : m[x];
        sc[t][2 * x] = ex2(sc[t][2 * x] - mu);
        sc[t][2 * x + 1] = ex2(sc[t][2 * x + 1] - mu);
        l[x] += sc[t][2 * x] + sc[t][2 * x + 1];
      }
  }
  // The warps' results together: res holds [warp][row][HS + 4] once every warp has written its own.
  template <int HS, typename T>
  __device__ __forceinline__ void join(const TokenParams& p, const float* res, float (*mx)[kTokenRows], float (*sm)[kTokenRows]) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
      if (c == 0) {
        mx[warp][g + 8 * x] = m[x];
        sm[warp][g + 8 * x] = l[x];
      }
    }
    __syncthreads();
    for (int at = threadIdx.x; at < p.rows * HS; at += 32 * kTokenWarps) {
      const int row = at / HS, h = at % HS;
      float all = -INFINITY, sum = 0.f, value = 0.f;
#pragma unroll
      for (int w = 0; w < kTokenWarps; ++w) all = fmaxf(all, mx[w][row]);
#pragma unroll
      for (int w = 0; w < kTokenWarps; ++w) {
        const float a = mx[w][row] == -INFINITY ? 0.f : ex2(mx[w][row] - all);
        sum += sm[w][row] * a;
        value += res[(w * p.rows + row) * (HS + 4) + h] * a;
      }
      if (p.splits == 1) {
        token_store<T>(p, batch, kv, row, h, value, all, sum);
      } else {
        const long long to = (unit * p.splits + split) * p.rows + row;
        p.part[to * HS + h] = value;
        if (h == 0) p.stat[to] = make_float2(all, sum);
      }
    }
  }
};

template <int HS>
__global__ void __launch_bounds__(32 * kTokenWarps, 2)
flash_token_kernel(const TokenParams p) {
  extern __shared__ float res[];  // [warp][row][HS + 4]
  __shared__ float mx[kTokenWarps][kTokenRows], sm[kTokenWarps][kTokenRows];
  pdl_wait();
  pdl_launch_dependents();
  TokenLane w(p);
  if (w.nothing(p)) return;
  const int g = w.g, c = w.c, end = w.end;
  uint32_t q[HS / 32][2][4];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int row = g + 8 * x;
    const __half* from = static_cast<const __half*>(p.q) + row % p.tq * p.ldq + (w.kv * p.group + row / p.tq) * p.shq + w.batch * p.sbq;
#pragma unroll
    for (int s = 0; s < HS / 32; ++s) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (row < p.rows && 32 * s + 8 * c < p.hs) v = *reinterpret_cast<const uint4*>(from + 32 * s + 8 * c);
      q[s][x][0] = v.x; q[s][x][1] = v.y; q[s][x][2] = v.z; q[s][x][3] = v.w;
    }
  }
  float acc[HS / 8][4];
#pragma unroll
  for (int e = 0; e < HS / 8; ++e) acc[e][0] = acc[e][1] = acc[e][2] = acc[e][3] = 0.f;
  const __half* kp = static_cast<const __half*>(p.k) + w.kv * p.shk + w.batch * p.sbk;
  const __half* vp = static_cast<const __half*>(p.v) + w.kv * p.shv + w.batch * p.sbv;
  uint4 kr[2][HS / 32], vr[HS / 64][4];
  auto load_k = [&](int j) {  // keys j + g and j + 8 + g, head elements 32 s + 8 c ..
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int s = 0; s < HS / 32; ++s) {
        const int key = j + 8 * t + g;
        kr[t][s] = make_uint4(0, 0, 0, 0);
        if (key < end && 32 * s + 8 * c < p.hs) kr[t][s] = load_stream(kp + key * p.ldk + 32 * s + 8 * c);
      }
  };
  auto load_v = [&](int j) {  // keys j + 2 c + {0, 1, 8, 9}, head elements 64 s + 8 g ..
#pragma unroll
    for (int s = 0; s < HS / 64; ++s)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int key = j + 2 * c + (t & 1) + 8 * (t >> 1);
        vr[s][t] = make_uint4(0, 0, 0, 0);
        if (key < end && 64 * s + 8 * g < p.hs) vr[s][t] = load_stream(vp + key * p.ldv + 64 * s + 8 * g);
      }
  };
  int j = w.begin + 16 * w.warp;
  if (j < end) {
    load_k(j);
    load_v(j);
  }
  for (; j < end; j += 16 * kTokenWarps) {
    float sc[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      sc[t][0] = sc[t][1] = sc[t][2] = sc[t][3] = 0.f;
#pragma unroll
      for (int s = 0; s < HS / 32; ++s) {
        mma_16816(sc[t], q[s][0][0], q[s][1][0], q[s][0][1], q[s][1][1], kr[t][s].x, kr[t][s].y);
        mma_16816(sc[t], q[s][0][2], q[s][1][2], q[s][0][3], q[s][1][3], kr[t][s].z, kr[t][s].w);
      }
    }
    const int next = j + 16 * kTokenWarps;
    if (next < end) load_k(next);
    w.softmax(p, j, sc, acc);
    uint32_t pr[2][2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int x = 0; x < 2; ++x) pr[t][x] = pack_half2(sc[t][2 * x], sc[t][2 * x + 1]);
#pragma unroll
    for (int s = 0; s < HS / 64; ++s) {
      const uint32_t v0[4] = {vr[s][0].x, vr[s][0].y, vr[s][0].z, vr[s][0].w}, v1[4] = {vr[s][1].x, vr[s][1].y, vr[s][1].z, vr[s][1].w};
      const uint32_t v8[4] = {vr[s][2].x, vr[s][2].y, vr[s][2].z, vr[s][2].w}, v9[4] = {vr[s][3].x, vr[s][3].y, vr[s][3].z, vr[s][3].w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {  // head element 64 s + 8 n + e for column n of the fragment
        const uint32_t pick = e & 1 ? 0x7632u : 0x5410u;
        mma_16816(acc[8 * s + e], pr[0][0], pr[0][1], pr[1][0], pr[1][1], __byte_perm(v0[e / 2], v1[e / 2], pick),
                  __byte_perm(v8[e / 2], v9[e / 2], pick));
      }
    }
    if (next < end) load_v(next);
  }
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int row = g + 8 * x;
    if (row >= p.rows) continue;
    // element k of a fragment: row g + 8 (k / 2), column n = 2 c + k % 2, head element 64 s + 8 n + e
    float* to = res + (w.warp * p.rows + row) * (HS + 4);
#pragma unroll
    for (int s = 0; s < HS / 64; ++s)
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < 8; e += 4)
          *reinterpret_cast<float4*>(to + 64 * s + 8 * (2 * c + k) + e) =
              make_float4(acc[8 * s + e][2 * x + k], acc[8 * s + e + 1][2 * x + k], acc[8 * s + e + 2][2 * x + k],
                          acc[8 * s + e + 3][2 * x + k]);
  }
  w.join<HS, __half>(p, res, mx, sm);
}

// fp32: three TF32 products per term on mma.m16n8k8, values split as they arrive (high: rounded to the
// upper 11 bits of the mantissa, low: the exact rest; what is not a number stays so through the rest).  A lane's four consecutive head elements of a key are its shares
// of two fragments, its four of a value those of four; the queries' two parts lie in shared memory.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi));
}
__device__ __forceinline__ void mma_1688(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int HS>
__global__ void __launch_bounds__(32 * kTokenWarps, 2)
flash_token32_kernel(const TokenParams p) {
  constexpr int M = HS > 64 ? 1 : 2, KEYS = 8 * M;  // keys per block: as many as the registers hold twice
  extern __shared__ float res[];  // [warp][row][HS + 4], then the queries: [part][row 16][HS + 4]
  __shared__ float mx[kTokenWarps][kTokenRows], sm[kTokenWarps][kTokenRows];
  constexpr int PITCH = HS + 4;
  float* qs = res + kTokenWarps * p.rows * PITCH;
  pdl_wait();
  pdl_launch_dependents();
  TokenLane w(p);
  if (w.nothing(p)) return;
  const int g = w.g, c = w.c, end = w.end;
  for (int at = threadIdx.x; at < kTokenRows * HS; at += 32 * kTokenWarps) {
    const int row = at / HS, h = at % HS;
    float v = 0.f;
    if (row < p.rows && h < p.hs)
      v = static_cast<const float*>(p.q)[h + row % p.tq * p.ldq + (w.kv * p.group + row / p.tq) * p.shq + w.batch * p.sbq];
    uint32_t hi, lo;
    split_tf32(v, hi, lo);
    qs[row * PITCH + h] = __uint_as_float(hi);
    qs[(kTokenRows + row) * PITCH + h] = __uint_as_float(lo);
  }
  __syncthreads();
  float acc[HS / 8][4];
#pragma unroll
  for (int e = 0; e < HS / 8; ++e) acc[e][0] = acc[e][1] = acc[e][2] = acc[e][3] = 0.f;
  const float* kp = static_cast<const float*>(p.k) + w.kv * p.shk + w.batch * p.sbk;
  const float* vp = static_cast<const float*>(p.v) + w.kv * p.shv + w.batch * p.sbv;
  float4 kr[M][HS / 16], vr[HS / 32][2 * M];
  auto load_k = [&](int j) {  // keys j + 8 t + g, head elements 16 s + 4 c ..
#pragma unroll
    for (int t = 0; t < M; ++t)
#pragma unroll
      for (int s = 0; s < HS / 16; ++s) {
        const int key = j + 8 * t + g, h = 16 * s + 4 * c;
        kr[t][s] = load_four(kp + key * p.ldk + h, key < end ? p.hs - h : 0, p.vec_k);
      }
  };
  auto load_v = [&](int j) {  // keys j + 8 t + 2 c and the next, head elements 32 s + 4 g ..
#pragma unroll
    for (int s = 0; s < HS / 32; ++s)
#pragma unroll
      for (int t = 0; t < 2 * M; ++t) {
        const int key = j + 2 * c + (t & 1) + 8 * (t >> 1), h = 32 * s + 4 * g;
        vr[s][t] = load_four(vp + key * p.ldv + h, key < end ? p.hs - h : 0, p.vec_v);
      }
  };
  int j = w.begin + KEYS * w.warp;
  if (j < end) {
    load_k(j);
    load_v(j);
  }
  for (; j < end; j += KEYS * kTokenWarps) {
    float sc[M][4];
#pragma unroll
    for (int t = 0; t < M; ++t) sc[t][0] = sc[t][1] = sc[t][2] = sc[t][3] = 0.f;
#pragma unroll
    for (int s = 0; s < HS / 16; ++s) {
      float4 q[2][2];  // [part][row g, g + 8]: elements 16 s + 4 c ..
#pragma unroll
      for (int part = 0; part < 2; ++part)
#pragma unroll
        for (int x = 0; x < 2; ++x)
          q[part][x] = *reinterpret_cast<const float4*>(qs + (part * kTokenRows + g + 8 * x) * PITCH + 16 * s + 4 * c);
#pragma unroll
      for (int t = 0; t < M; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u) {  // contraction indices c and c + 4: head elements 4 c + 2 u and the next
          uint32_t bh[2], bl[2], a[2][4];
          split_tf32(u ? kr[t][s].z : kr[t][s].x, bh[0], bl[0]);
          split_tf32(u ? kr[t][s].w : kr[t][s].y, bh[1], bl[1]);
#pragma unroll
          for (int part = 0; part < 2; ++part)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              a[part][x] = __float_as_uint(u ? q[part][x].z : q[part][x].x);
              a[part][2 + x] = __float_as_uint(u ? q[part][x].w : q[part][x].y);
            }
          mma_1688(sc[t], a[1][0], a[1][1], a[1][2], a[1][3], bh[0], bh[1]);
          mma_1688(sc[t], a[0][0], a[0][1], a[0][2], a[0][3], bl[0], bl[1]);
          mma_1688(sc[t], a[0][0], a[0][1], a[0][2], a[0][3], bh[0], bh[1]);
        }
    }
    const int next = j + KEYS * kTokenWarps;
    if (next < end) load_k(next);
    w.softmax(p, j, sc, acc);
#pragma unroll
    for (int t = 0; t < M; ++t) {  // keys j + 8 t ..: contraction index c is key 2 c, c + 4 is key 2 c + 1
      uint32_t ph[4], pl[4];       // rows g, g + 8 at key 2 c, then at 2 c + 1
      split_tf32(sc[t][0], ph[0], pl[0]);
      split_tf32(sc[t][2], ph[1], pl[1]);
      split_tf32(sc[t][1], ph[2], pl[2]);
      split_tf32(sc[t][3], ph[3], pl[3]);
#pragma unroll
      for (int s = 0; s < HS / 32; ++s) {
        const float4 v0 = vr[s][2 * t], v1 = vr[s][2 * t + 1];
        const float f0[4] = {v0.x, v0.y, v0.z, v0.w}, f1[4] = {v1.x, v1.y, v1.z, v1.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // head element 32 s + 4 n + e for column n of the fragment
          uint32_t bh[2], bl[2];
          split_tf32(f0[e], bh[0], bl[0]);
          split_tf32(f1[e], bh[1], bl[1]);
          mma_1688(acc[4 * s + e], pl[0], pl[1], pl[2], pl[3], bh[0], bh[1]);
          mma_1688(acc[4 * s + e], ph[0], ph[1], ph[2], ph[3], bl[0], bl[1]);
          mma_1688(acc[4 * s + e], ph[0], ph[1], ph[2], ph[3], bh[0], bh[1]);
        }
      }
    }
    if (next < end) load_v(next);
  }
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int row = g + 8 * x;
    if (row >= p.rows) continue;
    float* to = res + (w.warp * p.rows + row) * PITCH;
#pragma unroll
    for (int s = 0; s < HS / 32; ++s)
#pragma unroll
      for (int k = 0; k < 2; ++k)  // column n = 2 c + k
        *reinterpret_cast<float4*>(to + 32 * s + 4 * (2 * c + k)) =
            make_float4(acc[4 * s][2 * x + k], acc[4 * s + 1][2 * x + k], acc[4 * s + 2][2 * x + k], acc[4 * s + 3][2 * x + k]);
  }
  w.join<HS, float>(p, res, mx, sm);
}

// The splits' results together: one CTA per row of a (sequence, key head).  Every split's weight first, by
// all threads side by side, then the results, four threads to a head element with every fourth split each, joined
// in order.  (Two sequences of 16384 keys have 148 splits each: 60 us with one thread per element walking them, 27
// so.)
constexpr int kJoinParts = 4;
template <int HS, typename T>
__global__ void __launch_bounds__(kJoinParts * HS)
flash_token_join_kernel(const TokenParams p) {
  extern __shared__ float weight[];  // [split]; -1: no keys, its result was not written
  __shared__ float red[2][32], parts[kJoinParts][HS];
  pdl_wait();
  pdl_launch_dependents();
  const long long unit = blockIdx.x / p.rows;
  const int row = static_cast<int>(blockIdx.x % p.rows), h = threadIdx.x % HS, q = threadIdx.x / HS;
  const int batch = static_cast<int>(unit / p.kv_heads), kv = static_cast<int>(unit % p.kv_heads);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = kJoinParts * HS / 32;
  const float2* stat = p.stat + unit * p.splits * p.rows + row;
  float m = -INFINITY;
  for (int s = threadIdx.x; s < p.splits; s += kJoinParts * HS) m = fmaxf(m, stat[static_cast<long long>(s) * p.rows].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) red[0][warp] = m;
  __syncthreads();
  for (int w = 0; w < warps; ++w) m = fmaxf(m, red[0][w]);
  float l = 0.f;
  for (int s = threadIdx.x; s < p.splits; s += kJoinParts * HS) {
    const float2 st = stat[static_cast<long long>(s) * p.rows];
    const float a = st.x == -INFINITY ? (st.y == 0.f ? -1.f : 0.f) : ex2(st.x - m);
    weight[s] = a;
    if (a >= 0.f) l += st.y * a;
    else if (!(a < 0.f)) l = a;  // not a number
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  if (lane == 0) red[1][warp] = l;
  __syncthreads();
  l = 0.f;
  for (int w = 0; w < warps; ++w) l += red[1][w];
  const float* part = p.part + (unit * p.splits * p.rows + row) * HS + h;
  const long long step = static_cast<long long>(p.rows) * HS;
  float v = 0.f;
#pragma unroll 8
  for (int s = q; s < p.splits; s += kJoinParts) {
    const float a = weight[s];
    if (!(a < 0.f)) v += part[s * step] * a;
  }
  parts[q][h] = v;
  __syncthreads();
  if (q != 0) return;
  v = 0.f;
#pragma unroll
  for (int k = 0; k < kJoinParts; ++k) v += parts[k][h];
  token_store<T>(p, batch, kv, row, h, v, m, l);
}

// ---- backward -----------------------------------------------------------------------------------
//
// Two kernels of one shape: a CTA keeps 128 rows of two operands (A1, A2) in shared memory, streams
// tiles of 64 rows of two others (B1, B2), and holds up to two results in tensor memory.
//   rows = keys    : A1 = K, A2 = V, B1 = Q, B2 = dO;  X = K Q^T, Y = V dO^T;
//                    dV += P dO,  dK += dS Q   (over all query heads that share the keys)
//   rows = queries : A1 = Q, A2 = dO, B1 = K, B2 = V;  X = Q K^T, Y = dO V^T;  dQ += dS K,
//                    and the sums of dS by distance for the bias table
// with P = exp(X - lse), dS = P (Y - delta).  X and Y are formed twice in all (seven products instead of
// five), which keeps every sum inside one CTA: no atomics on dQ, the same bits every time.
// Two groups of 256 threads (two per row, 32 columns each) take the streamed tiles in turn; X and Y of
// the next tile are formed while they work.  Tensor memory: per group X (64 columns) and Y (64),
// overwritten by P and dS as fp16 left operands (each thread over the columns it has read); the results
// behind them.
//
// Range: P enters its product times 2^12 (probabilities down to 2^-26 stay normal numbers).  dS
// enters times a power of two that brings its bound 2 max|dO| max|v| (Cauchy-Schwarz, per sequence
// and key head) to 2^14, so neither large nor small upstream gradients leave a Half's range.
//
// What bounds it: the way of a tile from its products through the threads and back.  A streamed tile takes
// about 2800 cycles (16 heads of 4096 x 4096 x 128, causal: keys 185 us for 137 GFLOP, queries 167 us for
// 103, 0.74 and 0.62 PFLOP/s), its four products 1280 of them; two tiles are on that way at a time, and
// tensor memory has no room for a third beside the results.
constexpr int BN = 64;             // rows of a streamed tile
constexpr int BCHUNK = BN * 128;   // bytes of 64 rows x 64 halves
constexpr int kDistSmem = 1024;    // distances whose sums fit in shared memory (per group)

struct FlashBwdParams {
  CUtensorMap tmQ, tmK, tmV, tmDO;      // boxes of 128 rows
  CUtensorMap tmQ64, tmK64, tmV64, tmDO64;
  void *dq, *dk, *dv;
  long long lddq, shdq, sbdq, lddk, shdk, sbdk, lddv, shdv, sbdv;
  const float2* stats;        // [batch][heads][tq_pad]: lse * log2(e) (+inf = empty), delta
  float2* delta;              // the same, for the launch that corrects delta
  const unsigned* norms;      // [2][batch][kv heads]: bits of max |dO|^2, max |v|^2
  float* dist;                // [batch][heads][query tile][2][width] sums of dS by distance; null = not wanted
  const float* bias;
  const float *iq, *ik, *iv, *ido;  // split operands: inverse scales, [batch][kv heads]
  int tq, tk, hs, heads, kv_heads, group, batch, tq_pad, row_tiles, width;
  int vec_dq, vec_dk, vec_dv;       // the results' rows allow 16-byte accesses
  int wait_late;                    // the launch before this one is another of the same pass, see the kernel
  int reach, q_offset;
  const int* q_offsets;
  const int* q_lengths;
  const int* k_lengths;
  float scale, c1;
  int causal, accumulate;
};

// Power of two dS is multiplied with: the bound from the rows' norms or, where their squares leave fp32
// (split operands only), from the largest elements.
template <bool SPLIT>
__device__ __forceinline__ float ds_scale(const FlashBwdParams& p, int unit) {
  float e = 13.f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float q = __uint_as_float(p.norms[i * p.batch * p.kv_heads + unit]);
    if (q > 1e-36f && q < 1e36f) e -= 0.5f * log2f(q);
    else if (SPLIT) e -= 15.f + 3.5f + log2f((i == 0 ? p.ido : p.iv)[unit]);  // 128 elements below 2^15 as scaled
    else return 1.f;
  }
  return exp2f(floorf(fminf(fmaxf(e, -120.f), 120.f)));
}
// delta and lse of every query, and the largest norms of dO and v rows per key head.  Sixteen threads
// per row; a CTA takes 64 rows of one head, of dO (first `qparts` parts) or of v.
__global__ void __launch_bounds__(256)
flash_prepare_kernel(const __half* d_o, long long lddo, long long shdo, long long sbdo, const __half* o, long long ldo,
                     long long sho, long long sbo, const __half* v, long long ldv, long long shv, long long sbv,
                     const float* __restrict__ lse, const FlashBwdParams p, float2* __restrict__ stats,
                     unsigned* __restrict__ norms, int qparts, long long qblocks) {
  __shared__ float red[16];
  pdl_wait();
  pdl_launch_dependents();
  const int sub = threadIdx.x & 15, row16 = threadIdx.x >> 4;
  const bool queries = blockIdx.x < qblocks;
  const long long at = queries ? blockIdx.x : blockIdx.x - qblocks;
  const int parts = queries ? qparts : (p.tk + 63) / 64;
  const int hb = static_cast<int>(at / parts), part = static_cast<int>(at % parts);
  const int heads = queries ? p.heads : p.kv_heads;
  const int batch = hb / heads, head = hb - batch * heads;
  const int kv = queries ? head / p.group : head;
  const int len = queries ? rel_length(p.q_lengths, batch, p.tq) : rel_keys(p, batch);
  const int unit = batch * p.kv_heads + kv;
  auto widen = [&](uint4 w, float (&f)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 q = __half22float2(*reinterpret_cast<const __half2*>(&u[e]));
      f[2 * e] = q.x;
      f[2 * e + 1] = q.y;
    }
  };
  float norm[4], dot[4];
  {
    uint4 wa[4], wb[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {  // all loads before the first sum
      const int i = part * 64 + k * 16 + row16;
      wa[k] = wb[k] = make_uint4(0, 0, 0, 0);
      if (i < len && sub * 8 < p.hs) {
        wa[k] = *reinterpret_cast<const uint4*>(queries ? d_o + i * lddo + head * shdo + batch * sbdo + sub * 8
                                                        : v + i * ldv + head * shv + batch * sbv + sub * 8);
        if (queries) wb[k] = *reinterpret_cast<const uint4*>(o + i * ldo + head * sho + batch * sbo + sub * 8);
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float a[8], b[8];
      widen(wa[k], a);
      widen(wb[k], b);
      norm[k] = dot[k] = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        norm[k] += a[e] * a[e];
        dot[k] += a[e] * b[e];
      }
    }
  }
#pragma unroll
  for (int s = 8; s > 0; s >>= 1)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      norm[k] += __shfl_xor_sync(0xffffffffu, norm[k], s);
      dot[k] += __shfl_xor_sync(0xffffffffu, dot[k], s);
    }
  float most = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    // a row that is not a number or infinite makes the bound so (the integer order puts both last)
    most = __uint_as_float(max(__float_as_uint(most), __float_as_uint(norm[k])));
    const int i = part * 64 + k * 16 + row16;
    if (queries && sub == 0 && i < p.tq_pad) {
      float2 s = make_float2(INFINITY, 0.f);
      if (i < len) {
        const float x = lse[static_cast<long long>(hb) * p.tq + i];
        if (x != -INFINITY) s = make_float2(x * kLog2e, dot[k]);
      }
      stats[static_cast<long long>(hb) * p.tq_pad + i] = s;
    }
  }
  if (sub == 0) red[row16] = most;
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned m = 0;
    for (int k = 0; k < 16; ++k) m = max(m, __float_as_uint(red[k]));
    // a maximum of non-negative floats: the order of the updates does not matter
    atomicMax(norms + (queries ? 0 : p.batch * p.kv_heads) + unit, m);
  }
}

// MODE: what a launch forms.  128-wide split operands leave room in tensor memory for one result (with its
// cross terms) beside X and Y, and in shared memory for one stage: dK and dV are then two launches.
//
// DELTA runs before the others and adds sum_j P (Y - delta) to delta, which is what delta is off by: delta from the
// stored o carries o's rounding for Half and the truncation of o's accumulation for fp32.  A row's score gradients
// add up to zero; what delta is off by, they add up to, and keys with a mean of their own make that an error of dq,
// one that does not average out over the keys.  Relative to the gradient, operands of mean 1, as it is and corrected:
//   Half  dq 1.6e-3 and 3.8e-4 at 64 keys, 3.4e-3 and 3.6e-4 at 512, 9.9e-3 and 3.6e-4 at 4096
//   fp32  dq 2.4e-6 and 1.1e-6 at 64 keys, 4.6e-5 and 1.8e-6 at 256, 1.5e-4 and 2.4e-6 at 512 (plain sums 5.0e-6)
// and the table's gradient, whose terms all but cancel, shows it with operands of mean zero: Half, 2048 keys 4.5e-4
// and 2.2e-4.  So every pass that forms a score gradient takes the two extra products, except fp32 tiles that
// see at most kDeltaSplit keys.  They are a fifth to a third of it (backward pass, as it would be and is: Half 8 x 8 heads of
// 512 x 512 x 64 54 and 72 us, 4 heads of 4096 x 4096 x 64 117 and 159; fp32 256 heads of 256 x 256 x 64 152 and 186).
enum FlashMode { KEYS_BOTH = 0, QUERIES = 1, KEYS_DK = 2, KEYS_DV = 3, DELTA = 4 };
constexpr int kDeltaSplit = 64;

// What a CTA works on: 128 rows of one head of one sequence, and the streamed tiles first .. first + per - 1
// of every query head of the group.
template <int MODE, bool SPLIT>
struct FlashBwdTile {
  int tile, batch, head, kv, r0, qlen, klen, off, first = 0, per = 0;
  __device__ __forceinline__ explicit FlashBwdTile(const FlashBwdParams& p) {
    constexpr bool KEYS = MODE != QUERIES && MODE != DELTA;
    // the CTAs with the most work first: under a causal mask the first keys and the last queries
    const int heads = KEYS ? p.kv_heads : p.heads;
    const int hbs = heads * p.batch, hb = static_cast<int>(blockIdx.x) % hbs;
    tile = KEYS ? static_cast<int>(blockIdx.x) / hbs : p.row_tiles - 1 - static_cast<int>(blockIdx.x) / hbs;
    batch = hb / heads;
    head = hb - batch * heads;
    kv = KEYS ? head : head / p.group;
    r0 = tile * FT;
    qlen = rel_length(p.q_lengths, batch, p.tq);
    klen = rel_keys(p, batch);
    off = rel_offset(p.q_offset, p.q_offsets, batch);
    if (KEYS) {
      if (r0 < klen && qlen > 0) {
        int i = p.causal ? r0 - off : 0;  // the first query that sees key r0
        i = i < 0 ? 0 : i;
        if (i < qlen) {
          first = i / BN;
          per = (qlen + BN - 1) / BN - first;
        }
      }
    } else if (r0 < qlen) {
      const int last = r0 + FT - 1 < qlen - 1 ? r0 + FT - 1 : qlen - 1;
      per = (rel_visible(p.causal, last + off, klen) + BN - 1) / BN;
      if (MODE == DELTA && SPLIT && per <= kDeltaSplit / BN) per = 0;
    }
  }
};

// Number `it` of the streamed tiles as (query head of the group, tile), without a division per tile.
struct StreamWalk {
  int tile, head = 0, per;
  __device__ __forceinline__ StreamWalk(int it, int per_head) : tile(it), per(per_head) { next(0); }
  __device__ __forceinline__ void next(int by) {
    tile += by;
    while (per > 0 && tile >= per) {
      tile -= per;
      ++head;
    }
  }
};

// The launches of one pass behind the first are independent of it: dQ needs nothing of dK and dV.  They begin when
// the CTAs of the one before have all begun (which wait for what both read), fill the SMs that its last wave leaves
// idle, and wait for its end at theirs (wait_late), so that whoever waits for the last launch waits for all.
template <int HS, int MODE, int BSTAGES, bool SPLIT, bool CHAINS>
__global__ void __launch_bounds__(FTHREADS, 1)
flash_backward_kernel(const __grid_constant__ FlashBwdParams p, int* __restrict__ status) {
  constexpr bool KEYS = MODE != QUERIES && MODE != DELTA;
  constexpr bool WANT_P = MODE == KEYS_BOTH || MODE == KEYS_DV, WANT_D = MODE != KEYS_DV;
  constexpr int WIDE = HS / 64;           // 64-wide chunks of a plane
  constexpr int CHUNKS = (SPLIT ? 2 : 1) * WIDE;
  constexpr int PV_COL = MODE == KEYS_BOTH ? (SPLIT ? 2 * HS : HS) : 0;  // tensor memory: dV behind dK
  constexpr int ROWS = FCHUNK * CHUNKS;   // bytes of a resident operand
  constexpr int TILE = BCHUNK * CHUNKS;   // bytes of a streamed tile
  constexpr float PSHIFT = SPLIT ? 14.f : 12.f;  // P is formed times 2^PSHIFT
  constexpr float PINV = SPLIT ? 1.f / 16384.f : 1.f / 4096.f;
  constexpr int CUT = (SPLIT ? kChain : kChainHalf) / BN;  // streamed tiles to a chain
  static_assert(CUT % 2 == 0, "both groups have as many tiles in a chain");
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t rows_full, b_full[BSTAGES], b_empty[BSTAGES], x_full[2], p_full[2], acc_full, acc_empty;
  __shared__ uint32_t tmem_slot;
  __shared__ float window[2][2][256];
  __shared__ __align__(16) float colx[KEYS ? 2 : 1][2][BN], coly[KEYS ? 2 : 1][2][BN];
  __shared__ float diag[KEYS ? 1 : 16][64];
  __shared__ float dist_s[KEYS ? 1 : 2][KEYS ? 1 : kDistSmem];
  __shared__ float far_s[2][2][8];
  __shared__ float delta_s[MODE == DELTA ? 4 : 1][FT];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* base_ptr = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t a1_s = base, a2_s = base + ROWS, b_s = base + 2 * ROWS;  // stage: B1, B2

  if (MODE == DELTA) {  // some of its CTAs have nothing to do
    pdl_wait();
    if (FlashBwdTile<MODE, SPLIT>(p).per == 0) return;
  }
  if (warp == 1) {
    if (lane == 0) {
      mbar_init(smem_u32(&rows_full), 1);
      mbar_init(smem_u32(&acc_full), 1);
      mbar_init(smem_u32(&acc_empty), 512);
      for (int s = 0; s < BSTAGES; ++s) {
        mbar_init(smem_u32(&b_full[s]), 1);
        mbar_init(smem_u32(&b_empty[s]), 1);
      }
      for (int g = 0; g < 2; ++g) {
        mbar_init(smem_u32(&x_full[g]), 1);
        mbar_init(smem_u32(&p_full[g]), 256);
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
  if (!p.wait_late) pdl_wait();
  pdl_launch_dependents();

  const FlashBwdTile<MODE, SPLIT> w(p);
  const int tile = w.tile, batch = w.batch, head = w.head, kv = w.kv, r0 = w.r0, qlen = w.qlen, klen = w.klen;
  const int first = w.first, per = w.per, off = w.off;
  const int n = per * (KEYS ? p.group : 1);

  if (warp == 0) {
    // ===================== TMA producer =====================
    if (n > 0 && elect_one()) {
      mbar_arrive_expect_tx(smem_u32(&rows_full), 2 * ROWS);
      for (int c = 0; c < CHUNKS; ++c) {
        const int x = 64 * (c % WIDE), plane = batch + c / WIDE * p.batch;
        tma_load_4d(a1_s + c * FCHUNK, KEYS ? &p.tmK : &p.tmQ, smem_u32(&rows_full), x, r0, head, plane);
        tma_load_4d(a2_s + c * FCHUNK, KEYS ? &p.tmV : &p.tmDO, smem_u32(&rows_full), x, r0, head, plane);
      }
      StreamWalk walk(0, per);
      for (int it = 0; it < n; ++it, walk.next(1)) {
        const int s = it % BSTAGES;
        if (!mbar_wait(smem_u32(&b_empty[s]), ((it / BSTAGES) & 1) ^ 1u, status, DEV_TIMEOUT_EMPTY, 0xd00)) break;
        const uint32_t bar = smem_u32(&b_full[s]), dst = b_s + s * 2 * TILE;
        const int at = (first + walk.tile) * BN, h = KEYS ? head * p.group + walk.head : kv;
        mbar_arrive_expect_tx(bar, 2 * TILE);
        for (int c = 0; c < CHUNKS; ++c) {
          const int x = 64 * (c % WIDE), plane = batch + c / WIDE * p.batch;
          tma_load_4d(dst + c * BCHUNK, KEYS ? &p.tmQ64 : &p.tmK64, bar, x, at, h, plane);
          tma_load_4d(dst + TILE + c * BCHUNK, KEYS ? &p.tmDO64 : &p.tmV64, bar, x, at, h, plane);
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ===================== MMA issuer =====================
    constexpr uint32_t IDESC_X = make_idesc(0, 0, 0, FT, BN);
    constexpr uint32_t IDESC_ACC = make_idesc(0, 0, 1, FT, HS);
    const bool leader = elect_one();
    const int blen = KEYS ? qlen : klen, bt = KEYS ? p.tq : p.tk;
    bool ok = n == 0 || warp_wait(&rows_full, 0, status, DEV_TIMEOUT_FULL, 0xe00);
    StreamWalk walk(0, per);
    auto scores = [&](int it) {  // called for one tile after the other
      const int s = it % BSTAGES, at = (first + walk.tile) * BN;
      walk.next(1);
      ok = warp_wait(&b_full[s], (it / BSTAGES) & 1, status, DEV_TIMEOUT_FULL, 0xe01);
      if (!ok) return;
      tc_fence_after();
      if (!SPLIT && blen < bt && at + BN > blen) {
        // rows behind the sequence's end may hold anything: the second products meet them with
        // zeros, and so they have to be zero
        uint8_t* stage = base_ptr + (b_s - base) + s * 2 * TILE;
        const int from = blen - at;  // > 0: tiles behind the end are not streamed
        for (int x = lane * 16; x < (BN - from) * 128; x += 512)
          for (int c = 0; c < 2 * CHUNKS; ++c)
            *reinterpret_cast<uint4*>(stage + c * BCHUNK + from * 128 + x) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
      }
      if (leader) {
        const uint32_t b = b_s + s * 2 * TILE, d = tmem + (it & 1) * FT;
#pragma unroll
        for (int y = 0; y < (WANT_D ? 2 : 1); ++y)  // X = A1 B1^T, Y = A2 B2^T
#pragma unroll
          for (int term = 0; term < (SPLIT ? 3 : 1); ++term)
#pragma unroll
            for (int ks = 0; ks < HS / 16; ++ks) {
              const uint32_t aa = (ks / 4) * FCHUNK + (ks % 4) * 32 + (SPLIT && term == 0 ? WIDE * FCHUNK : 0);
              const uint32_t bb = (ks / 4) * BCHUNK + (ks % 4) * 32 + (SPLIT && term == 1 ? WIDE * BCHUNK : 0);
              mma_f16(d + y * BN, make_smem_desc((y ? a2_s : a1_s) + aa, 16, 1024), make_smem_desc(b + y * TILE + bb, 16, 1024),
                      IDESC_X, term > 0 || ks > 0);
            }
        tc_commit(smem_u32(&x_full[it & 1]));
      }
    };
    if (n > 0 && ok) scores(0);
    for (int it = 0; it < n && ok; ++it) {
      const int s = it % BSTAGES, g = it & 1;
      // overwrites P and dS of tile it - 1, whose products are issued; a single stage is still in use
      if (BSTAGES > 1 && it + 1 < n) scores(it + 1);
      ok = ok && warp_wait(&p_full[g], (it >> 1) & 1, status, DEV_TIMEOUT_FULL, 0xe02);
      if (CHAINS && it > 0 && it % CUT == 0)  // the chain before has left its place
        ok = ok && warp_wait(&acc_empty, (it / CUT - 1) & 1, status, DEV_TIMEOUT_EMPTY, 0xe03);
      if (!ok) break;
      tc_fence_after();
      if (leader) {
        const uint32_t b = b_s + s * 2 * TILE, a = tmem + g * FT;
        // the result behind a left operand at `a`, split operands' cross terms beside it
        auto product = [&](uint32_t d, uint32_t left, uint32_t right) {
#pragma unroll
          for (int ks = 0; ks < BN / 16; ++ks) {
            const uint32_t l = left + (ks / 2) * 32 + (ks % 2) * 8, add = ((CHAINS ? it % CUT : it) > 0 || ks > 0) ? 1u : 0u;
            mma_f16_ts(d, l, make_smem_desc(right + ks * 2048, BCHUNK, 1024), IDESC_ACC, add);
            if (SPLIT) {
              mma_f16_ts(d + HS, l, make_smem_desc(right + WIDE * BCHUNK + ks * 2048, BCHUNK, 1024), IDESC_ACC, add);
              mma_f16_ts(d + HS, l + 16, make_smem_desc(right + ks * 2048, BCHUNK, 1024), IDESC_ACC, 1u);
            }
          }
        };
        if (WANT_P) product(tmem + 2 * FT + PV_COL, a, b + TILE);  // dV += P dO
        if (WANT_D && MODE != DELTA) product(tmem + 2 * FT, a + BN, b);  // dK += dS Q,  dQ += dS K
        if (it + BSTAGES < n) tc_commit(smem_u32(&b_empty[s]));  // only where the producer waits for it
        if (it == n - 1 || (CHAINS && (it + 1) % CUT == 0)) tc_commit(smem_u32(&acc_full));
      }
      __syncwarp();
      if (BSTAGES == 1 && it + 1 < n) scores(it + 1);
    }
  } else if (warp >= 4) {
    // ===================== probabilities and their gradient =====================
    // thread: row r, columns 32 half .. 32 half + 31 of every streamed tile of group g
    const int g = (warp - 4) >> 3, half = ((warp - 4) >> 2) & 1;
    const int r = threadIdx.x & 127, gt = (threadIdx.x - 128) & 255;
    const int row = r0 + r;
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t x_col = lanes + g * FT + half * 32, y_col = x_col + BN;
    const int unit = batch * p.kv_heads + kv;
    const float c1 = SPLIT ? p.c1 * p.iq[unit] * p.ik[unit] : p.c1;
    const float up = ds_scale<SPLIT>(p, unit);
    const float f = up * PINV;  // on P, which is formed times 2^PSHIFT
    const float fy = SPLIT ? f * p.iv[unit] * p.ido[unit] : f;
    const bool dist_on = MODE == QUERIES && p.dist != nullptr;
    float2 mine = make_float2(INFINITY, 0.f);
    int vis = 0;
    if (!KEYS && row < p.tq) {
      mine = p.stats[(static_cast<long long>(batch) * p.heads + head) * p.tq_pad + row];
      vis = row < qlen ? rel_visible(p.causal, row + off, klen) : 0;
    }
    const int low = KEYS ? 0 : static_cast<int>(rel_dist_low(p.reach, r0 + FT - 1 + off));
    float* dist = nullptr;
    float far_lo = 0.f, far_hi = 0.f;
    if (dist_on) {
      float* out = p.dist + (((static_cast<long long>(batch) * p.heads + head) * p.row_tiles + tile) * 2 + g) * p.width;
      dist = p.width <= kDistSmem ? dist_s[g] : out;
      for (int e = gt; e < p.width; e += 256) dist[e] = 0.f;
      group_barrier(1 + g);
    }
    bool ok = true;
    StreamWalk walk(g, per);
    // statistics of a streamed query, loaded a tile ahead: the group's barrier waits for them
    auto stat = [&](const StreamWalk& w) {
      return p.stats[(static_cast<long long>(batch) * p.heads + head * p.group + w.head) * p.tq_pad + (first + w.tile) * BN + gt];
    };
    float2 ahead = make_float2(0.f, 0.f);
    if (KEYS && gt < BN && g < n) ahead = stat(walk);
    // What the chains that ended add up to, in local memory (see the forward kernel).
    float part[CHAINS ? HS / 2 : 1];
    int it = g;
    for (int chain = 0;; ++chain) {
      const int stop = CHAINS && n > (chain + 1) * CUT ? (chain + 1) * CUT : n;
      for (; it < stop; it += 2, walk.next(2)) {
        const int at = (first + walk.tile) * BN, turn = (it >> 1) & 1;
        const int h = KEYS ? head * p.group + walk.head : head;
        const float* bias = p.bias != nullptr ? p.bias + static_cast<long long>(h) * (2 * p.reach + 1) : nullptr;
        // distances of the tile's pairs: dlo .. dlo + 190
        const int dlo = KEYS ? r0 - (at + BN - 1 + off) : at - (r0 + FT - 1 + off);
        // one number for the whole tile (a masked score is -inf before it is scaled: c1 > 0), or a window
        const bool beyond = dlo >= p.reach || dlo + FT + BN - 2 <= -p.reach;
        const bool flat = c1 > 0.f && (bias == nullptr || beyond);
        float value = 0.f;
        float* win = window[g][turn];
        if (flat) {
          if (bias != nullptr) value = __ldg(bias + (dlo >= p.reach ? 2 * p.reach : 0));
        } else {
          int d = dlo + gt;
          d = d > p.reach ? p.reach : d < -p.reach ? -p.reach : d;
          win[gt] = bias != nullptr ? __ldg(bias + d + p.reach) : 0.f;
        }
        if (KEYS && gt < BN) {
          // per column: what is added to the scaled score, and to Y times f
          const float2 st = ahead;
          if (it + 2 < n) {
            StreamWalk then = walk;
            then.next(2);
            ahead = stat(then);
          }
          const bool alone = rel_visible(p.causal, at + gt + off, klen) <= 1;
          colx[KEYS ? g : 0][turn][gt] = (flat ? value : 0.f) + PSHIFT - st.x;
          coly[KEYS ? g : 0][turn][gt] = alone ? 0.f : -st.y * f;
        }
        if (KEYS || !flat) group_barrier(1 + g);
        // window[c - r + 127] for query rows, window[r - c + 63] for key rows
        const float* wrow = KEYS ? win + (BN - 1) + r - 32 * half : win + (FT - 1) - r + 32 * half;
        ok = ok && warp_wait(&x_full[g], turn, status, DEV_TIMEOUT_ACCUM, 0xf00 + g);
        // of this thread's columns those from lo to hi - 1 take part
        int lo = 0, hi = 32;
        if (KEYS) {
          hi = row < klen ? 32 : 0;
          if (p.causal) {
            const int from = row - off - at - 32 * half;
            lo = from < 0 ? 0 : from > 32 ? 32 : from;
          }
        } else {
          hi = vis - at - 32 * half;
        }
        const bool sweep = !KEYS && !beyond && p.reach > 0;  // sums along the diagonals
        F2 all(0.f, 0.f);
        if (ok) {
          tc_fence_after();
          const bool alone = !KEYS && vis <= 1;
          const float rx = (flat ? value : 0.f) + PSHIFT - mine.x, ry = alone ? 0.f : -mine.y * f;
          uint32_t x[32], y[32];
          tmem_ld32(x_col, x);
          if (WANT_D) tmem_ld32(y_col, y);
          tmem_ld_wait();
          if (!flat) {  // the window's bias joins the scores here, everything else below
#pragma unroll
            for (int e = 0; e < 32; ++e)
              x[e] = __float_as_uint(fmaf(__uint_as_float(x[e]), c1, KEYS ? wrow[-e] : wrow[e]));
          }
          if (__any_sync(0xffffffffu, lo > 0 || hi < 32)) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (e < lo || e >= hi) {
                x[e] = 0xff800000u;  // -inf
                if (WANT_D) y[e] = 0u;
              }
          }
          // A query that sees one key gives it all its weight whatever the score: dS is zero, not what is
          // left of two roundings.  The first query of a causal sequence, or every one over a single key.
          if (WANT_D && (KEYS ? klen <= 1 || (p.causal && at + off <= 0) : __any_sync(0xffffffffu, alone))) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (KEYS ? klen <= 1 || at + 32 * half + e + off <= 0 : alone) y[e] = 0u;
          }
          const float cx1 = flat ? c1 : 1.f;
          const F2 cx(cx1, cx1), f2(fy, fy);
          uint32_t pw[16], dw[16], plow[16], dlow[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            F2 sx(rx, rx), sy(ry, ry);
            if (KEYS) {
              const float2 ax = *reinterpret_cast<const float2*>(&colx[KEYS ? g : 0][turn][32 * half + e]);
              const float2 ay = *reinterpret_cast<const float2*>(&coly[KEYS ? g : 0][turn][32 * half + e]);
              sx = F2(ax.x, ax.y);
              sy = F2(ay.x, ay.y);
            }
            float p0, p1;
            fma2(F2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), cx, sx).get(p0, p1);
            p0 = ex2(p0);
            p1 = ex2(p1);
            if (WANT_P) {
              if (SPLIT) split_pair(p0, p1, pw[e / 2], plow[e / 2]);
              else pw[e / 2] = pack_half2(p0, p1);
            }
            if (WANT_D) {
              const F2 ds = mul2(F2(p0, p1), fma2(F2(__uint_as_float(y[e]), __uint_as_float(y[e + 1])), f2, sy));
              float d0, d1;
              ds.get(d0, d1);
              if (SPLIT) split_pair(d0, d1, dw[e / 2], dlow[e / 2]);
              else dw[e / 2] = pack_half2(d0, d1);
              if (!KEYS) {
                all = add2(all, ds);
                y[e] = __float_as_uint(d0);
                y[e + 1] = __float_as_uint(d1);
              }
            }
          }
          if (WANT_P) tmem_st16(x_col, pw);
          if (WANT_P && SPLIT) tmem_st16(x_col + 16, plow);
          if (WANT_D && MODE != DELTA) tmem_st16(y_col, dw);
          if (WANT_D && MODE != DELTA && SPLIT) tmem_st16(y_col + 16, dlow);
          tmem_st_wait();
          tc_fence_before();
          mbar_arrive(smem_u32(&p_full[g]));
          if (sweep && dist_on) {
            // the running sum of a diagonal moves down one lane per column; lane 31 ends it
            float run = 0.f;
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              run = __shfl_up_sync(0xffffffffu, run, 1);
              run = (lane == 0 ? 0.f : run) + __uint_as_float(y[e]);
              if (lane == 31) diag[KEYS ? 0 : warp - 4][e] = run;  // diagonal e - 31
            }
            if (lane < 31) diag[KEYS ? 0 : warp - 4][32 + lane] = run;  // diagonal 31 - lane
          }
        }
        if (MODE == DELTA) far_lo += all.sum();
        if (dist_on) {
          if (!sweep) {  // one side of the reach
            float a0, a1;
            all.get(a0, a1);
            if (dlo >= p.reach) far_hi += a0 + a1;
            else far_lo += a0 + a1;
          } else {
            group_barrier(1 + g);
            if (gt < FT + BN - 1) {
              const int w = gt;
              float sum = 0.f;
#pragma unroll
              for (int q = 0; q < 8; ++q) {
                // column - row = w - 127; warp q of the group: rows 32 (q % 4) + lane, columns 32 (q / 4) + e
                const int dg = w - (FT - 1) + 32 * (q & 3) - 32 * (q >> 2);  // e - lane
                if (dg >= -31 && dg <= 31) sum += diag[KEYS ? 0 : g * 8 + q][dg <= 0 ? dg + 31 : 32 + 31 - dg];
              }
              const int d = dlo + w;
              if (d >= p.reach) far_hi += sum;
              else if (d <= -p.reach) far_lo += sum;
              else if (d - low < p.width) dist[d - low] += sum;  // behind the last key: nothing, and no place
            }
            group_barrier(1 + g);
          }
        }
      }
      // ---- results: of two, group 0 writes dK and group 1 dV; a single one's columns are shared ----
      const bool last = !CHAINS || stop == n;
      if (MODE != DELTA && n > 0 && ok) {
        ok = warp_wait(&acc_full, chain & 1, status, DEV_TIMEOUT_ACCUM, 0xf10 + g);
        tc_fence_after();
      }
      using Out = typename std::conditional<SPLIT, float, __half>::type;
      constexpr bool SHARED = MODE != KEYS_BOTH;
      constexpr int COUNT = SHARED ? HS / 4 : HS / 2;                         // columns of this thread
      const bool values = MODE == KEYS_DV || (MODE == KEYS_BOTH && g == 1);  // it writes dV
      const int c_from = SHARED ? (2 * g + half) * COUNT : half * COUNT;
      Out* out = static_cast<Out*>(KEYS ? (values ? p.dv : p.dk) : p.dq);
      if (MODE != DELTA && ok && out != nullptr && (n > 0 || !p.accumulate)) {
        const long long ld = KEYS ? (values ? p.lddv : p.lddk) : p.lddq, sh = KEYS ? (values ? p.shdv : p.shdk) : p.shdq,
                        sb = KEYS ? (values ? p.sbdv : p.sbdk) : p.sbdq;
        const int vec = KEYS ? (values ? p.vec_dv : p.vec_dk) : p.vec_dq;
        const bool real = row < (KEYS ? p.tk : p.tq);
        out += row * ld + head * sh + batch * sb + c_from;
        float factor = values ? PINV : p.scale / up;
        if (SPLIT) factor *= KEYS ? (values ? p.ido[unit] : p.iq[unit]) : p.ik[unit];
        const uint32_t col0 = lanes + 2 * FT + (values ? PV_COL : 0) + c_from;
        auto eight = [&](int c) {
          uint32_t w[8], x[8];
          if (n > 0) {
            tmem_ld8(col0 + c, w);
            if (SPLIT) tmem_ld8(col0 + HS + c, x);
            tmem_ld_wait();
          }
          float res[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            res[e] = n > 0 ? (SPLIT ? __uint_as_float(w[e]) + __uint_as_float(x[e]) : __uint_as_float(w[e])) : 0.f;
            if (CHAINS && chain > 0) res[e] += part[CHAINS ? c + e : 0];
            if (!last) part[CHAINS ? c + e : 0] = res[e];
            res[e] *= factor;
          }
          if (last && real) store_row8(out + c, p.hs - c_from - c, vec, res, p.accumulate != 0);
        };
        if (CHAINS) {
#pragma unroll 1
          for (int c = 0; c < COUNT; c += 8) eight(c);
        } else {
          for (int c = 0; c < COUNT; c += 8) eight(c);
        }
      }
      if (last) break;
      tc_fence_before();
      mbar_arrive(smem_u32(&acc_empty));
    }
    // ---- sums by distance ----
    if (dist_on) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        far_lo += __shfl_xor_sync(0xffffffffu, far_lo, o);
        far_hi += __shfl_xor_sync(0xffffffffu, far_hi, o);
      }
      if (lane == 0) {
        far_s[g][0][(warp - 4) & 7] = far_lo;
        far_s[g][1][(warp - 4) & 7] = far_hi;
      }
      group_barrier(1 + g);
      if (gt == 0) {
        float s[2] = {0.f, 0.f};
        for (int k = 0; k < 16; ++k) s[k >> 3] += far_s[g][k >> 3][k & 7];
        if (-p.reach - low >= 0 && -p.reach - low < p.width) dist[-p.reach - low] += s[0];
        if (p.reach - low >= 0 && p.reach - low < p.width) dist[p.reach - low] += s[1];
      }
      group_barrier(1 + g);
      if (p.width <= kDistSmem) {
        float* out = p.dist + (((static_cast<long long>(batch) * p.heads + head) * p.row_tiles + tile) * 2 + g) * p.width;
        for (int e = gt; e < p.width; e += 256) out[e] = dist[e] * (1.f / up);
      } else {
        for (int e = gt; e < p.width; e += 256) dist[e] *= 1.f / up;
      }
    }
    if (MODE == DELTA) delta_s[2 * g + half][r] = ok ? far_lo / up : 0.f;
  }

  tc_fence_before();
  __syncthreads();
  if (MODE == DELTA && n > 0 && threadIdx.x < FT && r0 + threadIdx.x < qlen) {
    float2* st = p.delta + (static_cast<long long>(batch) * p.heads + head) * p.tq_pad + r0 + threadIdx.x;
    st->y += (delta_s[0][threadIdx.x] + delta_s[1][threadIdx.x]) + (delta_s[2][threadIdx.x] + delta_s[3][threadIdx.x]);
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (p.wait_late) pdl_wait();
}

bool heads_aligned(const FlashOperand& x, long long t, long long heads, long long batch) {
  if ((reinterpret_cast<uintptr_t>(x.p) & 15u) != 0) return false;
  const long long n[3] = {t, heads, batch}, s[3] = {x.ld, x.head, x.batch};
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && (s[i] % 8 != 0 || s[i] <= 0 || s[i] >= (1LL << 38))) return false;
  return true;
}

// Width of the kernels' operand tiles.
int flash_width(int hs) { return hs <= 64 ? 64 : 128; }
// Tensor map of an operand: Half as it lies, or the planes of a split one (twice the sequences).
bool encode_operand(CUtensorMap* map, const FlashOperand& x, int hs, int t, int heads, int batch, int rows, bool split) {
  const long long w = flash_width(hs);
  if (split) return encode_heads_tmap(map, x.planes, static_cast<int>(w), t, heads, 2LL * batch, w, w * t, w * t * heads, rows);
  return encode_heads_tmap(map, x.p, hs, t, heads, batch, x.ld, x.head, x.batch, rows);
}
// Rows allow 16-byte accesses (`n` elements).
int rows16(const FlashOperand& x, int n) {
  return (reinterpret_cast<uintptr_t>(x.p) & 15u) == 0 && x.ld % n == 0 && x.head % n == 0 && x.batch % n == 0;
}

bool fill_params(const FlashArgs& a, FlashParams* p) {
  std::memset(p, 0, sizeof(*p));
  const bool split = a.inverse != nullptr;
  if (!encode_operand(&p->tmQ, a.q, a.hs, a.tq, a.heads, a.batch, FT, split) ||
      !encode_operand(&p->tmK, a.k, a.hs, a.tk, a.kv_heads, a.batch, FT, split) ||
      !encode_operand(&p->tmV, a.v, a.hs, a.tk, a.kv_heads, a.batch, FT, split))
    return false;
  p->O = const_cast<void*>(a.o.p);
  p->vec = rows16(a.o, split ? 4 : 8);
  p->ldo = a.o.ld; p->sho = a.o.head; p->sbo = a.o.batch;
  p->lse = a.lse;
  p->bias = a.bias;
  const long long units = static_cast<long long>(a.batch) * a.kv_heads;
  p->iq = a.inverse; p->ik = a.inverse + units; p->iv = a.inverse + 2 * units;
  p->tq = a.tq; p->tk = a.tk; p->hs = a.hs; p->heads = a.heads; p->kv_heads = a.kv_heads; p->group = a.heads / a.kv_heads;
  p->batch = a.batch;
  p->reach = a.reach; p->q_offset = a.q_offset;
  p->q_offsets = a.q_offsets; p->q_lengths = a.q_lengths; p->k_lengths = a.k_lengths;
  p->c1 = a.scale * kLog2e;
  p->causal = a.causal;
  return true;
}

template <int HS, int NST, int NQ, bool SPLIT, bool CHAINS = false>
cudaError_t forward_hs(FlashParams& p, cudaStream_t stream, int* status) {
  const int smem = (NQ + 2 * NST) * FCHUNK * (SPLIT ? 2 : 1) * (HS / 64) + 1024;
  static unsigned long long smem_set = 0;  // per template instantiation
  auto kern = flash_forward_kernel<HS, NST, NQ, SPLIT, CHAINS>;
  cudaError_t e = set_smem_limit_once(reinterpret_cast<const void*>(kern), smem, &smem_set);
  if (e != cudaSuccess) return e;
  p.qblocks = (p.tq + NQ * FT - 1) / (NQ * FT);
  const long long grid = static_cast<long long>(p.qblocks) * p.heads * p.batch;
  if (grid > 0x7fffffffLL) return cudaErrorInvalidValue;
  return launch_kernel(kern, dim3(static_cast<unsigned>(grid)), dim3(128 + 256 * NQ), smem, stream, pdl_enabled(), p, status);
}

template <int HS, int MODE, int BSTAGES, bool SPLIT, bool CHAINS = false>
cudaError_t backward_hs(const FlashBwdParams& p, cudaStream_t stream, int* status) {
  constexpr bool keys = MODE != QUERIES && MODE != DELTA;
  if constexpr (!CHAINS && MODE != DELTA) {
    const long long tiles = keys ? (p.tq + BN - 1LL) / BN * p.group : (p.tk + BN - 1) / BN;
    if (tiles * BN > (SPLIT ? kChain : kChainHalf)) return backward_hs<HS, MODE, BSTAGES, SPLIT, true>(p, stream, status);
  }
  const int smem = (2 * FCHUNK + BSTAGES * 2 * BCHUNK) * (SPLIT ? 2 : 1) * (HS / 64) + 1024;
  static unsigned long long smem_set = 0;  // per template instantiation
  auto kern = flash_backward_kernel<HS, MODE, BSTAGES, SPLIT, CHAINS>;
  cudaError_t e = set_smem_limit_once(reinterpret_cast<const void*>(kern), smem, &smem_set);
  if (e != cudaSuccess) return e;
  FlashBwdParams q = p;
  q.row_tiles = ((keys ? p.tk : p.tq) + FT - 1) / FT;
  const long long grid = static_cast<long long>(q.row_tiles) * (keys ? p.kv_heads : p.heads) * p.batch;
  return launch_kernel(kern, dim3(static_cast<unsigned>(grid)), dim3(FTHREADS), smem, stream, pdl_enabled(), q, status);
}
template <int MODE>
cudaError_t backward_any(const FlashBwdParams& p, bool split, cudaStream_t stream, int* status) {
  if constexpr (MODE != KEYS_BOTH) {  // wide split operands take two launches instead
    if (split && p.hs > 64) return backward_hs<128, MODE, 1, true>(p, stream, status);
  }
  if (split) return backward_hs<64, MODE, 4, true>(p, stream, status);
  return p.hs <= 64 ? backward_hs<64, MODE, 4, false>(p, stream, status) : backward_hs<128, MODE, 4, false>(p, stream, status);
}

template <int MODE>
cudaError_t backward_wide(const FlashBwdParams& p, bool, cudaStream_t stream, int* status) {
  return backward_hs<128, MODE, 1, true>(p, stream, status);
}

cudaError_t prepare(const FlashArgs& a, const FlashGradArgs& g, const FlashBwdParams& p, float* stats, float* norms, int qparts,
                    cudaStream_t stream) {
  const long long qblocks = static_cast<long long>(qparts) * a.heads * a.batch,
                  blocks = qblocks + static_cast<long long>((a.tk + 63) / 64) * a.kv_heads * a.batch;
  return launch_kernel(flash_prepare_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, pdl_enabled(),
                       static_cast<const __half*>(g.d_o.p), g.d_o.ld, g.d_o.head, g.d_o.batch, static_cast<const __half*>(a.o.p),
                       a.o.ld, a.o.head, a.o.batch, static_cast<const __half*>(a.v.p), a.v.ld, a.v.head, a.v.batch,
                       static_cast<const float*>(a.lse), p, reinterpret_cast<float2*>(stats), reinterpret_cast<unsigned*>(norms),
                       qparts, qblocks);
}

}  // namespace

// Sizes the Half kernels take, wherever the operands lie.
bool flash_fits(const FlashArgs& a) {
  const auto fits = [](long long parts, long long heads, long long batch) { return parts * heads * batch <= 0x3fffffffLL; };
  return tmap_encoder_available() && a.hs <= 128 && fits((a.tq + 127) / 128 * 2, a.heads, a.batch) &&
         fits((a.tk + 63) / 64, a.kv_heads, a.batch);
}

bool flash_supported(const FlashArgs& a) {
  return flash_fits(a) && a.hs % 8 == 0 && heads_aligned(a.q, a.tq, a.heads, a.batch) &&
         heads_aligned(a.k, a.tk, a.kv_heads, a.batch) && heads_aligned(a.v, a.tk, a.kv_heads, a.batch) &&
         heads_aligned(a.o, a.tq, a.heads, a.batch);
}

cudaError_t launch_flash_forward(const FlashArgs& a, cudaStream_t stream, int* status) {
  FlashParams p;
  if (!fill_params(a, &p)) return cudaErrorInvalidValue;
  if (a.inverse != nullptr) {  // 64 wide, two tiles with two stages each: 16 heads of 2048 x 2048, causal, 103 us; one tile 85
    if (a.tk > kChain)
      return a.hs <= 64 ? forward_hs<64, 1, 1, true, true>(p, stream, status) : forward_hs<128, 1, 1, true, true>(p, stream, status);
    return a.hs <= 64 ? forward_hs<64, 1, 1, true>(p, stream, status) : forward_hs<128, 1, 1, true>(p, stream, status);
  }
  const bool chains = a.tk > kChainHalf;
  if (a.hs > 64) return chains ? forward_hs<128, 2, 2, false, true>(p, stream, status) : forward_hs<128, 2, 2, false>(p, stream, status);
  // Half, 64 wide: CTAs of one query tile where their work is uneven or short (16 heads of 2048 x 2048, causal:
  // 42 us with two tiles, 36 with one; 512 of 128 x 128: 25 and 21), of two where every tile walks all keys,
  // which are then read half as often (16 of 2048 x 2048, not causal: 43 and 46).
  if (a.causal || a.tq <= FT)
    return chains ? forward_hs<64, 2, 1, false, true>(p, stream, status) : forward_hs<64, 2, 1, false>(p, stream, status);
  return chains ? forward_hs<64, 3, 2, false, true>(p, stream, status) : forward_hs<64, 3, 2, false>(p, stream, status);
}

long long flash_packed(int hs, long long t, long long heads, long long batch) {
  return (flash_width(hs) * t * heads * batch + 1) / 2;
}

cudaError_t launch_flash_pack(FlashOperand* x, int hs, int t, int heads, int batch, float* to, int num_sms, cudaStream_t stream) {
  const long long rows = static_cast<long long>(t) * heads * batch, want = (rows + 7) / 8, most = 16LL * num_sms;
  const long long w = flash_width(hs);
  const cudaError_t e = launch_kernel(w == 64 ? flash_pack_kernel<64> : flash_pack_kernel<128>,
                                      dim3(static_cast<unsigned>(want < most ? want : most)), dim3(256), 0, stream, pdl_enabled(),
                                      static_cast<const __half*>(x->p), x->ld, x->head, x->batch, hs, t, heads, rows,
                                      reinterpret_cast<__half*>(to));
  x->p = to;
  x->ld = w; x->head = w * t; x->batch = w * t * heads;
  return e;
}

// fp32 through Half planes, at any length: chains keep sums of 8192 values of one sign within 6e-6 (the
// composed path's products 1.9e-5).
bool flash_split_supported(const FlashArgs& a) {
  const long long parts = (a.tq + 63) / 64 + (a.tk + 63) / 64;
  return tmap_encoder_available() && a.hs <= 128 && parts * a.heads * a.batch <= 0x1fffffffLL;
}
long long flash_planes(int hs, long long t, long long heads, long long batch) { return flash_width(hs) * t * heads * batch; }

// work: largest magnitudes of four operands, norms of d_o's and v's rows, inverse scales of four operands.
long long flash_split_work(const FlashArgs& a) { return 10LL * a.batch * a.kv_heads; }
long long flash_split_clear(const FlashArgs& a) { return 6LL * a.batch * a.kv_heads; }

cudaError_t launch_flash_split(FlashArgs* a, FlashOperand* d_o, float* work, float* stats, float** norms, cudaStream_t stream) {
  SplitParams p;
  std::memset(&p, 0, sizeof(p));
  const long long units = static_cast<long long>(a->batch) * a->kv_heads;
  p.extent = {a->tq, a->tk, a->causal, a->q_offset, a->q_offsets, a->q_lengths, a->k_lengths};
  p.count = d_o != nullptr ? 4 : 3;
  p.hs = a->hs; p.batch = a->batch; p.kv_heads = a->kv_heads;
  p.most = reinterpret_cast<unsigned*>(work);
  p.inverse = work + 6 * units;
  a->inverse = p.inverse;
  if (d_o != nullptr) {
    *norms = work + 4 * units;
    p.norms = reinterpret_cast<unsigned*>(*norms);
    p.o = static_cast<const float*>(a->o.p);
    p.ldo = a->o.ld; p.sho = a->o.head; p.sbo = a->o.batch;
    p.vec_o = rows16(a->o, 4);
    p.lse = a->lse;
    p.stats = reinterpret_cast<float2*>(stats);
    p.tq_pad = (a->tq + FT - 1) / FT * FT;
    static_assert(kSplitRows == FT, "the CTAs of d_o cover the padded queries");
  }
  FlashOperand* ops[4] = {&a->q, &a->k, &a->v, d_o};
  long long blocks = 0;
  for (int i = 0; i < p.count; ++i) {
    const bool query = i == 0 || i == 3;
    SplitOperand& o = p.op[i];
    o.x = static_cast<const float*>(ops[i]->p);
    o.ld = ops[i]->ld; o.head = ops[i]->head; o.batch = ops[i]->batch;
    o.planes = static_cast<__half*>(ops[i]->planes);
    o.query = query;
    o.t = query ? a->tq : a->tk;
    o.heads = query ? a->heads : a->kv_heads;
    o.per = query ? a->heads / a->kv_heads : 1;
    o.vec = rows16(*ops[i], 4);
    o.block0 = blocks;
    blocks += static_cast<long long>((o.t + kSplitRows - 1) / kSplitRows) * o.heads * a->batch;
  }
  const bool narrow = a->hs <= 64;
  const cudaError_t e = launch_kernel(narrow ? split_most_kernel<64> : split_most_kernel<128>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream,
                    pdl_enabled(), p);
  if (e != cudaSuccess) return e;
  return launch_kernel(narrow ? split_planes_kernel<64> : split_planes_kernel<128>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, pdl_enabled(), p);
}
int flash_token_splits(int dtype, const FlashArgs& a, int num_sms, long long* floats) {
  const long long rows = static_cast<long long>(a.heads / a.kv_heads) * a.tq;
  *floats = 0;
  if (rows > kTokenRows || a.hs > 128) return 0;
  // Eight CTAs' worth of work per SM, so that ragged lengths even out; a CTA takes at least 64 keys (one
  // block per warp), in multiples of that, and at most a chain, whatever the number of sequences.
  const long long units = static_cast<long long>(a.kv_heads) * a.batch, step = 16 * kTokenWarps;
  long long chunk = (a.tk * units + 8LL * num_sms - 1) / (8LL * num_sms);
  chunk = (chunk + step - 1) / step * step;
  const long long most = dtype == 0 ? kTokenChain : kTokenChainHalf;
  chunk = chunk < most ? chunk : most;
  const long long splits = (a.tk + chunk - 1) / chunk;
  if (splits * units > 0x7fffffffLL || units * rows > 0x7fffffffLL) return 0;
  if (splits > 1) *floats = units * splits * rows * ((a.hs <= 64 ? 64 : 128) + 2);
  return static_cast<int>(splits);
}

cudaError_t launch_flash_token(int dtype, const FlashArgs& a, int splits, float* scratch, int* launches, cudaStream_t stream) {
  TokenParams p;
  std::memset(&p, 0, sizeof(p));
  p.q = a.q.p;
  p.k = a.k.p;
  p.v = a.v.p;
  p.o = const_cast<void*>(a.o.p);
  p.vec_k = rows16(a.k, 4); p.vec_v = rows16(a.v, 4);
  p.ldq = a.q.ld; p.shq = a.q.head; p.sbq = a.q.batch;
  p.ldk = a.k.ld; p.shk = a.k.head; p.sbk = a.k.batch;
  p.ldv = a.v.ld; p.shv = a.v.head; p.sbv = a.v.batch;
  p.ldo = a.o.ld; p.sho = a.o.head; p.sbo = a.o.batch;
  p.lse = a.lse;
  p.bias = a.bias;
  p.tq = a.tq; p.tk = a.tk; p.hs = a.hs; p.heads = a.heads; p.kv_heads = a.kv_heads; p.group = a.heads / a.kv_heads;
  p.batch = a.batch;
  p.rows = p.group * a.tq;
  p.splits = splits;
  const int step = 16 * kTokenWarps;
  p.chunk = static_cast<int>(((a.tk + splits - 1LL) / splits + step - 1) / step * step);
  p.reach = a.reach; p.q_offset = a.q_offset;
  p.q_offsets = a.q_offsets; p.q_lengths = a.q_lengths; p.k_lengths = a.k_lengths;
  p.c1 = a.scale * kLog2e;
  p.causal = a.causal;
  const bool narrow = a.hs <= 64;
  const long long units = static_cast<long long>(a.kv_heads) * a.batch;
  if (splits > 1) {  // pairs first: their alignment does not depend on the head size
    p.stat = reinterpret_cast<float2*>(scratch);
    p.part = scratch + 2 * units * splits * p.rows;
  }
  *launches = 1;
  const bool half = dtype != 0;
  auto kern = half ? (narrow ? flash_token_kernel<64> : flash_token_kernel<128>)
                   : (narrow ? flash_token32_kernel<64> : flash_token32_kernel<128>);
  const int row_bytes = ((narrow ? 64 : 128) + 4) * static_cast<int>(sizeof(float));
  const int queries = half ? 0 : 2 * kTokenRows * row_bytes;
  static unsigned long long smem_set[4] = {};  // per kernel
  cudaError_t e = set_smem_limit_once(reinterpret_cast<const void*>(kern), kTokenRows * kTokenWarps * row_bytes + queries,
                                      &smem_set[half * 2 + narrow]);
  if (e != cudaSuccess) return e;
  e = launch_kernel(kern, dim3(static_cast<unsigned>(units * splits)), dim3(32 * kTokenWarps), p.rows * kTokenWarps * row_bytes + queries,
                    stream, pdl_enabled(), p);
  if (e != cudaSuccess || splits == 1) return e;
  *launches = 2;
  auto join = half ? (narrow ? flash_token_join_kernel<64, __half> : flash_token_join_kernel<128, __half>)
                   : (narrow ? flash_token_join_kernel<64, float> : flash_token_join_kernel<128, float>);
  return launch_kernel(join, dim3(static_cast<unsigned>(units * p.rows)), dim3(kJoinParts * (narrow ? 64 : 128)), splits * sizeof(float), stream,
                       pdl_enabled(), p);
}

bool flash_backward_supported(const FlashArgs& a, const FlashGradArgs& g) {
  return flash_supported(a) && heads_aligned(g.d_o, a.tq, a.heads, a.batch);
}

FlashScratch flash_backward_scratch(const FlashArgs& a, bool table) {
  FlashScratch s;
  const long long rows = static_cast<long long>(a.heads) * a.batch, tiles = (a.tq + FT - 1) / FT;
  s.stats = rows * tiles * FT * 2;
  s.norms = 2LL * a.batch * a.kv_heads;
  s.dist = table ? rows * tiles * 2 * rel_dist_width(a.reach, a.tk, FT) : 0;
  s.sums = table ? (2 * a.reach + 1) * a.heads : 0;
  return s;
}

cudaError_t launch_flash_backward(const FlashArgs& a, const FlashGradArgs& g, float* stats, float* norms, float* dist,
                                  float* sums, int* launches, cudaStream_t stream, int* status) {
  FlashBwdParams p;
  std::memset(&p, 0, sizeof(p));
  const bool split = a.inverse != nullptr;
  const struct {
    CUtensorMap* map;
    const FlashOperand* x;
    int t, heads, rows;
  } maps[] = {{&p.tmQ, &a.q, a.tq, a.heads, FT},   {&p.tmDO, &g.d_o, a.tq, a.heads, FT},
              {&p.tmK, &a.k, a.tk, a.kv_heads, FT}, {&p.tmV, &a.v, a.tk, a.kv_heads, FT},
              {&p.tmQ64, &a.q, a.tq, a.heads, BN},   {&p.tmDO64, &g.d_o, a.tq, a.heads, BN},
              {&p.tmK64, &a.k, a.tk, a.kv_heads, BN}, {&p.tmV64, &a.v, a.tk, a.kv_heads, BN}};
  for (const auto& m : maps)
    if (!encode_operand(m.map, *m.x, a.hs, m.t, m.heads, a.batch, m.rows, split)) return cudaErrorInvalidValue;
  const long long units = static_cast<long long>(a.batch) * a.kv_heads;
  p.iq = a.inverse; p.ik = a.inverse + units; p.iv = a.inverse + 2 * units; p.ido = a.inverse + 3 * units;
  const int per16 = split ? 4 : 8;
  p.vec_dq = rows16(g.dq, per16); p.vec_dk = rows16(g.dk, per16); p.vec_dv = rows16(g.dv, per16);
  p.dq = const_cast<void*>(g.dq.p);
  p.dk = const_cast<void*>(g.dk.p);
  p.dv = const_cast<void*>(g.dv.p);
  p.lddq = g.dq.ld; p.shdq = g.dq.head; p.sbdq = g.dq.batch;
  p.lddk = g.dk.ld; p.shdk = g.dk.head; p.sbdk = g.dk.batch;
  p.lddv = g.dv.ld; p.shdv = g.dv.head; p.sbdv = g.dv.batch;
  p.stats = reinterpret_cast<const float2*>(stats);
  p.norms = reinterpret_cast<const unsigned*>(norms);
  p.dist = dist;
  p.bias = a.bias;
  p.tq = a.tq; p.tk = a.tk; p.hs = a.hs; p.heads = a.heads; p.kv_heads = a.kv_heads; p.group = a.heads / a.kv_heads;
  p.batch = a.batch;
  const int qtiles = (a.tq + FT - 1) / FT;
  p.tq_pad = qtiles * FT;
  p.reach = a.reach; p.q_offset = a.q_offset;
  p.q_offsets = a.q_offsets; p.q_lengths = a.q_lengths; p.k_lengths = a.k_lengths;
  p.scale = a.scale;
  p.c1 = a.scale * kLog2e;
  p.causal = a.causal;
  p.accumulate = g.accumulate;
  p.width = rel_dist_width(a.reach, a.tk, FT);
  cudaError_t e = cudaSuccess;
  *launches = 0;
  if (!split) {  // split operands came with their statistics
    e = prepare(a, g, p, stats, norms, qtiles * 2, stream);
    *launches = 1;
    if (e != cudaSuccess) return e;
  }
  p.delta = reinterpret_cast<float2*>(stats);
  if (!(split && a.tk <= kDeltaSplit) && (p.dk != nullptr || p.dq != nullptr || dist != nullptr)) {
    e = backward_any<DELTA>(p, split, stream, status);
    ++*launches;
    if (e != cudaSuccess) return e;
  }
  const bool wide = split && a.hs > 64;
  auto launch = [&](cudaError_t (*kernel)(const FlashBwdParams&, bool, cudaStream_t, int*)) {
    const cudaError_t e = kernel(p, split, stream, status);
    ++*launches;
    p.wait_late = 1;
    return e;
  };
  if (!wide && (p.dk != nullptr || p.dv != nullptr)) e = launch(backward_any<KEYS_BOTH>);
  if (wide && p.dk != nullptr) e = launch(backward_wide<KEYS_DK>);
  if (e == cudaSuccess && wide && p.dv != nullptr) e = launch(backward_wide<KEYS_DV>);
  if (e == cudaSuccess && (p.dq != nullptr || dist != nullptr)) e = launch(backward_any<QUERIES>);
  if (e != cudaSuccess) return e;
  if (dist == nullptr) return cudaSuccess;
  RelDist d;
  d.dist = dist;
  d.batch = a.batch; d.heads = a.heads; d.tiles = qtiles; d.tile_rows = FT; d.slots = 2; d.width = p.width;
  d.reach = a.reach; d.q_offset = a.q_offset; d.q_offsets = a.q_offsets;
  *launches += 2;
  return launch_rel_table_grad(split ? 0 : 1, d, sums, g.map, g.buckets, g.accumulate, g.dtable, g.lddt, stream);
}

}  // namespace gb
