// Counter-based random masks (Philox4x32-10; J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel
// random numbers: as easy as 1, 2, 3", SC 2011).  A mask is a function of (seed, offset, element
// index) alone, so the backward pass forms it again instead of reading it.
//
// Element e of a rows x cols matrix (e = row + rows * col) belongs to block e / 8: counter words
// (e / 8 mod 2^32, e / 8 div 2^32, offset low, offset high), key words (seed low, seed high).
// The block's four output words are eight 16-bit numbers, low half first; element e takes number
// e % 8 and is kept when it is not below `threshold` = round(65536 p).  Sixteen bits per decision
// halve the generator's work against thirty-two (it would bound a Half dropout otherwise: ten
// rounds of two 32 x 32 -> 64 products for four elements of 4 bytes traffic each); the factor on
// kept elements is 65536 / (65536 - threshold), the exact inverse of the probability used.
#pragma once
#include <stdint.h>

namespace gb {

struct Dropout {
  uint32_t seed_lo = 0, seed_hi = 0;
  unsigned long long offset = 0;
  const unsigned long long* step = nullptr;  // device counter added to `offset`; may be null
  uint32_t threshold = 0;                    // 0: everything is kept
  float factor = 1.f;
};

// The generator of one launch, with the device counter already added.
struct Philox {
  uint32_t k0, k1, c2, c3, threshold;
  __device__ __forceinline__ explicit Philox(const Dropout& d)
      : k0(d.seed_lo), k1(d.seed_hi), threshold(d.threshold) {
    unsigned long long off = d.offset;
    if (d.step != nullptr && d.threshold != 0) off += *d.step;
    c2 = static_cast<uint32_t>(off);
    c3 = static_cast<uint32_t>(off >> 32);
  }
  // The four output words of a block.
  __device__ __forceinline__ uint4 words(unsigned long long block) const {
    uint32_t x0 = static_cast<uint32_t>(block), x1 = static_cast<uint32_t>(block >> 32), x2 = c2, x3 = c3;
    uint32_t a = k0, b = k1;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
      const unsigned long long p0 = static_cast<unsigned long long>(0xD2511F53u) * x0;
      const unsigned long long p1 = static_cast<unsigned long long>(0xCD9E8D57u) * x2;
      x0 = static_cast<uint32_t>(p1 >> 32) ^ x1 ^ a;
      x1 = static_cast<uint32_t>(p1);
      x2 = static_cast<uint32_t>(p0 >> 32) ^ x3 ^ b;
      x3 = static_cast<uint32_t>(p0);
      a += 0x9E3779B9u;
      b += 0xBB67AE85u;
    }
    return make_uint4(x0, x1, x2, x3);
  }
  // x[i] of element 8 * block + i: times `factor` when it is kept, 0 otherwise.  Both halves of a word
  // are compared in its upper sixteen bits.
  __device__ __forceinline__ void drop8(unsigned long long block, float factor, float (&x)[8]) const {
    apply(words(block), factor, x);
  }
  __device__ __forceinline__ void apply(const uint4 r, float factor, float (&x)[8]) const {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w}, limit = threshold << 16;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = (w[i] << 16) >= limit ? x[2 * i] * factor : 0.f;
      x[2 * i + 1] = w[i] >= limit ? x[2 * i + 1] * factor : 0.f;
    }
  }
  // Bit i of the result: element 8 * block + i is kept.
  __device__ __forceinline__ uint32_t keep8(unsigned long long block) const {
    const uint4 r = words(block);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w}, limit = threshold << 16;
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      bits |= ((w[i] << 16) >= limit ? 1u : 0u) << (2 * i);
      bits |= (w[i] >= limit ? 1u : 0u) << (2 * i + 1);
    }
    return bits;
  }
  // Keep bits of the eight elements first + lane + 32 i (i = 0..7) of a warp's 256 consecutive
  // elements, wherever `first` lies in its block.  Each lane forms one block and the 33rd is
  // formed by all, so that an element costs a quarter of a block instead of a whole one; the
  // whole warp calls this.
  __device__ __forceinline__ uint32_t keep_strided(unsigned long long first, int lane) const {
    const unsigned long long b0 = first >> 3;
    const int shift = static_cast<int>(first & 7u);
    const uint32_t mine = keep8(b0 + lane);
    const uint32_t last = shift != 0 ? keep8(b0 + 32) : 0u;  // uniform over the warp
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int at = shift + lane + 32 * i;
      const uint32_t got = __shfl_sync(0xffffffffu, mine, (at >> 3) & 31);
      const uint32_t m = (at >> 3) < 32 ? got : last;
      bits |= ((m >> (at & 7)) & 1u) << i;
    }
    return bits;
  }
};

}  // namespace gb
