// Shared description of attention with a relative position bias: which pairs of query and key
// take part, and at which distance.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace gb {

constexpr int kRelDiagonal = 32;  // queries whose sums by distance are formed together

// Scores of `matrices` (sequence, head) pairs from pair number `matrix0` on, queries q0 .. q0 + nq - 1
// of tq: s[matrix][query][ld], keys contiguous.
struct RelScores {
  float* s = nullptr;
  long long ld = 0, matrices = 0, matrix0 = 0;
  int nq = 0, q0 = 0, tq = 0, tk = 0, heads = 1;
  float scale = 1.f;
  int causal = 0;
  long long q_offset = 0;           // position of query 0, in keys
  const int* q_offsets = nullptr;   // per sequence instead
  const int* q_lengths = nullptr;   // queries / keys behind these take no part
  const int* k_lengths = nullptr;
  long long reach = 0;
};

__device__ __forceinline__ int rel_length(const int* lengths, int batch, int t) {
  if (lengths == nullptr) return t;
  const int n = lengths[batch];
  return n < 0 ? 0 : n < t ? n : t;
}
// Offsets are held within +-2^30, whatever the device array says, and tensors end before 2^29: positions and
// distances are ints.
__device__ __forceinline__ int rel_offset(long long offset, const int* offsets, int batch) {
  const int x = offsets != nullptr ? offsets[batch] : static_cast<int>(offset);
  return x > (1 << 30) ? 1 << 30 : x < -(1 << 30) ? -(1 << 30) : x;
}
// Number of keys 0 .. n - 1 the query at position `pos` sees.
__device__ __forceinline__ int rel_visible(int causal, int pos, int klen) {
  if (!causal || pos >= klen - 1) return klen;
  return pos < 0 ? 0 : pos + 1;
}

// Keys 0 .. n - 1 of a sequence that some query sees: under a causal mask those behind the last query's
// position are no more looked at than those behind the length (a cache that is filled so far, say).
template <typename P>
__device__ __forceinline__ int rel_keys(const P& p, int batch) {
  const int klen = rel_length(p.k_lengths, batch, p.tk);
  if (!p.causal) return klen;
  const int last = rel_length(p.q_lengths, batch, p.tq) + rel_offset(p.q_offset, p.q_offsets, batch);
  return last >= klen ? klen : last < 0 ? 0 : last;
}
// What rel_keys reads, for the passes that need nothing else of the attention.
struct RelExtent {
  int tq = 0, tk = 0, causal = 0;
  long long q_offset = 0;
  const int* q_offsets = nullptr;
  const int* q_lengths = nullptr;
  const int* k_lengths = nullptr;
};
__device__ __forceinline__ int rel_rows(const RelExtent& x, bool query, int batch) {
  return query ? rel_length(x.q_lengths, batch, x.tq) : rel_keys(x, batch);
}

// Sums of dS by distance as the backward kernels leave them: dist[sequence][head][tile][slot][width].
struct RelDist {
  const float* dist = nullptr;
  int batch = 0, heads = 0, tiles = 0, tile_rows = 1, slots = 1, width = 0;
  long long reach = 0, q_offset = 0;
  const int* q_offsets = nullptr;
};
// First distance (clamped to the reach) that a tile of queries keeps a sum of; `last`: position of
// its last query.
__device__ __forceinline__ long long rel_dist_low(long long reach, long long last) {
  return -last > reach ? reach : -last > -reach ? -last : -reach;
}
// Distances a tile of `rows` queries can need a sum for.
inline int rel_dist_width(long long reach, long long tk, int rows) {
  const long long w = tk + rows - 1;
  return static_cast<int>(2 * reach + 1 < w ? 2 * reach + 1 : w);
}

// The query of score column `col` of a RelScores.
struct RelQuery {
  long long matrix, local;  // within the scores of this call
  int batch, head, query, visible;
  int pos;                  // its position in keys
  __device__ __forceinline__ RelQuery(const RelScores& s, long long col) {
    matrix = col / s.nq;
    local = col - matrix * s.nq;
    query = s.q0 + static_cast<int>(local);
    batch = static_cast<int>((s.matrix0 + matrix) / s.heads);
    head = static_cast<int>((s.matrix0 + matrix) % s.heads);
    pos = query + rel_offset(s.q_offset, s.q_offsets, batch);
    const int klen = rel_length(s.k_lengths, batch, s.tk);
    visible = query < rel_length(s.q_lengths, batch, s.tq) ? rel_visible(s.causal, pos, klen) : 0;
  }
};

}  // namespace gb
