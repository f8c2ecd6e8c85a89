// The block selection of a decode step by one wave.
#pragma once
#include "nsa_common.hpp"

namespace nsa {

__device__ __forceinline__ float wave_reduce_max(float v) {
#pragma unroll
  for (int o = 1; o <= 32; o <<= 1) v = fmaxf(v, o == 1 ? dpp_quad_xor1(v) : o == 2 ? dpp_quad_xor2(v) : __shfl_xor(v, o, 64));
  return v;
}
__device__ __forceinline__ float wave_reduce_sum(float v) {
#pragma unroll
  for (int o = 1; o <= 32; o <<= 1) v += o == 1 ? dpp_quad_xor1(v) : o == 2 ? dpp_quad_xor2(v) : __shfl_xor(v, o, 64);
  return v;
}

// Block selection of one row by one wave (NSA.py:693-713, 721: softmax with the extra -1e3 column, the k largest in descending
// order, equal ones lower index first; a slot is live when its probability exceeds 1e-10).  nb <= 2048, k <= min(64, nb).
// Lane l holds entries l, l + 64, ...  The k-th largest of the 64 lanes' maxima (a bitwise search with ballots: 31 steps) is a
// lower bound of the k-th largest entry that only a few entries beyond the k reach; those are listed in LDS, a lane takes
// one and counts the listed ones that come before it: its slot.  (Extracting maxima one by one, k dependent rounds of a wave
// maximum and a re-scan: 16 us for 8 rows of 512 with k = 16.)  sel[slot] = block, or -1 for a dead slot.
__device__ __forceinline__ void wave_topk(const float* __restrict__ row, int nb, int k, int lane, float* __restrict__ cand_p, int* __restrict__ cand_j,
                                          int* __restrict__ sel, int* __restrict__ idx_out, unsigned char* __restrict__ fm_out) {
  const int vpl = (nb + 63) >> 6;
  float x[32];
  float mx = -1e3f;
#pragma unroll
  for (int c = 0; c < 32; c += 8) {
    if (c >= vpl) continue;                               // wave-uniform
#pragma unroll
    for (int r = c; r < c + 8; ++r) x[r] = r * 64 + lane < nb ? row[r * 64 + lane] : -INFINITY;
  }
#pragma unroll
  for (int c = 0; c < 32; c += 8) {
    if (c >= vpl) continue;
#pragma unroll
    for (int r = c; r < c + 8; ++r) mx = fmaxf(mx, x[r]);
  }
  mx = wave_reduce_max(mx);
  float sum = 0.f;
#pragma unroll
  for (int c = 0; c < 32; c += 8) {
    if (c >= vpl) continue;
#pragma unroll
    for (int r = c; r < c + 8; ++r) { x[r] = __expf(x[r] - mx); sum += x[r]; }
  }
  sum = wave_reduce_sum(sum) + __expf(-1e3f - mx);
  const float inv = 1.0f / sum;
  int top = 0;                                             // probabilities as integers: same order, padding negative
#pragma unroll
  for (int c = 0; c < 32; c += 8) {
    if (c >= vpl) continue;
#pragma unroll
    for (int r = c; r < c + 8; ++r) {
      float p = x[r] * inv;
      p = (p == p) ? p : INFINITY;                         // NaN (a diverged row): ordered first, like torch.topk
      p = r * 64 + lane < nb ? p : -1.0f;
      x[r] = p;
      top = max(top, __builtin_bit_cast(int, p));
    }
  }
  int T = 0;
  for (int bit = 30; bit >= 0; --bit) {
    const int c = T | (1 << bit);
    if ((int)__popcll(__ballot(top >= c)) >= k) T = c;
  }
  auto count = [&](int v) {                                // entries >= v
    int n = 0;
#pragma unroll
    for (int c = 0; c < 32; c += 8) {
      if (c >= vpl) continue;
#pragma unroll
      for (int r = c; r < c + 8; ++r) n += (int)__popcll(__ballot(__builtin_bit_cast(int, x[r]) >= v));
    }
    return n;
  };
  int ties = 64;                                           // entries equal to T that are listed
  if (count(T) > 64) {                                     // (many equal entries, or the k largest in few lanes: the exact k-th largest)
    T = 0;
    for (int bit = 30; bit >= 0; --bit) {
      const int c = T | (1 << bit);
      if (count(c) >= k) T = c;
    }
    ties = k - count(T + 1);
  }
  int listed = 0;
  const unsigned long long below = (1ull << lane) - 1;
#pragma unroll
  for (int c = 0; c < 32; c += 8) {
    if (c >= vpl) continue;
#pragma unroll
    for (int r = c; r < c + 8; ++r) {
      const int v = __builtin_bit_cast(int, x[r]);
      const unsigned long long eq = __ballot(v == T);
      const bool keep = v > T || (v == T && (int)__popcll(eq & below) < ties);
      const unsigned long long kept = __ballot(keep);
      const int at = listed + (int)__popcll(kept & below);
      if (keep && at < 64) { cand_p[at] = x[r]; cand_j[at] = r * 64 + lane; }
      listed += (int)__popcll(kept);
      ties -= (int)__popcll(eq);
    }
  }
  __builtin_amdgcn_wave_barrier();                         // LDS operations of one wave execute in order
  listed = min(listed, 64);
  const float p = lane < listed ? cand_p[lane] : -1.0f;
  const int j = lane < listed ? cand_j[lane] : 0;
  int rank = 0;
  for (int i = 0; i < listed; ++i) {
    const float pi = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, p), i));
    rank += (pi > p) | ((pi == p) & (i < lane));           // the list is in index order
  }
  if (lane < listed && rank < k) {
    const bool live = p < INFINITY && p > 1e-10f;
    sel[rank] = live ? j : -1;
    if (idx_out != nullptr) { idx_out[rank] = j; fm_out[rank] = live ? 1 : 0; }
  }
}

}  // namespace nsa
