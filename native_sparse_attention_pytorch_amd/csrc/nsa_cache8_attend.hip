// One token of each sequence attends the 8-bit key / value cache: all its keys, its newest ones, or selected blocks of them and its own.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(scale log2(e) q . k_j - m),  v_j and k_j code times scale
//
// HBM-bound: a row of the cache is read once for all query heads of its kv head, 2 D bytes against 4 D G operations.  What is there to be arranged is
// that nothing between the loads and the matrix cores waits: every wave works by itself, with its own running maximum and sum, on tiles of 32 keys,
// and nothing passes through LDS on the way.
//   S^T = K Q^T  (16x16x32, keys as rows, the query heads as columns): a lane holds 16 consecutive codes of a key's row.  Which features the matrix
//     core takes as its k-th ones is free as long as K and Q agree, so a row's 16 bytes become two operands as they lie.
//   O^T = V^T P^T: the scores of four consecutive keys that a lane holds, of two tiles of 16, are the operand that the second product wants.  Of V a lane
//     holds D / 16 consecutive features of those eight keys: bytes are transposed four by four (v_perm) and converted in pairs.
// Codes become bf16 exactly; a key's scale goes into the conversion, a value's into its probability, both powers of two.  Queries are sums of bf16
// parts (one of bf16, two of fp16, three of fp32: exact), probabilities of two (three for fp32 results): 2^-17 (2^-24) of each.  At 16 columns
// the matrix cores have the time for it: they are busy for up to 12 % of the times below.  Two parts for results of 16 bits: of 32768 in bf16 some 47 then round the other
// way than with exact probabilities, with three some 11, which 17 tiles of 64 features do not get for nothing (10.3 us instead of 9.9; 32768 keys 20.2 instead of 20.0).
//
// Measured in a trace (this kernel, then the merge of the shares; a copy reaches 4.7 TB/s): one sequence of 524287 keys, 16 heads on 2 of 128 features, 51.1 us
// (5.3 TB/s) and 5.8; of 32768 keys, 32 heads on 8, 16.5 us (4.1 TB/s) and 4.0; 48 sequences of 1 to 16384 keys, 38.7 us (4.4 TB/s) and 4.8; 16 blocks of 64 keys
// and the newest of 32 sequences, 16 heads on 4 of 64 features, 10.0 us, and of one sequence, 32 heads on 8 of 128, 11.2 us: a few CUs have it all, and one
// takes 64 KB in 1.4 us, by eight waves or by sixteen (the same within 0.2 us).
// More than 16 query heads of a kv head are two groups of columns, each converted for by waves of its own: 26 sequences of 3 to 9339 keys, 4 kv heads, take
// 30 us with 32 query heads each and 23 with 16.
#include <type_traits>

#include "nsa_cache8.hpp"
#include "nsa_decode_topk.hpp"

namespace nsa {

struct Attend8Args {
  Cache8Args c;
  const void* q;
  long q0, q1;
  int g, units, gc;                    // units: kv heads, or query heads that have blocks of their own; gc: query heads of a unit
  int window, sel_block, num_sel, idx64, per_block;      // per_block: sel_block / 16
  const void* idx;
  const uint8_t* fmask;
  float scale;
  int block_shift;
  int batch;
  int shared;                          // work-groups share the tiles of all units, else each has a unit
  int most;                            // tiles of a unit at most
  float* part;                         // shared: two records for each work-group, [gc][D] sums, [gc] maxima, [gc] weights, rec floats each
  int groups;                          // work-groups of the first launch
  int parts, per, records;             // else: of a unit, tiles of each; records: leave one for each part
  const int* compressed;               // keys cached so far, of which num_sel is not more than ... / per_compressed, where they are known to the device
  int per_compressed, most_compressed;
  const float* pooled;                 // logits of the blocks, from which the work-group makes its unit's selection itself
  long pooled_stride;
  int rec, table;                      // table: where in LDS the sequences' first tiles are, in bytes
  void* out;
};

typedef __attribute__((__vector_size__(2 * sizeof(float)))) float floatx2;

constexpr int kTile = 32, kTable = 2048, kListed = 64;      // kTable: sequences of a launch; kListed: tiles whose rows are in LDS
// see Shares.  kUnit: of 4, 48 ragged sequences take 55 us instead of 47; of 12, 48.  kShare: of 16, 57 to 125 tiles of 8 units take 12.0 to 13.6 us instead of
// 10.1 to 10.5
constexpr int kUnit = 8, kShare = 4;
// Tiles of a unit up to which it has a work-group for itself and no merge follows.  us alone / shared, replayed from a graph and, in brackets, as calls: of 128 features
// and scales of 32 rows, 34 tiles of 8 units 11.5 / 10.4 (11.2 / 15.4), 50 tiles 14.4 / 10.4 (13.7 / 15.1), 42 of 64 units 14.1 / 14.8 (13.1 / 14.8), 50 tiles 15.8 / 15.3
// (14.7 / 14.9); of 64 features, 50 of 16 units 11.6 / 9.6 (11.1 / 14.9); 41 of 512 units of lengths from 10 keys on 14.3 / 21.4 (13.1 / 20.2), 91 tiles 23.3 / 25.2 (22.1 /
// 23.8), 125 tiles 30.5 / 28.4 (29.4 / 27.0).  With few units the kernels alone would be shared from 34 tiles on; a call has a second launch and a workspace more then.
__host__ inline int alone_up_to(long units) { return units >= 256 ? 96 : 50; }

__device__ __forceinline__ floatx4 mfma16(bf16x8 a, bf16x8 b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// maximum / sum over the lanes l, l ^ 16, l ^ 32, l ^ 48 (as swap_halves: inline assembly with its wait states)
__device__ __forceinline__ void swap_quarters(float& a, float& b) { asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b)); }
__device__ __forceinline__ float quarters_max(float v) {
  v = halves_max(v);
  float a = v, b = v;
  swap_quarters(a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float quarters_sum(float v) {
  v = halves_sum(v);
  float a = v, b = v;
  swap_quarters(a, b);
  return a + b;
}

// the keys of a unit: places 0 .. places - 1, each with a row of the cache or none
struct Keys8 {
  int len, first, base, places;
};
__device__ __forceinline__ Keys8 keys_of(const Attend8Args& A, int len) {
  Keys8 K;
  K.len = len;
  K.first = A.window > 0 && A.sel_block == 0 ? max(0, K.len - A.window) : 0;
  K.base = K.first & ~15;
  K.places = A.sel_block > 0 ? (K.len > 0 ? (A.num_sel + 1) * A.sel_block : 0) : K.len - K.base;
  return K;
}
__device__ __forceinline__ int tiles_of(const Attend8Args& A, int b) { return (keys_of(A, cache8_length(A.c, b)).places + kTile - 1) / kTile; }
// the row of a place of a selection; without one ~ of the newest key's, which is attended: what is there may be read in its place
__device__ __forceinline__ int selected_row(const Attend8Args& A, const Keys8& K, long unit, int place, int filled, const int* sel) {
  const int none = ~max(K.len - 1, 0);
  if (place >= K.places) return none;
  const int slot = place / A.sel_block, own = (K.len - 1) / A.sel_block;
  long blk = own;
  if (slot < A.num_sel) {
    if (slot >= filled) return none;
    if (sel != nullptr) {
      blk = sel[slot];
    } else {
      const long e = unit * A.num_sel + slot;
      const uint8_t live = A.fmask[e];
      blk = A.idx64 ? reinterpret_cast<const long*>(A.idx)[e] : (long)reinterpret_cast<const int*>(A.idx)[e];
      blk = live != 0 ? blk : -1;
    }
    if (blk < 0 || blk > own) return none;
  }
  const long row = blk * A.sel_block + (place - slot * A.sel_block);
  return row < K.len ? (int)row : none;
}

template <class T>
struct Parts8;
template <> struct Parts8<__bf16> { static constexpr int Q = 1, P = 2; };
template <> struct Parts8<_Float16> { static constexpr int Q = 2, P = 2; };
template <> struct Parts8<float> { static constexpr int Q = 3, P = 3; };

// x as the sum of N bf16 values
template <int N>
__device__ __forceinline__ void split_parts(const float (&x)[8], bf16x8 (&to)[N]) {
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    float r0 = x[e], r1 = x[e + 1];
#pragma unroll
    for (int p = 0; p < N; ++p) {
      const bf16x2 h = __builtin_convertvector((floatx2{r0, r1}), bf16x2);      // (as one instruction)
      const uint32_t w = __builtin_bit_cast(uint32_t, h);
      to[p][e] = h[0];
      to[p][e + 1] = h[1];
      r0 -= __builtin_bit_cast(float, w << 16);
      r1 -= __builtin_bit_cast(float, w & 0xffff0000u);
    }
  }
}

// eight codes as bf16 times `scale`, a power of two
__device__ __forceinline__ bf16x8 bf16_of_codes(uint32_t lo, uint32_t hi, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// bytes of four words: word i of the result holds byte i of each
__device__ __forceinline__ void transpose_bytes(const uint32_t (&d)[4], uint32_t (&t)[4]) {
  // v_perm(hi, lo, sel): bytes 0 .. 3 are lo's, 4 .. 7 hi's
  const uint32_t a = __builtin_amdgcn_perm(d[1], d[0], 0x05010400u), b = __builtin_amdgcn_perm(d[1], d[0], 0x07030602u);
  const uint32_t c = __builtin_amdgcn_perm(d[3], d[2], 0x05010400u), e = __builtin_amdgcn_perm(d[3], d[2], 0x07030602u);
  t[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
  t[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
  t[2] = __builtin_amdgcn_perm(e, b, 0x05040100u);
  t[3] = __builtin_amdgcn_perm(e, b, 0x07060302u);
}

// Where a unit's keys are: a range of rows; selected blocks of a multiple of 16 keys; selected blocks of any size.
enum { kRange = 0, kBlocks = 1, kPacked = 2 };

// a float at an address that is the same in all lanes, through the scalar cache: it waits for no other load
__device__ __forceinline__ float of_all(const float* p) {
  return *reinterpret_cast<const __attribute__((address_space(4))) float*>(reinterpret_cast<uintptr_t>(p));
}

template <int D>
struct Tile8 {                         // what a lane holds of 32 keys
  uintx4 k[2][D / 64];                 // key n of each 16: 16 codes
  typedef __attribute__((__vector_size__(D / 16))) uint32_t words;
  words v[2][4];                       // keys 4 q + e: D / 16 codes
  float ks[2], vs[2];                  // ks: of key n.  vs: one for all 16 keys (kPacked reads them from LDS where it needs them)
};

// a value that is the same in all lanes, for the compiler too
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ long uniform(long x) { return (long)((unsigned long)(unsigned)uniform((int)(x >> 32)) << 32 | (unsigned)uniform((int)x)); }

// n / d of n below 2^50, the same in all lanes: by the division of doubles, put right where that is rounded up (one of 64-bit integers takes 150 instructions)
__device__ __forceinline__ long quotient(long n, long d) {
  long q = (long)((double)n / (double)d);
  q -= q * d > n;
  return uniform(q + (n - q * d >= d));
}

// Shared tiles.  A sequence's tiles are as many as its length has, known to the device only.  All units lie one after the other on a line, each as long as its
// tiles and kUnit more (what a unit costs besides them), and the line is cut into equal shares, one for each work-group, whatever the lengths are.  A unit whose
// tiles lie in one share is finished there; of the others each share leaves a record, and the merge finds them by the same arithmetic.  (Parts of a fixed
// size for each unit, sized for the capacity: 48 sequences of 1 to 16384 keys took 105 us where these take 48; most work-groups had nothing to do,
// and a few too much.)
struct Shares {
  long total, share;                   // the line's length, a work-group's part of it
  __device__ __forceinline__ void set(long all, int groups) {
    total = all;
    share = max(quotient(all + groups - 1, groups), (long)kShare);
  }
};

// slots of a selection that are filled
__device__ __forceinline__ int filled_slots(const Attend8Args& A) {
  return A.compressed == nullptr ? A.num_sel : min(A.num_sel, min(max(A.compressed[0], 0), A.most_compressed) / A.per_compressed);
}

__device__ __forceinline__ long length_on_line(long tiles) { return tiles > 0 ? tiles + kUnit : 0; }

// where the sequences' first units begin, in units' lengths before each, into `first` (batch + 1 of them); a sequence without tiles takes none
template <int NT>
__device__ __forceinline__ void first_tiles(const Attend8Args& A, long* first) {
  __shared__ long sum_s[NT / 64];
  const int tid = threadIdx.x, each = (A.batch + NT - 1) / NT, b0 = min(A.batch, tid * each), b1 = min(A.batch, b0 + each);
  long mine = 0;
  for (int b = b0; b < b1; ++b) mine += length_on_line(tiles_of(A, b));
  long up = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const long x = __shfl_up(up, o, 64);
    if ((tid & 63) >= o) up += x;
  }
  if ((tid & 63) == 63) sum_s[tid >> 6] = up;
  __syncthreads();
  long at = up - mine;
  for (int w = 0; w < (tid >> 6); ++w) at += sum_s[w];
  for (int b = b0; b < b1; ++b) {
    first[b] = at;
    at += length_on_line(tiles_of(A, b));
  }
  if (b1 == A.batch && b0 < b1) first[A.batch] = at;
  __syncthreads();
}
// all sequences have as many tiles
__device__ __forceinline__ bool alike(const Attend8Args& A) { return A.sel_block > 0 || A.c.lengths == nullptr || A.c.length_stride == 0; }

// A work-group: SHARED, its share of all units' tiles; else the unit, or the part of one, that is its own.  CHOOSE: it selects the blocks itself, into sel_s (64
// of them, and 128 words besides).
template <class T, int D, int MODE, int kWaves, bool SHARED, bool CHOOSE = false>
__device__ __forceinline__ void attend8_body(const Attend8Args& A, const int group_id, const int groups_all, char* lds, int* sel_s = nullptr) {
  constexpr int QP = Parts8<T>::Q, PP = Parts8<T>::P, KS = D / 32, DT = D / 16;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15, q4 = lane >> 4;
  // (the length of a sequence without keys counts for a selection: no tile of it has any)
  long pos = 0, end = 0, each = 0;
  Shares all;
  const long* first = reinterpret_cast<const long*>(lds + A.table);
  if constexpr (SHARED) {
    if (alike(A)) {
      each = uniform(length_on_line(A.sel_block > 0 ? A.most : tiles_of(A, 0)));
      all.set(each * A.batch * A.units, groups_all);
    } else {
      first_tiles<64 * kWaves>(A, const_cast<long*>(first));
      all.set(uniform(first[A.batch]) * A.units, groups_all);
    }
    pos = group_id * all.share;
    end = min(all.total, pos + all.share);
    if (pos >= end) return;
  }
  int seq = -1;
  do {
  int b, u, t0, t1, tiles;
  if constexpr (SHARED) {
    long at, length = each;            // of the unit that `pos` lies in: where it begins, how long it is
    if (each > 0) {
      const long unit = quotient(pos, each);
      b = (int)unit / A.units;
      u = (int)unit - b * A.units;
      at = unit * each;
    } else {
      if (seq < 0) {                   // the last sequence that begins here or before
        int lo = 0, hi = A.batch - 1;
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (uniform(first[mid]) * A.units <= pos) lo = mid;
          else hi = mid - 1;
        }
        seq = lo;
      } else {
        while (uniform(first[seq + 1]) * A.units <= pos) ++seq;
      }
      b = seq;
      const long before = uniform(first[b]);
      length = uniform(first[b + 1]) - before;
      u = (int)quotient(pos - before * A.units, length);
      at = before * A.units + u * length;
    }
    tiles = (int)(length - kUnit);
    t0 = (int)max(0L, pos - at - kUnit);
    t1 = (int)min((long)tiles, end - at - kUnit);
    pos = at + length;
    if (t0 >= t1) continue;            // (its tiles are all in the next share)
  } else {
    const int own = group_id / A.parts;
    b = own / A.units;
    u = own - b * A.units;
    t0 = (group_id - own * A.parts) * A.per;
    t1 = min(A.most, t0 + A.per);
    tiles = A.records ? -1 : A.most;
  }
  const bool whole_unit = t0 == 0 && t1 == tiles;
  const long unit = (long)b * A.units + u;
  const int hk = A.units == A.c.hk ? u : u / A.g, head0 = A.units == A.c.hk ? u * A.g : u;

  // more than 16 query heads: half of the waves for the first 16
  const int groups = A.gc > 16 ? 2 : 1, nw = kWaves / groups, group = wave / nw, w0 = wave - group * nw;
  const int cols = min(16, A.gc - 16 * group);

  bf16x8 Q[KS][QP];
  {
    const T* qp = reinterpret_cast<const T*>(A.q) + b * A.q0 + (long)(head0 + 16 * group + min(n, cols - 1)) * A.q1;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      typedef __attribute__((__vector_size__(8 * sizeof(T)))) T vec;
      const vec x = *reinterpret_cast<const vec*>(qp + 16 * (q4 + 4 * (s >> 1)) + 8 * (s & 1));
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = n < cols ? (float)x[e] : 0.f;
      split_parts(f, Q[s]);
    }
  }

  const Keys8 K = keys_of(A, uniform(cache8_length(A.c, b)));
  const int last = K.len - 1;
  if constexpr (MODE == kRange) t1 = min(t1, (K.places + kTile - 1) / kTile);

  const float sc = A.scale * kLog2e;
  const uint8_t* kb = A.c.keys + b * A.c.s0 + hk * A.c.s1;
  const uint8_t* vb = A.c.values + b * A.c.s0 + hk * A.c.s1;
  const float* kz = A.c.key_scales + b * A.c.z0 + hk * A.c.z1;
  const float* vz = A.c.value_scales + b * A.c.z0 + hk * A.c.z1;
  const long s2 = A.c.s2;
  const uint32_t k_lane = 16 * q4, v_lane = DT * n;

  int* row_s = reinterpret_cast<int*>(lds);
  float* ks_s = reinterpret_cast<float*>(lds) + kListed * kTile;
  float* vs_s = ks_s + kListed * kTile;

  float m = -INFINITY, l = 0.f;
  floatx4 O[DT];
#pragma unroll
  for (int c = 0; c < DT; ++c) O[c] = floatx4{0.f, 0.f, 0.f, 0.f};

  const int filled = MODE == kRange ? 0 : filled_slots(A);
  if constexpr (CHOOSE) {
    if (filled > 0) {                  // (at most 64)
      const int blocks = min(max(A.compressed[0], 0), A.most_compressed) / A.per_compressed;
      if (wave == 0) wave_topk(A.pooled + unit * A.pooled_stride, blocks, filled, lane, reinterpret_cast<float*>(sel_s + 64), sel_s + 128, sel_s, nullptr, nullptr);
      __syncthreads();
    }
  }
  // tiles c0 .. c1 - 1 at a time: as many as there are lanes, or room in LDS, for where their rows are
  const int chunk = MODE == kBlocks ? 32 * nw : MODE == kPacked ? kListed : t1 - t0;
  int c0 = t0, lane_row = -1;
  // the first row of the 16 keys i of the wave's tile r, -1: there is none
  auto row0 = [&](int r, int i) {
    if constexpr (MODE == kBlocks) return __builtin_amdgcn_readlane(lane_row, 2 * r + i);
    const int x = K.base + (c0 + w0 + r * nw) * kTile + 16 * i;
    return x <= last ? x : -1;
  };
  auto there = [&](int r0, int x) { return (r0 >= 0) & (x >= K.first) & (x <= last); };
  auto whole = [&](int r0) { return r0 >= K.first && r0 + 15 <= last; };
  // Of 16 keys that begin with row r0 and may not all be there: key x is read where it is or, in its place, the nearest that is (the newest where none is).
  // Addresses are one for the wave and 32 bits of a lane's own.
  auto beyond = [&](int r0, int x) { return r0 < 0 ? 0u : (uint32_t)((min(max(r0 + x, K.first), last) - r0) * s2); };
  using words = typename Tile8<D>::words;
  auto load_k = [&](int r, Tile8<D>& X) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (MODE == kPacked) {
        const int at = (w0 + r * nw) * kTile + 16 * i + n, x = row_s[at];
        X.ks[i] = ks_s[at];
        const uint8_t* p = kb + (long)(x ^ (x >> 31)) * s2 + k_lane;
#pragma unroll
        for (int j = 0; j < D / 64; ++j) X.k[i][j] = *reinterpret_cast<const uintx4*>(p + 64 * j);
      } else {
        const int r0 = row0(r, i), rb = r0 < 0 ? last : r0;
        X.ks[i] = of_all(kz + (rb >> A.block_shift));
        const uint8_t* p = kb + rb * s2;
        const uint32_t off = (whole(r0) ? n * (uint32_t)s2 : beyond(r0, n)) + k_lane;
#pragma unroll
        for (int j = 0; j < D / 64; ++j) X.k[i][j] = *reinterpret_cast<const uintx4*>(p + 64 * j + off);
      }
    }
  };
  auto load_v = [&](int r, Tile8<D>& X) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (MODE == kPacked) {
        const intx4 rv = *reinterpret_cast<const intx4*>(row_s + (w0 + r * nw) * kTile + 16 * i + 4 * q4);
#pragma unroll
        for (int e = 0; e < 4; ++e) X.v[i][e] = *reinterpret_cast<const words*>(vb + (long)(rv[e] ^ (rv[e] >> 31)) * s2 + v_lane);
      } else {
        const int r0 = row0(r, i), rb = r0 < 0 ? last : r0;
        X.vs[i] = of_all(vz + (rb >> A.block_shift));
        const uint8_t* p = vb + rb * s2;
        if (whole(r0)) {
          const uint32_t off = 4 * q4 * (uint32_t)s2 + v_lane;
#pragma unroll
          for (int e = 0; e < 4; ++e) X.v[i][e] = *reinterpret_cast<const words*>(p + e * s2 + off);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) X.v[i][e] = *reinterpret_cast<const words*>(p + (beyond(r0, 4 * q4 + e) + v_lane));
        }
      }
    }
  };

  float s[8];
  auto scores = [&](int r, const Tile8<D>& X) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      floatx4 S = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < D / 64; ++j) {
        const bf16x8 k0 = bf16_of_codes(X.k[i][j][0], X.k[i][j][1], X.ks[i]), k1 = bf16_of_codes(X.k[i][j][2], X.k[i][j][3], X.ks[i]);
#pragma unroll
        for (int p = QP - 1; p >= 0; --p) {      // (small parts first)
          S = mfma16(k0, Q[2 * j][p], S);
          S = mfma16(k1, Q[2 * j + 1][p], S);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) s[4 * i + e] = S[e] * sc;
      if constexpr (MODE == kPacked) {
        const intx4 rv = *reinterpret_cast<const intx4*>(row_s + (w0 + r * nw) * kTile + 16 * i + 4 * q4);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[4 * i + e] = rv[e] >= 0 ? s[4 * i + e] : -INFINITY;
      } else {
        const int r0 = row0(r, i);
        if (!whole(r0)) {
#pragma unroll
          for (int e = 0; e < 4; ++e) s[4 * i + e] = there(r0, r0 + 4 * q4 + e) ? s[4 * i + e] : -INFINITY;
        }
      }
    }
  };
  auto probabilities = [&](int r, const Tile8<D>& X, bf16x8 (&P)[PP]) {
    float mx = s[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) mx = fmaxf(mx, s[e]);
    mx = quarters_max(mx);
    if (__any(mx > m)) {                         // (a NaN raises no maximum: it reaches the sum by itself)
      const float mn = fmaxf(m, mx), by = m == -INFINITY ? 0.f : fast_exp2(m - mn);
      m = mn;
      l *= by;
#pragma unroll
      for (int c = 0; c < DT; ++c) O[c] *= by;
    }
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      floatx4 v;
      if constexpr (MODE == kPacked) v = *reinterpret_cast<const floatx4*>(vs_s + (w0 + r * nw) * kTile + 16 * i + 4 * q4);
      else v = floatx4{X.vs[i], X.vs[i], X.vs[i], X.vs[i]};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = fast_exp2(s[4 * i + e] - ref);
        l += p;
        s[4 * i + e] = p * v[e];
      }
    }
    split_parts(s, P);
  };
  auto products = [&](const Tile8<D>& X, const bf16x8 (&P)[PP]) {
#pragma unroll
    for (int j = 0; j < D / 64; ++j) {
      uint32_t tr[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t d[4] = {X.v[i][0][j], X.v[i][1][j], X.v[i][2][j], X.v[i][3][j]};
        transpose_bytes(d, tr[i]);
      }
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        const bf16x8 V = bf16_of_codes(tr[0][f], tr[1][f], 1.0f);
#pragma unroll
        for (int p = PP - 1; p >= 0; --p) O[4 * j + f] = mfma16(V, P[p], O[4 * j + f]);
      }
    }
  };

  // the wave's tiles; those of a selection whose blocks are not there are passed over.  The next tile's keys are asked for as soon as this one's
  // are operands, its values likewise: one set of registers (with two, and loads a tile further ahead, 32768 keys take 21.9 us instead of 20.8, 524287 72
  // instead of 67, 17 blocks of 64 12.9 instead of 12.1)
  for (; c0 < t1; c0 += chunk) {
    const int c1 = min(t1, c0 + chunk), rounds = c0 + w0 < c1 ? (c1 - c0 - w0 + nw - 1) / nw : 0;
    if constexpr (MODE == kBlocks) {
      // lane 2 r + i: keys 16 i .. 16 i + 15 of tile c0 + w0 + r nw
      const int at = 2 * (c0 + w0 + (lane >> 1) * nw) + (lane & 1), slot = at / A.per_block;
      long blk = -1;
      if (slot < filled) {
        if constexpr (CHOOSE) {
          blk = sel_s[slot];
        } else {
          const long e = unit * A.num_sel + slot;
          const uint8_t live = A.fmask[e];
          blk = A.idx64 ? reinterpret_cast<const long*>(A.idx)[e] : (long)reinterpret_cast<const int*>(A.idx)[e];
          blk = live != 0 && blk >= 0 && blk < 1L << 30 ? blk : -1;
        }
      } else if (slot == A.num_sel && last >= 0) {
        blk = last / A.sel_block;      // the newest key's
      }
      const long x = blk * A.sel_block + 16 * (at - slot * A.per_block);
      lane_row = blk < 0 || x > last ? -1 : (int)x;
    } else if constexpr (MODE == kPacked) {
      if (c0 > t0) __syncthreads();
      for (int i = tid; i < (c1 - c0) * kTile; i += 64 * kWaves) {
        const int r = selected_row(A, K, unit, c0 * kTile + i, filled, CHOOSE ? sel_s : nullptr), at = (r ^ (r >> 31)) >> A.block_shift;
        row_s[i] = r;
        ks_s[i] = kz[at];
        vs_s[i] = vz[at];
      }
      __syncthreads();
    }
    auto next = [&](int r) {
      if constexpr (MODE == kBlocks) {
        while (r < rounds && row0(r, 0) < 0 && row0(r, 1) < 0) ++r;
      } else if constexpr (MODE == kPacked) {
        while (r < rounds && !__any(row_s[(w0 + r * nw) * kTile + (lane & 31)] >= 0)) ++r;
      }
      return r;
    };
    Tile8<D> X;
    bf16x8 P[PP];
    int r = next(0);
    if (r < rounds) {
      load_k(r, X);
      load_v(r, X);
      // (the last tile by itself: a load that may be there or not is one that the compiler can only wait for together with all others)
      for (int rn = next(r + 1); rn < rounds; rn = next(r + 1)) {
        scores(r, X);
        load_k(rn, X);
        probabilities(r, X, P);
        products(X, P);
        load_v(rn, X);
        r = rn;
      }
      scores(r, X);
      probabilities(r, X, P);
      products(X, P);
    }
  }
  l = quarters_sum(l);

  // The waves' results as one, weighted by their maxima, by whoever sums them: all of a head's are asked for at once.  NW: waves of a group of columns; X: of four
  // quarters of a lane's features, how many go through LDS at a time.
  if constexpr (MODE == kPacked) __syncthreads();          // (the lists of rows are read no more)
  float* m_s = reinterpret_cast<float*>(lds);
  float* l_s = m_s + kWaves * 16;
  float* o_s = l_s + kWaves * 16;                // [wave][cols of a group][RO]
  const int most = min(16, A.gc);
  if (q4 == 0) { m_s[wave * 16 + n] = m; l_s[wave * 16 + n] = l; }
  auto merge = [&](auto nw_, auto x_) {
    constexpr int NW = decltype(nw_)::value, X = decltype(x_)::value, H = D * X / 4, RO = H + 4;
#pragma unroll
    for (int part = 0; part < 4 / X; ++part) {
      // (place f of a part: feature DT (4 (f / X DT) + X part) + f % X DT)
      if (n < cols) {
        float* o = o_s + (wave * most + n) * RO + X * DT * q4;
#pragma unroll
        for (int i = 0; i < X; ++i)
#pragma unroll
          for (int c = 0; c < DT; c += 4) {
            const int x = X * part + i;
            *reinterpret_cast<floatx4*>(o + DT * i + c) = floatx4{O[c][x], O[c + 1][x], O[c + 2][x], O[c + 3][x]};
          }
      }
      __syncthreads();
      for (int i = tid; i < A.gc * (H / 4); i += 64 * kWaves) {
        const int g = i / (H / 4), at = i % (H / 4) * 4, w0 = (g >> 4) * NW, c = g & 15, f = DT * (4 * (at / (X * DT)) + X * part) + at % (X * DT);
        float mw[NW], lw[NW], M = -INFINITY, L = 0.f;
        floatx4 ow[NW], o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          mw[w] = m_s[(w0 + w) * 16 + c];
          lw[w] = l_s[(w0 + w) * 16 + c];
          ow[w] = *reinterpret_cast<const floatx4*>(o_s + ((w0 + w) * most + c) * RO + at);
          M = fmaxf(M, mw[w]);
        }
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          const float by = mw[w] == -INFINITY ? 0.f : fast_exp2(mw[w] - M);
          L += mw[w] == -INFINITY ? lw[w] : by * lw[w];    // (a NaN that raised no maximum)
          o += ow[w] * by;
        }
        if (whole_unit) {
          typedef __attribute__((__vector_size__(4 * sizeof(T)))) T vec;
          *reinterpret_cast<vec*>(reinterpret_cast<T*>(A.out) + ((long)b * A.c.hk * A.g + head0 + g) * D + f) =
              L == 0.f ? vec{(T)0.f, (T)0.f, (T)0.f, (T)0.f} : vec{(T)(o[0] / L), (T)(o[1] / L), (T)(o[2] / L), (T)(o[3] / L)};
        } else {
          float* rec = A.part + (SHARED ? 2L * group_id + (t0 == 0) : group_id) * A.rec;
          *reinterpret_cast<floatx4*>(rec + g * D + f) = o;
          if (f == 0) {
            rec[A.gc * D + g] = M;
            rec[A.gc * D + A.gc + g] = L;
          }
        }
      }
      if (part + 1 < 4 / X) __syncthreads();
    }
  };
  if (groups == 1 && A.gc <= 8) merge(std::integral_constant<int, kWaves>{}, std::integral_constant<int, 4>{});
  else if (groups == 1) merge(std::integral_constant<int, kWaves>{}, std::integral_constant<int, 2>{});
  else merge(std::integral_constant<int, kWaves / 2>{}, std::integral_constant<int, 2>{});
  if (pos < end) __syncthreads();      // (LDS is used again)
  } while (pos < end);
}

// (shared tiles of 64 features: registers for the four work-groups of a CU that are launched; fp32, 20000 keys of 8 sequences 28.4 -> 26.7 us)
template <class T, int D, int MODE, int W, bool SHARED>
__global__ __launch_bounds__(64 * W, SHARED && D == 64 && W == 4 ? 4 : 1) void cache8_attend_kernel(const Attend8Args A) {
  extern __shared__ __align__(16) char lds[];
  attend8_body<T, D, MODE, W, SHARED>(A, blockIdx.x, gridDim.x, lds);
}

// The sliding window and the selected blocks of a step in one launch: neither waits for the other.
template <int D, int MODE, bool CHOOSE>
__global__ __launch_bounds__(512) void cache8_step_kernel(const Attend8Args S, const Attend8Args F, const int groups) {
  extern __shared__ __align__(16) char lds[];
  __shared__ int sel_s[192];
  // (the blocks' work-groups first: choosing comes before their attention)
  const int later = gridDim.x - groups;
  if ((int)blockIdx.x < later) attend8_body<__bf16, D, MODE, 8, false, CHOOSE>(F, blockIdx.x, later, lds, sel_s);
  else attend8_body<__bf16, D, kRange, 8, false>(S, blockIdx.x - later, groups, lds);
}

// the parts of a head, weighted by their maxima
template <class T, int D, int kMerge>
__global__ __launch_bounds__(kMerge) void cache8_merge_kernel(const Attend8Args A) {
  constexpr int LPP = D / 4, PPR = kMerge / LPP;
  __shared__ __align__(16) float acc_s[PPR][D];
  __shared__ float m_s[PPR], l_s[PPR];
  const int tid = threadIdx.x, heads = A.c.hk * A.g;
  const long bh = blockIdx.x;
  const int b = (int)(bh / heads), head = (int)(bh % heads);
  const int u = A.units == A.c.hk ? head / A.g : head, gi = A.units == A.c.hk ? head % A.g : 0;
  extern __shared__ __align__(16) char lds[];
  Shares all;
  long at, length;
  if (alike(A)) {
    length = length_on_line(A.sel_block > 0 ? A.most : tiles_of(A, b));
    all.set(length * A.batch * A.units, A.groups);
    at = ((long)b * A.units + u) * length;
  } else {
    long* first = reinterpret_cast<long*>(lds);
    first_tiles<kMerge>(A, first);
    all.set(first[A.batch] * A.units, A.groups);
    length = first[b + 1] - first[b];
    at = first[b] * A.units + u * length;
  }
  T* out = reinterpret_cast<T*>(A.out) + bh * D;
  if (length == 0) {
    if (tid < D) out[tid] = (T)0.f;
    return;
  }
  const long g0 = quotient(at + kUnit, all.share), g1 = quotient(at + length - 1, all.share);
  if (g0 == g1) return;                // finished by its work-group
  // a share has a record of the unit that it begins inside of and one of the unit that begins in it
  const int parts = (int)(g1 - g0) + 1;
  const float* base = A.part + 2 * g0 * A.rec;
  auto record = [&](int p) { return base + (2L * p + (p == 0)) * A.rec; };
  const int om = A.gc * D + gi, f = 4 * (tid % LPP);
  floatx4 acc = {0.f, 0.f, 0.f, 0.f};
  float M = -INFINITY, L = 0.f;
  for (int p0 = tid / LPP; p0 < parts; p0 += 4 * PPR) {
    float mp[4], lp[4];
    floatx4 o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int p = p0 + i * PPR;
      mp[i] = -INFINITY; lp[i] = 0.f; o[i] = floatx4{0.f, 0.f, 0.f, 0.f};
      if (p < parts) {
        const float* rec = record(p);
        mp[i] = rec[om]; lp[i] = rec[om + A.gc];
        o[i] = *reinterpret_cast<const floatx4*>(rec + gi * D + f);
      }
    }
    const float mn = fmaxf(fmaxf(fmaxf(mp[0], mp[1]), fmaxf(mp[2], mp[3])), M), by = M == -INFINITY ? 1.f : fast_exp2(M - mn);
    M = mn;
    L *= by;
    acc *= by;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float w = mp[i] == -INFINITY ? 1.f : fast_exp2(mp[i] - mn);      // (without a maximum there is nothing, or a NaN)
      L += w * lp[i];
      acc += w * o[i];
    }
  }
  *reinterpret_cast<floatx4*>(&acc_s[tid / LPP][f]) = acc;
  if (tid % LPP == 0) { m_s[tid / LPP] = M; l_s[tid / LPP] = L; }
  __syncthreads();
  if (tid < D) {
    float o = 0.f, l = 0.f, top = -INFINITY;
#pragma unroll
    for (int r = 0; r < PPR; ++r) top = fmaxf(top, m_s[r]);
#pragma unroll
    for (int r = 0; r < PPR; ++r) {
      const float w = m_s[r] == -INFINITY ? 1.f : fast_exp2(m_s[r] - top);
      o += w * acc_s[r][tid];
      l += w * l_s[r];
    }
    out[tid] = (T)(l == 0.f ? 0.f : o / l);
  }
}

// units, parts and records of a call
static int attend8_plan(const nsa_cache8_desc* d, Attend8Args& A, size_t& bytes) {
  if (!cache8_check(d) || d->group <= 0 || d->window < 0 || d->sel_block < 0 || d->num_sel < 0) return NSA_E_ARG;
  if (!cache8_supported(d) || d->group > 32 || d->num_sel > 1 << 20 || ((long)d->num_sel + 1) * d->sel_block >= 1L << 30 || d->kv_stride[2] >= 1L << 28)
    return NSA_E_UNSUPPORTED;
  const bool per_head = d->sel_block > 0 && d->per_head_sel;
  A.g = d->group;
  A.units = per_head ? d->kv_heads * d->group : d->kv_heads;
  A.gc = per_head ? 1 : d->group;
  A.rec = A.gc * d->dim_head + ((2 * A.gc + 3) & ~3);
  A.block_shift = __builtin_ctz(d->block);
  const long units = (long)d->batch * A.units;
  long places = d->sel_block > 0 ? ((long)d->num_sel + 1) * d->sel_block : d->capacity;
  if (d->sel_block == 0 && d->window > 0 && d->window + 15L < places) places = d->window + 15L;
  const long tiles = (places + kTile - 1) / kTile;
  if ((long)d->batch * d->kv_heads * d->group >= 1L << 23) return NSA_E_UNSUPPORTED;
  A.most = (int)tiles;
  A.shared = tiles > alone_up_to(units);
  // (work-groups of a CU: with three of 128 features 32768 keys take 22.8 us instead of 20.8, 48 ragged sequences 49.5 instead of 48; five of 64 the same)
  const int resident = d->dim_head == 64 ? 4 : 2;
  // (and of a unit 256, whose records are merged: with 512, 131072 keys of one kv head take 21.0 us instead of 18.3)
  long most = ((tiles + kUnit) * (units < 1L << 20 ? units : 1L << 20) + kShare - 1) / kShare;
  most = most < 256 * resident ? most : 256 * resident;
  A.groups = A.shared ? (int)(most < 256 * units ? most : 256 * units) : 0;
  bytes = A.shared ? 2 * (size_t)A.groups * A.rec * sizeof(float) : 0;
  return 0;
}

// bytes of LDS besides the table of first tiles
template <int D>
static int attend8_lds(const Attend8Args& A, int waves, bool lists) {
  const int cols = A.gc < 16 ? A.gc : 16, merge = (waves * 32 + waves * cols * ((cols <= 8 ? D : D / 2) + 4)) * 4, rows = lists ? kListed * kTile * 12 : 0;
  return ((merge > rows ? merge : rows) + 15) / 16 * 16;
}

template <class T, int D, int MODE, int W, bool SHARED>
static void attend8_mode(const Attend8Args& A, hipStream_t st) {
  Attend8Args B = A;
  B.table = attend8_lds<D>(A, W, MODE == kPacked);
  B.parts = 1; B.per = A.most;
  const int table = SHARED && A.sel_block == 0 && A.c.lengths && A.c.length_stride ? (A.batch + 1) * 8 : 0;
  const dim3 grid((unsigned)(SHARED ? A.groups : A.batch * A.units));
  hipLaunchKernelGGL((cache8_attend_kernel<T, D, MODE, W, SHARED>), grid, dim3(64 * W), B.table + table, st, B);
  if (!SHARED) return;
  // few heads have many parts each; of many heads, most are finished, and a work-group finds out no more than that
  const unsigned heads = (unsigned)(A.batch * A.c.hk * A.g);
  if (heads <= 128) hipLaunchKernelGGL((cache8_merge_kernel<T, D, 512>), dim3(heads), dim3(512), table, st, B);
  else hipLaunchKernelGGL((cache8_merge_kernel<T, D, 128>), dim3(heads), dim3(128), table, st, B);
}

template <class T, int D>
static int attend8_launch(const Attend8Args& A, hipStream_t st) {
  // (the first tiles of a launch's sequences lie in LDS)
  for (int b = 0; b < A.batch; b += kTable) {
    Attend8Args B = A;
    B.batch = A.batch - b < kTable ? A.batch - b : kTable;
    B.q = reinterpret_cast<const T*>(A.q) + b * A.q0;
    B.out = reinterpret_cast<T*>(A.out) + (long)b * A.c.hk * A.g * D;
    B.c.keys += b * A.c.s0; B.c.values += b * A.c.s0; B.c.key_scales += b * A.c.z0; B.c.value_scales += b * A.c.z0;
    if (A.c.lengths) B.c.lengths += (long)b * A.c.length_stride;
    const long rows = (long)b * A.units * A.num_sel;
    if (A.idx) B.idx = A.idx64 ? (const void*)(reinterpret_cast<const long*>(A.idx) + rows) : (const void*)(reinterpret_cast<const int*>(A.idx) + rows);
    if (A.fmask) B.fmask += rows;
    // Work-groups of two waves where a unit has not tiles enough for eight, or the chip not room: it holds one of eight on a CU with 128 features, two with 64.
    // us with eight / two: 3 tiles of 800 units 18.6 / 8.7, 10 of 320 14.9 / 12.8, 10 of 640 21.4 / 13.7, 32 of 640 44 / 41; 43 of 296 17 / 28, 79 of 256 37 / 63.
    const int units = B.batch * A.units, slots = D == 64 ? 512 : 256;
    const bool few = A.most <= 4 || (units > slots && A.most <= 12) || units > 2 * slots;
    if (A.sel_block == 0) {
      if (A.shared) attend8_mode<T, D, kRange, 4, true>(B, st);
      else if (few) attend8_mode<T, D, kRange, 2, false>(B, st);
      else attend8_mode<T, D, kRange, 8, false>(B, st);
    } else if (A.sel_block % 16 == 0) {
      if (A.shared) attend8_mode<T, D, kBlocks, 4, true>(B, st);
      else if (few) attend8_mode<T, D, kBlocks, 2, false>(B, st);
      else attend8_mode<T, D, kBlocks, 8, false>(B, st);
    } else {
      if (A.shared) attend8_mode<T, D, kPacked, 8, true>(B, st);
      else attend8_mode<T, D, kPacked, 8, false>(B, st);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  return 0;
}

// ------------------------------------------------------------------------------------------------------------
// The window and the blocks of a step, as records: parts of eight tiles, one for each wave, while the chip has room for them.
static void step8_branches(const Step8& s, Attend8Args& S, Attend8Args& F) {
  const nsa_cache8_desc* d = s.d;
  auto branch = [&](Attend8Args& A, bool per_head, long places) {
    A.batch = d->batch; A.g = d->group;
    A.units = per_head ? d->kv_heads * d->group : d->kv_heads;
    A.gc = per_head ? 1 : d->group;
    A.rec = A.gc * d->dim_head + ((2 * A.gc + 3) & ~3);
    A.most = (int)((places + kTile - 1) / kTile);
    const long units = (long)d->batch * A.units;
    int per = 8;
    while (per < A.most && (A.most + per - 1) / per * units > 512) per += 8;
    while ((A.most + per - 1) / per > 128) per += 8;      // (records that the merge takes)
    A.per = per; A.parts = (A.most + per - 1) / per; A.records = 1;
    A.block_shift = __builtin_ctz(d->block);
    A.scale = d->scale;
  };
  const long window = (long)s.window + 15 < d->capacity ? s.window + 15L : d->capacity;
  branch(S, false, window);
  S.window = s.window;
  branch(F, s.per_head, ((long)s.num_sel + 1) * s.sel_block);
  F.sel_block = s.sel_block; F.num_sel = s.num_sel; F.per_block = s.sel_block / 16;
}

void cache8_step_parts(const Step8& s, int parts[2], int rec[2]) {
  Attend8Args S{}, F{};
  step8_branches(s, S, F);
  parts[0] = S.parts; parts[1] = F.parts; rec[0] = S.rec; rec[1] = F.rec;
}

template <int D>
static void step8_launch(const Attend8Args& S, const Attend8Args& F, hipStream_t st) {
  const int a = attend8_lds<D>(S, 8, false), b = attend8_lds<D>(F, 8, F.sel_block % 16 != 0);
  const int groups = S.batch * S.units * S.parts, all = groups + F.batch * F.units * F.parts;
  const unsigned bytes = a > b ? a : b;
  const dim3 grid((unsigned)all), block(512);
  const bool blocks = F.sel_block % 16 == 0;
  if (blocks && F.pooled) hipLaunchKernelGGL((cache8_step_kernel<D, kBlocks, true>), grid, block, bytes, st, S, F, groups);
  else if (blocks) hipLaunchKernelGGL((cache8_step_kernel<D, kBlocks, false>), grid, block, bytes, st, S, F, groups);
  else if (F.pooled) hipLaunchKernelGGL((cache8_step_kernel<D, kPacked, true>), grid, block, bytes, st, S, F, groups);
  else hipLaunchKernelGGL((cache8_step_kernel<D, kPacked, false>), grid, block, bytes, st, S, F, groups);
}

int cache8_step_attend(const Step8& s, const void* rq, const int32_t* idx, const uint8_t* fmask, const float* pooled, long pooled_stride,
                       float* window_records, float* block_records, void* stream) {
  const nsa_cache8_desc* d = s.d;
  Attend8Args S{}, F{};
  step8_branches(s, S, F);
  for (Attend8Args* A : {&S, &F}) {
    A->c = cache8_args(d, s.keys, s.values, s.key_scales, s.value_scales, s.state);
    A->c.length = 1;                   // the new token is in the cache
    A->c.length_stride = 0;
    A->c.cap = s.rows;
    A->q = rq; A->q0 = (long)d->kv_heads * d->group * d->dim_head; A->q1 = d->dim_head;
  }
  S.part = window_records;
  F.part = block_records;
  F.idx = idx; F.fmask = fmask; F.pooled = pooled; F.pooled_stride = pooled_stride;
  F.compressed = s.state + 1; F.per_compressed = s.per_block; F.most_compressed = s.compressed;
  if (d->dim_head == 64) step8_launch<64>(S, F, (hipStream_t)stream);
  else step8_launch<128>(S, F, (hipStream_t)stream);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : (int)e;
}

}  // namespace nsa

extern "C" int nsa_cache8_workspace_bytes(const nsa_cache8_desc* d, size_t* bytes) {
  nsa::Attend8Args A{};
  if (!bytes) return NSA_E_ARG;
  return nsa::attend8_plan(d, A, *bytes);
}

extern "C" int nsa_cache8_attend(const nsa_cache8_desc* d, const void* q, const void* keys, const void* values, const float* key_scales,
                                 const float* value_scales, const int32_t* lengths, const void* idx, const uint8_t* fmask, void* ws, size_t ws_bytes,
                                 void* out, void* stream) {
  using namespace nsa;
  Attend8Args A{};
  size_t need = 0;
  if (int e = attend8_plan(d, A, need)) return e;
  if (!q || !keys || !values || !key_scales || !value_scales || !out || ((uintptr_t)keys | (uintptr_t)values | (uintptr_t)q) % 16) return NSA_E_ARG;
  if ((d->q_stride[0] | d->q_stride[1]) & 7) return NSA_E_ARG;
  if (d->sel_block > 0 && d->num_sel > 0 && (!idx || !fmask)) return NSA_E_ARG;
  if (need > 0 && (!ws || (uintptr_t)ws % 16)) return NSA_E_ARG;
  if (ws_bytes < need) return NSA_E_WORKSPACE;
  A.c = cache8_args(d, keys, values, key_scales, value_scales, lengths);
  A.q = q; A.q0 = d->q_stride[0]; A.q1 = d->q_stride[1];
  A.window = d->window; A.sel_block = d->sel_block; A.num_sel = d->num_sel; A.idx64 = d->idx_is_int64; A.per_block = d->sel_block / 16;
  A.idx = idx; A.fmask = fmask; A.scale = d->scale; A.part = (float*)ws; A.out = out;
  A.batch = d->batch;
  hipStream_t st = (hipStream_t)stream;
  if (d->dim_head == 64)
    return d->dtype == 0 ? attend8_launch<__bf16, 64>(A, st) : d->dtype == 1 ? attend8_launch<_Float16, 64>(A, st) : attend8_launch<float, 64>(A, st);
  return d->dtype == 0 ? attend8_launch<__bf16, 128>(A, st) : d->dtype == 1 ? attend8_launch<_Float16, 128>(A, st) : attend8_launch<float, 128>(A, st);
}
