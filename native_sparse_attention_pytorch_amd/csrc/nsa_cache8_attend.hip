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
// the matrix cores have the time for it.
#include "nsa_cache8.hpp"

namespace nsa {

struct Attend8Args {
  Cache8Args c;
  const void* q;
  long q0, q1;
  int g, units, gc;                    // units: kv heads, or query heads that have blocks of their own; gc: query heads of a unit
  int window, sel_block, num_sel, idx64;
  const void* idx;
  const uint8_t* fmask;
  float scale;
  int block_shift;
  int nparts, tiles;                   // a part: this many tiles of 32 keys
  float* part;                         // records [gc][D] sums, [gc] maxima, [gc] weights, rec floats each
  int rec;
  void* out;
};

constexpr int kTile = 32, kWaves = 8;

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
__device__ __forceinline__ Keys8 keys_of(const Attend8Args& A, int b) {
  Keys8 K;
  K.len = cache8_length(A.c, b);
  K.first = A.window > 0 && A.sel_block == 0 ? max(0, K.len - A.window) : 0;
  K.base = K.first & ~15;
  K.places = A.sel_block > 0 ? (K.len > 0 ? (A.num_sel + 1) * A.sel_block : 0) : K.len - K.base;
  return K;
}
// the row of a place of a selection; without one ~ of the newest key's, which is attended: what is there may be read in its place
__device__ __forceinline__ int selected_row(const Attend8Args& A, const Keys8& K, long unit, int place) {
  const int none = ~(K.len - 1);
  if (place >= K.places) return none;
  const int slot = place / A.sel_block, own = (K.len - 1) / A.sel_block;
  long blk = own;
  if (slot < A.num_sel) {
    const long e = unit * A.num_sel + slot;
    const uint8_t live = A.fmask[e];
    blk = A.idx64 ? reinterpret_cast<const long*>(A.idx)[e] : (long)reinterpret_cast<const int*>(A.idx)[e];
    if (live == 0 || blk < 0 || blk > own) return none;
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
  for (int e = 0; e < 8; ++e) {
    float r = x[e];
#pragma unroll
    for (int p = 0; p < N; ++p) {
      const __bf16 h = (__bf16)r;
      to[p][e] = h;
      r -= (float)h;
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

template <int D>
struct Tile8 {                         // what a lane holds of 32 keys
  uintx4 k[2][D / 64];                 // key n of each 16: 16 codes
  uint32_t v[2][4][D / 64];            // keys 4 q + e: D / 16 codes
  float ks[2];
  floatx4 vs[2];
};

template <class T, int D, bool SEL>
__global__ __launch_bounds__(64 * kWaves) void cache8_attend_kernel(const Attend8Args A) {
  constexpr int QP = Parts8<T>::Q, PP = Parts8<T>::P, KS = D / 32, DT = D / 16;
  extern __shared__ __align__(16) char lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, q4 = lane >> 4;
  const long unit = blockIdx.x / A.nparts;
  const int part = (int)(blockIdx.x - unit * A.nparts);
  const int b = (int)(unit / A.units), u = (int)(unit - (long)b * A.units);
  const int hk = A.units == A.c.hk ? u : u / A.g, head0 = A.units == A.c.hk ? u * A.g : u;
  const Keys8 K = keys_of(A, b);
  const int tiles = (K.places + kTile - 1) / kTile, t0 = part * A.tiles, t1 = min(tiles, t0 + A.tiles);
  if (t0 >= t1 && part > 0) return;    // (the merge knows how many parts there are)

  // more than 16 query heads: half of the waves for the first 16
  const int groups = A.gc > 16 ? 2 : 1, group = groups == 2 ? wave & 1 : 0;
  const int w0 = groups == 2 ? wave >> 1 : wave, nw = kWaves / groups;
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
  const float sc = A.scale * kLog2e;
  const uint8_t* kb = A.c.keys + b * A.c.s0 + hk * A.c.s1 + 16 * q4;
  const uint8_t* vb = A.c.values + b * A.c.s0 + hk * A.c.s1 + DT * n;
  const float* kz = A.c.key_scales + b * A.c.z0 + hk * A.c.z1;
  const float* vz = A.c.value_scales + b * A.c.z0 + hk * A.c.z1;
  const uint32_t s2 = (uint32_t)A.c.s2;

  int* row_s = reinterpret_cast<int*>(lds);
  float* ks_s = reinterpret_cast<float*>(lds) + A.tiles * kTile;
  float* vs_s = ks_s + A.tiles * kTile;
  if constexpr (SEL) {
    for (int i = tid; i < (t1 - t0) * kTile; i += 64 * kWaves) {
      const int r = selected_row(A, K, unit, t0 * kTile + i), at = (r < 0 ? ~r : r) >> A.block_shift;
      row_s[i] = r;
      ks_s[i] = kz[at];
      vs_s[i] = vz[at];
    }
    __syncthreads();
  }

  float m = -INFINITY, l = 0.f;
  floatx4 O[DT];
#pragma unroll
  for (int c = 0; c < DT; ++c) O[c] = floatx4{0.f, 0.f, 0.f, 0.f};

  auto load = [&](int t, Tile8<D>& X) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (SEL) {
        const int at = (t - t0) * kTile + 16 * i;
        int r = row_s[at + n];
        r = r < 0 ? ~r : r;
        X.ks[i] = ks_s[at + n];
#pragma unroll
        for (int j = 0; j < D / 64; ++j) X.k[i][j] = *reinterpret_cast<const uintx4*>(kb + (uint64_t)(uint32_t)r * s2 + 64 * j);
        const intx4 rv = *reinterpret_cast<const intx4*>(row_s + at + 4 * q4);
        X.vs[i] = *reinterpret_cast<const floatx4*>(vs_s + at + 4 * q4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int x = rv[e] < 0 ? ~rv[e] : rv[e];
          const uint32_t* p = reinterpret_cast<const uint32_t*>(vb + (uint64_t)(uint32_t)x * s2);
#pragma unroll
          for (int j = 0; j < D / 64; ++j) X.v[i][e][j] = p[j];
        }
      } else {
        // (a place without a key: the newest one, which is attended, is read instead)
        const int r0 = K.base + t * kTile + 16 * i, last = K.len - 1;
        const int z = min(r0, last) >> A.block_shift;
        X.ks[i] = kz[z];
        const float s = vz[z];
        X.vs[i] = floatx4{s, s, s, s};
        int r = r0 + n;
        r = r < K.first || r > last ? last : r;
#pragma unroll
        for (int j = 0; j < D / 64; ++j) X.k[i][j] = *reinterpret_cast<const uintx4*>(kb + (uint64_t)(uint32_t)r * s2 + 64 * j);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          int x = r0 + 4 * q4 + e;
          x = x < K.first || x > last ? last : x;
          const uint32_t* p = reinterpret_cast<const uint32_t*>(vb + (uint64_t)(uint32_t)x * s2);
#pragma unroll
          for (int j = 0; j < D / 64; ++j) X.v[i][e][j] = p[j];
        }
      }
    }
  };

  auto work = [&](int t, const Tile8<D>& X) {
    float s[8];
    float mx = -INFINITY;
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
      intx4 rows;
      if constexpr (SEL) rows = *reinterpret_cast<const intx4*>(row_s + (t - t0) * kTile + 16 * i + 4 * q4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        bool live;
        if constexpr (SEL) live = rows[e] >= 0;
        else {
          const int r = K.base + t * kTile + 16 * i + 4 * q4 + e;
          live = r >= K.first && r < K.len;
        }
        const float v = live ? S[e] * sc : -INFINITY;
        s[4 * i + e] = v;
        mx = fmaxf(mx, v);
      }
    }
    mx = quarters_max(mx);
    if (__any(mx > m)) {                         // (a NaN raises no maximum: it reaches the sum by itself)
      const float mn = fmaxf(m, mx), a = fast_exp2(m - mn);
      const float by = m == -INFINITY ? 0.f : a;
      m = mn;
      l *= by;
#pragma unroll
      for (int c = 0; c < DT; ++c) O[c] *= by;
    }
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float p = fast_exp2(s[e] - ref);
      l += p;
      s[e] = p * X.vs[e >> 2][e & 3];
    }
    bf16x8 P[PP];
    split_parts(s, P);
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

  // (tiles of a selection whose blocks are not there are passed over)
  auto next = [&](int t) {
    for (; t < t1; t += nw) {
      if constexpr (SEL) {
        if (!__any(row_s[(t - t0) * kTile + (lane & 31)] >= 0)) continue;
      }
      break;
    }
    return t;
  };
  Tile8<D> X, Y;
  int t = next(t0 + w0);
  if (t < t1) load(t, X);
  while (t < t1) {
    const int tn = next(t + nw);
    if (tn < t1) load(tn, Y);
    work(t, X);
    X = Y;
    t = tn;
  }
  l = quarters_sum(l);

  // the waves' results as one
  __syncthreads();                               // (the lists of rows are read no more)
  constexpr int H = D / 2, RO = H + 4;           // half of the features at a time: 36 KB at 16 columns
  float* m_s = reinterpret_cast<float*>(lds);
  float* l_s = m_s + kWaves * 16;
  float* o_s = l_s + kWaves * 16;                // [wave][cols of a group][RO]
  const int most = min(16, A.gc);
  if (q4 == 0) { m_s[wave * 16 + n] = m; l_s[wave * 16 + n] = l; }
  __syncthreads();
  float M = -INFINITY;
  for (int w = group; w < kWaves; w += groups) M = fmaxf(M, m_s[w * 16 + n]);
  const float by = m == -INFINITY ? 0.f : fast_exp2(m - M);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    // (place f of the half: feature DT (4 (f / 2 DT) + 2 half) + f % 2 DT)
    if (n < cols) {
      float* o = o_s + (wave * most + n) * RO + 2 * DT * q4;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int c = 0; c < DT; c += 4) {
          const int r = 2 * half + i;
          *reinterpret_cast<floatx4*>(o + DT * i + c) = floatx4{O[c][r] * by, O[c + 1][r] * by, O[c + 2][r] * by, O[c + 3][r] * by};
        }
    }
    __syncthreads();
    for (int i = tid; i < A.gc * (H / 4); i += 64 * kWaves) {
      const int g = i / (H / 4), at = i % (H / 4) * 4, gr = g >> 4, c = g & 15, f = DT * (4 * (at / (2 * DT)) + 2 * half) + at % (2 * DT);
      floatx4 o = {0.f, 0.f, 0.f, 0.f};
      float Mg = -INFINITY, L = 0.f;
      for (int w = gr; w < kWaves; w += groups) Mg = fmaxf(Mg, m_s[w * 16 + c]);
      for (int w = gr; w < kWaves; w += groups) {
        const float mw = m_s[w * 16 + c];
        L += (mw == -INFINITY ? 1.f : fast_exp2(mw - Mg)) * l_s[w * 16 + c];
        o += *reinterpret_cast<const floatx4*>(o_s + (w * most + c) * RO + at);
      }
      if (A.nparts == 1) {
        T* to = reinterpret_cast<T*>(A.out) + ((long)b * A.c.hk * A.g + head0 + g) * D + f;
#pragma unroll
        for (int e = 0; e < 4; ++e) to[e] = (T)(L == 0.f ? 0.f : o[e] / L);
      } else {
        float* rec = A.part + blockIdx.x * (long)A.rec;
        *reinterpret_cast<floatx4*>(rec + g * D + f) = o;
        if (f == 0) { rec[A.gc * D + g] = Mg; rec[A.gc * D + A.gc + g] = L; }
      }
    }
    if (half == 0) __syncthreads();
  }
}

// the parts of a head, weighted by their maxima
template <class T, int D>
__global__ __launch_bounds__(256) void cache8_merge_kernel(const Attend8Args A) {
  constexpr int LPP = D / 4, PPR = 256 / LPP;
  __shared__ float red_s[4];
  __shared__ __align__(16) float acc_s[PPR][D];
  __shared__ float l_s[PPR];
  const int tid = threadIdx.x, heads = A.c.hk * A.g;
  const long bh = blockIdx.x;
  const int b = (int)(bh / heads), head = (int)(bh % heads);
  const int u = A.units == A.c.hk ? head / A.g : head, gi = A.units == A.c.hk ? head % A.g : 0;
  const Keys8 K = keys_of(A, b);
  const int parts = max(1, ((K.places + kTile - 1) / kTile + A.tiles - 1) / A.tiles);
  const float* base = A.part + ((long)b * A.units + u) * A.nparts * A.rec;
  const int om = A.gc * D + gi;
  float M = -INFINITY;
  for (int p = tid; p < parts; p += 256) M = fmaxf(M, base[(long)p * A.rec + om]);
#pragma unroll
  for (int o = 1; o <= 32; o <<= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
  if ((tid & 63) == 0) red_s[tid >> 6] = M;
  __syncthreads();
  M = fmaxf(fmaxf(red_s[0], red_s[1]), fmaxf(red_s[2], red_s[3]));
  floatx4 acc = {0.f, 0.f, 0.f, 0.f};
  float L = 0.f;
  for (int p = tid / LPP; p < parts; p += PPR) {
    const float* rec = base + (long)p * A.rec;
    const float mp = rec[om], w = mp == -INFINITY ? 1.f : fast_exp2(mp - M);      // (a part without a number for its maximum: NaN or nothing)
    L += w * rec[om + A.gc];
    acc += w * *reinterpret_cast<const floatx4*>(rec + gi * D + 4 * (tid % LPP));
  }
  *reinterpret_cast<floatx4*>(&acc_s[tid / LPP][4 * (tid % LPP)]) = acc;
  if (tid % LPP == 0) l_s[tid / LPP] = L;
  __syncthreads();
  if (tid < D) {
    float o = 0.f, l = 0.f;
#pragma unroll
    for (int r = 0; r < PPR; ++r) { o += acc_s[r][tid]; l += l_s[r]; }
    reinterpret_cast<T*>(A.out)[bh * D + tid] = (T)(l == 0.f ? 0.f : o / l);
  }
}

// units, parts and records of a call
static int attend8_plan(const nsa_cache8_desc* d, Attend8Args& A, size_t& bytes) {
  if (!cache8_check(d) || d->group <= 0 || d->window < 0 || d->sel_block < 0 || d->num_sel < 0) return NSA_E_ARG;
  if (!cache8_supported(d) || d->group > 32 || d->num_sel > 1 << 20 || ((long)d->num_sel + 1) * d->sel_block >= 1L << 30 || d->kv_stride[2] >= 1L << 31)
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
  long per = (tiles * units + 511) / 512;
  per = per < kWaves ? kWaves : (per + kWaves - 1) / kWaves * kWaves;
  if (d->sel_block > 0 && per > 64) per = 64;    // (the lists of rows and scales in LDS)
  if (tiles <= 5 * kWaves) per = 5 * kWaves;
  A.tiles = (int)per;
  A.nparts = (int)((tiles + per - 1) / per);
  if (units * A.nparts >= 1L << 23 || (long)d->batch * d->kv_heads * d->group >= 1L << 24) return NSA_E_UNSUPPORTED;
  bytes = A.nparts > 1 ? (size_t)units * A.nparts * A.rec * sizeof(float) : 0;
  return 0;
}

template <class T, int D>
static int attend8_launch(const Attend8Args& A, long units, hipStream_t st) {
  const size_t merge = (kWaves * 32 + (size_t)kWaves * (A.gc < 16 ? A.gc : 16) * (D / 2 + 4)) * 4, lists = A.sel_block > 0 ? (size_t)A.tiles * kTile * 12 : 0;
  const unsigned bytes = (unsigned)(merge > lists ? merge : lists);
  const dim3 grid((unsigned)(units * A.nparts)), block(64 * kWaves);
  if (A.sel_block > 0) hipLaunchKernelGGL((cache8_attend_kernel<T, D, true>), grid, block, bytes, st, A);
  else hipLaunchKernelGGL((cache8_attend_kernel<T, D, false>), grid, block, bytes, st, A);
  if (A.nparts > 1) hipLaunchKernelGGL((cache8_merge_kernel<T, D>), dim3((unsigned)(units / A.units * A.c.hk * A.g)), dim3(256), 0, st, A);
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
  A.window = d->window; A.sel_block = d->sel_block; A.num_sel = d->num_sel; A.idx64 = d->idx_is_int64;
  A.idx = idx; A.fmask = fmask; A.scale = d->scale; A.part = (float*)ws; A.out = out;
  const long units = (long)d->batch * A.units;
  hipStream_t st = (hipStream_t)stream;
  if (d->dim_head == 64)
    return d->dtype == 0 ? attend8_launch<__bf16, 64>(A, units, st) : d->dtype == 1 ? attend8_launch<_Float16, 64>(A, units, st) : attend8_launch<float, 64>(A, units, st);
  return d->dtype == 0 ? attend8_launch<__bf16, 128>(A, units, st) : d->dtype == 1 ? attend8_launch<_Float16, 128>(A, units, st) : attend8_launch<float, 128>(A, units, st);
}
