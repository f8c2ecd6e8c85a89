// One token of each sequence attends the 8-bit key / value cache: all its keys, its newest ones, or selected blocks of them and its own.
#include "nsa_cache8.hpp"

namespace nsa {

struct Attend8Args {
  Cache8Args c;
  const void* q;
  long q0, q1;
  int dtype, g, units, gc;             // units: kv heads, or query heads that have blocks of their own; gc: query heads of a unit
  int window, sel_block, num_sel, idx64;
  const void* idx;
  const uint8_t* fmask;
  float scale;
  int nparts, tiles;                   // a part: this many tiles of 32 keys
  float* part;                         // records [gc][D] sums, [gc] maxima, [gc] weights, rec floats each
  int rec;
  void* out;
};

template <class T>
__device__ __forceinline__ float to_float(T x) { return (float)x; }

constexpr int kTile = 32;

// the keys of a unit: places 0 .. places - 1, each with a row of the cache or none
struct Keys8 {
  int len, first, base, places;
};
__device__ __forceinline__ Keys8 keys_of(const Attend8Args& A, int b) {
  Keys8 K;
  K.len = cache8_length(A.c, b);
  K.first = A.window > 0 && A.sel_block == 0 ? max(0, K.len - A.window) : 0;
  K.base = K.first / 16 * 16;
  K.places = A.sel_block > 0 ? (K.len > 0 ? (A.num_sel + 1) * A.sel_block : 0) : K.len - K.base;
  return K;
}
// the row of a place, -1 for none
__device__ __forceinline__ int row_of(const Attend8Args& A, const Keys8& K, long unit, int place) {
  if (place >= K.places) return -1;
  long row = K.base + (long)place;
  if (A.sel_block > 0) {
    const int slot = place / A.sel_block;
    long blk = (K.len - 1) / A.sel_block;
    if (slot < A.num_sel) {
      const long e = unit * A.num_sel + slot;
      blk = A.idx64 ? reinterpret_cast<const long*>(A.idx)[e] : (long)reinterpret_cast<const int*>(A.idx)[e];
      if (A.fmask[e] == 0 || blk < 0 || blk > K.len / A.sel_block) return -1;
    }
    row = blk * A.sel_block + place % A.sel_block;
  }
  return row >= K.first && row < K.len ? (int)row : -1;
}

template <class T, int D>
__global__ __launch_bounds__(256) void cache8_attend_kernel(const Attend8Args A) {
  __shared__ float q_s[32 * D], p_s[32][64];
  __shared__ int row_s[64];
  __shared__ float ks_s[64], vs_s[64], m_s[32], l_s[32], a_s[32];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long unit = blockIdx.y + (long)blockIdx.z * gridDim.y;
  const int b = (int)(unit / A.units), u = (int)(unit % A.units);
  const int hk = A.units == A.c.hk ? u : u / A.g, head0 = A.units == A.c.hk ? u * A.g : u;
  const Keys8 K = keys_of(A, b);
  const int p0 = blockIdx.x * A.tiles * kTile, p1 = min(K.places, p0 + A.tiles * kTile);
  for (int i = tid; i < A.gc * D; i += 256) q_s[i] = to_float(reinterpret_cast<const T*>(A.q)[b * A.q0 + (head0 + i / D) * A.q1 + i % D]) * A.scale * kLog2e;
  if (tid < 32) { m_s[tid] = -INFINITY; l_s[tid] = 0.f; }
  float acc[32 * D / 256];
#pragma unroll
  for (int i = 0; i < 32 * D / 256; ++i) acc[i] = 0.f;
  const uint8_t* kb = A.c.keys + b * A.c.s0 + hk * A.c.s1;
  const uint8_t* vb = A.c.values + b * A.c.s0 + hk * A.c.s1;
  const float* kz = A.c.key_scales + b * A.c.z0 + hk * A.c.z1;
  const float* vz = A.c.value_scales + b * A.c.z0 + hk * A.c.z1;
  for (int p = p0; p < p1; p += 64) {
    __syncthreads();
    if (tid < 64) {
      const int r = row_of(A, K, unit, p + tid < p1 ? p + tid : K.places);
      row_s[tid] = r;
      ks_s[tid] = r < 0 ? 0.f : kz[r / A.c.block];
      vs_s[tid] = r < 0 ? 0.f : vz[r / A.c.block];
    }
    __syncthreads();
    for (int i = tid; i < A.gc * 64; i += 256) {
      const int g = i / 64, j = i % 64, r = row_s[j];
      float s = -INFINITY;
      if (r >= 0) {
        s = 0.f;
        for (int f = 0; f < D; f += 4) {
          const int w = *reinterpret_cast<const int*>(kb + (long)r * A.c.s2 + f);
          s += q_s[g * D + f] * __builtin_amdgcn_cvt_f32_fp8(w, 0) + q_s[g * D + f + 1] * __builtin_amdgcn_cvt_f32_fp8(w, 1) +
               q_s[g * D + f + 2] * __builtin_amdgcn_cvt_f32_fp8(w, 2) + q_s[g * D + f + 3] * __builtin_amdgcn_cvt_f32_fp8(w, 3);
        }
        s *= ks_s[j];
      }
      p_s[g][j] = s;
    }
    __syncthreads();
    for (int g = wave; g < A.gc; g += 4) {
      const float s = p_s[g][lane];
      float mx = s;
      for (int o = 1; o <= 32; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
      const float mn = fmaxf(m_s[g], mx), ref = mn > -INFINITY ? mn : 0.f;
      const float e = fast_exp2(s - ref);
      float sum = e;
      for (int o = 1; o <= 32; o <<= 1) sum += __shfl_xor(sum, o, 64);
      p_s[g][lane] = e;
      if (lane == 0) {
        a_s[g] = fast_exp2(m_s[g] - ref);
        l_s[g] = l_s[g] * a_s[g] + sum;
        m_s[g] = mn;
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 32 * D / 256; ++i) {
      const int at = i * 256 + tid, g = at / D, f = at % D;
      if (g >= A.gc) continue;
      float a = acc[i] * a_s[g];
      for (int j = 0; j < 64; ++j)
        if (row_s[j] >= 0) a += p_s[g][j] * (__builtin_amdgcn_cvt_f32_fp8(vb[(long)row_s[j] * A.c.s2 + f], 0) * vs_s[j]);
      acc[i] = a;
    }
  }
  __syncthreads();
  float* rec = A.part + (unit * A.nparts + blockIdx.x) * A.rec;
#pragma unroll
  for (int i = 0; i < 32 * D / 256; ++i) {
    const int at = i * 256 + tid;
    if (at / D < A.gc) rec[at] = acc[i];
  }
  if (tid < A.gc) { rec[A.gc * D + tid] = m_s[tid]; rec[A.gc * D + A.gc + tid] = l_s[tid]; }
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
  const int parts = (K.places + A.tiles * kTile - 1) / (A.tiles * kTile);
  const float* base = A.part + ((long)b * A.units + u) * A.nparts * A.rec;
  const int om = A.gc * D + gi;
  float M = -INFINITY;
  for (int p = tid; p < parts; p += 256) M = fmaxf(M, base[(long)p * A.rec + om]);
#pragma unroll
  for (int o = 1; o <= 32; o <<= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
  if ((tid & 63) == 0) red_s[tid >> 6] = M;
  __syncthreads();
  M = fmaxf(fmaxf(red_s[0], red_s[1]), fmaxf(red_s[2], red_s[3]));
  const float ref = M > -INFINITY ? M : 0.f;
  floatx4 acc = {0.f, 0.f, 0.f, 0.f};
  float L = 0.f;
  for (int p = tid / LPP; p < parts; p += PPR) {
    const float* rec = base + (long)p * A.rec;
    const float w = fast_exp2(rec[om] - ref);
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
  if (!cache8_supported(d) || d->group > 32 || d->num_sel > 1 << 20 || ((long)d->num_sel + 1) * d->sel_block >= 1L << 30) return NSA_E_UNSUPPORTED;
  const bool per_head = d->sel_block > 0 && d->per_head_sel;
  A.g = d->group;
  A.units = per_head ? d->kv_heads * d->group : d->kv_heads;
  A.gc = per_head ? 1 : d->group;
  A.rec = A.gc * d->dim_head + ((2 * A.gc + 3) & ~3);
  const long units = (long)d->batch * A.units;
  if (units > 1L << 24) return NSA_E_UNSUPPORTED;
  long places = d->sel_block > 0 ? ((long)d->num_sel + 1) * d->sel_block : d->capacity;
  if (d->sel_block == 0 && d->window > 0 && d->window + 15L < places) places = d->window + 15L;
  const long tiles = (places + kTile - 1) / kTile;
  long per = (tiles * units + 1023) / 1024;
  per = per < 2 ? 2 : per;
  A.tiles = (int)per;
  A.nparts = (int)((tiles + per - 1) / per);
  bytes = (size_t)units * A.nparts * A.rec * sizeof(float);
  return 0;
}

template <class T, int D>
static int attend8_launch(const Attend8Args& A, long units, hipStream_t st) {
  const long z = (units + 32767) / 32768, y = (units + z - 1) / z;
  if (z * y != units) {                // (a grid has no ragged end: one plane after another)
    return NSA_E_UNSUPPORTED;
  }
  hipLaunchKernelGGL((cache8_attend_kernel<T, D>), dim3(A.nparts, (unsigned)y, (unsigned)z), dim3(256), 0, st, A);
  const long heads = units / A.units * A.c.hk * A.g;
  hipLaunchKernelGGL((cache8_merge_kernel<T, D>), dim3((unsigned)heads), dim3(256), 0, st, A);
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
  if (!q || !keys || !values || !key_scales || !value_scales || !out || ((uintptr_t)keys | (uintptr_t)values) % 16) return NSA_E_ARG;
  if (d->sel_block > 0 && d->num_sel > 0 && (!idx || !fmask)) return NSA_E_ARG;
  if (!ws || (uintptr_t)ws % 16) return NSA_E_ARG;
  if (ws_bytes < need) return NSA_E_WORKSPACE;
  A.c = cache8_args(d, keys, values, key_scales, value_scales, lengths);
  A.q = q; A.q0 = d->q_stride[0]; A.q1 = d->q_stride[1];
  A.dtype = d->dtype; A.window = d->window; A.sel_block = d->sel_block; A.num_sel = d->num_sel; A.idx64 = d->idx_is_int64;
  A.idx = idx; A.fmask = fmask; A.scale = d->scale; A.part = (float*)ws; A.out = out;
  const long units = (long)d->batch * A.units;
  hipStream_t st = (hipStream_t)stream;
  if (d->dim_head == 64)
    return d->dtype == 0 ? attend8_launch<__bf16, 64>(A, units, st) : d->dtype == 1 ? attend8_launch<_Float16, 64>(A, units, st) : attend8_launch<float, 64>(A, units, st);
  return d->dtype == 0 ? attend8_launch<__bf16, 128>(A, units, st) : d->dtype == 1 ? attend8_launch<_Float16, 128>(A, units, st) : attend8_launch<float, 128>(A, units, st);
}
