// Rows that go into the 8-bit key / value cache.  The values of a block of tokens and a kv head are code x scale with e4m3 codes and a scale that is a
// power of two: e4m3 is a floating type, so a finer scale would only move where its smallest values end, and with powers of two neither the
// division by the scale nor a later change of it rounds anything that the codes' own rounding does not.
//
// HBM-bound: a row is read once (16 bits or 32 a value) and written once (8).  A block's largest value has to be known before any of its codes: the
// block's new rows are held in registers in between, 32 values a lane, by one wave up to 2048 values and by up to eight for 128 rows of 128.  A
// block that holds rows already is read too, and its rows are written again only where the scale grows.
//
// Measured in a trace: a prompt of 30011 tokens, 4 heads of 64 bf16 features, 11.6 us (46 MB: 4.0 TB/s; a copy of as much takes 10); six chunks of 1021 tokens, 5
// heads of 128 fp32 features, 8.8 us (31 MB); one token for each of 64 sequences, 8 heads, 4.6 us, most of it the launch.  Blocks that are new as a whole have
// loads without a branch between them (replayed from a graph 11.4, 8.7 and 4.3 us; with the test of each row 12.7 and 9.4; with rows outside read as their neighbours in
// all blocks 12.1, 8.6 and 4.6).
#include "nsa_cache8.hpp"

namespace nsa {

struct AppendArgs {
  Cache8Args c;
  const void *k, *v;
  long k0, k1, k2, v0, v1, v2;
  const int* counts;
  int rows, touched;                   // rows handed in for each sequence, blocks that they may touch
  unsigned total;                      // (sequence, kv head, keys or values, block)
};

template <int D, int B>
struct AppendShape {
  static constexpr int CHUNKS = D * B / 8;                            // of eight values
  static constexpr int PER = CHUNKS / 64 < 4 ? CHUNKS / 64 : 4;       // a lane
  static constexpr int WAVES = CHUNKS / 64 / PER;                     // a block
  static constexpr int BLOCKS = WAVES < 4 ? 4 / WAVES : 1, THREADS = 64 * WAVES * BLOCKS;
};

template <class T, int D, int B>
__global__ __launch_bounds__((AppendShape<D, B>::THREADS)) void cache8_append_kernel(const AppendArgs A) {
  using S = AppendShape<D, B>;
  constexpr int LPR = D / 8;
  __shared__ float top_s[S::BLOCKS * S::WAVES];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = wave % S::WAVES;
  const unsigned id = blockIdx.x * S::BLOCKS + wave / S::WAVES;
  const bool here = id < A.total;
  const unsigned rest = here ? id / (unsigned)A.touched : 0;
  const int t = here ? (int)(id - rest * A.touched) : 0;
  const bool is_v = rest & 1;
  const int unit = (int)(rest >> 1), b = unit / A.c.hk, h = unit - b * A.c.hk;
  const int start = cache8_length(A.c, b);
  const int n = A.counts != nullptr ? min(max(A.counts[b], 0), A.rows) : A.rows;
  const int row0 = (start / B + t) * B, first = start - row0, last = (int)min((long)start + n, (long)A.c.cap) - row0;      // of the block, and its new rows
  const bool any = here && last > 0 && last > first;

  const T* src = (is_v ? reinterpret_cast<const T*>(A.v) + b * A.v0 + h * A.v1 : reinterpret_cast<const T*>(A.k) + b * A.k0 + h * A.k1);
  const long s_row = is_v ? A.v2 : A.k2;
  uint8_t* dst = (is_v ? A.c.values : A.c.keys) + b * A.c.s0 + h * A.c.s1 + row0 * A.c.s2;
  float* scale = (is_v ? A.c.value_scales : A.c.key_scales) + b * A.c.z0 + h * A.c.z1 + row0 / B;
  // chunk c of a lane: row part * RPW + c * STEP + lane / LPR, values 8 (lane % LPR) ..
  constexpr int RPW = 64 / LPR, STEP = RPW * S::WAVES;
  const int mine = part * RPW + lane / LPR, f = lane % LPR * 8;

  // All loads before the first value is looked at; of the rows of a load that are not there the nearest that is is read
  typedef __attribute__((__vector_size__(8 * sizeof(T)))) T vec;
  vec x[S::PER];
  uintx2 old[S::PER];
  float top = 0.f, s_old = 0.f;
  const bool held = first > 0;
  const bool all_new = !held && last >= B;       // no row is asked about
  auto fresh = [&](int row) { return row >= first && row < last; };
  auto some = [&](int c) { return part * RPW + c * STEP < last && part * RPW + c * STEP + RPW > first; };      // of a load's rows
  auto largest = [&](int c, bool in) {
    const floatx8 y = __builtin_convertvector(x[c], floatx8);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float m = fabsf(y[e]);
      top = fmaxf(top, in && m < INFINITY ? m : 0.f);
    }
  };
  if (any) {
    const T* from = src + f;
    if (all_new) {
#pragma unroll
      for (int c = 0; c < S::PER; ++c) x[c] = *reinterpret_cast<const vec*>(from + (long)(mine + c * STEP - first) * s_row);
#pragma unroll
      for (int c = 0; c < S::PER; ++c) largest(c, true);
    } else {
#pragma unroll
      for (int c = 0; c < S::PER; ++c)
        if (some(c)) x[c] = *reinterpret_cast<const vec*>(from + (long)(min(max(mine + c * STEP, first), last - 1) - first) * s_row);
      if (held) {
        s_old = *scale;
#pragma unroll
        for (int c = 0; c < S::PER; ++c)
          if (part * RPW + c * STEP < first) old[c] = *reinterpret_cast<const uintx2*>(dst + min(mine + c * STEP, first - 1) * A.c.s2 + f);
      }
#pragma unroll
      for (int c = 0; c < S::PER; ++c)
        if (some(c)) largest(c, fresh(mine + c * STEP));
    }
    top = wave_max(top);
  }
  if constexpr (S::WAVES > 1) {
    if (lane == 0) top_s[wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < S::WAVES; ++w) top = fmaxf(top, top_s[wave - part + w]);
  }
  if (!any) return;
  float s_new = power_of_two(scale_exponent(bits_of(top)));
  if (held) s_new = fmaxf(s_new, s_old);
  const float inv = 1.0f / s_new;      // (of a power of two: exact)
  if (lane == 0 && part == 0) *scale = s_new;
#pragma unroll
  for (int c = 0; c < S::PER; ++c) {
    const int row = mine + c * STEP;
    uintx2* to = reinterpret_cast<uintx2*>(dst + row * A.c.s2 + f);
    if (all_new || fresh(row)) *to = codes_of(__builtin_convertvector(x[c], floatx8), inv);
    else if (row < first && s_new != s_old) *to = codes_of(values_of(old[c]), s_old * inv);
  }
}

template <class T, int D, int B>
static int append_launch(const AppendArgs& A, hipStream_t st) {
  using S = AppendShape<D, B>;
  const unsigned groups = (A.total + S::BLOCKS - 1) / S::BLOCKS;
  if ((unsigned long)groups * S::THREADS >= 1UL << 32) return NSA_E_UNSUPPORTED;
  hipLaunchKernelGGL((cache8_append_kernel<T, D, B>), dim3(groups), dim3(S::THREADS), 0, st, A);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : (int)e;
}
template <class T, int D>
static int append_block(const AppendArgs& A, hipStream_t st) {
  switch (A.c.block) {
    case 16: return append_launch<T, D, 16>(A, st);
    case 32: return append_launch<T, D, 32>(A, st);
    case 64: return append_launch<T, D, 64>(A, st);
    default: return append_launch<T, D, 128>(A, st);
  }
}
template <class T>
static int append_dim(const AppendArgs& A, int d, hipStream_t st) { return d == 64 ? append_block<T, 64>(A, st) : append_block<T, 128>(A, st); }

}  // namespace nsa

extern "C" int nsa_cache8_append(const nsa_cache8_desc* d, int32_t rows, const void* k, const int64_t* k_stride, const void* v, const int64_t* v_stride,
                                 const int32_t* lengths, const int32_t* counts, void* keys, void* values, float* key_scales, float* value_scales,
                                 void* stream) {
  using namespace nsa;
  if (!cache8_check(d) || rows < 0 || !keys || !values || !key_scales || !value_scales || ((uintptr_t)keys | (uintptr_t)values) % 16) return NSA_E_ARG;
  if (!cache8_supported(d)) return NSA_E_UNSUPPORTED;
  if (rows == 0) return 0;
  if (!k || !v || !k_stride || !v_stride || ((uintptr_t)k | (uintptr_t)v) % 16) return NSA_E_ARG;
  const int per16 = d->dtype == 2 ? 4 : 8;
  for (int i = 0; i < 3; ++i)
    if (k_stride[i] % per16 || v_stride[i] % per16) return NSA_E_ARG;
  AppendArgs A{};
  A.c = cache8_args(d, keys, values, key_scales, value_scales, lengths);
  A.k = k; A.v = v;
  A.k0 = k_stride[0]; A.k1 = k_stride[1]; A.k2 = k_stride[2];
  A.v0 = v_stride[0]; A.v1 = v_stride[1]; A.v2 = v_stride[2];
  A.counts = counts; A.rows = rows;
  // (rows that begin anywhere in a block)
  A.touched = (int)(((long)rows + d->block - 2) / d->block + 1);
  A.touched = A.touched < d->capacity / d->block ? A.touched : d->capacity / d->block;
  const long units = (long)d->batch * d->kv_heads;
  if (units > 1L << 24 || units * 2 * A.touched >= 1L << 31) return NSA_E_UNSUPPORTED;
  A.total = (unsigned)(units * 2 * A.touched);
  hipStream_t st = (hipStream_t)stream;
  return d->dtype == 0 ? append_dim<__bf16>(A, d->dim_head, st) : d->dtype == 1 ? append_dim<_Float16>(A, d->dim_head, st) : append_dim<float>(A, d->dim_head, st);
}
