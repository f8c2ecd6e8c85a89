// Sizes and addresses of the 8-bit key / value cache that its writer and its readers share.
#pragma once
#include "nsa_common.hpp"
#include "../../include/nsa_hip.h"

namespace nsa {

struct Cache8Args {
  uint8_t *keys, *values;
  float *key_scales, *value_scales;
  long s0, s1, s2, z0, z1;             // strides of the codes {batch, head, row} and of the scales {batch, head}
  int hk, block, cap;
  const int* lengths;
  int length, length_stride;
};

__device__ __forceinline__ int cache8_length(const Cache8Args& C, int b) {
  const long n = C.length + (C.lengths != nullptr ? (long)C.lengths[(long)b * C.length_stride] : 0);
  return (int)(n < 0 ? 0 : n > C.cap ? C.cap : n);
}

template <class T>
__device__ __forceinline__ floatx8 load_values(const T* p) {
  typedef __attribute__((__vector_size__(8 * sizeof(T)))) T vec;
  return __builtin_convertvector(*reinterpret_cast<const vec*>(p), floatx8);
}

// (a bit cast of a vector's element itself takes the vector's first)
__device__ __forceinline__ uint32_t bits_of(float x) { return __builtin_bit_cast(uint32_t, x); }

// Eight values times `inv`, which is a power of two, as e4m3 codes: nearest, halves to even, beyond 448 to 448, what is no finite number as NaN.
__device__ __forceinline__ uintx2 codes_of(const floatx8& x, float inv) {
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float v = x[e];
    const bool finite = (bits_of(v) & 0x7f800000u) != 0x7f800000u;
    y[e] = finite ? fminf(fmaxf(v * inv, -448.f), 448.f) : __builtin_nanf("");
  }
  uintx2 r;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h], y[4 * h + 1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h + 2], y[4 * h + 3], w, true);
    r[h] = (uint32_t)w;
  }
  return r;
}

__device__ __forceinline__ floatx8 values_of(const uintx2& c) {
  floatx8 x;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int w = (int)c[h];
    x[4 * h] = __builtin_amdgcn_cvt_f32_fp8(w, 0);
    x[4 * h + 1] = __builtin_amdgcn_cvt_f32_fp8(w, 1);
    x[4 * h + 2] = __builtin_amdgcn_cvt_f32_fp8(w, 2);
    x[4 * h + 3] = __builtin_amdgcn_cvt_f32_fp8(w, 3);
  }
  return x;
}

// the exponent of the smallest power of two that takes a finite value of these bits to 448 = 1.75 x 2^8 or less
__device__ __forceinline__ int scale_exponent(uint32_t bits) {
  const int e = (int)(bits >> 23) - 127, k = e - 8 + ((bits & 0x7fffffu) > 0x600000u);
  return min(max(k, -110), 119);
}
__device__ __forceinline__ float power_of_two(int k) { return __builtin_bit_cast(float, (uint32_t)(k + 127) << 23); }

// maximum over the wave, in all lanes; mirrors of eight and sixteen lanes reach the other half of each
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, dpp_quad_xor1(v));
  v = fmaxf(v, dpp_quad_xor2(v));
  v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x141, 0xF, 0xF, true)));
  v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x140, 0xF, 0xF, true)));
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return halves_max(v);
}

inline bool cache8_check(const nsa_cache8_desc* d) {
  return d && d->batch > 0 && d->kv_heads > 0 && d->capacity > 0 && d->block > 0 && d->capacity % d->block == 0 && d->dtype >= 0 && d->dtype <= 2 &&
         d->reserved == 0 && !((d->kv_stride[0] | d->kv_stride[1] | d->kv_stride[2]) & 15) && d->kv_stride[2] >= d->dim_head;
}
inline bool cache8_supported(const nsa_cache8_desc* d) {
  return (d->dim_head == 64 || d->dim_head == 128) && (d->block == 16 || d->block == 32 || d->block == 64 || d->block == 128) &&
         d->capacity <= 1 << 30;
}

inline Cache8Args cache8_args(const nsa_cache8_desc* d, const void* keys, const void* values, const float* key_scales, const float* value_scales,
                              const int32_t* lengths) {
  Cache8Args C{};
  C.keys = (uint8_t*)keys; C.values = (uint8_t*)values; C.key_scales = (float*)key_scales; C.value_scales = (float*)value_scales;
  C.s0 = d->kv_stride[0]; C.s1 = d->kv_stride[1]; C.s2 = d->kv_stride[2]; C.z0 = d->scale_stride[0]; C.z1 = d->scale_stride[1];
  C.hk = d->kv_heads; C.block = d->block; C.cap = d->capacity;
  C.lengths = lengths; C.length = d->length; C.length_stride = d->length_stride;
  return C;
}

// The parts of a decode step over an 8-bit cache whose lengths are read from `state` = {rows held, compressed keys}: nsa_decode_step8_dyn has the rest.
struct Step8 {
  const nsa_cache8_desc* d;            // (q_stride, lengths and the selection are not read)
  void *keys, *values;
  float *key_scales, *value_scales;
  const int* state;
  int rows;                            // that the caches may hold: a token beyond them is left out
  int window, sel_block, num_sel, per_block, compressed;      // per_block: compressed keys of a selected block; compressed: that the caches may hold
  bool per_head;
};
// The new token: its queries rotated to rq, its key and value into the cache, both unrotated into the ring.
struct StepPrepArgs {
  Cache8Args c;
  int rows, g, ring;
  const __bf16 *q, *k, *v;
  long q0, q1, k0, k1, v0, v1;
  const float* freqs;
  __bf16 *rq, *krun, *vrun;
  long ku0, ku1, ku_row, vu0, vu1, vu_row;
};

// A work-group of two waves for each sequence and kv head, `unit`: the group's queries by both, then the key by one and the value by the other.  A lane
// has a pair of features.
template <int D>
__device__ __forceinline__ void step8_prep(const StepPrepArgs& A, const int unit) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = unit / A.c.hk, h = unit - b * A.c.hk, pos = A.c.lengths[0];
  if (lane >= D / 2) return;
  float sn, cs;
  sincosf((float)pos * A.freqs[lane], &sn, &cs);
  // (rounded to bf16 as the rotation by itself does)
  auto rotated = [&](bf16x2 x) {
    const float a = (float)x[0], c = (float)x[1];
    return bf16x2{(__bf16)(a * cs - c * sn), (__bf16)(c * cs + a * sn)};
  };
  for (int i = wave; i < A.g; i += 2) {
    const int head = h * A.g + i;
    const bf16x2 y = *reinterpret_cast<const bf16x2*>(A.q + b * A.q0 + head * A.q1 + 2 * lane);
    *reinterpret_cast<bf16x2*>(A.rq + ((long)b * A.c.hk * A.g + head) * D + 2 * lane) = rotated(y);
  }
  if (pos < 0 || pos >= A.rows) return;
  const bool is_v = wave == 1;
  bf16x2 x = *reinterpret_cast<const bf16x2*>((is_v ? A.v + b * A.v0 + h * A.v1 : A.k + b * A.k0 + h * A.k1) + 2 * lane);
  __bf16* run = is_v ? A.vrun : A.krun;
  if (run != nullptr) {
    const long at = pos % A.ring;
    *reinterpret_cast<bf16x2*>(run + (is_v ? b * A.vu0 + h * A.vu1 + at * A.vu_row : b * A.ku0 + h * A.ku1 + at * A.ku_row) + 2 * lane) = x;
  }
  if (!is_v) x = rotated(x);
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const float m = fabsf((float)x[e]);
    top = fmaxf(top, m < INFINITY ? m : 0.f);
  }
  // (of the lanes that have features: half a wave with 64)
#pragma unroll
  for (int o = 1; o < D / 2; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  const int held = pos % A.c.block;
  uint8_t* codes = (is_v ? A.c.values : A.c.keys) + b * A.c.s0 + h * A.c.s1 + (long)(pos - held) * A.c.s2;
  float* scale = (is_v ? A.c.value_scales : A.c.key_scales) + b * A.c.z0 + h * A.c.z1 + pos / A.c.block;
  const float s_old = held > 0 ? *scale : 0.f, s_new = fmaxf(power_of_two(scale_exponent(bits_of(top))), s_old), inv = 1.0f / s_new;
  if (held > 0 && s_new != s_old) {
    for (int i = lane; i < held * (D / 8); i += D / 2) {
      uintx2* at = reinterpret_cast<uintx2*>(codes + (i / (D / 8)) * A.c.s2 + i % (D / 8) * 8);
      *at = codes_of(values_of(*at), s_old * inv);
    }
  }
  if (lane == 0) *scale = s_new;
  const uintx2 both = codes_of(floatx8{(float)x[0], (float)x[1], 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, inv);
  *reinterpret_cast<uint16_t*>(codes + held * A.c.s2 + 2 * lane) = (uint16_t)both[0];
}

inline StepPrepArgs step8_prep_args(const Step8& s, const void* q, const int64_t* q_stride, const void* k, const int64_t* k_stride, const void* v, const int64_t* v_stride,
                     const float* freqs, void* rq, void* krun, const int64_t* krun_stride, int64_t krun_row, void* vrun, const int64_t* vrun_stride,
                     int64_t vrun_row, int ring) {
  const nsa_cache8_desc* d = s.d;
  StepPrepArgs A{};
  A.c = cache8_args(d, s.keys, s.values, s.key_scales, s.value_scales, s.state);
  A.rows = s.rows; A.g = d->group; A.ring = ring;
  A.q = (const __bf16*)q; A.k = (const __bf16*)k; A.v = (const __bf16*)v;
  A.q0 = q_stride[0]; A.q1 = q_stride[1]; A.k0 = k_stride[0]; A.k1 = k_stride[1]; A.v0 = v_stride[0]; A.v1 = v_stride[1];
  A.freqs = freqs; A.rq = (__bf16*)rq; A.krun = (__bf16*)krun; A.vrun = (__bf16*)vrun;
  if (krun) {
    A.ku0 = krun_stride[0]; A.ku1 = krun_stride[1]; A.ku_row = krun_row; A.vu0 = vrun_stride[0]; A.vu1 = vrun_stride[1]; A.vu_row = vrun_row;
  }
  return A;
}
// Parts and floats of a record of each unit, {sliding window, selected blocks}: records [gc][D] sums, [gc] maxima, [gc] weights, as nsa_decode_combine takes them.
void cache8_step_parts(const Step8& s, int parts[2], int rec[2]);
// The blocks are idx where fmask is set, or the ones that the work-groups choose themselves from `pooled` [batch, rows of the selection, pooled_stride].
int cache8_step_attend(const Step8& s, const void* rq, const int32_t* idx, const uint8_t* fmask, const float* pooled, long pooled_stride,
                       float* window_records, float* block_records, void* stream);

}  // namespace nsa
