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
// the new token: its queries rotated to rq, its key and value into the cache, both unrotated into the ring
int cache8_step_prep(const Step8& s, const void* q, const int64_t* q_stride, const void* k, const int64_t* k_stride, const void* v, const int64_t* v_stride,
                     const float* freqs, void* rq, void* krun, const int64_t* krun_stride, int64_t krun_row, void* vrun, const int64_t* vrun_stride,
                     int64_t vrun_row, int ring, void* stream);
// Parts and floats of a record of each unit, {sliding window, selected blocks}: records [gc][D] sums, [gc] maxima, [gc] weights, as nsa_decode_combine takes them.
void cache8_step_parts(const Step8& s, int parts[2], int rec[2]);
int cache8_step_attend(const Step8& s, const void* rq, const int32_t* idx, const uint8_t* fmask, float* window_records, float* block_records, void* stream);

}  // namespace nsa
