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

}  // namespace nsa
