// What is done to logits before a token is drawn: penalties for tokens that the sequence holds, a bias, the temperature, which tokens are allowed.
//
// HBM-bound: an entry is read once and written once.  A work-group takes one row's slice of the vocabulary, counts the row's history into LDS - the
// tokens that fall into the slice, by integer additions, so that their order changes nothing - and then passes over the slice: no counts in memory
// and one launch, for a history that every slice reads again (from L2).
#include "nsa_common.hpp"
#include "../../include/nsa_hip.h"

// every step of the chain rounds by itself
#pragma clang fp contract(off)

namespace nsa {

struct LogitsArgs {
  const void* x;
  long row_stride;
  int vocab, slice, slices;
  const void* history;
  long length;
  int history64;
  const int* history_lengths;
  const float *repetition, *frequency, *presence, *temperature, *bias;
  int rs, fs, ps, ts;
  float rep, freq, pres, temp;         // of all rows, where there is no address
  long bias_stride;
  const void* allowed;
  int allowed_kind;
  long allowed_stride;
  float* out;
};

constexpr int kLogitsSlice = 1024;

template <class T>
__global__ __launch_bounds__(256) void adjust_logits_kernel(const LogitsArgs A) {
  __shared__ int count_s[kLogitsSlice];
  const long r = blockIdx.x / A.slices;
  const int v0 = (int)(blockIdx.x % A.slices) * kLogitsSlice, v1 = min(A.vocab, v0 + kLogitsSlice);
  const long n = A.history == nullptr ? 0 : A.history_lengths != nullptr ? min(max((long)A.history_lengths[r], 0L), A.length) : A.length;
  if (n > 0) {
    for (int i = threadIdx.x; i < kLogitsSlice; i += 256) count_s[i] = 0;
    __syncthreads();
    for (long i = threadIdx.x; i < n; i += 256) {
      const long t = A.history64 ? reinterpret_cast<const long*>(A.history)[r * A.length + i] : (long)reinterpret_cast<const int*>(A.history)[r * A.length + i];
      if (t >= v0 && t < v1) atomicAdd(&count_s[t - v0], 1);
    }
    __syncthreads();
  }
  const float rep = A.repetition ? A.repetition[r * A.rs] : A.rep, freq = A.frequency ? A.frequency[r * A.fs] : A.freq;
  const float pres = A.presence ? A.presence[r * A.ps] : A.pres, temp = A.temperature ? A.temperature[r * A.ts] : A.temp;
  for (int i = v0 + threadIdx.x; i < v1; i += 256) {
    float x = (float)reinterpret_cast<const T*>(A.x)[r * A.row_stride + i];
    if (n > 0) {
      const int c = count_s[i - v0];
      if (c > 0) {
        x = x > 0.f ? x / rep : x * rep;
        x = x - freq * (float)c;
        x = x - pres;
      }
    }
    if (A.bias) x = x + A.bias[r * A.bias_stride + i];
    x = x / temp;
    bool ok = true;
    if (A.allowed_kind == 1) ok = reinterpret_cast<const uint8_t*>(A.allowed)[r * A.allowed_stride + i] != 0;
    else if (A.allowed_kind == 2) ok = (reinterpret_cast<const uint32_t*>(A.allowed)[r * A.allowed_stride + (i >> 5)] >> (i & 31)) & 1u;
    A.out[r * A.vocab + i] = ok ? x : -INFINITY;
  }
}

}  // namespace nsa

extern "C" int nsa_adjust_logits(const nsa_logits_desc* d, const void* x, const void* history, const int32_t* history_lengths, const float* repetition,
                                 const float* frequency, const float* presence, const float* bias, const void* allowed, const float* temperature,
                                 float* out, void* stream) {
  using namespace nsa;
  if (!d || d->rows < 0 || d->vocab <= 0 || d->dtype < 0 || d->dtype > 2 || d->history < 0 || d->allowed_kind < 0 || d->allowed_kind > 2) return NSA_E_ARG;
  if (d->rows == 0) return 0;
  if (!x || !out || (d->history > 0 && !history) || (d->allowed_kind != 0 && !allowed)) return NSA_E_ARG;
  const long slices = (d->vocab + kLogitsSlice - 1) / kLogitsSlice;
  if (d->rows > 1L << 30 || d->vocab > 1 << 30 || 4 * d->rows * slices >= 1L << 31) return NSA_E_UNSUPPORTED;
  LogitsArgs A{};
  A.x = x; A.row_stride = d->row_stride; A.vocab = d->vocab; A.slices = (int)slices;
  A.history = d->history > 0 ? history : nullptr; A.length = d->history; A.history64 = d->history_int64; A.history_lengths = history_lengths;
  A.repetition = repetition; A.frequency = frequency; A.presence = presence; A.temperature = temperature; A.bias = bias;
  A.rs = d->repetition_stride; A.fs = d->frequency_stride; A.ps = d->presence_stride; A.ts = d->temperature_stride;
  A.rep = d->repetition; A.freq = d->frequency; A.pres = d->presence; A.temp = d->temperature;
  A.bias_stride = d->bias_stride; A.allowed = allowed; A.allowed_kind = d->allowed_kind; A.allowed_stride = d->allowed_stride;
  A.out = out;
  const dim3 grid((unsigned)(d->rows * slices)), block(256);
  hipStream_t st = (hipStream_t)stream;
  if (d->dtype == 0) hipLaunchKernelGGL((adjust_logits_kernel<__bf16>), grid, block, 0, st, A);
  else if (d->dtype == 1) hipLaunchKernelGGL((adjust_logits_kernel<_Float16>), grid, block, 0, st, A);
  else hipLaunchKernelGGL((adjust_logits_kernel<float>), grid, block, 0, st, A);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : (int)e;
}
