// What is done to logits before a token is drawn: penalties for tokens that the sequence holds, a bias, the temperature, which tokens are allowed.
//
// HBM-bound: an entry is read once and written once, four bytes of it.  A work-group takes one row's slice of the vocabulary, counts the row's history
// into LDS - the tokens that fall into the slice, by integer additions, so that their order changes nothing - and then passes over the slice: no
// counts in memory and one launch, for a history that every slice reads again (from L2).
//
// Measured in a trace: 64 rows of 128000 bf16 logits, 4096 tokens of history, a bit mask, 16.6 us (52 MB: 3.1 TB/s; 11 without history and mask: all work-groups are on the
// chip at once and write only when they have counted); 300 rows of 50021 fp32 ones with a bias, 34.2 us (137 MB: 4.0 TB/s); 8 rows of 256, 4.6 us.
// Slices of 256 threads are up to 2 us faster with a history of some hundred tokens (300 rows of 50021: 24.6 and 25.7) and slower with thousands (256 rows of
// 32000 with 4096: 20.4 and 16.8).  Asking for the history before the entries changed nothing (17.3 and 33.9 us), and neither did divisions of five instructions by reciprocals (17.3 and
// 34.4): neither the one wait nor the arithmetic is what it waits for.
#include <algorithm>

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

constexpr int kLogitsThreads = 512, kRun = 8, kSweeps = 2;         // kRun: entries of a thread at a time; kSweeps: of a slice, at most

// n consecutive values of any alignment (that of the type at least)
template <class T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Run { T v[N]; };

template <class T, class I>
__global__ __launch_bounds__(kLogitsThreads) void adjust_logits_kernel(const LogitsArgs A) {
  extern __shared__ __align__(16) int count_s[];
  constexpr int V = kRun;
  const int tid = threadIdx.x;
  const long r = blockIdx.x / A.slices;
  const int v0 = (int)(blockIdx.x - r * A.slices) * A.slice, v1 = min(A.vocab, v0 + A.slice);
  const T* x = reinterpret_cast<const T*>(A.x) + r * A.row_stride;
  const float* bias = A.bias ? A.bias + r * A.bias_stride : nullptr;
  float* out = A.out + r * A.vocab;
  const long n = A.history == nullptr ? 0 : A.history_lengths != nullptr ? min(max((long)A.history_lengths[r], 0L), A.length) : A.length;
  const float rep = A.repetition ? A.repetition[r * A.rs] : A.rep, freq = A.frequency ? A.frequency[r * A.fs] : A.freq;
  const float pres = A.presence ? A.presence[r * A.ps] : A.pres, temp = A.temperature ? A.temperature[r * A.ts] : A.temp;
  // the entries and their mask are asked for before the history is read
  Run<T, V> a[kSweeps];
  uint32_t ok[kSweeps];
#pragma unroll
  for (int k = 0; k < kSweeps; ++k) {
    const int i = v0 + (k * kLogitsThreads + tid) * V;
    ok[k] = ~0u;
    if (i + V > v1) continue;
    a[k] = *reinterpret_cast<const Run<T, V>*>(x + i);
    if (A.allowed_kind == 1) {
      const Run<uint8_t, V> t = *reinterpret_cast<const Run<uint8_t, V>*>(reinterpret_cast<const uint8_t*>(A.allowed) + r * A.allowed_stride + i);
      ok[k] = 0;
#pragma unroll
      for (int e = 0; e < V; ++e) ok[k] |= (unsigned)(t.v[e] != 0) << e;
    } else if (A.allowed_kind == 2) {            // (slices begin at words, runs of eight lie in one)
      ok[k] = reinterpret_cast<const uint32_t*>(A.allowed)[r * A.allowed_stride + (i >> 5)] >> (i & 31);
    }
  }
  if (n > 0) {
    for (int i = tid * 4; i < A.slice; i += kLogitsThreads * 4) *reinterpret_cast<intx4*>(count_s + i) = intx4{0, 0, 0, 0};
    __syncthreads();
    const I* h = reinterpret_cast<const I*>(A.history) + r * A.length;
    const unsigned size = (unsigned)(v1 - v0);
    constexpr int H = 16 / sizeof(I), U = 4;     // tokens of a load, loads at once
    auto tally = [&](I t) {
      const unsigned long at = (unsigned long)((long)t - v0);
      if (at < size) atomicAdd(&count_s[at], 1);
    };
    const long whole = n / H * H;
    for (long i = (long)tid * H; i < whole; i += (long)U * kLogitsThreads * H) {
      Run<I, H> t[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long at = i + (long)u * kLogitsThreads * H;
        if (at < whole) t[u] = *reinterpret_cast<const Run<I, H>*>(h + at);
        else
#pragma unroll
          for (int e = 0; e < H; ++e) t[u].v[e] = (I)-1;
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < H; ++e) tally(t[u].v[e]);
    }
    if (whole + tid < n) tally(h[whole + tid]);
    __syncthreads();
  }
  // (a branch that all lanes take alike, for what there is no need of)
  auto entry = [&](float v, int c, float b, bool ok) {
    if (c > 0) {
      v = v > 0.f ? v / rep : v * rep;
      v = v - freq * (float)c;
      v = v - pres;
    }
    if (bias) v = v + b;
    if (temp != 1.f) v = v / temp;
    return ok ? v : -INFINITY;
  };
#pragma unroll
  for (int k = 0; k < kSweeps; ++k) {
    const int i = v0 + (k * kLogitsThreads + tid) * V;
    if (i + V <= v1) {
      Run<float, V> o, b;
      int c[V];
#pragma unroll
      for (int e = 0; e < V; ++e) c[e] = 0, b.v[e] = 0.f;
      if (bias) b = *reinterpret_cast<const Run<float, V>*>(bias + i);
      if (n > 0) {
        const intx4 c0 = *reinterpret_cast<const intx4*>(count_s + i - v0), c1 = *reinterpret_cast<const intx4*>(count_s + i - v0 + 4);
#pragma unroll
        for (int e = 0; e < V; ++e) c[e] = e < 4 ? c0[e & 3] : c1[e & 3];
      }
#pragma unroll
      for (int e = 0; e < V; ++e) o.v[e] = entry((float)a[k].v[e], c[e], b.v[e], ok[k] >> e & 1);
      *reinterpret_cast<Run<float, V>*>(out + i) = o;
    } else {
      for (int j = i; j < v1; ++j) {
        bool allow = true;
        if (A.allowed_kind == 1) allow = reinterpret_cast<const uint8_t*>(A.allowed)[r * A.allowed_stride + j] != 0;
        else if (A.allowed_kind == 2) allow = (reinterpret_cast<const uint32_t*>(A.allowed)[r * A.allowed_stride + (j >> 5)] >> (j & 31)) & 1u;
        out[j] = entry((float)x[j], n > 0 ? count_s[j - v0] : 0, bias ? bias[j] : 0.f, allow);
      }
    }
  }
}

template <class T>
static void logits_launch(const LogitsArgs& A, bool wide, unsigned groups, hipStream_t st) {
  const unsigned lds = A.history ? (unsigned)A.slice * 4 : 0;
  if (wide) hipLaunchKernelGGL((adjust_logits_kernel<T, int64_t>), dim3(groups), dim3(kLogitsThreads), lds, st, A);
  else hipLaunchKernelGGL((adjust_logits_kernel<T, int32_t>), dim3(groups), dim3(kLogitsThreads), lds, st, A);
}

}  // namespace nsa

extern "C" int nsa_adjust_logits(const nsa_logits_desc* d, const void* x, const void* history, const int32_t* history_lengths, const float* repetition,
                                 const float* frequency, const float* presence, const float* bias, const void* allowed, const float* temperature,
                                 float* out, void* stream) {
  using namespace nsa;
  if (!d || d->rows < 0 || d->vocab <= 0 || d->dtype < 0 || d->dtype > 2 || d->history < 0 || d->allowed_kind < 0 || d->allowed_kind > 2) return NSA_E_ARG;
  if (d->rows == 0) return 0;
  if (!x || !out || (d->history > 0 && !history) || (d->allowed_kind != 0 && !allowed)) return NSA_E_ARG;
  if (d->rows > 1L << 30 || d->vocab > 1 << 30) return NSA_E_UNSUPPORTED;
  // A slice: work-groups enough for the chip several times over, whole sweeps of the threads, two of them where there are rows enough
  const int sweep = kLogitsThreads * kRun;
  long slice = ((long)d->rows * d->vocab / 1024 + sweep - 1) / sweep * sweep;
  slice = std::max<long>(sweep, std::min<long>(slice, kSweeps * sweep));
  const long slices = (d->vocab + slice - 1) / slice;
  if (d->rows * slices >= 1L << 23) return NSA_E_UNSUPPORTED;
  LogitsArgs A{};
  A.x = x; A.row_stride = d->row_stride; A.vocab = d->vocab; A.slice = (int)slice; A.slices = (int)slices;
  A.history = d->history > 0 ? history : nullptr; A.length = d->history; A.history_lengths = history_lengths;
  A.repetition = repetition; A.frequency = frequency; A.presence = presence; A.temperature = temperature; A.bias = bias;
  A.rs = d->repetition_stride; A.fs = d->frequency_stride; A.ps = d->presence_stride; A.ts = d->temperature_stride;
  A.rep = d->repetition; A.freq = d->frequency; A.pres = d->presence; A.temp = d->temperature;
  A.bias_stride = d->bias_stride; A.allowed = allowed; A.allowed_kind = d->allowed_kind; A.allowed_stride = d->allowed_stride;
  A.out = out;
  hipStream_t st = (hipStream_t)stream;
  const unsigned groups = (unsigned)(d->rows * slices);
  const bool wide = d->history_int64 != 0;
  if (d->dtype == 0) logits_launch<__bf16>(A, wide, groups, st);
  else if (d->dtype == 1) logits_launch<_Float16>(A, wide, groups, st);
  else logits_launch<float>(A, wide, groups, st);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : (int)e;
}
