// Softmax cross entropy of a projection onto a vocabulary, l = x w^T, and its gradients, without the logits in memory.
//
//   loss_i = log sum_v exp(l[i][v] - l[i][t_i]),  G[i][v] = g_i (p[i][v] - [v == t_i]),  p[i][v] = exp(l[i][v]) / sum_u exp(l[i][u]),
//   dx = G w,  dw = G^T x
//
// Rows whose label is `ignore` are left out of everything: the others are gathered first (their order kept), so work goes by their number,
// which stays on the device, and what an ignored row holds (a NaN) reaches nothing.
// Where the label is the likely entry, its loss and its G are small beside what they are differences of.  So the other entries are summed by
// themselves: with the sum r of exp(l[i][v] - l[i][t_i]) over them, loss_i = log(1 + r) and the label's G is -g_i r / (1 + r) (a loss below 1e-6 was
// noise before, fp32 gradients of likely labels 1.8e-6 off instead of 2.5e-7).  An r that 64 bits do not tell from nothing beside 1 is nothing, as
// in a softmax computed in them: loss and the label's G are zero.  No G of a row is larger than g_i r / (1 + r), and each row's G is scaled by a
// power of two of its own, from that.  The row's maximum and the logarithm of its sum stay two numbers for the others' G.
//
// Forward: a tile of logits is made with the vocabulary along the registers of a lane and the tokens along the lanes, so a token's maximum
// and sum over a wave's 64 or 128 logits are a lane's own and one exchange of the wave's halves; the pairs (maximum, sum) of all waves'
// parts are merged by a second kernel.  Backward, piece by piece of the vocabulary: the logits again, G as fp16 (below), then both products.
//
// G in fp16: G 2^14 / max |G| of its row has 11 bits down to 2^-28 of the row's largest, against bf16's 8: with
// a bf16 G the gradients of a bf16 model were off by 1.4 times their own rounding, with this by 1.01.  dx, whose rows are sums along rows of G, takes
// the row's power of two out again; for dw, a sum over rows, a second copy of x is multiplied by what it is beside the largest row's.  (With one
// power of two for all rows, a row whose label is likely, or whose g is small, lost its others' G: a row with r = 1.2e-8 beside one with a loss
// near 1 had a dx off by several times its norm.)  The other operands of those products, w and x, are scaled by powers of two into fp16's range and
// lose nothing that is above 2^-29 of their largest value.
// fp32 operands are two fp16 planes each, G too (nsa_tiles.hpp); fp16 ones are exact in one beside two of G.
#include <algorithm>
#include <cmath>
#include "nsa_tiles.hpp"
#include "../../include/nsa_hip.h"

namespace nsa {

constexpr float kNothing = 0x1p-53f;      // beside 1
// A row's G is held times 2 to the power of this (up to 120: the exponential of a row whose g is zero stays finite)
__device__ __forceinline__ int grad_shift(unsigned largest) { return min(120, 14 - plane_exponent(largest)); }
// and a row of x for dw times 2 to the power of this: what the row's G has more than that of the row with the largest
__device__ __forceinline__ int weight_shift(int largest_rows, int row) { return min(0, largest_rows - row); }
// device words, of the state and of a backward pass: rows that count; bits of the largest finite |x|, |w| and |G|; slices of dx
enum { CELL_ROWS, CELL_X, CELL_W, CELL_G, CELL_SLICES, CELLS = 64 };
// Behind those of the state, for 16-bit types, the bits of the largest finite |x| that work-groups have found, each in one of 16 words 64 bytes apart: one word
// for all held up the copy of 8184 rows of 512 by 11 us.
constexpr int kMost = 16, kParts = 1024;
// the largest of `count` words is that of a matrix
struct LossFound {
  const unsigned* words;
  int count, stride;
};

// How logits are made: FEW rows as loss_few_kernel has them, the others by tiles of 64, 128 or 256 (loss_plan)
enum LossSize { FEW, TINY, MIDDLE, WIDE };

struct LossPlan {
  int n, npad, kp;                        // rows and their capacity (a multiple of 64), features padded to 64
  int P, grad_P;                          // planes of the operands of the forward, of the backward (ONE_BY_TWO: one of w and x, two of G)
  LossSize size;
  bool in_place;                          // the forward reads the weight where it lies
  int tile, part;                         // entries of the vocabulary of a tile, of a pair (maximum, sum)
  int fwd_rows, bwd_rows;                 // entries of a piece
  int w_splits, last_splits;              // slices of the rows that dw of a piece, of the last one, is summed from
  size_t state, fwd, bwd;                 // bytes
  size_t s_map, s_place, s_label, s_norm, s_own;                            // offsets in the state
  size_t f_part, f_target, f_loss, f_x, f_w, f_most, f_count;               // in the forward's workspace
  size_t b_cells, b_most, b_g, b_shift, b_x, b_xg, b_w, b_grad, b_dx, b_dw;  // in the backward's
};

static size_t up(size_t v, size_t to) { return (v + to - 1) / to * to; }

constexpr int kMaxSlices = 32, kSliceTiles = 512;      // of dx
constexpr int kRowsUncounted = 32768;                  // loss_rows_kernel

static int loss_plan(const nsa_loss_desc* d, const void* weight, LossPlan& p) {
  if (!d || d->rows < 0 || d->dim <= 0 || d->vocab <= 0 || d->dtype < 0 || d->dtype > 2 || d->reduction < 0 || d->reduction > 2) return NSA_E_ARG;
  if (d->x_stride < d->dim || d->w_stride < d->dim) return NSA_E_ARG;
  if (d->rows > (1 << 24) || d->dim > (1 << 16) || d->vocab > (1 << 24) || std::max<long>(d->rows, d->vocab) * up(d->dim, 64) >> 33) return NSA_E_UNSUPPORTED;
  p.n = (int)d->rows;
  p.npad = (int)up(std::max<size_t>(p.n, 1), 64);
  p.kp = (int)up(d->dim, 64);
  p.P = d->dtype == 2 ? 2 : 1;
  // fp16 results have as many bits as an fp16 G, and hang on single entries of it, the labels': its rounding would make them up to 1.41 times as far
  // off as their own alone, so fp16 takes two halves of G, a product more for dx and dw each.  (2047 rows, 768 features, 32000 entries: 720-760 us;
  // 475 with one half, and dw off by 1.2 times its own rounding.)  bf16 results have an eighth of G's bits: 1.01 times their rounding with one half.
  p.grad_P = d->dtype == 2 ? 2 : d->dtype == 1 ? ONE_BY_TWO : 1;
  // The tiles whose rounds end first: time of a round on all places, in us for each feature and beside that (products measured from 512 to 4096
  // features, the maxima and sums of a tile beside them).  256 x 256 tiles have no registers for sums in pieces (TileProduct::PIECES), so long
  // fp32 rows do without them: at 2066 features the gradients were 2.8e-6 off, 7 times as much as fp32 products by the library.  (4095 rows, 32000
  // entries: at 1088 features 4425 us and dx 2.0e-7 off, with 256 x 256 tiles 4002 us and 6.3e-7; at 2048 7073 and 2.0e-7, 5946 and 7.7e-7.  1021 rows of
  // 1024 features, forward: 265 us as 256 x 256 tiles, dx 4.1e-7 off; rows of 1088: 348 us without them, 304 with.)
  struct Cost { LossSize size; int tile, places; double each, beside; };
  static constexpr Cost one[3] = {{WIDE, 256, 256, 0.0272, 13.0}, {MIDDLE, 128, 256, 0.0085, 5.0}, {TINY, 64, 512, 0.0060, 3.5}};
  static constexpr Cost two[3] = {{WIDE, 256, 256, 0.0785, 13.0}, {MIDDLE, 128, 256, 0.0238, 5.0}, {TINY, 64, 512, 0.0210, 3.5}};
  // Up to 32 rows: loss_few_kernel (32 rows, 1024 features, 32000 entries: 20 us in bf16 and 35 in fp32, as tiles of 64 rows 30 and 105; 4096 features,
  // 131072 entries: 191 and 412 us, 196 and 1830).
  double least = 0.;
  p.size = FEW;
  for (const Cost& c : p.P == 2 ? two : one) {
    if (p.n <= 32 || (c.size == WIDE && p.P == 2 && p.kp > 1024)) continue;
    const double tiles = (double)(up(d->vocab, c.tile) / c.tile) * (up(p.npad, c.tile) / c.tile), time = std::ceil(tiles / c.places) * (p.kp * c.each + c.beside);
    if (p.size == FEW || time < least) {
      p.size = c.size;
      least = time;
    }
  }
  // Few rows: tiles of 32 entries, whose waves share the features, where those of 128 leave half the CUs idle.  (7 rows, 3542 features, 3870 entries in
  // fp32: 80 us with 128, 35 with 32; 24, 4096, 16000 in bf16: 41 and 41; 30000: 59 and 66.)
  const bool narrow = p.size == FEW && d->vocab < 16384;
  p.tile = p.size == WIDE ? 256 : p.size == TINY ? 64 : narrow ? 32 : 128;
  p.part = narrow || p.size == TINY ? 32 : p.size == MIDDLE ? 64 : 128;
  p.in_place = d->dtype != 2 && d->dim % 8 == 0 && d->dim >= 64 && d->w_stride % 8 == 0 && d->w_stride < (1 << 20) && ((uintptr_t)weight & 15) == 0;
  const size_t v256 = up(d->vocab, 256), v64 = up(d->vocab, 64), row = (size_t)p.kp * 2;
  p.fwd_rows = (int)std::min(v256, std::max<size_t>(256, ((size_t)256 << 20) / (row * p.P) / 256 * 256));
  // (a launch has fewer than 2^32 threads; backward pieces of more than 1024 entries are no larger than 2^27 values, others than 2^34)
  if (p.size != FEW) {
    const size_t entries = p.in_place ? d->vocab : std::min<size_t>(p.fwd_rows, d->vocab), side = p.tile;
    if ((up(entries, side) / side) * (up(p.n, side) / side) * (p.size == TINY ? 256 : 512) >> 32) return NSA_E_UNSUPPORTED;
  }
  const int planes = p.grad_P == 2 ? 2 : 1, g_planes = p.grad_P == 1 ? 1 : 2;
  // a piece's G: up to 256 MB
  p.bwd_rows = (int)std::min(v256, std::max<size_t>(1024, ((size_t)256 << 20) / ((size_t)g_planes * p.npad * 2) / 1024 * 1024));
  // gradients: tiles of 256 where the logits have them, else 128; as many slices as give every CU a tile
  const size_t tile = p.size == WIDE ? 256 : 128, piece = std::min<size_t>(p.bwd_rows, v64), last = (v64 - 1) % p.bwd_rows + 1;
  auto w_slices = [&](size_t entries) {
    return (int)std::max<size_t>(1, std::min<size_t>({kMaxSlices, 256 / (up(p.kp, tile) / tile * (up(entries, tile) / tile)), (size_t)p.npad / 256}));
  };
  p.w_splits = w_slices(piece);
  p.last_splits = w_slices(last);
  size_t at = CELLS * 4 + kMost * 64;
  auto take = [&](size_t bytes) { const size_t here = at; at = up(at + bytes, 256); return here; };
  p.s_map = take((size_t)p.npad * 4);
  p.s_place = take((size_t)p.npad * 4);
  p.s_label = take((size_t)p.npad * 4);
  p.s_norm = take((size_t)p.npad * 8);
  p.s_own = take((size_t)p.npad * 4);
  p.state = at;
  at = 0;
  p.f_part = take(up(d->vocab, p.tile) / p.part * (size_t)p.npad * 8);
  p.f_target = take((size_t)p.npad * 4);
  p.f_loss = take((size_t)p.npad * 4);
  p.f_x = take(p.size == FEW ? 0 : p.npad * row * p.P);
  p.f_w = take(p.size == FEW || p.in_place ? 0 : p.fwd_rows * row * p.P);
  p.f_most = take(d->dtype == 2 ? 2 * kParts * 4 : 0);
  p.f_count = take(p.n > kRowsUncounted ? (size_t)(p.npad + 1023) / 1024 * 4 : 0);
  p.fwd = at;
  at = 0;
  p.b_cells = take(CELLS * 4);
  p.b_most = take((2 * kParts + (size_t)(p.npad + 1023) / 1024) * 4);
  p.b_g = take((size_t)p.npad * 4);
  p.b_shift = take((size_t)p.npad * 4);
  p.b_x = take(p.npad * row * planes);
  p.b_xg = take(p.npad * row * planes);
  p.b_w = take(p.bwd_rows * row * planes);
  p.b_grad = take((size_t)g_planes * p.npad * p.bwd_rows * 2);
  // (rows of the slices: no more than kSliceTiles tiles of them where there are two or more)
  p.b_dx = take(std::max<size_t>((size_t)p.npad * p.kp, std::min<size_t>((size_t)kMaxSlices * p.npad * p.kp, kSliceTiles * tile * tile)) * 4);
  p.b_dw = take(std::max<size_t>(p.w_splits > 1 ? p.w_splits * piece : 0, p.last_splits > 1 ? p.last_splits * last : 0) * p.kp * 4);
  p.bwd = at;
  return 0;
}

// ------------------------------------------------------------------------------------ rows that count

__device__ __forceinline__ long label_at(const void* labels, int is64, int i) { return is64 ? ((const long*)labels)[i] : (long)((const int*)labels)[i]; }
// counts[b]: rows among 1024 b .. 1024 b + 1023 that count
__global__ __launch_bounds__(256) void loss_count_kernel(const void* labels, int is64, int n, long ignore, int* counts) {
  __shared__ int sums[4];
  const int tid = threadIdx.x;
  int count = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int row = blockIdx.x * 1024 + e * 256 + tid;
    count += row < n && label_at(labels, is64, row) != ignore;
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) count += __shfl_xor(count, o);
  if ((tid & 63) == 0) sums[tid >> 6] = count;
  __syncthreads();
  if (tid == 0) counts[blockIdx.x] = sums[0] + sums[1] + sums[2] + sums[3];
}
// map[c] = row of the c-th row that counts, label[c] = its label (-1: outside the vocabulary), place[row] = c or -1.  A work-group takes
// 1024 rows; how many count before them it finds out itself, from the labels (8 bytes a row from L2, and no second launch) or, of
// many rows, from counts of 1024 each.  (From labels 16384 rows take 7 us, 32768 10, 65536 17, 4194304 5.7 ms; from counts, with their kernel,
// 65536 6 us and 4194304 29.)
__global__ __launch_bounds__(256) void loss_rows_kernel(const void* labels, int is64, int n, int vocab, long ignore, const int* counts, int* map, int* place,
                                                        int* label, unsigned* cells, float* losses) {
  __shared__ int sums[8];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, first = blockIdx.x * 1024;
  auto at = [&](int i) { return label_at(labels, is64, i); };
  int before = 0;
  if (counts != nullptr) {
#pragma unroll 8
    for (int i = tid; i < (int)blockIdx.x; i += 256) before += counts[i];
  } else {
#pragma unroll 8
    for (int i = tid; i < first; i += 256) before += at(i) != ignore;
  }
  long mine[4];
  int count = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int row = first + 4 * tid + e;
    mine[e] = row < n ? at(row) : ignore;
    count += mine[e] != ignore;
  }
  int upto = count;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    before += __shfl_xor(before, o);
    const int other = __shfl_up(upto, o);
    if (lane >= o) upto += other;
  }
  if (lane == 63) { sums[wave] = before; sums[4 + wave] = upto; }
  __syncthreads();
  int c = sums[0] + sums[1] + sums[2] + sums[3] + upto - count, total = sums[0] + sums[1] + sums[2] + sums[3];
  for (int w = 0; w < 4; ++w) {
    c += w < wave ? sums[4 + w] : 0;
    total += sums[4 + w];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int row = first + 4 * tid + e;
    if (row >= n) break;
    const bool counts = mine[e] != ignore;
    place[row] = counts ? c : -1;
    if (counts) {
      map[c] = row;
      label[c] = mine[e] >= 0 && mine[e] < vocab ? (int)mine[e] : -1;
      ++c;
    } else if (losses != nullptr) {
      losses[row] = 0.f;
    }
  }
  if (blockIdx.x == gridDim.x - 1 && tid == 0) cells[CELL_ROWS] = (unsigned)total;
  if (blockIdx.x == 0 && tid < kMost) cells[CELLS + 16 * tid] = 0;
}

// up to 8 values of a row, zeros past its end
template <class S> __device__ __forceinline__ void load_values(const S* p, int have, float (&v)[8]) {
  if (have >= 8) {
    const auto a = load_any<16 / sizeof(S)>(p), b = load_any<16 / sizeof(S)>(p + 8 - 16 / sizeof(S));      // (of 16 bits: the same)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)(e < (int)(16 / sizeof(S)) ? a[e] : b[e - (8 - 16 / (int)sizeof(S))]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < have ? (float)p[e] : 0.f;
  }
}

__device__ __forceinline__ unsigned finite_bits(float v) {
  const unsigned u = __builtin_bit_cast(unsigned, v) & 0x7fffffffu;
  return u < 0x7f800000u ? u : 0u;
}
// the largest of the work-group's values
__device__ __forceinline__ unsigned largest_of(unsigned best) {
  __shared__ unsigned best_s[4];
  __syncthreads();
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) best = max(best, (unsigned)__shfl_xor((int)best, o));
  if ((threadIdx.x & 63) == 0) best_s[threadIdx.x >> 6] = best;
  __syncthreads();
  return max(max(best_s[0], best_s[1]), max(best_s[2], best_s[3]));
}
__device__ __forceinline__ unsigned largest_of(const LossFound& f) {
  if (f.count == 1) return *f.words;
  unsigned best = 0;
  for (int i = threadIdx.x; i < f.count; i += 256) best = max(best, f.words[i * f.stride]);
  return largest_of(best);
}
// Into one of `words`.  (Whoever finds a larger one there already has nothing to say: with an atomic a wave, 16384 of them on one address, the
// kernel took 100 us for 8 MB.)
__device__ __forceinline__ void largest_into(unsigned best, unsigned* words, int block) {
  best = largest_of(best);
  unsigned* word = words + 16 * (block % kMost);
  if (threadIdx.x == 0 && best > __hip_atomic_load(word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) atomicMax(word, best);
}

// A matrix, or the rows of it that map names, whose largest finite |value| is to be known: that of each work-group's part
struct LossMost {
  const void* src;
  long ld;
  int rows, cols;
  const int* map;
  const unsigned* count;
  unsigned* parts;
  int blocks;
};
struct LossBegin {
  LossMost of[2];
  // the backward's weights (work-groups behind those): g of the rows that count, the power of two that their G is scaled by, and of each 1024 of
  // them the bits of the largest finite |G|
  const float* dloss;
  int reduction;
  const int* map;
  const unsigned* count;
  const float* own;
  float* g;
  int* row_shift;
  unsigned* most;
};
// What has to be known of the operands before they are copied
template <class S>
__global__ __launch_bounds__(256) void loss_begin_kernel(const LossBegin G) {
  const int second = (int)blockIdx.x - G.of[0].blocks, third = second - G.of[1].blocks;
  unsigned best = 0;
  if (third >= 0) {
    const int live = (int)*G.count;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = third * 1024 + e * 256 + threadIdx.x;
      if (i >= live) break;
      const float v = G.reduction == 0 ? G.dloss[G.map[i]] : G.reduction == 1 ? G.dloss[0] / (float)live : G.dloss[0];
      G.g[i] = v;
      const float size = v * G.own[i];
      const unsigned bits = finite_bits(size);
      G.row_shift[i] = bits != 0 || size == 0.f ? grad_shift(bits) : 0;      // (what is not finite stays that)
      best = max(best, bits);
    }
    best = largest_of(best);
    if (threadIdx.x == 0) G.most[third] = best;
    return;
  }
  const LossMost& M = G.of[second >= 0];
  const int block = second >= 0 ? second : (int)blockIdx.x;
  const S* src = (const S*)M.src;
  const int live = M.count != nullptr ? (int)*M.count : M.rows;
  const bool flat = M.map == nullptr && M.ld == M.cols;      // one run of values
  const unsigned per = (M.cols + 7) / 8;
  const long total = (long)live * M.cols, pieces = flat ? (total + 7) / 8 : (long)live * per;
#pragma unroll 4
  for (long i = (long)block * 256 + threadIdx.x; i < pieces; i += (long)M.blocks * 256) {
    float v[8];
    if (flat) {
      load_values(src + 8 * i, (int)min(8L, total - 8 * i), v);
    } else {
      const unsigned r = (unsigned)i / per, c = ((unsigned)i - r * per) * 8;
      load_values(src + (M.map != nullptr ? M.map[r] : (int)r) * M.ld + c, M.cols - (int)c, v);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) best = max(best, finite_bits(v[e]));
  }
  best = largest_of(best);
  if (threadIdx.x == 0) M.parts[block] = best;
}

// Rows (named by map, or all) as planes of kp columns, those past `cols` zero; rows past the last one up to a multiple of 64 zero too.
// found: the values are scaled below 2^15 by the power of two that suits the largest (none, or as_is: they are not).  most: their own largest
// goes there.  weighted: a second copy, scaled, of rows times what they weigh in dw (weight_shift).  back: the last 64 columns end with the row's
// last value, `back` zeros before what is left (TileProduct::run).
struct LossRows {
  const void* src;
  long ld;
  int rows, cols;
  const int* map;
  const unsigned* count;
  LossFound found;
  void* dst;
  long plane;
  unsigned* most;
  int back, blocks;
  bool as_is;
  void* weighted;
  const int* row_shift;
  LossFound rows_most;      // of |G|
};
struct LossCopy {
  LossRows of[2];
  int kp;
  // The first copy of a pass: one more work-group leaves the largest of both matrices here, and in a backward pass that of G (`most`: of
  // each 1024) and the slices of a piece's entries that dx is summed from
  unsigned* cells;
  LossFound most;
  const unsigned* count;
  int tiles_m, tile, piece;
};
// Slices of dx: those whose rounds on 256 CUs end first, where a tile's beginning and end, and its share of the sum of slices, cost as much as 512
// entries.  The rows that count decide, so they are chosen here.  (8192 rows, 40 % of them ignored, 1024 features, 50021 entries: 80 tiles in 2 slices
// as for all rows 695 us, in 3 of them 600.)
__device__ __forceinline__ void loss_cells(const LossCopy& G) {
  const int tid = threadIdx.x;
  for (int i = 0; i < 2; ++i)
    if (G.of[i].found.words != nullptr) {
      const unsigned best = largest_of(G.of[i].found);
      if (tid == 0) G.cells[i == 0 ? CELL_X : CELL_W] = best;
    }
  if (G.most.words == nullptr) return;
  const int live = (int)*G.count;
  const unsigned best = largest_of(G.most);
  if (tid == 0) G.cells[CELL_G] = best;
  if (tid < kMaxSlices) {
    const int n = tid + 1, tiles = G.tiles_m * ((live + G.tile - 1) / G.tile), rounds = (tiles * n + 255) / 256;
    long time = n > 1 && (tiles * n > kSliceTiles || G.piece / n < 512) ? 1L << 50 : (long)rounds * (G.piece / n + 512);
    time = time * 64 + n;
#pragma unroll
    for (int o = 1; o < kMaxSlices; o <<= 1) time = min(time, (long)__shfl_xor(time, o));
    if (tid == 0) G.cells[CELL_SLICES] = (unsigned)(time & 63);
  }
}
// (four times 8 values a thread: with one, finding the scale was a fifth of the time)
constexpr int kCopies = 4;
template <class S, class D, int P>
__global__ __launch_bounds__(256) void loss_planes_kernel(const LossCopy G) {
  if (G.cells != nullptr && (int)blockIdx.x == G.of[0].blocks + G.of[1].blocks) {
    loss_cells(G);
    return;
  }
  const bool second = (int)blockIdx.x >= G.of[0].blocks;
  const LossRows& M = G.of[second];
  const unsigned block = blockIdx.x - (second ? G.of[0].blocks : 0), per = G.kp / 8, first = block * kCopies * 256 + threadIdx.x;      // (below 2^31: loss_plan)
  const int live = M.count != nullptr ? (int)*M.count : M.rows, pad = (live + 63) / 64 * 64;
  if (block * kCopies * 256 / per >= (unsigned)pad) return;
  float v[kCopies][8];
  unsigned best = 0;
#pragma unroll
  for (int u = 0; u < kCopies; ++u) {
    const unsigned i = first + u * 256;
    const int r = (int)(i / per), c = (int)(i - r * per) * 8, from = M.back > 0 && c >= G.kp - 64 ? c - M.back : c;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[u][e] = 0.f;
    if (r < live && from < M.cols && (from == c || from >= G.kp - 64))
      load_values((const S*)M.src + (M.map != nullptr ? M.map[r] : r) * M.ld + from, M.cols - from, v[u]);
  }
  if (M.most != nullptr) {
#pragma unroll
    for (int u = 0; u < kCopies; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) best = max(best, finite_bits(v[u][e]));
    largest_into(best, M.most, block);
  }
  const int scale = M.found.words != nullptr ? plane_shift(largest_of(M.found)) : 0, shift = M.as_is ? 0 : scale;
  auto store = [&](void* dst, int u, int r, int c, int by) {
    typename PlaneVec<D>::x8 hi, lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = by != 0 ? __builtin_ldexpf(v[u][e], by) : v[u][e];
      if constexpr (P == 2) {
        const Halves s = halves_of(x);
        hi[e] = s.hi;
        lo[e] = s.lo;
      } else {
        hi[e] = (D)x;
      }
    }
    D* to = (D*)dst + (long)r * G.kp + c;
    *reinterpret_cast<decltype(hi)*>(to) = hi;
    if (P == 2) *reinterpret_cast<decltype(lo)*>(to + M.plane) = lo;
  };
  const int largest_rows = M.weighted != nullptr ? grad_shift(largest_of(M.rows_most)) : 0;
#pragma unroll
  for (int u = 0; u < kCopies; ++u) {
    const unsigned i = first + u * 256;
    const int r = (int)(i / per), c = (int)(i - r * per) * 8;
    if (r >= pad) break;
    store(M.dst, u, r, c, shift);
    if (M.weighted != nullptr) store(M.weighted, u, r, c, scale + (r < live ? weight_shift(largest_rows, M.row_shift[r]) : 0));
  }
}

// ------------------------------------------------------------------------------------ tiles of logits

struct LossTileArgs {
  const void *w, *x;
  long w_plane, w_ld, x_plane;
  int kp, v0, vend;                        // the piece: entries v0 .. vend - 1
  int tail, back;                          // see TileProduct::run; tail in features
  int n, tiles_m;
  const unsigned *count, *x_cell, *w_cell;  // cells: null where the planes are not scaled
  const int* label;
  float2* part;                            // [parts][npad]
  float* target;
  int npad;
  // backward
  const float2* norm;                      // maximum, log2 of the sum
  const float *own, *g;                    // -r / (1 + r)
  const int* row_shift;
  _Float16* grad;                          // [grad_planes][npad][grad_ld]
  long grad_plane;
  int grad_ld, grad_planes;
};

// One tile: TM entries of the vocabulary (registers) by TN tokens (lanes).  GRAD: G of the tile; else its maxima, sums and the labels' logits.
template <class Tiles, bool GRAD>
__global__ __launch_bounds__(Tiles::THREADS, 2) void loss_tile_kernel(const LossTileArgs G) {
  typedef typename Tiles::T T;
  __shared__ __align__(1024) char shared[Tiles::LDS];
  // (the grid is for all rows; of the tiles that have any, each XCD gets its share)
  const int live = (int)*G.count, tiles_n = ((GRAD ? (live + 63) / 64 * 64 : live) + Tiles::TN - 1) / Tiles::TN;
  if ((int)blockIdx.x >= G.tiles_m * tiles_n) return;
  const TileAt tile = tile_at(blockIdx.x, G.tiles_m, tiles_n, 4);
  const int m0 = G.v0 + tile.m * Tiles::TM, n0 = tile.n * Tiles::TN;
  if (n0 >= live) {
    // rows of G up to a multiple of 64 are read as the contraction index of dw
    if (GRAD) {
      const int width = min(Tiles::TM, G.grad_ld - tile.m * Tiles::TM) / 8;
      for (int i = threadIdx.x; i < G.grad_planes * Tiles::TN * width; i += Tiles::THREADS) {
        const int row = i / width % Tiles::TN, plane = i / width / Tiles::TN;
        *reinterpret_cast<uintx4*>(G.grad + plane * G.grad_plane + (size_t)(n0 + row) * G.grad_ld + tile.m * Tiles::TM + i % width * 8) = uintx4{0u, 0u, 0u, 0u};
      }
    }
    return;
  }
  Tiles t;
  t.init(shared);
  t.operand_a((const T*)G.w, G.w_plane, G.w_ld, tile.m * Tiles::TM, G.vend - G.v0);
  t.operand_b((const T*)G.x, G.x_plane, G.kp, n0, live);
  t.run(G.kp / Tiles::BK, 0, G.back > 0 ? G.tail / Tiles::BK : -1, G.back);

  constexpr bool SCALED = Tiles::P == 2 || GRAD;
  const int unscale = SCALED && G.x_cell != nullptr ? -(plane_shift(*G.x_cell) + plane_shift(*G.w_cell)) : 0;
  const bool cut = m0 + Tiles::TM > G.vend;      // entries past the last one
  constexpr int PART = Tiles::TM / Tiles::WM;
#pragma unroll
  for (int j = 0; j < Tiles::NI; ++j) {
    const int token = n0 + t.col_of(j);
    const bool ok = token < live;
    const int label = ok ? G.label[token] : -1, own = label - (m0 + t.wm * PART);      // in this wave's part
    const bool hit = label >= 0 && own >= 0 && own < PART && ((own >> 2) & 1) == (t.lane >> 5);
    if (SCALED) {
#pragma unroll
      for (int i = 0; i < Tiles::MI; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) t.acc[i][j][e] = __builtin_ldexpf(t.acc[i][j][e], unscale);
    }
    if (!GRAD) {
      if (cut) {
#pragma unroll
        for (int i = 0; i < Tiles::MI; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (m0 + t.row_of(i, e >> 2) + (e & 3) >= G.vend) t.acc[i][j][e] = -INFINITY;
      }
      if (__any(hit)) {
        float found = 0.f;
#pragma unroll
        for (int i = 0; i < Tiles::MI; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) {      // (the label is none of the entries that are summed)
            const bool it = hit && own == 32 * i + 8 * (e >> 2) + 4 * (t.lane >> 5) + (e & 3);
            found = it ? t.acc[i][j][e] : found;
            t.acc[i][j][e] = it ? -INFINITY : t.acc[i][j][e];
          }
        if (hit) G.target[token] = found;
      }
      float top = t.acc[0][j][0];
#pragma unroll
      for (int i = 0; i < Tiles::MI; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, t.acc[i][j][e]);
      top = halves_max(top);
      const float from = top > -INFINITY ? top : 0.f;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < Tiles::MI; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) sum += fast_exp2((t.acc[i][j][e] - from) * kLog2e);
      sum = halves_sum(sum);
      if (ok && t.lane < 32) G.part[(size_t)((m0 / PART) + t.wm) * G.npad + token] = make_float2(top, sum);
    } else {
      const int pad = (live + 63) / 64 * 64;
      const float2 norm = ok ? G.norm[token] : make_float2(0.f, 0.f);
      const int g_shift = ok ? G.row_shift[token] : 0;
      const float g = ok ? G.g[token] : 0.f, shift = (float)g_shift - norm.y;
#pragma unroll
      for (int i = 0; i < Tiles::MI; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) t.acc[i][j][e] = ok ? g * fast_exp2(__builtin_fmaf(t.acc[i][j][e] - norm.x, kLog2e, shift)) : 0.f;
      if (__any(hit)) {
        const float of_label = hit ? G.own[token] : 0.f, at_label = __builtin_fabsf(of_label) < kNothing ? 0.f : __builtin_ldexpf(g * of_label, g_shift);
#pragma unroll
        for (int i = 0; i < Tiles::MI; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (hit && own == 32 * i + 8 * (e >> 2) + 4 * (t.lane >> 5) + (e & 3)) t.acc[i][j][e] = at_label;
      }
      if (cut) {
#pragma unroll
        for (int i = 0; i < Tiles::MI; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (m0 + t.row_of(i, e >> 2) + (e & 3) >= G.vend) t.acc[i][j][e] = 0.f;
      }
      if (token >= pad) continue;
#pragma unroll
      for (int i = 0; i < Tiles::MI; ++i) {
        const int col = tile.m * Tiles::TM + t.wm * PART + 32 * i;
        if (col >= G.grad_ld) break;
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
          f16x4 hi[2], lo[2];
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float v = t.acc[i][j][4 * (q + u) + e];
              const Halves s = halves_of(v);
              hi[u][e] = s.hi;
              lo[u][e] = s.lo;
            }
          _Float16* at = G.grad + (size_t)token * G.grad_ld + col + 8 * q + 8 * (t.lane >> 5);
          *reinterpret_cast<uintx4*>(at) = join_quads(__builtin_bit_cast(uintx2, hi[0]), __builtin_bit_cast(uintx2, hi[1]));
          if (G.grad_planes == 2) *reinterpret_cast<uintx4*>(at + G.grad_plane) = join_quads(__builtin_bit_cast(uintx2, lo[0]), __builtin_bit_cast(uintx2, lo[1]));
        }
      }
    }
  }
}

// ------------------------------------------------------------------------------------ few rows

// Up to 32 rows (scoring, decoding): one pass over the weight where it lies, of any type and alignment, is all their time.  Tiles of 128 entries by
// 32 rows, 128 bytes of each at a time in LDS (swizzled as TileOperand's); NARROW: of 32 entries, 128 bytes for each wave at a time.  Rows that begin at multiples of 16 bytes are copied there three
// stages ahead of their use (24 rows of 4096 features, 131072 entries in bf16, 1.07 GB: 5.8 TB/s); others go through registers, a stage ahead
// (a row of 1675, 88295 entries in fp16: 3.7 TB/s with three work-groups a CU, 3.4 with two).  fp32 takes fp32 products (32 x 32 x 2: half the time that the weight takes from memory), so there are no planes.  Every
// work-group finds out the rows that count by itself.
struct LossFewArgs {
  const void *x, *w, *labels;
  long x_ld, w_ld, ignore;
  int is64, n, dim, vocab, npad;
  int *map, *place, *label;
  unsigned* cells;
  float2* part;
  float *target, *losses;
};
template <class S, bool ALIGNED, bool NARROW>
__global__ __launch_bounds__(256, ALIGNED || NARROW ? 2 : 3) void loss_few_kernel(const LossFewArgs G) {
  // rows of 128 bytes: entries, then rows of x, of NARROW for each wave.  (All of LDS is the stages: two work-groups fit into a CU, one if NARROW)
  constexpr int STAGES = ALIGNED ? 4 : 2, LOADS = NARROW ? 8 : 5, STAGE = LOADS * 32 * 128;
  __shared__ __align__(1024) char stage_s[STAGES][STAGE];
  int* map_s = reinterpret_cast<int*>(stage_s[0]);
  float(*top_s)[32] = reinterpret_cast<float(*)[32]>(stage_s[0]), (*sum_s)[32] = top_s + 4;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5, token = lane & 31;
  const long given = lane < G.n ? (G.is64 ? ((const long*)G.labels)[lane] : (long)((const int*)G.labels)[lane]) : G.ignore;
  const bool counts = given != G.ignore;
  const unsigned long mask = __ballot(counts);
  const int live = __popcll(mask), c = __popcll(mask & ((1ul << lane) - 1)), label = given >= 0 && given < G.vocab ? (int)given : -1;
  if (wave == 0 && counts) {
    map_s[c] = lane;
    map_s[32 + c] = label;
  }
  if (blockIdx.x == 0 && wave == 0) {
    if (lane < G.n) G.place[lane] = counts ? c : -1;
    if (counts) {
      G.map[c] = lane;
      G.label[c] = label;
    } else if (G.losses != nullptr && lane < G.n) {
      G.losses[lane] = 0.f;
    }
    if (lane == 0) G.cells[CELL_ROWS] = (unsigned)live;
  }
  if (live == 0) return;
  __syncthreads();

  // (an XCD takes neighbouring tiles: 4.8 TB/s with every eighth of them)
  const int tile = xcd_run(blockIdx.x, gridDim.x), first = tile * (NARROW ? 32 : 128), m0 = first + (NARROW ? 0 : 32 * wave), dim = G.dim;
  constexpr int V = 16 / sizeof(S), K = 8 * V, BK = NARROW ? 4 * K : K;      // values of 16 bytes, of 128, of a stage
  typedef decltype(load_any<V>((const S*)nullptr)) vec;
  // this thread's 16 bytes of each load: of every 32nd entry and one row of x, or of one entry and one row of x, 128 bytes on for each wave
  const int r0 = tid >> 3, swz = (r0 >> 1) & 7, chunk = ALIGNED ? (tid & 7) ^ swz : tid & 7;
  const S *src[LOADS], *x_row = (const S*)G.x + (long)map_s[min(r0, live - 1)] * G.x_ld + chunk * V;
#pragma unroll
  for (int u = 0; u < LOADS; ++u) {
    const bool of_x = NARROW ? u & 1 : u == 4;
    src[u] = of_x ? x_row : (const S*)G.w + (long)min(first + r0 + (NARROW ? 0 : 32 * u), G.vocab - 1) * G.w_ld + chunk * V;
    if (NARROW) src[u] += (u >> 1) * K;
  }
  const int own = token < live ? map_s[32 + token] - m0 : -1;
  __syncthreads();
  char* to = &stage_s[0][0] + r0 * 128 + 16 * (chunk ^ swz);
  vec held[2][LOADS];
  floatx16 part[4], acc = zero_acc();      // sums in parts: each of 64 products, then theirs
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) part[ks] = zero_acc();
  auto store = [&](const vec (&v)[LOADS], int buf) {
#pragma unroll
    for (int u = 0; u < LOADS; ++u) *reinterpret_cast<vec*>(to + buf * STAGE + u * 32 * 128) = v[u];
  };
  auto products = [&](int buf) {
    const char *row = stage_s[buf] + token * 128 + (NARROW ? wave * 64 * 128 : 0), *entry = row + (NARROW ? 0 : wave * 32 * 128), *x = row + (NARROW ? 32 : 128) * 128;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      const int at = 16 * ((2 * ks + h) ^ ((token >> 1) & 7));
      const vec a = *reinterpret_cast<const vec*>(entry + at), b = *reinterpret_cast<const vec*>(x + at);
      if constexpr (sizeof(S) == 4) {
#pragma unroll
        for (int e = 0; e < 4; ++e) part[ks] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], part[ks], 0, 0, 0);
      } else {
        part[ks] = mma(a, b, part[ks]);
      }
    }
  };
  auto piece = [&](int k) {      // (sums in pieces: see TileProduct::PIECES)
    if (k % (NARROW ? 1024 : 256) == 0) {
      acc += (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) part[ks] = zero_acc();
    }
  };
  int k = 0;
  if constexpr (ALIGNED) {
    typedef __attribute__((address_space(3))) void* lds_p;
    const unsigned mine = __builtin_amdgcn_readfirstlane((unsigned)(unsigned long)(lds_p)stage_s + wave * 1024);
    const int stages = dim / BK;
    // (a stage past the last one: no lane takes part)
    auto copy = [&](int t) {
      const unsigned lanes = __builtin_amdgcn_readfirstlane(t < stages ? ~0u : 0u);
#pragma unroll
      for (int u = 0; u < LOADS; ++u)
        asm volatile("s_mov_b32 m0, %0\n\ts_mov_b64 vcc, exec\n\ts_mov_b32 exec_lo, %2\n\ts_mov_b32 exec_hi, %2\n\ts_nop 0\n\t"
                     "global_load_lds_dwordx4 %1, off\n\ts_mov_b64 exec, vcc"
                     :: "s"(mine + (t & 3) * STAGE + u * 32 * 128), "v"(src[u] + t * BK), "s"(lanes) : "memory", "m0", "vcc");
    };
#pragma unroll
    for (int t = 0; t < 3; ++t) copy(t);
    for (int t = 0; t < stages; ++t, k += BK) {
      fence();
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(2 * LOADS) : "memory");
      fence();
      copy(t + 3);
      products(t & 3);
      piece(k + BK);
    }
    fence();
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    fence();
  } else {
    // (No branch around a load - behind the last one it is read again - or every use of one waits for all of them.  A buffer is written again
    // when all have passed the barrier behind its reading.)
    const int pairs = dim / (2 * BK) * (2 * BK);
    auto load = [&](int at, vec (&into)[LOADS]) {
#pragma unroll
      for (int u = 0; u < LOADS; ++u) into[u] = load_any<V>(src[u] + at);
    };
    if (pairs > 0) {
      load(0, held[0]);
      load(BK, held[1]);
      for (; k < pairs; k += 2 * BK) {
        const int next = min(k + 2 * BK, pairs - 2 * BK);
        store(held[0], 0);
        load(next, held[0]);
        __syncthreads();
        products(0);
        store(held[1], 1);
        load(next + BK, held[1]);
        __syncthreads();
        products(1);
        piece(k + 2 * BK);
      }
    }
  }
  for (; k < dim; k += BK) {      // what is left of the rows
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      const int have = dim - (k + (NARROW ? (u >> 1) * K : 0) + chunk * V);
      if (have >= V) {
        held[0][u] = load_any<V>(src[u] + k);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) held[0][u][e] = e < have ? src[u][k + e] : (S)0.f;
      }
    }
    __syncthreads();
    store(held[0], 0);
    __syncthreads();
    products(0);
  }
  acc += (part[0] + part[1]) + (part[2] + part[3]);
  if (NARROW) {
    // the waves' parts of the sums, in their order
    float* sums = reinterpret_cast<float*>(stage_s[0]) + lane;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 16; ++e) sums[(wave * 16 + e) * 64] = acc[e];
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = (sums[e * 64] + sums[(16 + e) * 64]) + (sums[(32 + e) * 64] + sums[(48 + e) * 64]);
  }

  float top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int row = 8 * (e >> 2) + 4 * h + (e & 3);
    if (row == own && (!NARROW || wave == 0)) G.target[token] = acc[e];
    if (row == own || m0 + row >= G.vocab) acc[e] = -INFINITY;      // (the label is none of the entries that are summed)
    top = fmaxf(top, acc[e]);
  }
  top = halves_max(top);
  const float from = top > -INFINITY ? top : 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) sum += fast_exp2((acc[e] - from) * kLog2e);
  sum = halves_sum(sum);
  __syncthreads();
  if (h == 0) {
    top_s[wave][token] = top;
    sum_s[wave][token] = sum;
  }
  __syncthreads();
  if (tid >= live) return;
  float most = -INFINITY, s = 0.f;
#pragma unroll
  for (int v = 0; v < (NARROW ? 1 : 4); ++v) most = fmaxf(most, top_s[v][tid]);
  const float at = most > -INFINITY ? most : 0.f;
#pragma unroll
  for (int v = 0; v < (NARROW ? 1 : 4); ++v) s += sum_s[v][tid] * fast_exp2((top_s[v][tid] - at) * kLog2e);
  G.part[(size_t)blockIdx.x * G.npad + tid] = make_float2(most, s);
}

// norm and loss of TOKENS tokens from the parts' maxima and sums: 256 / TOKENS threads a token.  (8 of them read whole 64 bytes; 2 end a long
// vocabulary's parts sooner where there are not many: 24 tokens, 4096 parts 16 -> 6 us.)
template <int TOKENS>
__global__ __launch_bounds__(256) void loss_merge_kernel(const float2* part, int parts, int npad, const unsigned* count, const int* map, const int* label,
                                                         const float* target, float2* norm, float* own, float* loss, float* losses) {
  constexpr int LANES = 256 / TOKENS;
  __shared__ float top_s[LANES][TOKENS], sum_s[LANES][TOKENS];
  const int live = (int)*count, tid = threadIdx.x, at = tid % TOKENS, lane = tid / TOKENS, token = blockIdx.x * TOKENS + at;
  if (blockIdx.x * TOKENS >= (unsigned)live) return;
  float top = -INFINITY, sum = 0.f;
  auto add = [&](float m, float s) {
    const float most = fmaxf(top, m), from = most > -INFINITY ? most : 0.f;
    sum = sum * fast_exp2((top - from) * kLog2e) + s * fast_exp2((m - from) * kLog2e);
    top = most;
  };
  if (token < live) {
#pragma unroll 8
    for (int p = lane; p < parts; p += LANES) {
      const float2 v = part[(size_t)p * npad + token];
      add(v.x, v.y);
    }
  }
  top_s[lane][at] = top;
  sum_s[lane][at] = sum;
  for (int half = LANES / 2; half > 0; half /= 2) {
    __syncthreads();
    if (lane < half) {
      add(top_s[lane + half][at], sum_s[lane + half][at]);
      top_s[lane][at] = top;
      sum_s[lane][at] = sum;
    }
  }
  if (lane != 0 || token >= live) return;
  // the others' sum and the label's exponential, both from the larger maximum (no entry of the vocabulary: NaN, in the loss and all gradients; an
  // infinite logit too)
  const float at_label = label[token] < 0 ? __builtin_nanf("") : target[token], from = fmaxf(top, at_label) + (at_label - at_label);
  const float others = sum > 0.f ? sum * expf(top - from) : sum, all = others + expf(at_label - from);
  const float value = at_label >= top ? (others < kNothing ? 0.f : log1pf(others)) + (at_label - at_label) : (top - at_label) + logf(all);
  norm[token] = make_float2(from, log2f(all));
  own[token] = -others / all;
  loss[token] = value;
  if (losses != nullptr) losses[map[token]] = value;
}

// the sum of the losses, or their mean (of none: NaN)
__global__ __launch_bounds__(1024) void loss_sum_kernel(const float* loss, const unsigned* count, int mean, float* out) {
  __shared__ double sums[16];
  const int live = (int)*count;
  double s = 0.0;
#pragma unroll 4
  for (int i = threadIdx.x; i < live; i += 1024) s += loss[i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < 16; ++w) s += sums[w];
  *out = (float)(mean ? s / live : s);
}

// ------------------------------------------------------------------------------------ gradients

struct LossGradArgs {
  const _Float16 *grad, *w, *x;       // G [npad][grad_ld]; w [piece][kp]; x [npad][kp], weighted
  long grad_plane, w_plane, x_plane;
  int grad_ld, kp, tiles_m, entries;
  const unsigned *count, *w_cell, *x_cell, *g_cell;
  const int* row_shift;
  // dx
  float* sums;                        // [slices][live rows up to a multiple of 64][kp]
  int first;                          // first piece
  const unsigned* slices;
  // dw: the first dw_tiles work-groups
  int dw_tiles, tiles_n, splits, dim;
  void* dw;
  long dw_ld;
};

// dx, one slice of the piece's vocabulary: features (registers) by tokens (lanes), unscaled, added to what the pieces before gave
template <class Tiles>
__device__ __forceinline__ void loss_dx(const LossGradArgs& G, char* shared) {
  const int live = (int)*G.count, tiles_n = (live + Tiles::TN - 1) / Tiles::TN, tiles = G.tiles_m * tiles_n, splits = (int)*G.slices;
  const int id = (int)blockIdx.x - G.dw_tiles;
  if (id >= tiles * splits) return;
  const int nth = xcd_run(id, tiles * splits), split = nth / tiles;
  const TileAt tile = tile_in(nth % tiles, G.tiles_m, tiles_n, 4);
  const int m0 = tile.m * Tiles::TM, n0 = tile.n * Tiles::TN;
  const int all = G.grad_ld / Tiles::BK, per = (all + splits - 1) / splits, from = min(split * per, all), steps = min(per, all - from);
  if (steps <= 0 && !G.first) return;
  Tiles t;
  t.init(shared);
  t.operand_a(G.w, G.w_plane, G.kp, m0, G.kp);
  t.operand_b(G.grad, G.grad_plane, G.grad_ld, n0, live);
  t.run(steps, from);
  const int of_w = G.w_cell != nullptr ? plane_shift(*G.w_cell) : 0;
  float* sums = G.sums + (size_t)split * ((live + 63) / 64 * 64) * G.kp;
#pragma unroll
  for (int j = 0; j < Tiles::NI; ++j) {
    const int shift = -G.row_shift[min(n0 + t.col_of(j), live - 1)] - of_w;
    t.template rows_of<float>(shared, [&](int i, int e) { return __builtin_ldexpf(t.acc[i][j][e], shift); }, [&](int r, int c, floatx4 v) {
      const int token = n0 + t.col_of(j) - (t.lane & 31) + r, col = m0 + t.wm * Tiles::W + c;
      if (token >= live || col >= G.kp) return;
      floatx4* at = reinterpret_cast<floatx4*>(sums + (size_t)token * G.kp + col);
      *at = G.first ? v : *at + v;
    });
  }
}

// dw of the piece: features (registers) by entries of the vocabulary (lanes), over all rows or (SLICES, unscaled fp32 [splits][entries][kp]) a slice of them
template <class Tiles, class O, bool SLICES>
__device__ __forceinline__ void loss_dw(const LossGradArgs& G, char* shared) {
  const int tiles = G.tiles_m * G.tiles_n, nth = xcd_run(blockIdx.x, G.dw_tiles), split = SLICES ? nth / tiles : 0;
  const TileAt tile = tile_in(SLICES ? nth % tiles : nth, G.tiles_m, G.tiles_n, 4);
  const int m0 = tile.m * Tiles::TM, n0 = tile.n * Tiles::TN, live = (int)*G.count, steps = (live + Tiles::BK - 1) / Tiles::BK;
  Tiles t;
  t.init(shared);
  t.operand_a(G.x, G.x_plane, G.kp, m0, G.kp);
  t.operand_b(G.grad, G.grad_plane, G.grad_ld, n0, G.grad_ld);
  if (SLICES) {
    const int per = (steps + G.splits - 1) / G.splits, from = min(steps, split * per);
    t.run(min(per, steps - from), from);
  } else {
    t.run(steps);
  }
  const int shift = -grad_shift(*G.g_cell) - plane_shift(*G.x_cell);
  O* dw = (O*)G.dw + (SLICES ? (size_t)split * G.entries * G.dw_ld : 0);
#pragma unroll
  for (int j = 0; j < Tiles::NI; ++j)
    t.template rows_of<O>(shared, [&](int i, int e) { return __builtin_ldexpf(t.acc[i][j][e], shift); }, [&](int r, int c, auto v) {
      const int entry = n0 + t.col_of(j) - (t.lane & 31) + r, col = m0 + t.wm * Tiles::W + c;
      if (entry >= G.entries || col >= G.dim) return;
      O* at = dw + (size_t)entry * G.dw_ld + col;
      if (col + (int)(16 / sizeof(O)) <= G.dim) {
        store_any(at, v);
      } else {
#pragma unroll
        for (int e = 0; e < (int)(16 / sizeof(O)); ++e)
          if (col + e < G.dim) at[e] = v[e];
      }
    });
}

// Both products of a piece's G in one launch: neither waits for the other's last tiles.
template <class TilesX, class TilesW, class O, bool SLICES>
__global__ __launch_bounds__(TilesX::THREADS, 2) void loss_products_kernel(const LossGradArgs G) {
  static_assert(TilesX::THREADS == TilesW::THREADS, "");
  __shared__ __align__(1024) char shared[TilesX::LDS > TilesW::LDS ? TilesX::LDS : TilesW::LDS];
  if ((int)blockIdx.x < G.dw_tiles) loss_dw<TilesW, O, SLICES>(G, shared);
  else loss_dx<TilesX>(G, shared);
}

// rows of dx or dw [n][dim] from `splits` slices [size][kp].  dx: place is the slices' row of each, -1: zeros, and
// `slices` of them have the rows that count up to a multiple of 64.
template <class O>
__global__ __launch_bounds__(256) void loss_rows_of_slices_kernel(const float* sums, int splits, int size, int kp, int n, int dim, const int* place, const unsigned* count,
                                                                  const unsigned* slices, O* to) {
  const unsigned per = (dim + 3) / 4, i = blockIdx.x * 256 + threadIdx.x;      // (below 2^31: loss_plan)
  const unsigned row = i / per, c = (i - row * per) * 4;
  if (row >= (unsigned)n) return;
  const int at = place != nullptr ? place[row] : (int)row;
  floatx4 v = {0.f, 0.f, 0.f, 0.f};
  if (place != nullptr) {
    splits = (int)*slices;
    size = ((int)*count + 63) / 64 * 64;
  }
  if (at >= 0) {
#pragma unroll 8
    for (int s = 0; s < splits; ++s) v += *reinterpret_cast<const floatx4*>(sums + ((size_t)s * size + at) * kp + c);
  }
  O* p = to + (size_t)row * dim + c;
  typedef __attribute__((__vector_size__(4 * sizeof(O)))) O o4;
  o4 o;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = (O)v[e];
  if ((int)c + 4 <= dim) {
    store_any(p, o);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if ((int)c + e < dim) p[e] = o[e];
  }
}

// ------------------------------------------------------------------------------------ launches

typedef __bf16 B16;
typedef _Float16 H16;
template <class T, int P> struct LogitTiles {
  typedef TileProduct<T, P, ROWS, ROWS, 256, 256, 2, 4, 32, P == 2 ? 2 : 4> Wide;
  typedef TileProduct<T, P, ROWS, ROWS, 128, 128, 2, 4, P == 2 ? 32 : 64, 4> Middle;
  typedef TileProduct<T, P, ROWS, ROWS, 64, 64, 2, 2, 64, P == 2 ? 2 : 4> Tiny;
  typedef TileProduct<T, P, ROWS, ROWS, 128, 32, 4, 1, 64, P == 2 ? 2 : 4> Few;
};
template <int P> struct GradTiles {
  static constexpr int WIDE_STAGES = P == 1 ? 4 : P == 2 ? 2 : 3, BK = P == 1 ? 64 : 32, FEW_STAGES = P == ONE_BY_TWO ? 3 : 2;
  typedef TileProduct<H16, P, COLUMNS, ROWS, 256, 256, 2, 4, 32, WIDE_STAGES> WideX;
  typedef TileProduct<H16, P, COLUMNS, ROWS, 128, 128, 2, 4, BK, 4> MiddleX;
  typedef TileProduct<H16, P, COLUMNS, COLUMNS, 256, 256, 2, 4, 32, WIDE_STAGES> WideW;
  typedef TileProduct<H16, P, COLUMNS, COLUMNS, 128, 128, 2, 4, BK, 4> MiddleW;
  typedef TileProduct<H16, P, COLUMNS, ROWS, 128, 128, 2, 4, BK, FEW_STAGES> FewX;
  typedef TileProduct<H16, P, COLUMNS, COLUMNS, 128, 128, 2, 4, BK, FEW_STAGES> FewW;
};

template <class Tiles, bool GRAD>
static void launch_tile(LossTileArgs a, hipStream_t st) {
  a.tiles_m = (a.vend - a.v0 + Tiles::TM - 1) / Tiles::TM;
  const int tiles_n = ((GRAD ? a.npad : a.n) + Tiles::TN - 1) / Tiles::TN;
  hipLaunchKernelGGL((loss_tile_kernel<Tiles, GRAD>), dim3((unsigned)(a.tiles_m * tiles_n)), dim3(Tiles::THREADS), 0, st, a);
}
template <class T, int P, bool GRAD>
static void launch_tiles(const LossPlan& p, const LossTileArgs& a, hipStream_t st) {
  typedef LogitTiles<T, P> L;
  if (p.size == WIDE) launch_tile<typename L::Wide, GRAD>(a, st);
  else if (p.size == MIDDLE) launch_tile<typename L::Middle, GRAD>(a, st);
  else if (p.size == TINY) launch_tile<typename L::Tiny, GRAD>(a, st);
  else if constexpr (GRAD) launch_tile<typename L::Few, GRAD>(a, st);      // (the forward of few rows: loss_few_kernel)
}

template <class S>
static auto few_kernel(bool aligned, bool narrow) {
  return aligned ? narrow ? loss_few_kernel<S, true, true> : loss_few_kernel<S, true, false> : narrow ? loss_few_kernel<S, false, true> : loss_few_kernel<S, false, false>;
}
static bool misaligned(std::initializer_list<const void*> all, size_t to) {
  for (const void* p : all)
    if ((uintptr_t)p % to) return true;
  return false;
}
static unsigned blocks_for(long work) { return (unsigned)std::max<long>(1, (work + 255) / 256); }

static LossMost most_to(const void* src, long ld, int rows, int cols, const int* map, const unsigned* count, unsigned* parts) {
  return LossMost{src, ld, rows, cols, map, count, parts, (int)std::min<unsigned>(kParts, blocks_for((long)rows * ((cols + 7) / 8)))};
}
static LossFound found(const LossMost& m) { return LossFound{m.parts, m.blocks, 1}; }
static LossFound found(const unsigned* cell) { return LossFound{cell, 1, 0}; }
static void begin(const nsa_loss_desc* d, const LossBegin& a, int blocks, hipStream_t st) {
  const dim3 grid((unsigned)(a.of[0].blocks + a.of[1].blocks + blocks)), block(256);
  if (d->dtype == 0) hipLaunchKernelGGL((loss_begin_kernel<B16>), grid, block, 0, st, a);
  else if (d->dtype == 1) hipLaunchKernelGGL((loss_begin_kernel<H16>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((loss_begin_kernel<float>), grid, block, 0, st, a);
}
static LossRows rows_to(const LossPlan& p, const void* src, long ld, int rows, int cols, const int* map, const unsigned* count, const LossFound& found, void* dst,
                        long plane, unsigned* most = nullptr, int back = 0) {
  return LossRows{src, ld, rows, cols, map, count, found, dst, plane, most, back, (int)blocks_for(((long)up(rows, 64) * p.kp / 8 + kCopies - 1) / kCopies), false, nullptr, nullptr, LossFound{}};
}
template <class S, class D, int P>
static void copy(const LossCopy& a, hipStream_t st) {
  const unsigned blocks = (unsigned)(a.of[0].blocks + a.of[1].blocks + (a.cells != nullptr));
  if (blocks > 0) hipLaunchKernelGGL((loss_planes_kernel<S, D, P>), dim3(blocks), dim3(256), 0, st, a);
}

template <int P, class O, bool SLICES>
static void products(const LossPlan& p, const LossGradArgs& q, bool dx, hipStream_t st) {
  typedef GradTiles<P> T;
  const int tile = p.size == WIDE ? 256 : 128, all = q.tiles_m * ((p.n + tile - 1) / tile);
  const dim3 grid((unsigned)(q.dw_tiles + (dx ? std::max(all, std::min(kMaxSlices * all, kSliceTiles)) : 0))), block(512);
  // few rows: nothing to read ahead, so two work-groups a CU that write in turn (25 rows, 1917 features, 21120 entries in bf16: 36 -> 24 us)
  if constexpr (!SLICES)
    if (p.size == FEW) {
      hipLaunchKernelGGL((loss_products_kernel<typename T::FewX, typename T::FewW, O, SLICES>), grid, block, 0, st, q);
      return;
    }
  if (p.size == WIDE) hipLaunchKernelGGL((loss_products_kernel<typename T::WideX, typename T::WideW, O, SLICES>), grid, block, 0, st, q);
  else hipLaunchKernelGGL((loss_products_kernel<typename T::MiddleX, typename T::MiddleW, O, SLICES>), grid, block, 0, st, q);
}
static void rows_of_slices(const nsa_loss_desc* d, const LossGradArgs& q, const float* sums, int size, int n, const int* place, void* to, hipStream_t st) {
  const dim3 grid(blocks_for((long)n * ((d->dim + 3) / 4)));
  auto go = [&](auto kernel, auto* out) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, sums, q.splits, size, q.kp, n, d->dim, place, q.count, q.slices, out);
  };
  if (d->dtype == 0) go(loss_rows_of_slices_kernel<B16>, (B16*)to);
  else if (d->dtype == 1) go(loss_rows_of_slices_kernel<H16>, (H16*)to);
  else go(loss_rows_of_slices_kernel<float>, (float*)to);
}

}  // namespace nsa

using namespace nsa;

extern "C" int nsa_loss_workspace_bytes(const nsa_loss_desc* d, const void* weight, size_t* state_bytes, size_t* fwd_bytes, size_t* bwd_bytes) {
  LossPlan p;
  if (!state_bytes || !fwd_bytes || !bwd_bytes) return NSA_E_ARG;
  if (int rc = loss_plan(d, weight, p)) return rc;
  *state_bytes = p.state;
  *fwd_bytes = p.fwd;
  *bwd_bytes = p.bwd;
  return 0;
}

extern "C" int nsa_loss_fwd(const nsa_loss_desc* d, const void* x, const void* weight, const void* labels, void* state, size_t state_bytes, void* ws,
                            size_t ws_bytes, float* loss, void* stream) {
  LossPlan p;
  if (int rc = loss_plan(d, weight, p)) return rc;
  if (!weight || !state || !ws || !loss || (p.n > 0 && (!x || !labels))) return NSA_E_ARG;
  if (misaligned({x, weight}, d->dtype == 2 ? 4 : 2) || misaligned({state, ws}, 256) || misaligned({loss}, 4) || misaligned({labels}, d->labels_int64 ? 8 : 4))
    return NSA_E_ARG;
  if (state_bytes < p.state || ws_bytes < p.fwd) return NSA_E_WORKSPACE;
  hipStream_t st = (hipStream_t)stream;
  char *s = (char*)state, *w = (char*)ws;
  unsigned* cells = (unsigned*)s;
  int *map = (int*)(s + p.s_map), *place = (int*)(s + p.s_place), *label = (int*)(s + p.s_label);
  float2* norm = (float2*)(s + p.s_norm);
  float *own = (float*)(s + p.s_own), *each = (float*)(w + p.f_loss), *target = (float*)(w + p.f_target);
  float* losses = d->reduction == 0 ? loss : nullptr;
  float2* part = (float2*)(w + p.f_part);
  const unsigned* count = cells + CELL_ROWS;
  const int each_bytes = d->dtype == 2 ? 4 : 2;
  if (p.size == FEW) {
    LossFewArgs a{x, weight, labels, (long)d->x_stride, (long)d->w_stride, (long)d->ignore_index, (int)d->labels_int64, p.n, d->dim, d->vocab, p.npad,
                  map, place, label, cells, part, target, losses};
    const dim3 grid((unsigned)((d->vocab + p.tile - 1) / p.tile));
    const bool aligned = (((uintptr_t)x | (uintptr_t)weight) & 15) == 0 && d->x_stride * each_bytes % 16 == 0 && d->w_stride * each_bytes % 16 == 0;
    const auto kernel = d->dtype == 0 ? few_kernel<B16>(aligned, p.tile == 32) : d->dtype == 1 ? few_kernel<H16>(aligned, p.tile == 32) : few_kernel<float>(aligned, p.tile == 32);
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, a);
  } else {
    const dim3 grid((unsigned)((p.n + 1023) / 1024));
    int* counts = p.n > kRowsUncounted ? (int*)(w + p.f_count) : nullptr;
    if (counts) hipLaunchKernelGGL(loss_count_kernel, grid, dim3(256), 0, st, labels, (int)d->labels_int64, p.n, (long)d->ignore_index, counts);
    hipLaunchKernelGGL(loss_rows_kernel, grid, dim3(256), 0, st, labels, (int)d->labels_int64, p.n, d->vocab, (long)d->ignore_index, (const int*)counts, map,
                       place, label, cells, losses);
    const long x_plane = (long)p.npad * p.kp;
    const int back = p.in_place ? p.kp - d->dim : 0;
    const bool scaled = d->dtype == 2;
    LossFound of_x{}, of_w{};
    if (scaled) {
      unsigned* parts = (unsigned*)(w + p.f_most);
      LossBegin a{};
      a.of[0] = most_to(x, d->x_stride, p.n, d->dim, map, count, parts);
      a.of[1] = most_to(weight, d->w_stride, d->vocab, d->dim, nullptr, nullptr, parts + kParts);
      begin(d, a, 0, st);
      of_x = found(a.of[0]);
      of_w = found(a.of[1]);
    }
    const int rows = p.in_place ? d->vocab : p.fwd_rows;
    for (long v0 = 0; v0 < d->vocab; v0 += rows) {
      LossTileArgs a{};
      a.v0 = (int)v0;
      a.vend = (int)std::min<long>(d->vocab, v0 + rows);
      LossCopy c{};
      c.kp = p.kp;
      if (v0 == 0) {
        // (a 16-bit backward pass wants to know the largest |x|)
        c.of[0] = rows_to(p, x, d->x_stride, p.n, d->dim, map, count, of_x, w + p.f_x, x_plane, scaled ? nullptr : cells + CELLS, back);
        c.cells = scaled ? cells : nullptr;
      }
      if (p.in_place) {
        a.w = weight;
        a.w_ld = d->w_stride;
        a.tail = p.kp - 64;
        a.back = back;
      } else {
        a.w = w + p.f_w;
        a.w_ld = p.kp;
        a.w_plane = (long)p.kp * up(a.vend - a.v0, 64);
        c.of[1] = rows_to(p, (const char*)weight + v0 * d->w_stride * each_bytes, d->w_stride, a.vend - a.v0, d->dim, nullptr, nullptr, of_w,
                          w + p.f_w, a.w_plane);
      }
      if (d->dtype == 0) copy<B16, B16, 1>(c, st);
      else if (d->dtype == 1) copy<H16, H16, 1>(c, st);
      else copy<float, H16, 2>(c, st);
      if (scaled) of_w = found(cells + CELL_W);
      a.x = w + p.f_x; a.x_plane = x_plane; a.kp = p.kp; a.n = p.n; a.npad = p.npad;
      a.count = count; a.x_cell = scaled ? cells + CELL_X : nullptr; a.w_cell = cells + CELL_W; a.label = label; a.part = part; a.target = target;
      if (d->dtype == 0) launch_tiles<B16, 1, false>(p, a, st);
      else if (d->dtype == 1) launch_tiles<H16, 1, false>(p, a, st);
      else launch_tiles<H16, 2, false>(p, a, st);
    }
  }
  if (p.n > 0) {
    const int parts = (int)(up(d->vocab, p.tile) / p.part);
    const auto merge = p.n <= 2048 ? loss_merge_kernel<2> : loss_merge_kernel<8>;
    hipLaunchKernelGGL(merge, dim3((unsigned)(p.n <= 2048 ? (p.n + 1) / 2 : (p.n + 7) / 8)), dim3(256), 0, st, (const float2*)part, parts, p.npad, count,
                       (const int*)map, (const int*)label, (const float*)target, norm, own, each, losses);
  }
  if (d->reduction != 0)
    hipLaunchKernelGGL(loss_sum_kernel, dim3(1), dim3(1024), 0, st, (const float*)each, count, (int)(d->reduction == 1), loss);
  return (int)hipGetLastError();
}

extern "C" int nsa_loss_bwd(const nsa_loss_desc* d, const void* x, const void* weight, const void* state, size_t state_bytes, const float* dloss, void* ws,
                            size_t ws_bytes, void* dx, void* dw, void* stream) {
  LossPlan p;
  if (int rc = loss_plan(d, weight, p)) return rc;
  if (!x || !weight || !state || !dloss || !ws || (!dx && !dw) || p.n == 0) return NSA_E_ARG;
  if (misaligned({x, weight, dx, dw}, d->dtype == 2 ? 4 : 2) || misaligned({state, ws}, 256) || misaligned({dloss}, 4)) return NSA_E_ARG;
  if (state_bytes < p.state || ws_bytes < p.bwd) return NSA_E_WORKSPACE;
  hipStream_t st = (hipStream_t)stream;
  const char* s = (const char*)state;
  char* w = (char*)ws;
  const unsigned* kept = (const unsigned*)s;
  unsigned *cells = (unsigned*)(w + p.b_cells), *parts = (unsigned*)(w + p.b_most), *g_most = parts + 2 * kParts;
  const int *map = (const int*)(s + p.s_map), *place = (const int*)(s + p.s_place), *label = (const int*)(s + p.s_label);
  const unsigned* count = kept + CELL_ROWS;
  float* g = (float*)(w + p.b_g);
  const int each = d->dtype == 2 ? 4 : 2, tile = p.size == WIDE ? 256 : 128, tiles_m = (p.kp + tile - 1) / tile;
  int* row_shift = (int*)(w + p.b_shift);
  // All operands in fp16: x once (for the logits as it is where it is fp16, for dw weighted), w with each piece.  Magnitudes: those the forward has
  // found, else here.
  const bool scaled = d->dtype != 1;
  LossBegin b{};
  LossFound of_x{}, of_w{};
  if (p.size != FEW) {
    of_x = d->dtype == 2 ? found(kept + CELL_X) : LossFound{kept + CELLS, kMost, 16};
  } else {
    b.of[0] = most_to(x, d->x_stride, p.n, d->dim, map, count, parts);
    of_x = found(b.of[0]);
  }
  if (d->dtype == 2 && p.size != FEW) {
    of_w = found(kept + CELL_W);
  } else if (scaled) {
    b.of[1] = most_to(weight, d->w_stride, d->vocab, d->dim, nullptr, nullptr, parts + kParts);
    of_w = found(b.of[1]);
  }
  b.dloss = dloss; b.reduction = d->reduction; b.map = map; b.count = count; b.own = (const float*)(s + p.s_own); b.g = g; b.row_shift = row_shift; b.most = g_most;
  begin(d, b, (p.n + 1023) / 1024, st);
  const long x_plane = (long)p.npad * p.kp;
  LossGradArgs q{};
  q.kp = p.kp; q.count = count; q.g_cell = cells + CELL_G; q.row_shift = row_shift; q.tiles_m = tiles_m; q.slices = cells + CELL_SLICES;
  q.x = (const H16*)(w + p.b_xg); q.x_plane = x_plane; q.x_cell = cells + CELL_X; q.w = (const H16*)(w + p.b_w); q.w_cell = scaled ? cells + CELL_W : nullptr; q.sums = (float*)(w + p.b_dx);
  for (long v0 = 0; v0 < d->vocab; v0 += p.bwd_rows) {
    LossTileArgs a{};
    a.v0 = (int)v0;
    a.vend = (int)std::min<long>(d->vocab, v0 + p.bwd_rows);
    const int entries = a.vend - a.v0, ld = (int)up(entries, 64);
    const long w_plane = (long)p.kp * ld;
    void* wg = w + p.b_w;
    LossCopy c{};
    c.kp = p.kp;
    if (v0 == 0) {
      c.of[0] = rows_to(p, x, d->x_stride, p.n, d->dim, map, count, of_x, w + p.b_x, x_plane);
      c.of[0].as_is = !scaled; c.of[0].weighted = dw ? w + p.b_xg : nullptr; c.of[0].row_shift = row_shift;
      c.most = c.of[0].rows_most = LossFound{g_most, (p.n + 1023) / 1024, 1};
      c.count = count; c.cells = cells; c.tiles_m = tiles_m; c.tile = tile; c.piece = std::min(p.bwd_rows, (int)up(d->vocab, 64));
    }
    c.of[1] = rows_to(p, (const char*)weight + v0 * d->w_stride * each, d->w_stride, entries, d->dim, nullptr, nullptr, of_w, wg, w_plane);
    auto make = [&](const LossCopy& a) {
      if (d->dtype == 0) copy<B16, H16, 1>(a, st);
      else if (d->dtype == 2) copy<float, H16, 2>(a, st);
      else copy<H16, H16, 1>(a, st);
    };
    if (v0 == 0 && c.most.count > 64) {      // (many words for every work-group to read: once, in a launch before)
      LossCopy only = c;
      only.of[0].blocks = only.of[1].blocks = 0;
      make(only);
      c.cells = nullptr;
      c.of[0].rows_most = found(cells + CELL_G);
    }
    make(c);
    if (scaled) of_w = found(cells + CELL_W);
    a.w = wg; a.w_ld = p.kp; a.w_plane = w_plane;
    a.x = w + p.b_x; a.x_plane = x_plane; a.kp = p.kp; a.n = p.n; a.npad = p.npad;
    a.count = count; a.x_cell = scaled ? q.x_cell : nullptr; a.w_cell = q.w_cell; a.label = label;
    a.norm = (const float2*)(s + p.s_norm); a.own = (const float*)(s + p.s_own); a.g = g; a.row_shift = row_shift;
    a.grad = (H16*)(w + p.b_grad); a.grad_plane = (long)p.npad * ld; a.grad_ld = ld; a.grad_planes = p.grad_P == 1 ? 1 : 2;
    if (p.grad_P == 2) launch_tiles<H16, 2, true>(p, a, st);
    else launch_tiles<H16, 1, true>(p, a, st);

    q.grad = a.grad; q.grad_plane = a.grad_plane; q.grad_ld = ld; q.w_plane = w_plane; q.entries = entries; q.first = v0 == 0;
    q.tiles_n = (entries + tile - 1) / tile;
    q.splits = !dw ? 1 : a.vend == d->vocab ? p.last_splits : p.w_splits;
    q.dw_tiles = dw ? tiles_m * q.tiles_n * q.splits : 0;
    const bool slices = q.splits > 1;
    char* to = (char*)dw + v0 * d->dim * each;
    q.dw = slices ? w + p.b_dw : to; q.dw_ld = q.dim = slices ? p.kp : d->dim;
    if (slices && p.grad_P == 1) products<1, float, true>(p, q, dx, st);
    else if (slices && p.grad_P == 2) products<2, float, true>(p, q, dx, st);
    else if (slices) products<ONE_BY_TWO, float, true>(p, q, dx, st);
    else if (d->dtype == 0) products<1, B16, false>(p, q, dx, st);
    else if (d->dtype == 2) products<2, float, false>(p, q, dx, st);
    else products<ONE_BY_TWO, H16, false>(p, q, dx, st);
    if (slices) rows_of_slices(d, q, (const float*)(w + p.b_dw), entries, entries, nullptr, to, st);
  }
  if (dx) rows_of_slices(d, q, (const float*)(w + p.b_dx), 0, p.n, place, dx, st);
  return (int)hipGetLastError();
}
