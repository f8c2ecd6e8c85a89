// Orthogonalised updates: the polar factor of a matrix by Newton-Schulz products,
//
//   X <- G / (|G| + eps) (turned so that it is not taller than wide), `steps` times:  A = X X^T,  B = a + b A + c A A,  X <- B X,
//
// for a list of matrices of any sizes, all of them in each launch: the norms, the first planes, then three launches a step.
//
// X, A and B are held as two fp16 halves each (22 bits; nsa_tiles.hpp).  Directions of small singular values grow by a = 3.4 a step, and what
// a step's rounding adds to them grows alike: against 64 bits the result is 4e-5 off with bf16 halves, 3 % with bf16 alone, and 6e-7 with
// these, less than with fp32 products (1.6e-6 at 512 x 512).  a stands on the diagonal of B and not beside the product: one pass over X less, and
// a rounding of what is left of a + b A + c A A, not of its parts.  A bf16 result is itself rounded to 2^-9, so its last two steps, after which little grows,
// take the first halves alone, at a third of the matrix instructions: that adds at most a tenth to the result's error (1.66e-3 of its norm
// from rounding, 1.83e-3 with two such steps, 2.0e-3 with three, 2.1e-3 with all five).  And a matrix of 16 bits begins as itself times a power of
// two, one half and exact; what it is short of G / (|G| + eps) is a factor of the first A and B X.  Scales: X 2^(12 + s), A 2^(10 + 2 s), B 2^10.  s is 0 unless |G| is small beside eps:
// then X starts so small that fp16 would lose it, and s is what brings its norm to 1; it falls by the bits of a with each step, so nothing grows out
// of range.  The entry checks that singular values up to 1 stay below 4 for the given coefficients.
//
// A and B are symmetric: only tiles on and below the diagonal are made, and stored twice.
#include <algorithm>
#include <cmath>
#include "nsa_tiles.hpp"
#include "../../include/nsa_hip.h"

namespace nsa {

constexpr int kNewtonMany = 56, kNormChunks = 512;      // matrices of one launch (their table is a kernel argument)

struct NewtonMatrix {
  const void* in;
  void* out;
  long stride;                // of the rows of `in`
  unsigned at;                // of its planes in the workspace, in units of 256 bytes
  int rows, cols;             // as given
};
struct NewtonTable {
  NewtonMatrix of[kNewtonMany];
  // The launch at hand: every XCD (work-groups go to them in turn) has a queue of places; entry e has those from first[e] on, and begins
  // with matrix base[e].  One matrix, spread over all XCDs, or eight of them, one to an XCD (its operands are then read by that one alone).
  int first[kNewtonMany + 1];
  uint8_t base[kNewtonMany], kind[kNewtonMany];      // kind: spread, eight, eight in reverse
  int entries, many, chunks;
  char* ws;
  double* partial;                 // [many][kNormChunks]
  int* shift;                      // s of each
  float* factor;                   // what the first X is short of
};

__host__ __device__ inline long up64(long v) { return (v + 63) / 64 * 64; }
// X [2 buffers][2 halves][mp][np], then A and B [2 halves][mp][mp]
struct NewtonPlanes {
  int m, n, mp, np;
  bool turned;
  __host__ __device__ NewtonPlanes(int rows, int cols) {
    turned = rows > cols;
    m = turned ? cols : rows;
    n = turned ? rows : cols;
    mp = (int)up64(m);
    np = (int)up64(n);
  }
  __host__ __device__ long x_plane() const { return (long)mp * np; }
  __host__ __device__ long a_plane() const { return (long)mp * mp; }
  __host__ __device__ long halves() const { return 4 * x_plane() + 4 * a_plane(); }
};
__device__ __forceinline__ _Float16* planes_of(const NewtonTable& t, int k) { return (_Float16*)(t.ws + (size_t)t.of[k].at * 256); }

enum { SPREAD, EIGHT, REVERSED };
// The matrix (-1: none) and its tile that a work-group makes; count(planes): tiles of a matrix
struct NewtonPlace { int k, nth; };
template <class Count>
__device__ __forceinline__ NewtonPlace place_of(const NewtonTable& t, Count count) {
  const int i = blockIdx.x >> 3, x = blockIdx.x & 7;
  int e = 0, past = t.entries;
  while (past - e > 1) {
    const int mid = (e + past) / 2;
    if (i >= t.first[mid]) e = mid;
    else past = mid;
  }
  const int at = i - t.first[e], base = t.base[e], kind = t.kind[e], k = kind == SPREAD ? base : base + (kind == EIGHT ? x : 7 - x);
  const int total = count(NewtonPlanes(t.of[k].rows, t.of[k].cols));
  if (kind != SPREAD) return NewtonPlace{at < total ? k : -1, at};
  // (turned by the entry: small ones do not all begin on the same XCD)
  const int turn = (x + e) & 7, per = total / 8, rest = total % 8;
  return NewtonPlace{at < per + (turn < rest) ? k : -1, turn * per + min(turn, rest) + at};
}
__host__ __device__ inline int square_tiles(const NewtonPlanes& p, int size) {
  const int t = (p.m + size - 1) / size;
  return t * (t + 1) / 2;
}
__host__ __device__ inline int update_tiles(const NewtonPlanes& p, int size) { return (p.np + size - 1) / size * ((p.mp + size - 1) / size); }

template <class S>
__global__ __launch_bounds__(256) void newton_norm_kernel(const NewtonTable G) {
  __shared__ double sums[4];
  const int k = blockIdx.y, tid = threadIdx.x;
  const NewtonMatrix M = G.of[k];
  const S* in = (const S*)M.in;
  const bool whole = M.stride == M.cols;      // one run of values
  double sum = 0.0;
  const long total = (long)M.rows * M.cols, per = ((total + G.chunks - 1) / G.chunks + 2047) / 2048 * 2048, first = blockIdx.x * per, last = min(total, first + per);
  if (whole) {
    constexpr int V = 16 / sizeof(S);
    for (long i = first + tid * V; i < last; i += 256 * V) {
      if (i + V <= last) {
        const auto v = load_any<V>(in + i);
#pragma unroll
        for (int e = 0; e < V; ++e) sum += (double)(float)v[e] * (double)(float)v[e];
      } else {
        for (long e = i; e < last; ++e) sum += (double)(float)in[e] * (double)(float)in[e];
      }
    }
  } else {
    for (long i = first + tid; i < last; i += 256) {
      const double v = (double)(float)in[i / M.cols * M.stride + i % M.cols];
      sum += v * v;
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  if ((tid & 63) == 0) sums[tid >> 6] = sum;
  __syncthreads();
  if (tid == 0) G.partial[k * kNormChunks + blockIdx.x] = sums[0] + sums[1] + sums[2] + sums[3];
}

// kBeginTiles tiles of 64 x 64 of the first X, scaled, with zeros up to whole multiples of 64
constexpr int kBeginTiles = 2;
__host__ __device__ inline int begin_parts(const NewtonPlanes& p, int size) { return (update_tiles(p, size) + kBeginTiles - 1) / kBeginTiles; }
template <class S>
__global__ __launch_bounds__(256) void newton_begin_kernel(const NewtonTable G, float eps, int exact) {
  __shared__ float tile_s[64][65];
  __shared__ double sums[4], scale_s;
  const NewtonPlace place = place_of(G, [](const NewtonPlanes& p) { return begin_parts(p, 64); });
  if (place.k < 0) return;
  const int k = place.k, tid = threadIdx.x;
  const NewtonMatrix M = G.of[k];
  const NewtonPlanes L(M.rows, M.cols);
  double sum = 0.0;
  for (int i = tid; i < G.chunks; i += 256) sum += G.partial[k * kNormChunks + i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  if ((tid & 63) == 0) sums[tid >> 6] = sum;
  __syncthreads();
  if (tid == 0) {
    const double norm = sqrt(sums[0] + sums[1] + sums[2] + sums[3]), part = norm / (norm + eps);
    // (a norm of zero, and one that is no number: s = 0)
    const int s = part > 0.0 && part < 1.0 ? min(100, -(ilogb(part) + 1)) : 0;
    double scale = ldexp(1.0 / (norm + eps), 12 + s), factor = 1.0;
    if (exact && scale > 0.0 && scale < INFINITY) {
      int bits;
      factor = 2.0 * frexp(scale, &bits);
      scale = ldexp(1.0, bits - 1);
    }
    scale_s = scale;
    if (place.nth == 0) {
      G.shift[k] = s;
      G.factor[k] = (float)factor;
    }
  }
  const S* in = (const S*)M.in;
  const int wide = L.np / 64, r = tid >> 2, c = (tid & 3) * 16;
  for (int at = place.nth * kBeginTiles; at < min((place.nth + 1) * kBeginTiles, wide * (L.mp / 64)); ++at) {
    // (turned: the tile's rows are columns of the matrix)
    const int r0 = at / wide * 64, c0 = at % wide * 64, first = L.turned ? c0 : r0, col = (L.turned ? r0 : c0) + (tid & 63);
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int row = first + 4 * i + (tid >> 6);
      v[i] = row < M.rows && col < M.cols ? (float)in[row * M.stride + col] : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; ++i) tile_s[4 * i + (tid >> 6)][tid & 63] = v[i];
    __syncthreads();
    const double scale = scale_s;
    _Float16* x = planes_of(G, k) + (long)(r0 + r) * L.np + c0 + c;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      f16x8 hi, lo;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int cc = c + 8 * u + e;
        const Halves h = halves_of((float)((double)(L.turned ? tile_s[cc][r] : tile_s[r][cc]) * scale));
        hi[e] = h.hi;
        lo[e] = h.lo;
      }
      *reinterpret_cast<f16x8*>(x + 8 * u) = hi;
      if (!exact) *reinterpret_cast<f16x8*>(x + 8 * u + L.x_plane()) = lo;
    }
  }
}

struct NewtonStep {
  int step, growth, from;      // growth: bits that a step takes off s; from: the buffer of X that is read
  int both_x, both_a;          // second halves are wanted of the next X, of A and B
  float a, b, c;
};
__device__ __forceinline__ int shift_at(const NewtonTable& G, const NewtonStep& S, int k, int step) { return max(0, G.shift[k] - S.growth * step); }

// four consecutive values of P planes
template <int P> __device__ __forceinline__ floatx4 load_halves(const _Float16* p, long plane) {
  const f16x4 hi = *reinterpret_cast<const f16x4*>(p), lo = *reinterpret_cast<const f16x4*>(p + (P == 2 ? plane : 0));
  floatx4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = P == 2 ? (float)hi[e] + (float)lo[e] : (float)hi[e];
  return v;
}
__device__ __forceinline__ void store_halves(_Float16* p, long plane, floatx4 v, bool both) {
  f16x4 hi, lo;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const Halves h = halves_of(v[e]);
    hi[e] = h.hi;
    lo[e] = h.lo;
  }
  *reinterpret_cast<f16x4*>(p) = hi;
  if (both) *reinterpret_cast<f16x4*>(p + plane) = lo;
}

// POLY 0: A = X X^T; 1: B = a + b A + c A A.  Tiles on and below the diagonal.
template <class Tiles, bool POLY>
__global__ __launch_bounds__(Tiles::THREADS, 2) void newton_square_kernel(const NewtonTable G, const NewtonStep S) {
  __shared__ __align__(1024) char shared[Tiles::LDS];
  const NewtonPlace place = place_of(G, [](const NewtonPlanes& p) { return square_tiles(p, Tiles::TM); });
  if (place.k < 0) return;
  const int k = place.k;
  const NewtonPlanes L(G.of[k].rows, G.of[k].cols);
  const TileAt tile = triangle_in(place.nth, (L.m + Tiles::TM - 1) / Tiles::TM);
  const int m0 = tile.m * Tiles::TM, n0 = tile.n * Tiles::TN;
  _Float16* base = planes_of(G, k);
  const _Float16* x = base + (S.from ? 2 * L.x_plane() : 0);
  _Float16* A = base + 4 * L.x_plane();
  _Float16* out = POLY ? A + 2 * L.a_plane() : A;
  Tiles t;
  t.init(shared);
  if (POLY) {
    t.operand_a(A, L.a_plane(), L.mp, m0, L.m);
    t.operand_b(A, L.a_plane(), L.mp, n0, L.m);
    t.run(L.mp / Tiles::BK);
  } else {
    t.operand_a(x, L.x_plane(), L.np, m0, L.m);
    t.operand_b(x, L.x_plane(), L.np, n0, L.m);
    t.run(L.np / Tiles::BK);
  }
  const int s = POLY ? shift_at(G, S, k, S.step) : 0;
  const float factor = !POLY && S.step == 0 ? G.factor[k] : 1.f;
  const float unit = POLY ? __builtin_ldexpf(S.c, -10 - 4 * s) : 0x1p-14f * factor * factor, linear = __builtin_ldexpf(S.b, -2 * s), diagonal = S.a * 0x1p10f;
#pragma unroll
  for (int j = 0; j < Tiles::NI; ++j) {
    const int col0 = n0 + t.col_of(j) - (t.lane & 31), row0 = m0 + t.wm * Tiles::W;
    t.template rows_of<float>(shared, [&](int i, int e) { return t.acc[i][j][e]; }, [&](int r, int c, floatx4& v) {
      const int col = col0 + r, row = row0 + c;
      const bool ok = col < L.m && row < L.mp;
      const long at = (long)col * L.mp + row;
      floatx4 old = {0.f, 0.f, 0.f, 0.f};
      if (POLY && ok) old = load_halves<Tiles::P>(A + at, L.a_plane());
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] *= unit;
        if (POLY) v[e] = __builtin_fmaf(linear, old[e], v[e]) + (row + e == col ? diagonal : 0.f);
        if (row + e >= L.m || col >= L.m) v[e] = 0.f;
      }
      if (ok) store_halves(out + at, L.a_plane(), v, S.both_a);
    });
    if (tile.m != tile.n)      // the other side of the diagonal
      t.turned_of(shared, [&](int r, int c, floatx4 v) {
        if (row0 + c < L.m && col0 + r < L.mp) store_halves(out + (long)(row0 + c) * L.mp + col0 + r, L.a_plane(), v, S.both_a);
      });
  }
}

// X <- B X (the other buffer; LAST: the result as it was given), columns of X (registers) by its rows (lanes)
template <class Tiles, bool LAST, class O>
__global__ __launch_bounds__(Tiles::THREADS, 2) void newton_update_kernel(const NewtonTable G, const NewtonStep S) {
  __shared__ __align__(1024) char shared[Tiles::LDS];
  const NewtonPlace place = place_of(G, [](const NewtonPlanes& p) { return update_tiles(p, Tiles::TM); });
  if (place.k < 0) return;
  const int k = place.k;
  const NewtonMatrix M = G.of[k];
  const NewtonPlanes L(M.rows, M.cols);
  const int tiles_n = (L.mp + Tiles::TN - 1) / Tiles::TN, tiles_m = (L.np + Tiles::TM - 1) / Tiles::TM;
  const TileAt tile = tile_in(place.nth, tiles_m, tiles_n, 4);
  const int m0 = tile.m * Tiles::TM, n0 = tile.n * Tiles::TN;
  _Float16* base = planes_of(G, k);
  const _Float16* x = base + (S.from ? 2 * L.x_plane() : 0);
  _Float16* next = base + (S.from ? 0 : 2 * L.x_plane());
  const _Float16* B = base + 4 * L.x_plane() + 2 * L.a_plane();
  Tiles t;
  t.init(shared);
  t.operand_a(x, L.x_plane(), L.np, m0, L.np);
  t.operand_b(B, L.a_plane(), L.mp, n0, L.m);
  t.run(L.mp / Tiles::BK);
  const int s = shift_at(G, S, k, S.step), s2 = shift_at(G, S, k, S.step + 1);
  const float unit = __builtin_ldexpf(S.step == 0 ? G.factor[k] : 1.f, -10 + (LAST ? -12 - s : s2 - s));
#pragma unroll
  for (int j = 0; j < Tiles::NI; ++j) {
    if (LAST && L.turned) {
      // a register's value of 32 lanes is a run of a row of the result
      const int row = n0 + t.col_of(j);
      if (row >= L.m) continue;
#pragma unroll
      for (int i = 0; i < Tiles::MI; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int col = m0 + t.row_of(i, q);
          if (col >= L.n) continue;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (col + e < L.n) ((O*)M.out)[(long)(col + e) * M.cols + row] = (O)(t.acc[i][j][4 * q + e] * unit);
        }
      continue;
    }
    t.template rows_of<float>(shared, [&](int i, int e) { return t.acc[i][j][e]; }, [&](int r, int c, floatx4 v) {
      const int row = n0 + t.col_of(j) - (t.lane & 31) + r, col = m0 + t.wm * Tiles::W + c;
      if (row >= (LAST ? L.m : L.mp) || col >= (LAST ? L.n : L.np)) return;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = row < L.m ? v[e] * unit : 0.f;      // (rows past the last one are zeros)
      if (!LAST) {
        store_halves(next + (long)row * L.np + col, L.x_plane(), v, S.both_x);
        return;
      }
      O* p = (O*)M.out + (long)row * M.cols + col;
      typedef __attribute__((__vector_size__(4 * sizeof(O)))) O ox4;
      ox4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = (O)v[e];
      if (col + 4 <= L.n) {
        store_any(p, o);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < L.n) p[e] = o[e];
      }
    });
  }
}

// ------------------------------------------------------------------------------------ small matrices

// A matrix of up to 64 rows that fits a CU's LDS, all steps in one work-group, in fp32 throughout (32 x 32 x 2 products): the launches of the
// other kernels would be all of its time (a 24 x 512 matrix took 99 us with them, 39 so), and sums this short show that halves have a bit or two less
// than fp32.  X lies in LDS for the whole time; a step is A (the columns of X split over the waves and summed), B, and X, 32 columns a
// wave, in place.  A and B lie there in blocks of 32 x 32 as the matrix instructions leave them, four values of a lane together: what is a
// result's element of row 8 g + 4 h + e in column l is the operand's of column 8 g + 4 h + e in row l, and both are symmetric.
constexpr int kSmallFloats = 40960 - 4 * 8, kSmallWaves = 8, kSmallPart = kSmallWaves * 1024;      // (floats)
__host__ __device__ inline int up32(int v) { return (v + 31) / 32 * 32; }
__host__ __device__ inline bool newton_small(int m, int n) {
  if (m > 64) return false;
  const int M = up32(m);
  return (long)M * (up32(n) + 4) + 2 * M * M + kSmallPart <= kSmallFloats;
}
__device__ __forceinline__ floatx16 mma_f32(floatx4 a, floatx4 b, floatx16 c) {
#pragma unroll
  for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
  return c;
}

__device__ __forceinline__ floatx4 quad(const floatx16& v, int g) { return floatx4{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]}; }
// X <- a X + B X of 32 columns, from this lane's on.  (An operand's values are those that the result's registers stand for.)
template <int SIDE>
__device__ __forceinline__ void small_update(float* col, int xp, const floatx4* B, float a) {
  floatx16 acc[SIDE];
  floatx4 v[4 * SIDE];
#pragma unroll
  for (int bi = 0; bi < SIDE; ++bi) acc[bi] = zero_acc();
#pragma unroll
  for (int g = 0; g < 4 * SIDE; ++g)
#pragma unroll
    for (int e = 0; e < 4; ++e) v[g][e] = col[(8 * g + e) * xp];
#pragma unroll
  for (int g = 0; g < 4 * SIDE; ++g)
#pragma unroll
    for (int bi = 0; bi < SIDE; ++bi) acc[bi] = mma_f32(B[((g >> 2) * SIDE + bi) * 256 + (g & 3) * 64], v[g], acc[bi]);
#pragma unroll
  for (int g = 0; g < 4 * SIDE; ++g)
#pragma unroll
    for (int e = 0; e < 4; ++e) col[(8 * g + e) * xp] = __builtin_fmaf(a, v[g][e], acc[g >> 2][4 * (g & 3) + e]);
}

template <class S>
__global__ __launch_bounds__(64 * kSmallWaves) void newton_small_kernel(const NewtonTable G, const NewtonStep T, int steps, float eps) {
  __shared__ __align__(16) float lds[kSmallFloats];
  __shared__ double sums[kSmallWaves];
  const NewtonMatrix K = G.of[blockIdx.x];
  const NewtonPlanes L(K.rows, K.cols);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5, l = lane & 31;
  const int M = up32(L.m), N = up32(L.n), xp = N + 4, side = M / 32, blocks = side * side, splits = kSmallWaves / blocks;
  float* x = lds;
  floatx4 *A = reinterpret_cast<floatx4*>(x + M * xp), *B = A + blocks * 256, *part = B + blocks * 256;      // [block][g][lane]

  for (int i = tid; i < M * xp; i += 64 * kSmallWaves) x[i] = 0.f;
  __syncthreads();
  double sum = 0.0;
  constexpr int THREADS = 64 * kSmallWaves;
  const int total = K.rows * K.cols;
  // row and column of every THREADS-th value, one after the other (a division for each was a tenth of the kernel's time)
  struct Place {
    int cols, rows_on, cols_on, r, c;
    __device__ __forceinline__ Place(int at, int cols_) : cols(cols_), rows_on(THREADS / cols_), cols_on(THREADS % cols_), r(at / cols_), c(at % cols_) {}
    __device__ __forceinline__ void next() {
      r += rows_on;
      c += cols_on;
      if (c >= cols) {
        c -= cols;
        ++r;
      }
    }
  };
  Place from(tid, K.cols), to = from;
  for (int first = tid; first < total; first += 8 * THREADS) {
    float v[8];      // (eight loads in flight: one by one, 24 rounds of them were a third of the kernel's time)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = first + e * THREADS < total ? (float)((const S*)K.in)[from.r * K.stride + from.c] : 0.f;
      from.next();
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (first + e * THREADS < total) x[L.turned ? to.c * xp + to.r : to.r * xp + to.c] = v[e];
      sum += (double)v[e] * (double)v[e];
      to.next();
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  if (lane == 0) sums[wave] = sum;
  __syncthreads();
  sum = 0.0;
  for (int w = 0; w < kSmallWaves; ++w) sum += sums[w];
  const double scale = 1.0 / (sqrt(sum) + eps);
  for (int i = tid; i < M * xp; i += 64 * kSmallWaves) x[i] = (float)((double)x[i] * scale);
  __syncthreads();

  for (int step = 0; step < steps; ++step) {
    {
      const int blk = wave % blocks, split = wave / blocks, bi = blk / side, bj = blk % side, groups = N / 8;
      const int per = (groups + splits - 1) / splits;
      const float *xi = x + (32 * bi + l) * xp + 4 * h, *xj = x + (32 * bj + l) * xp + 4 * h;
      floatx16 acc = zero_acc();
#pragma unroll 4
      for (int g = split * per; g < min(groups, (split + 1) * per); ++g)
        acc = mma_f32(*reinterpret_cast<const floatx4*>(xi + 8 * g), *reinterpret_cast<const floatx4*>(xj + 8 * g), acc);
#pragma unroll
      for (int g = 0; g < 4; ++g) part[wave * 256 + g * 64 + lane] = quad(acc, g);
    }
    __syncthreads();
    for (int i = tid; i < blocks * 256; i += 64 * kSmallWaves) {
      floatx4 v = part[i];
      for (int s = 1; s < splits; ++s) v += part[s * blocks * 256 + i];
      A[i] = v;
    }
    __syncthreads();
    if (wave < blocks) {
      const int bi = wave / side, bj = wave % side;
      floatx16 acc = zero_acc();
      for (int bk = 0; bk < side; ++bk)
#pragma unroll
        for (int g = 0; g < 4; ++g) acc = mma_f32(A[(bk * side + bi) * 256 + g * 64 + lane], A[(bk * side + bj) * 256 + g * 64 + lane], acc);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int at = wave * 256 + g * 64 + lane;
        B[at] = T.b * A[at] + T.c * quad(acc, g);
      }
    }
    __syncthreads();
    for (int cb = wave; cb < N / 32; cb += kSmallWaves) {
      float* col = x + 32 * cb + l + 4 * h * xp;
      if (side == 1) small_update<1>(col, xp, B + lane, T.a);
      else small_update<2>(col, xp, B + lane, T.a);
    }
    __syncthreads();
  }
  Place out(tid, K.cols);
#pragma unroll 4
  for (int i = tid; i < total; i += THREADS) {
    ((S*)K.out)[i] = (S)x[L.turned ? out.c * xp + out.r : out.r * xp + out.c];
    out.next();
  }
}

// ------------------------------------------------------------------------------------ launches

typedef _Float16 H16;
// Tiles of a launch.  Time of a round of them on all places, in us for each of the contraction index and beside that (measured from 512 to 4096).
// 128: eight waves and four stages in one work-group a CU, as fast as two work-groups of four and two (1.05 PFLOP/s) with half the time to a
// round; 64: two work-groups a CU, or (DEEP) one of four stages where there are no more tiles than CUs (31 us instead of 52 at 4096); what they read is
// near what an L2 gives (64 bytes a clock to each CU), so theirs is the time with operands that do not all lie there.
enum NewtonSize { WIDE, MIDDLE, SMALL, DEEP, SIZES };
struct SizeCost { int tile, places; double each, beside; };
static constexpr SizeCost kSizes[SIZES] = {{256, 256, 0.0785, 7.0}, {128, 256, 0.0238, 3.5}, {64, 512, 0.021, 2.7}, {64, 256, 0.0089, 3.4}};
template <int SIZE, int P> struct NewtonTiles;
template <int P> struct NewtonTiles<WIDE, P> {
  template <int FORM_A> using Of = TileProduct<H16, P, FORM_A, ROWS, 256, 256, 2, 4, 32, P == 2 ? 2 : P == 1 ? 4 : 3>;
};
template <int P> struct NewtonTiles<MIDDLE, P> {
  template <int FORM_A> using Of = TileProduct<H16, P, FORM_A, ROWS, 128, 128, 4, 2, P == 1 ? 64 : 32, 4>;
};
template <int P> struct NewtonTiles<SMALL, P> {
  template <int FORM_A> using Of = TileProduct<H16, P, FORM_A, ROWS, 64, 64, 2, 2, 64, P == 1 ? 4 : 2>;
};
template <int P> struct NewtonTiles<DEEP, P> {
  template <int FORM_A> using Of = TileProduct<H16, P, FORM_A, ROWS, 64, 64, 2, 2, 64, P == 1 ? 8 : 4>;
};

// The queues of a launch with tiles of kSizes[size], and their length.  Matrices go to the XCDs by eights, back and forth, where that leaves no XCD with
// more than an eighth above the mean; what is over, and large ones, are spread.  (The byte-level model's 24: 1.04 -> 1.00 ms for all five steps.)
template <class Count, class Steps>
static int fill(NewtonTable& t, int size, Count count, Steps steps) {
  const SizeCost& c = kSizes[size];
  double load[8] = {}, sum = 0.;
  const int eights = t.many / 8;
  for (int k = 0; k < 8 * eights; ++k) {
    const NewtonPlanes p(t.of[k].rows, t.of[k].cols);
    const double time = (steps(p) * c.each + c.beside) * count(p, c.tile);
    load[k / 8 % 2 ? 7 - k % 8 : k % 8] += time;
    sum += time;
  }
  const bool by_eights = eights > 0 && *std::max_element(load, load + 8) <= sum / 8 * 1.125;
  int at = 0;
  t.entries = 0;
  for (int k = 0; k < t.many;) {
    const bool eight = by_eights && k < 8 * eights;
    int places = 0;
    for (int i = k; i < k + (eight ? 8 : 1); ++i) {
      const int tiles = count(NewtonPlanes(t.of[i].rows, t.of[i].cols), c.tile);
      places = std::max(places, eight ? tiles : (tiles + 7) / 8);
    }
    t.first[t.entries] = at;
    t.base[t.entries] = (uint8_t)k;
    t.kind[t.entries++] = !eight ? SPREAD : k / 8 % 2 ? REVERSED : EIGHT;
    at += places;
    k += eight ? 8 : 1;
  }
  t.first[t.entries] = at;
  return at;
}
// The tiles whose launch should end first: all tiles' time over the places, in rounds of the shortest, not less than the longest.
template <class Count, class Steps>
static int tile_size(const NewtonTable& t, Count count, Steps steps) {
  int best = 0;
  double least = 0.;
  for (int size = 0; size < SIZES; ++size) {
    const SizeCost& c = kSizes[size];
    double sum = 0., longest = 0., shortest = 1e30;
    for (int k = 0; k < t.many; ++k) {
      const NewtonPlanes p(t.of[k].rows, t.of[k].cols);
      const double one = steps(p) * c.each + c.beside;
      sum += one * count(p, c.tile);
      longest = std::max(longest, one);
      shortest = std::min(shortest, one);
    }
    const double time = std::max(longest, std::ceil(sum / c.places / shortest) * shortest);
    if (size == 0 || time < least) {
      best = size;
      least = time;
    }
  }
  return best;
}

static double long_side(const NewtonPlanes& p) { return p.np; }
static double short_side(const NewtonPlanes& p) { return p.mp; }
template <int SIZE, int P, bool POLY>
static void square(NewtonTable& t, const NewtonStep& s, hipStream_t st) {
  typedef typename NewtonTiles<SIZE, P>::template Of<ROWS> Tiles;
  const int places = fill(t, SIZE, square_tiles, POLY ? short_side : long_side);
  hipLaunchKernelGGL((newton_square_kernel<Tiles, POLY>), dim3(8u * places), dim3(Tiles::THREADS), 0, st, t, s);
}
template <int P, bool POLY>
static void square_any(int size, NewtonTable& t, const NewtonStep& s, hipStream_t st) {
  if (size == WIDE) square<WIDE, P, POLY>(t, s, st);
  else if (size == MIDDLE) square<MIDDLE, P, POLY>(t, s, st);
  else if (size == SMALL) square<SMALL, P, POLY>(t, s, st);
  else square<DEEP, P, POLY>(t, s, st);
}
template <int SIZE, int P, bool LAST, class O>
static void update(NewtonTable& t, const NewtonStep& s, hipStream_t st) {
  typedef typename NewtonTiles<SIZE, P>::template Of<COLUMNS> Tiles;
  const int places = fill(t, SIZE, update_tiles, short_side);
  hipLaunchKernelGGL((newton_update_kernel<Tiles, LAST, O>), dim3(8u * places), dim3(Tiles::THREADS), 0, st, t, s);
}
template <int P, bool LAST, class O>
static void update_any(int size, NewtonTable& t, const NewtonStep& s, hipStream_t st) {
  if (size == WIDE) update<WIDE, P, LAST, O>(t, s, st);
  else if (size == MIDDLE) update<MIDDLE, P, LAST, O>(t, s, st);
  else if (size == SMALL) update<SMALL, P, LAST, O>(t, s, st);
  else update<DEEP, P, LAST, O>(t, s, st);
}

template <class S>
static void newton(NewtonTable& t, NewtonStep s, int steps, float eps, hipStream_t st) {
  hipLaunchKernelGGL((newton_norm_kernel<S>), dim3((unsigned)t.chunks, (unsigned)t.many), dim3(256), 0, st, t);
  const int begin = fill(t, SMALL, begin_parts, short_side);
  // (steps >= 3: the first is none of the last two)
  const int exact = sizeof(S) == 2 && steps >= 3;
  hipLaunchKernelGGL((newton_begin_kernel<S>), dim3(8u * begin), dim3(256), 0, st, t, eps, exact);
  constexpr int LAST_P = std::is_same<S, __bf16>::value ? 1 : 2;      // planes of the last two steps
  const int gram = tile_size(t, square_tiles, long_side), poly = tile_size(t, square_tiles, short_side), un = tile_size(t, update_tiles, short_side);
  for (s.step = 0; s.step < steps; ++s.step) {
    const bool last = s.step == steps - 1;
    s.from = s.step & 1;
    s.both_a = LAST_P == 2 || s.step + 2 < steps;
    s.both_x = LAST_P == 2 || s.step + 3 < steps;
    if (s.both_a && !(s.step == 0 && exact)) square_any<2, false>(gram, t, s, st);
    else square_any<1, false>(gram, t, s, st);
    if (s.both_a) square_any<2, true>(poly, t, s, st);
    else square_any<1, true>(poly, t, s, st);
    if (last) update_any<LAST_P, true, S>(un, t, s, st);
    else if (!s.both_a) update_any<1, false, H16>(un, t, s, st);
    else if (s.step == 0 && exact) update_any<ONE_BY_TWO, false, H16>(un, t, s, st);
    else update_any<2, false, H16>(un, t, s, st);
  }
}

// bytes before the planes: sums of squares, shifts and factors
static size_t newton_head() { return (size_t)kNewtonMany * kNormChunks * 8 + 512; }

}  // namespace nsa

using namespace nsa;

static bool is_small(int rows, int cols) { return newton_small(std::min(rows, cols), std::max(rows, cols)); }

extern "C" int nsa_newton_workspace_bytes(int32_t many, const int32_t* rows, const int32_t* cols, size_t* bytes) {
  if (many < 0 || (many > 0 && (!rows || !cols)) || !bytes) return NSA_E_ARG;
  size_t most = 0, now = 0;
  int large = 0;
  for (int32_t k = 0; k < many; ++k) {
    if (rows[k] <= 0 || cols[k] <= 0) return NSA_E_ARG;
    if (rows[k] > (1 << 20) || cols[k] > (1 << 20) || std::min(rows[k], cols[k]) > (1 << 15)) return NSA_E_UNSUPPORTED;
    if (is_small(rows[k], cols[k])) continue;
    if (large++ % kNewtonMany == 0) now = 0;
    now += (NewtonPlanes(rows[k], cols[k]).halves() * 2 + 255) / 256 * 256;
    most = std::max(most, now);
  }
  if (most >> 40) return NSA_E_UNSUPPORTED;
  *bytes = newton_head() + most;
  return 0;
}

extern "C" int nsa_newton_schulz(int32_t many, const int32_t* rows, const int32_t* cols, const void* const* in, const int64_t* in_stride, void* const* out,
                                 int32_t dtype, int32_t steps, float a, float b, float c, float eps, void* ws, size_t ws_bytes, void* stream) {
  size_t need = 0;
  if (int rc = nsa_newton_workspace_bytes(many, rows, cols, &need)) return rc;
  if (many == 0) return 0;
  if (!in || !in_stride || !out || !ws || (uintptr_t)ws % 256 || dtype < 0 || dtype > 2 || steps < 1 || steps > 100 || !(eps >= 0.f)) return NSA_E_ARG;
  if (ws_bytes < need) return NSA_E_WORKSPACE;
  // singular values start in [0, 1]: where the polynomial takes them has to stay in the planes' range
  for (int i = 0; i <= 1024; ++i) {
    double x = i / 1024.0;
    for (int s = 0; s < steps; ++s) {
      const double l = x * x, f = b * l + c * l * l;
      if (!(std::fabs(f) <= 30.0)) return NSA_E_UNSUPPORTED;
      x = x * (a + f);
      if (!(std::fabs(x) <= 4.0)) return NSA_E_UNSUPPORTED;
    }
  }
  const int each = dtype == 2 ? 4 : 2;
  for (int32_t k = 0; k < many; ++k) {
    if (!in[k] || !out[k] || in_stride[k] < cols[k] || ((uintptr_t)in[k] | (uintptr_t)out[k]) % each) return NSA_E_ARG;
  }
  NewtonStep s{};
  s.a = a; s.b = b; s.c = c;
  s.growth = std::max(0, (int)std::ceil(std::log2(std::max(1e-6f, std::fabs(a)))));
  hipStream_t st = (hipStream_t)stream;
  for (int small = 0; small < 2; ++small)
    for (int32_t k = 0; k < many;) {
      NewtonTable t{};
      t.partial = (double*)ws;
      t.shift = (int*)((char*)ws + (size_t)kNewtonMany * kNormChunks * 8);
      t.factor = (float*)(t.shift + 64);
      t.ws = (char*)ws + newton_head();
      size_t at = 0;
      long largest = 0;
      for (; k < many && t.many < kNewtonMany; ++k) {
        if (is_small(rows[k], cols[k]) != (small == 1)) continue;
        t.of[t.many++] = NewtonMatrix{in[k], out[k], (long)in_stride[k], (unsigned)(at / 256), rows[k], cols[k]};
        at += (NewtonPlanes(rows[k], cols[k]).halves() * 2 + 255) / 256 * 256;
        largest = std::max(largest, (long)rows[k] * cols[k]);
      }
      if (t.many == 0) break;
      // (long contractions first: what is left at the end of a launch is short)
      std::stable_sort(t.of, t.of + t.many, [](const NewtonMatrix& u, const NewtonMatrix& v) { return std::max(u.rows, u.cols) > std::max(v.rows, v.cols); });
      if (small) {
        const dim3 grid((unsigned)t.many), block(64 * kSmallWaves);
        if (dtype == 0) hipLaunchKernelGGL((newton_small_kernel<__bf16>), grid, block, 0, st, t, s, steps, eps);
        else if (dtype == 1) hipLaunchKernelGGL((newton_small_kernel<_Float16>), grid, block, 0, st, t, s, steps, eps);
        else hipLaunchKernelGGL((newton_small_kernel<float>), grid, block, 0, st, t, s, steps, eps);
      } else {
        t.chunks = (int)std::max<long>(1, std::min<long>(kNormChunks, largest / 16384));
        if (dtype == 0) newton<__bf16>(t, s, steps, eps, st);
        else if (dtype == 1) newton<_Float16>(t, s, steps, eps, st);
        else newton<float>(t, s, steps, eps, st);
      }
      if (hipError_t e = hipGetLastError()) return (int)e;
    }
  return 0;
}
