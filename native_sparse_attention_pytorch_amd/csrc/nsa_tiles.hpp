// Tiles of matrix products c[m][n] = sum over k of a(m, k) b(n, k) with fp32 sums, for operands of one or two 16-bit planes.
//
// Two planes are the two halves of a number: hi, it rounded to fp16, and lo, what is left of it rounded to fp16 - 22 bits of significand in
// all.  Three products (hi hi, hi lo, lo hi; the fourth is 2^-22 of the first) then cost a third of the matrix rate, against a sixteenth for
// the fp32 matrix instructions.  The range is fp16's, so who makes the planes scales by a power of two (plane_shift).
//
// A work-group of WM x WN waves makes a TM x TN tile, BK of the contraction index at a time.  All planes' tiles of both operands are copied
// straight into swizzled LDS (global_load_lds: no registers, no store instructions) while the matrix instructions of the stage in use run.
// An operand whose rows run along k (ROWS) is read 16 bytes a lane; one whose rows are k (COLUMNS) through the transposing reads, so no
// operand is laid out anew in memory.  LDS reads bound the tile shape: a wave of 128 x 64 reads 6 KB for 8 products of 32 x 32 x 16, 75 % of
// what LDS gives while they run; with two planes 12 KB feed 24.
//
// Two stages: a stage is waited for at its own start and the next one is copied meanwhile.  Three and more: the first operands of the next
// stage are read at the end of this one, so no LDS latency follows the barrier, and a copy has a stage longer to arrive.
#pragma once
#include "nsa_pipe.hpp"

namespace nsa {

typedef __attribute__((__vector_size__(8 * sizeof(_Float16)))) _Float16 f16x8;
typedef __attribute__((__vector_size__(4 * sizeof(_Float16)))) _Float16 f16x4;
template <class T> struct PlaneVec;
template <> struct PlaneVec<__bf16> { typedef bf16x8 x8; };
template <> struct PlaneVec<_Float16> { typedef f16x8 x8; };

__device__ __forceinline__ floatx16 mma(bf16x8 a, bf16x8 b, floatx16 c) { return mfma32(a, b, c); }
__device__ __forceinline__ floatx16 mma(f16x8 a, f16x8 b, floatx16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// N values from or to an address that is aligned to one of them only: global memory takes wide accesses there as well, and rows of any length
// are read and written as others are
template <class S, int N> struct AnyVec { typedef __attribute__((__vector_size__(N * sizeof(S)), aligned(sizeof(S)))) S type; };
template <int N, class S> __device__ __forceinline__ auto load_any(const S* p) {
  typedef __attribute__((__vector_size__(N * sizeof(S)))) S vec;
  return (vec)*reinterpret_cast<const typename AnyVec<S, N>::type*>(p);
}
template <class S, class V> __device__ __forceinline__ void store_any(S* p, V v) { *reinterpret_cast<typename AnyVec<S, sizeof(V) / sizeof(S)>::type*>(p) = v; }

enum { ROWS = 0, COLUMNS = 1 };

// One operand's tile: R result rows by BK of k.  ROWS: `limit` rows exist (those past it are read as the last one: callers drop their
// results), rows are `ld` apart and hold whole multiples of BK.  COLUMNS: `limit` columns exist (a multiple of 64), whole multiples of BK rows.
template <class T, int FORM, int R, int BK, int WAVES>
struct TileOperand {
  static constexpr int LROW = FORM == COLUMNS ? 64 : BK, CPR = LROW / 8, SEG = 64 / CPR;      // LDS row; rows of one wave's 1 KB copy
  static constexpr unsigned PLANE = R * BK * 2;
  static constexpr int ROUNDS = PLANE / 1024 / WAVES;
  static_assert(ROUNDS * WAVES * 1024 == PLANE && (FORM == ROWS || R % 64 == 0) && (BK == 32 || BK == 64), "the waves copy whole kilobytes");
  static constexpr int READS = FORM == COLUMNS ? 4 : BK / 16;
  unsigned voff[ROUNDS];      // byte offsets of this lane's 16 bytes from the tile's first row (column)
  unsigned at[READS];         // LDS byte offsets of this lane's operand reads
  const T* base;
  long plane, step;

  // chunk c of an LDS row r is at c ^ swz(r): 16 lanes that read the same chunk of 16 rows meet all 64 banks (ROWS); COLUMNS as the
  // transposing reads want it (lds_swz)
  __device__ __forceinline__ static int swz(int r) { return FORM == COLUMNS ? lds_swz(r) : BK == 64 ? (r >> 1) & 7 : (r >> 2) & 3; }

  // first: of the tile, below limit; frag0: the first 32 rows (columns) of this wave in the tile, in units of 32
  __device__ __forceinline__ void init(const T* p, long plane_, long ld, int first, int limit, int frag0, int wave, int lane) {
    plane = plane_;
    base = FORM == COLUMNS ? p + first : p + (long)first * ld;
    step = FORM == COLUMNS ? (long)BK * ld : BK;
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      const int seg = wave + WAVES * r;
      if (FORM == COLUMNS) {
        const int k = seg % (BK / 8) * 8 + lane / 8, col = min(first + seg / (BK / 8) * 64 + 8 * ((lane & 7) ^ swz(k)), limit - 8) - first;
        voff[r] = (unsigned)((long)k * ld + col) * 2u;
      } else {
        const int row = seg * SEG + lane / CPR, src = min(first + row, limit - 1) - first;
        voff[r] = (unsigned)((long)src * ld + 8 * ((lane % CPR) ^ swz(row))) * 2u;
      }
    }
    const int h = lane >> 5;
    if (FORM == COLUMNS) {
      const int ll = lane & 15, e = ll >> 2, qq = ll & 3, mh = (lane >> 4) & 1;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int f = frag0 + (i >> 1), k = 8 * h + e + 4 * (i & 1), chunk = 4 * (f & 1) + 2 * mh + (qq >> 1);
        at[i] = (unsigned)(((f >> 1) * BK + k) * 64 + 8 * (chunk ^ swz(k)) + 4 * (qq & 1)) * 2u;
      }
    } else {
      const int m = lane & 31;
#pragma unroll
      for (int ks = 0; ks < BK / 16; ++ks) at[ks] = (unsigned)((32 * frag0 + m) * BK + 8 * ((2 * ks + h) ^ swz(m))) * 2u;
    }
  }
  // Round r of plane p of the tile at `from` (wave-uniform, as lds is: this wave's first kilobyte of the plane).  lanes: all ones, or zero: no
  // lane takes part then, nothing is read or written and `from` may point anywhere, but the copy counts among those outstanding.  So the
  // last stages need no branch: with one, the compiler kept a second set of sums and spilled registers.
  __device__ __forceinline__ void copy(const T* from, int p, int r, unsigned lds, unsigned lanes) const {
    asm volatile("s_mov_b32 m0, %0\n\ts_mov_b64 vcc, exec\n\ts_mov_b32 exec_lo, %3\n\ts_mov_b32 exec_hi, %3\n\ts_nop 0\n\t"
                 "global_load_lds_dwordx4 %1, %2\n\ts_mov_b64 exec, vcc"
                 :: "s"(lds + p * PLANE + r * WAVES * 1024), "v"(voff[r]), "s"(from + p * plane), "s"(__builtin_amdgcn_readfirstlane(lanes))
                 : "memory", "m0", "vcc");
  }
  // this wave's operand f (of 32 rows or columns; FRAGS of them, an even number or one) of step ks of the plane at lds
  __device__ __forceinline__ typename PlaneVec<T>::x8 read(unsigned lds, int f, int ks) const {
    if (FORM == COLUMNS) {
      const unsigned o = lds + (f >> 1) * BK * 128 + ks * 2048;
      return __builtin_bit_cast(typename PlaneVec<T>::x8, lds_read8_tr(at[2 * (f & 1)] + o, at[2 * (f & 1) + 1] + o));
    }
    return __builtin_bit_cast(typename PlaneVec<T>::x8, lds_read8(at[ks] + lds + f * 64 * BK));
  }
};

// P: planes of both operands, 1 or 2 (three products then), or ONE_BY_TWO: one of a, two of b, and two products
enum { ONE_BY_TWO = 3 };
template <class T_, int P_, int FORM_A, int FORM_B, int TM_, int TN_, int WM_, int WN_, int BK_, int STAGES_>
struct TileProduct {
  typedef T_ T;
  typedef typename PlaneVec<T>::x8 x8;
  static constexpr int P = P_, PA = P == 2 ? 2 : 1, PB = P == 1 ? 1 : 2, TM = TM_, TN = TN_, WM = WM_, WN = WN_, BK = BK_, STAGES = STAGES_, WAVES = WM * WN, THREADS = 64 * WAVES;
  static constexpr int MI = TM / WM / 32, NI = TN / WN / 32, KS = BK / 16, PRODUCTS = PA + PB - 1;
  typedef TileOperand<T, FORM_A, TM, BK, WAVES> OpA;
  typedef TileOperand<T, FORM_B, TN, BK, WAVES> OpB;
  static constexpr unsigned A_BYTES = PA * OpA::PLANE, STAGE = A_BYTES + PB * OpB::PLANE, LDS = STAGES * STAGE;
  static constexpr int LOADS = PA * OpA::ROUNDS + PB * OpB::ROUNDS, MFMAS = KS * PRODUCTS * MI * NI;
  static_assert((MI == 1 || MI % 2 == 0) && (NI == 1 || NI % 2 == 0) && STAGES >= 2 && (STAGES == 2 || (STAGES - 2) * LOADS < 64), "");

  OpA A;
  OpB B;
  floatx16 acc[MI][NI];      // lane l, register e of acc[i][j]: result row row_of(i, e), column col_of(j)
  int lane, wm, wn;
  unsigned lds, mine;        // of the work-group's LDS; of this wave's part in each copy

  __device__ __forceinline__ void init(const void* shared) {
    typedef __attribute__((address_space(3))) const void* lds_p;
    const int tid = threadIdx.x, wave = tid >> 6;
    lane = tid & 63;
    wm = wave / WN;
    wn = wave % WN;
    lds = (unsigned)(unsigned long)(lds_p)shared;
    mine = __builtin_amdgcn_readfirstlane(lds + wave * 1024);
  }
  __device__ __forceinline__ void operand_a(const T* p, long plane, long ld, int first, int limit) { A.init(p, plane, ld, first, limit, wm * MI, threadIdx.x >> 6, lane); }
  __device__ __forceinline__ void operand_b(const T* p, long plane, long ld, int first, int limit) { B.init(p, plane, ld, first, limit, wn * NI, threadIdx.x >> 6, lane); }
  // in the tile: the first of four consecutive rows of registers 4 q .. 4 q + 3, and this lane's column
  __device__ __forceinline__ int row_of(int i, int q) const { return wm * (TM / WM) + 32 * i + 8 * q + 4 * (lane >> 5); }
  __device__ __forceinline__ int col_of(int j) const { return wn * (TN / WN) + 32 * j + (lane & 31); }

  __device__ __forceinline__ void copy(int i, const T* a, const T* b, unsigned to, unsigned lanes) const {
    if (i < PA * OpA::ROUNDS) A.copy(a, i / OpA::ROUNDS, i % OpA::ROUNDS, to, lanes);
    else B.copy(b, (i - PA * OpA::ROUNDS) / OpB::ROUNDS, (i - PA * OpA::ROUNDS) % OpB::ROUNDS, to + A_BYTES, lanes);
  }
  template <int OUTSTANDING>
  __device__ __forceinline__ static void meet() {
    fence();
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(OUTSTANDING) : "memory");
    fence();
  }

  // Columns col_of(j) of the result, each W = TM / WM consecutive values of a row in memory from row_of(0, 0) on: value(i, e) is that of register
  // e of acc[i][j], store(r, c, v) takes the 16 bytes from value c on of column r of this wave's 32 - consecutive lanes consecutive
  // bytes, W of a row together, where lanes as they are would write 16 bytes of 32 rows at a time.  Through this wave's own part of LDS, where
  // what `store` makes of v stays for turned_of.
  static constexpr int W = TM / WM;
  template <class O> static constexpr int PER = 16 / sizeof(O);
  template <class O>
  __device__ __forceinline__ char* own_at(char* shared, int r, int c) const {
    constexpr int CHUNKS = W / PER<O>, MASK = (CHUNKS < 16 ? CHUNKS : 16) - 1;
    return shared + ((wm * WN + wn) * 32 + r) * W * sizeof(O) + 16 * ((c / PER<O>) ^ (r & MASK)) + c % PER<O> * sizeof(O);
  }
  template <class O, class Value, class Store>
  __device__ __forceinline__ void rows_of(char* shared, Value value, Store store) const {
    constexpr int CHUNKS = W / PER<O>;
    static_assert(WAVES * 32 * W * sizeof(O) <= LDS, "");
    typedef __attribute__((__vector_size__(16))) O ox;
    typedef __attribute__((__vector_size__(4 * sizeof(O)))) O o4;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        o4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (O)value(i, 4 * q + e);
        *reinterpret_cast<o4*>(own_at<O>(shared, lane & 31, 32 * i + 8 * q + 4 * (lane >> 5))) = v;
      }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int n = 0; n < 32 * CHUNKS / 64; ++n) {
      const int r = (64 * n + lane) / CHUNKS, c = (64 * n + lane) % CHUNKS * PER<O>;
      ox* at = reinterpret_cast<ox*>(own_at<O>(shared, r, c));
      ox v = *at;
      store(r, c, v);
      *at = v;
    }
    __builtin_amdgcn_wave_barrier();
  }
  // The same values (of floats) the other way: store(r, c, v) takes those of row c of this wave's W in columns r .. r + 3 of its 32.
  template <class Store>
  __device__ __forceinline__ void turned_of(char* shared, Store store) const {
#pragma unroll
    for (int n = 0; n < W / 8; ++n) {
      const int c = 8 * n + (lane >> 3), r = 4 * (lane & 7);
      floatx4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = *reinterpret_cast<const float*>(own_at<float>(shared, r + e, c));
      store(r, c, v);
    }
    __builtin_amdgcn_wave_barrier();
  }

  // two planes: the small products are summed by themselves, where there are registers for it, so that a leading sum is rounded once a
  // product of 16 and not three times; and where there are more, every 256 of the contraction index are a sum of their own (sums of 2048 and
  // 4096 are then off by 1.2e-7 and 1.6e-7 of their size instead of 3e-7 and 4e-7)
  static constexpr bool APART = PB == 2 && MI * NI <= 4, PIECES = PB == 2 && MI * NI <= 2;

  // `steps` times BK of the contraction index from k0 * BK on.  All waves of the work-group; LDS is free again behind it.
  // From stage `tail` on, operand a is read `back` elements before its place: rows that end `back` short of a whole number of stages (the other
  // operand holds zeros in the place of what comes twice).
  __device__ __forceinline__ void run(int steps, int k0 = 0, int tail = -1, int back = 0) {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = zero_acc();
    floatx16 small[APART ? MI : 1][APART ? NI : 1], whole[PIECES ? MI : 1][PIECES ? NI : 1];
    if (APART) {
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) small[APART ? i : 0][APART ? j : 0] = whole[PIECES ? i : 0][PIECES ? j : 0] = zero_acc();
    }
    const T* a = A.base + k0 * A.step;
    const T* b = B.base + k0 * B.step;
    constexpr int FIRST = STAGES - 1;
    constexpr bool AHEAD = STAGES > 2;
#pragma unroll
    for (int s = 0; s < FIRST; ++s) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) copy(i, a, b, mine + s * STAGE, s < steps ? ~0u : 0u);
      a += A.step;
      b += B.step;
      if (s + 1 == tail) a -= back;
    }
    x8 fa[2][PA][MI], fb[2][PB][NI];
    // the operand with fewer parts first, and with all of it each part of the other: products begin as soon as their operands arrive
    constexpr bool A_FIRST = MI <= NI;
    auto read = [&](unsigned stage, int ks, int into) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int p = 0; p < (A_FIRST == (u == 0) ? PA : PB); ++p) {
          if (A_FIRST == (u == 0)) {
#pragma unroll
            for (int i = 0; i < MI; ++i) fa[into][p][i] = A.read(stage + p * OpA::PLANE, i, ks);
          } else {
#pragma unroll
            for (int j = 0; j < NI; ++j) fb[into][p][j] = B.read(stage + A_BYTES + p * OpB::PLANE, j, ks);
          }
        }
      }
    };
    if (AHEAD) {
      meet<(FIRST - 1) * LOADS>();
      read(lds, 0, 0);
    }
    int use = 0, fill = FIRST;      // stage in use, stage to be filled next
    for (int t = 0; t < steps; ++t) {
      meet<(AHEAD ? STAGES - 3 : 0) * LOADS>();
      const unsigned stage = lds + use * STAGE, to = mine + fill * STAGE, lanes = t + FIRST < steps ? ~0u : 0u;
      use = use + 1 == STAGES ? 0 : use + 1;
      fill = fill + 1 == STAGES ? 0 : fill + 1;
      const unsigned next = lds + use * STAGE;
      if (!AHEAD) read(stage, 0, 0);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if (ks + 1 < KS) read(stage, ks + 1, (ks + 1) & 1);
        else if (AHEAD) read(next, 0, 0);
#pragma unroll
        for (int q = 0; q < PRODUCTS; ++q)
#pragma unroll
          for (int v = 0; v < MI * NI; ++v) {
            const int i = A_FIRST ? v % MI : v / NI, j = A_FIRST ? v / MI : v % NI, n = (ks * PRODUCTS + q) * MI * NI + v;
            floatx16& sum = APART && q > 0 ? small[APART ? i : 0][APART ? j : 0] : acc[i][j];
            sum = mma(fa[ks & 1][q == 2 ? PA - 1 : 0][i], fb[ks & 1][q == 1 ? PB - 1 : 0][j], sum);
#pragma unroll
            for (int c = n * LOADS / MFMAS; c < (n + 1) * LOADS / MFMAS; ++c) copy(c, a, b, to, lanes);
          }
      }
      a += A.step;
      b += B.step;
      if (t + FIRST + 1 == tail) a -= back;
      if (PIECES && t % (256 / BK) == 256 / BK - 1) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int j = 0; j < NI; ++j) {
            whole[PIECES ? i : 0][PIECES ? j : 0] += acc[i][j] + small[APART ? i : 0][APART ? j : 0];
            acc[i][j] = small[APART ? i : 0][APART ? j : 0] = zero_acc();
          }
      }
    }
    if (APART) {
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) {
          acc[i][j] += small[APART ? i : 0][APART ? j : 0];
          if (PIECES) acc[i][j] += whole[PIECES ? i : 0][PIECES ? j : 0];
        }
    }
    meet<0>();      // (copies without lanes too; LDS is free)
  }
};

// Of `total` tiles, work-group id's: one run of them to each XCD (work-groups go to the 8 XCDs in turn, each with an L2 of its own).
__device__ __forceinline__ int xcd_run(int id, int total) {
  const int per = total / 8, rest = total % 8, x = id & 7;
  return x * per + min(x, rest) + (id >> 3);
}
// Tile `id` of a grid of tiles_m x tiles_n, in bands of `band` columns, along the rows of the band first: the CUs of an XCD share the operands of
// a few rows and columns of tiles.
struct TileAt { int m, n; };
__device__ __forceinline__ TileAt tile_in(int nth, int tiles_m, int tiles_n, int band) {
  const int g = nth / (band * tiles_m), in = nth - g * band * tiles_m, width = min(band, tiles_n - g * band);
  return TileAt{in / width, g * band + in % width};
}
__device__ __forceinline__ TileAt tile_at(int id, int tiles_m, int tiles_n, int band) { return tile_in(xcd_run(id, tiles_m * tiles_n), tiles_m, tiles_n, band); }
// The same of the tiles on and below the diagonal of `tiles` rows: bands of 8 rows, column by column, then the triangle at the band's end.
__device__ __forceinline__ TileAt triangle_in(int nth, int tiles) {
  int g = (int)(sqrtf((float)nth) * 0.176776695f);      // 32 g^2 + 4 g tiles lie before band g
  while (32 * (g + 1) * (g + 1) + 4 * (g + 1) <= nth) ++g;
  while (32 * g * g + 4 * g > nth) --g;
  const int in = nth - 32 * g * g - 4 * g, rows = min(8, tiles - 8 * g);
  if (in < rows * 8 * g) return TileAt{8 * g + in % rows, in / rows};
  int left = in - rows * 8 * g, c = 0;
  while (left >= rows - c) left -= rows - c++;
  return TileAt{8 * g + c + left, 8 * g + c};
}

// The power of two (its exponent) that scales values below the given magnitude (bits of an fp32, finite) to below 2^15
__device__ __forceinline__ int plane_exponent(unsigned bits) { return (int)(bits >> 23) - 126; }
__device__ __forceinline__ int plane_shift(unsigned bits) { return 15 - plane_exponent(bits); }

struct Halves { _Float16 hi, lo; };
__device__ __forceinline__ Halves halves_of(float x) {
  const _Float16 hi = (_Float16)x;
  const float back = (float)hi;
  return Halves{hi, fabsf(back) < INFINITY ? (_Float16)(x - back) : (_Float16)0.f};      // (an infinity or NaN is in the first half alone)
}

// 8 consecutive 16-bit values a lane from the 4 + 4 of two register quads of a 32 x 32 result: before, lanes of the lower half hold values
// 0-3 (a) and 8-11 (b), those of the upper half 4-7 and 12-15; after, the lower half holds 0-7, the upper 8-15.
__device__ __forceinline__ uintx4 join_quads(uintx2 a, uintx2 b) {
#pragma unroll
  for (int i = 0; i < 2; ++i) asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a[i]), "+v"(b[i]));
  return uintx4{a[0], a[1], b[0], b[1]};
}

}  // namespace nsa
