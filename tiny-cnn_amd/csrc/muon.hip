// muon.hip — the update of a matrix by its orthogonalised momentum (K. Jordan et al., "Muon: an optimizer for hidden layers in neural networks", 2024).
//
// X = U / (|U| + eps), then a few times X <- a X + (b A + c A^2) X with the Gram matrix A of the shorter side (m of min(rows, cols)): A = X X^T, or
// where there are more rows than columns A = X^T X and the product on the right. Nothing is transposed for that: gemm16.h reads an operand
// along either index, and A and A^2 are symmetric.
//
// What a step multiplies is A - alpha I rather than A: with beta = b alpha + c alpha^2
//   b A + c A^2 = beta I + (b + 2 c alpha) (A - alpha I) + c (A - alpha I)^2,   X <- (a + beta) X + (that without beta I) X,
// the same for any alpha. alpha is what the diagonal of A is where all singular values are equal, and then there is little left to round.
//
// Operands are fp16, whose range is enough since every magnitude is known beforehand (bounds of the singular values): X is held as hi + lo times a power
// of two, 22 bits of it, and so are the Gram matrices. A product of hi with hi alone is TDH_F16; with lo's share of both operands, three products, TDH_F32:
// what is left out is 2^-22 of a product. X and all sums are of either kind as precise as that: lo is kept beside hi.
#include "gemm16.h"

#include <cfloat>
#include <cmath>

namespace tdh {

namespace {

constexpr int MU_NT = 256;

// ------------------------------------------------------------------ products

// C = A B of operands in two fp16 parts, p and p + plane, as hi hi + hi lo + lo hi. Tiles of 32 reduction indices of all four, two of
// them in turns; the products of TOGETHER tiles are summed from zero and then added in fp32, since the matrix instruction drops what falls off the end
// of a long sum. 4096^3, us, and the result's error against 64 bits after one step and after five: added after every tile 425; every 8
// 392, 5.6e-7 and 1.1e-6; every 32 384, 9.4e-7 and 1.5e-6; at the end 377, 2.1e-6 and 4.7e-6. Products in fp32 are off by 4e-6 to 7e-6. 4.1e11
// multiplications and additions in 384 us, 1.07 PFLOP/s of fp16, where the library's product of this size reaches 1.12; the counters have the matrix units busy for 62 to 66% of
// the time, and nothing shows what the rest waits for. Tiles of 256 x 128 on eight waves take the same time.
template <int WM, int WN, int TM, int TN, bool A_KC, bool B_KC, class Tiles, class Epi>
__global__ void __launch_bounds__(64 * WM * WN, 2)
gemm16x2_kernel(const G16Matrix A, const G16Matrix B, const long a_plane, const long b_plane, const Epi epi, const int tiles_m, const int tiles_n,
                const int K, const int k_per_split) {
  constexpr int NT = 64 * WM * WN, BM = 32 * TM * WM, BN = 32 * TN * WN, BK = 32, TOGETHER = 32;
  using SideA = G16Side<BM, A_KC, false, NT, BK>;
  using SideB = G16Side<BN, B_KC, false, NT, BK>;
  constexpr int STAGE = 2 * (SideA::BYTES + SideB::BYTES);
  __shared__ __align__(1024) char lds[2][STAGE];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave % WM, wn = wave / WM;
  int id = xcd_compact_id(blockIdx.x, gridDim.x), tm, tn;
  const int split = id / epi.tiles_here;
  id -= split * epi.tiles_here;
  Tiles::place(id + epi.first_tile, tiles_m, tiles_n, tm, tn);
  const int m0 = tm * BM, n0 = tn * BN, kbeg = split * k_per_split, kend = min(K, kbeg + k_per_split);
  SideA sa;
  SideB sb;
  sa.plan(A, m0, tid);
  sb.plan(B, n0, tid);
  g16_f32x16 acc[TM][TN], sum[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = sum[i][j] = g16_f32x16{};
  int oa[TM], ob[TN];
#pragma unroll
  for (int i = 0; i < TM; ++i) oa[i] = SideA::lane_offset(lane, 32 * (wm * TM + i));
#pragma unroll
  for (int j = 0; j < TN; ++j) ob[j] = 2 * SideA::BYTES + SideB::lane_offset(lane, 32 * (wn * TN + j));
  auto fetch = [&](int k0, int buf) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      SideA a = sa;
      SideB b = sb;
      a.base += 2 * p * a_plane;
      b.base += 2 * p * b_plane;
      a.fetch(A, lds[buf] + p * SideA::BYTES, k0, kend - k0, tid);
      b.fetch(B, lds[buf] + 2 * SideA::BYTES + p * SideB::BYTES, k0, kend - k0, tid);
    }
  };
  fetch(kbeg, 0);
  int buf = 0;
#pragma unroll 1
  for (int k0 = kbeg; k0 < kend; k0 += BK) {
    g16_arrived<0>();
    __syncthreads();   // this tile has arrived, and everyone has read the one before
    if (k0 + BK < kend) fetch(k0 + BK, buf ^ 1);
    const char *at = lds[buf];
    g16_s16x8 a[2][TM][2], b[2][TN][2];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
#pragma unroll
        for (int i = 0; i < TM; ++i) a[s][i][p] = SideA::read(at + p * SideA::BYTES, oa[i], lane, s);
#pragma unroll
        for (int j = 0; j < TN; ++j) b[s][j][p] = SideB::read(at + p * SideB::BYTES, ob[j], lane, s);
      }
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int q = 0; q < 3; ++q)   // the small ones first
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int j = 0; j < TN; ++j) sum[i][j] = mfma16(f16(), a[s][i][q == 0], b[s][j][q == 1], sum[i][j]);
    if ((k0 - kbeg) / BK % TOGETHER == TOGETHER - 1 || k0 + BK >= kend)
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            acc[i][j][r] += sum[i][j][r];
            sum[i][j][r] = 0.0f;
          }
    buf ^= 1;
  }
  static_assert(sizeof(lds) >= WM * WN * G16Turn<32 * TN>::BYTES, "");
  __syncthreads();
  epi.template done<TM, TN>(acc, m0 + 32 * TM * wm, n0 + 32 * TN * wn, lane, split, reinterpret_cast<float *>(lds[0] + wave * G16Turn<32 * TN>::BYTES));
}

// A matrix in two fp16 planes, rows of `ld` (a multiple of 8, zero behind `cols`).
struct Planes {
  uint16_t *p;
  long plane;   // elements from hi to lo
  int rows, cols, ld;
  G16Matrix matrix() const { return G16Matrix{p, ld, rows, ld}; }
};
struct Halves {
  uint4 hi, lo;
};
// eight neighbours times `scale`
__device__ __forceinline__ Halves split_halves(const float (&v)[8], const float scale) {
  float h[8], l[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float s = v[e] * scale;
    h[e] = s;
    l[e] = s - static_cast<float>(static_cast<_Float16>(s));
  }
  return Halves{Word<f16>::from(h).raw, Word<f16>::from(l).raw};
}
__device__ __forceinline__ void join_halves(const uint4 hi, const uint4 lo, const float scale, float (&v)[8]) {
  const Word<f16> h{hi}, l{lo};
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (h[e] + l[e]) * scale;
}

// Gives a wave's sums to F in rows: finish(row, column of the first, eight sums). SYM: the tiles above the diagonal get their mirror images.
template <class F, bool SYM>
struct EpiRows {
  F f;
  int rows, cols, tile;          // of C; of a side of the workgroup's tile
  int first_tile, tiles_here;    // of the launch
  float *partial;                // where the tiles are split along k: [split][tile of the launch][tile][tile], which rest_kernel() takes up
  template <int TM, int TN>
  __device__ __forceinline__ void done(const g16_f32x16 (&acc)[TM][TN], const int m0, const int n0, const int lane, const int split, float *lds) const {
    if (partial) {
      const int slot = xcd_compact_id(blockIdx.x, gridDim.x);   // split * tiles_here + the tile
      float *p = partial + static_cast<size_t>(slot) * tile * tile + (m0 % tile + 4 * (lane >> 5)) * tile + n0 % tile + (lane & 31);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r)
#pragma unroll
          for (int j = 0; j < TN; ++j) p[(32 * i + 8 * (r >> 2) + (r & 3)) * tile + 32 * j] = acc[i][j][r];
      return;
    }
    const G16Turn<32 * TN> turn{lds};
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
      for (int j = 0; j < TN; ++j) turn.put(lane, j, [&](int r) { return acc[i][j][r]; });
      turn.rows(lane, [&](int row, int col, const float (&v)[8]) {
        if (m0 + 32 * i + row < rows && n0 + col < cols) f.finish(m0 + 32 * i + row, n0 + col, v);
      });
    }
    if constexpr (SYM) {
      if (m0 / tile == n0 / tile) return;
      constexpr int PART = TM < 2 ? 1 : 2;   // blocks of 32 rows at a time, which become columns
      static_assert(PART <= TN, "");
      const G16Turn<32 * PART> across{lds};
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int i = 0; i < TM; i += PART) {
          const int half = lane >> 5, l32 = lane & 31;
#pragma unroll
          for (int q = 0; q < PART; ++q)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
              *reinterpret_cast<float4 *>(lds + l32 * G16Turn<32 * PART>::STRIDE + 32 * q + 2 * r + 4 * half) =
                  make_float4(acc[i + q][j][r], acc[i + q][j][r + 1], acc[i + q][j][r + 2], acc[i + q][j][r + 3]);
          across.rows(lane, [&](int row, int col, const float (&v)[8]) {
            if (n0 + 32 * j + row < rows && m0 + 32 * i + col < cols) f.finish(n0 + 32 * j + row, m0 + 32 * i + col, v);
          });
        }
    }
  }
};

// The tiles that were split along k: their parts added up, in order, and finished. Bound by reading them.
template <class F, bool SYM, class Tiles>
__global__ void __launch_bounds__(MU_NT)
muon_rest_kernel(const EpiRows<F, SYM> epi, const int tiles_m, const int tiles_n, const int parts) {
  const int side = epi.tile, at = blockIdx.y * MU_NT + threadIdx.x;   // of eight elements
  int tm, tn;
  Tiles::place(blockIdx.x + epi.first_tile, tiles_m, tiles_n, tm, tn);
  const size_t slice = static_cast<size_t>(epi.tiles_here) * side * side;
  const float *p = epi.partial + static_cast<size_t>(blockIdx.x) * side * side;
  {
    const int row = at / (side / 8), col = at % (side / 8) * 8;
    if (tm * side + row < epi.rows && tn * side + col < epi.cols) {
      float v[8] = {};
      for (int s = 0; s < parts; ++s) {
        float o[8];
        load8(p + s * slice + row * side + col, o);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += o[e];
      }
      epi.f.finish(tm * side + row, tn * side + col, v);
    }
  }
  if (!SYM || tm == tn) return;
  const int row = at % side, col = at / side * 8;   // of the mirror image
  if (tn * side + row < epi.rows && tm * side + col < epi.cols) {
    float v[8] = {};
    for (int s = 0; s < parts; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += p[s * slice + (col + e) * side + row];
    epi.f.finish(tn * side + row, tm * side + col, v);
  }
}

__device__ __forceinline__ void put_halves(const Planes &out, const int row, const int col, const Halves &h, const bool lo) {
  uint16_t *p = out.p + static_cast<long>(row) * out.ld + col;
  *reinterpret_cast<uint4 *>(p) = h.hi;
  if (lo) *reinterpret_cast<uint4 *>(p + out.plane) = h.lo;
}
// what lies behind the last column is zero
__device__ __forceinline__ void clear_behind(float (&v)[8], const int col, const int cols) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = col + e < cols ? v[e] : 0.0f;
}

// A - alpha I, times `scale`, from sums that are `from` times A
struct GramFinish {
  Planes out;
  float from, alpha, scale;
  bool lo;
  __device__ __forceinline__ void finish(const int row, const int col, const float (&acc)[8]) const {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = acc[e] * from - (row == col + e ? alpha : 0.0f);
    clear_behind(v, col, out.cols);
    put_halves(out, row, col, split_halves(v, scale), lo);
  }
};
// one * A + sums * square, times `scale`
struct PolyFinish {
  Planes out, gram;
  float one, square, scale;
  bool lo;
  __device__ __forceinline__ void finish(const int row, const int col, const float (&acc)[8]) const {
    const uint16_t *p = gram.p + static_cast<long>(row) * gram.ld + col;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    float v[8];
    join_halves(*reinterpret_cast<const uint4 *>(p), lo ? *reinterpret_cast<const uint4 *>(p + gram.plane) : zero, one, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = __builtin_fmaf(acc[e], square, v[e]);
    clear_behind(v, col, out.cols);
    put_halves(out, row, col, split_halves(v, scale), lo);
  }
};

// What becomes of X after the last step: w = keep * w + take * X (w fp32), or y = X.
template <class T>
struct Apply {
  T *out;
  int cols;
  bool add;
  float keep, take;
  __device__ __forceinline__ void one(const int row, const int col, const float v) const {
    T *p = out + static_cast<long>(row) * cols + col;
    *p = from_f32<T>(add ? keep * to_f32(*p) + take * v : v);
  }
  __device__ __forceinline__ void operator()(const int row, const int col, const float (&v)[8]) const {
    T *p = out + static_cast<long>(row) * cols + col;
    float o[8];
    if (col + 8 <= cols) {
      if (add) load8(p, o);
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = add ? keep * o[e] + take * v[e] : v[e];
      return store8(p, o);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (col + e < cols) p[e] = from_f32<T>(add ? keep * to_f32(p[e]) + take * v[e] : v[e]);
  }
};
// keep * X + sums * part, `keep` of the planes as they are
__device__ __forceinline__ void next_x(const Planes &x, const float keep, const float part, const int row, const int col, const float (&acc)[8],
                                       float (&v)[8]) {
  const uint16_t *p = x.p + static_cast<long>(row) * x.ld + col;
  join_halves(*reinterpret_cast<const uint4 *>(p), *reinterpret_cast<const uint4 *>(p + x.plane), keep, v);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = __builtin_fmaf(acc[e], part, v[e]);
}
struct StepFinish {
  Planes x, next;
  float keep, part, scale;
  __device__ __forceinline__ void finish(const int row, const int col, const float (&acc)[8]) const {
    float v[8];
    next_x(x, keep, part, row, col, acc, v);
    clear_behind(v, col, x.cols);
    put_halves(next, row, col, split_halves(v, scale), true);
  }
};
template <class T>
struct LastFinish {
  Planes x;
  float keep, part;
  Apply<T> apply;
  __device__ __forceinline__ void finish(const int row, const int col, const float (&acc)[8]) const {
    float v[8];
    next_x(x, keep, part, row, col, acc, v);
    apply(row, col, v);
  }
};

// Tiles, by the size of the product: a side, the workgroups that a compute unit holds, us of 64 reduction indices and beside them. Whole rounds
// of workgroups take whole tiles; the tiles of a last round that is not half full are split along k, which takes two more launches (4096 x 4096 of
// two parts, symmetric: 528 tiles of 128 on 512 places 235 us, unsplit 314). Of the tiles and splits at eleven sizes from 160^2 to 1024 x 4096 the
// rule's choices take 4.6% longer than the best of each.
struct MuTile {
  int side, per_cu;
  double us, round_us;
};
constexpr MuTile MU_TILES[] = {{256, 1, 1.65, 8.0}, {128, 2, 0.92, 5.0}, {64, 4, 0.78, 3.0}};    // hi alone
constexpr MuTile MU_TILES2[] = {{128, 2, 2.6, 6.0}, {64, 4, 2.2, 4.0}};                          // three products
struct MuSplit {
  int side, whole, parts, k_per_part;   // whole: tiles that are not split
};
template <int N>
MuSplit mu_plan(const MuTile (&tiles)[N], int M, int Ncols, int K, bool sym) {
  const long cus = std::max(1, ctx().compute_units);
  MuSplit best{};
  double best_us = 1e30;
  const int ktiles = ceil_div(K, 64);
  for (const MuTile &t : tiles) {
    const long tm = ceil_div(M, t.side), tn = ceil_div(Ncols, t.side), all = sym ? tm * (tm + 1) / 2 : tm * tn, places = cus * t.per_cu;
    const long rounds = all / places, rest = all % places;
    const double round_us = ktiles * t.us + t.round_us;
    auto take = [&](double us, const MuSplit &s) {
      if (us < best_us) {
        best_us = us;
        best    = s;
      }
    };
    take((rounds + (rest ? 1 : 0)) * round_us, MuSplit{t.side, static_cast<int>(all), 1, ktiles * 64});
    if (!rest) continue;
    const int per = ceil_div(ktiles, static_cast<int>(std::min<long>(std::max(1l, places / rest), std::min(16, std::max(1, ktiles / 2)))));
    const int parts = ceil_div(ktiles, per);
    if (parts < 2) continue;
    const double bytes = 8.0 * rest * parts * t.side * t.side;
    take(rounds * round_us + per * t.us + t.round_us + 8.0 + bytes / 4e6, MuSplit{t.side, static_cast<int>(all - rest), parts, per * 64});
  }
  return best;
}
MuSplit mu_plan(bool two, int M, int N, int K, bool sym) { return two ? mu_plan(MU_TILES2, M, N, K, sym) : mu_plan(MU_TILES, M, N, K, sym); }
int mu_tiles(const MuSplit &s, int M, int N, bool sym) {
  const int tm = ceil_div(M, s.side), tn = ceil_div(N, s.side);
  return sym ? G16LowerTiles::count(tm, tn) : G16AllTiles::count(tm, tn);
}
size_t mu_partial_bytes(bool two, int M, int N, int K, bool sym) {
  const MuSplit s = mu_plan(two, M, N, K, sym);
  return s.parts > 1 ? ws_align(4 * static_cast<size_t>(mu_tiles(s, M, N, sym) - s.whole) * s.parts * s.side * s.side) : 0;
}

template <bool A_KC, bool B_KC, bool SYM, class F>
int mu_gemm(bool two, const Planes &a, const Planes &b, const F &f, int M, int N, int K, float *partial, const char *tag) {
  ProfScope prof(tag, M, N, K);
  using Tiles = typename std::conditional<SYM, G16LowerTiles, G16AllTiles>::type;
  using Epi   = EpiRows<F, SYM>;
  const MuSplit plan = mu_plan(two, M, N, K, SYM);
  const int side = plan.side, tm = ceil_div(M, side), tn = ceil_div(N, side), rest = mu_tiles(plan, M, N, SYM) - plan.whole;
  const G16Matrix A = a.matrix(), B = b.matrix();
  auto launch = [&](const Epi &epi, int parts, int k_per_part) {
    const dim3 grid(static_cast<unsigned>(epi.tiles_here * parts));
    if (two) {
      if (side == 128)
        TDH_LAUNCH((gemm16x2_kernel<2, 2, 2, 2, A_KC, B_KC, Tiles, Epi>), grid, dim3(256), 0, ctx().stream, A, B, a.plane, b.plane, epi, tm, tn, K, k_per_part);
      else
        TDH_LAUNCH((gemm16x2_kernel<2, 1, 1, 2, A_KC, B_KC, Tiles, Epi>), grid, dim3(128), 0, ctx().stream, A, B, a.plane, b.plane, epi, tm, tn, K, k_per_part);
    } else {
      if (side == 256)
        TDH_LAUNCH((gemm16_kernel<f16, 2, 4, 4, 2, 2, A_KC, B_KC, false, Epi, Tiles>), grid, dim3(512), 0, ctx().stream, A, B, epi, tm, tn, K, k_per_part);
      else if (side == 128)
        TDH_LAUNCH((gemm16_kernel<f16, 2, 2, 2, 2, 2, A_KC, B_KC, false, Epi, Tiles>), grid, dim3(256), 0, ctx().stream, A, B, epi, tm, tn, K, k_per_part);
      else
        TDH_LAUNCH((gemm16_kernel<f16, 2, 1, 1, 2, 2, A_KC, B_KC, false, Epi, Tiles>), grid, dim3(128), 0, ctx().stream, A, B, epi, tm, tn, K, k_per_part);
    }
    TDH_LAUNCH_CHECK();
    return static_cast<int>(TDH_OK);
  };
  if (plan.whole) TDH_TRY(launch(Epi{f, M, N, side, 0, plan.whole, nullptr}, 1, ceil_div(K, 64) * 64));
  if (!rest) return TDH_OK;
  const Epi epi{f, M, N, side, plan.whole, rest, partial};
  TDH_TRY(launch(epi, plan.parts, plan.k_per_part));
  TDH_LAUNCH((muon_rest_kernel<F, SYM, Tiles>), dim3(rest, side * side / 8 / MU_NT), dim3(MU_NT), 0, ctx().stream, epi, tm, tn, plan.parts);
  TDH_LAUNCH_CHECK();
  return TDH_OK;
}

// -------------------------------------------------------------- U and its size
// U of eight elements from `at`, of `n` in all (zero behind them): the gradient itself, or the momentum that it goes into, and with nesterov on to
// what the next gradient would be. FIRST: the momentum is still the one before.
template <class T>
struct Momentum {
  const T *g;
  float *momentum;   // or null: U is g
  float grad_scale, mu;
  bool nesterov;
  // one element, with the momentum's update
  __device__ __forceinline__ float one(const size_t at) const {
    const float v = to_f32(g[at]);
    if (!momentum) return v;
    const float s = v * grad_scale, m = mu * momentum[at] + s;
    momentum[at] = m;
    return nesterov ? s + mu * m : m;
  }
  template <bool FIRST>
  __device__ __forceinline__ void get(const size_t at, const int n, float (&u)[8]) const {
    float m[8];
    if (n >= 8) {
      load8(g + at, u);
      if (momentum) load8(momentum + at, m);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        u[e] = e < n ? to_f32(g[at + e]) : 0.0f;
        m[e] = e < n && momentum ? momentum[at + e] : 0.0f;
      }
    }
    if (!momentum) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float s = u[e] * grad_scale;
      if (FIRST) m[e] = mu * m[e] + s;
      u[e] = nesterov ? s + mu * m[e] : m[e];
    }
    if (!FIRST) return;
    if (n >= 8) return store8(momentum + at, m);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) momentum[at + e] = m[e];
  }
};

constexpr int MU_PARTS = 1024;   // workgroups of the first pass at most
// the sum of squares, in 64 bits: U may be of any size. Bound by memory.
template <class T>
__global__ void __launch_bounds__(MU_NT)
muon_norm_kernel(const Momentum<T> u, const size_t n, double *__restrict__ partial) {
  __shared__ double waves[MU_NT / 64];
  double s = 0.0;
  const size_t items = (n + 7) / 8, step = static_cast<size_t>(gridDim.x) * MU_NT;
  for (size_t i = static_cast<size_t>(blockIdx.x) * MU_NT + threadIdx.x; i < items; i += step) {
    float v[8];
    u.template get<true>(8 * i, static_cast<int>(n - 8 * i < 8 ? n - 8 * i : 8), v);
#pragma unroll
    for (int e = 0; e < 8; ++e) s = __builtin_fma(static_cast<double>(v[e]), static_cast<double>(v[e]), s);
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < MU_NT / 64; ++w) s += waves[w];
    partial[blockIdx.x] = s;
  }
}
// one over the size, from the partial sums, by every workgroup for itself
__device__ __forceinline__ double inverse_norm(const double *__restrict__ partial, const int parts, const double eps) {
  __shared__ double waves[MU_NT / 64];
  double s = 0.0;
  for (int i = threadIdx.x; i < parts; i += MU_NT) s += partial[i];
#pragma unroll
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = s;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int w = 0; w < MU_NT / 64; ++w) s += waves[w];
  return 1.0 / (sqrt(s) + eps);
}
// X = U / (|U| + eps) in its planes
template <class T>
__global__ void __launch_bounds__(MU_NT)
muon_start_kernel(const Momentum<T> u, const Planes x, const float scale, const double *__restrict__ partial, const int parts, const double eps) {
  const double inverse = inverse_norm(partial, parts, eps);
  const long words = x.ld / 8, total = words * x.rows;
  for (long i = static_cast<long>(blockIdx.x) * MU_NT + threadIdx.x; i < total; i += static_cast<long>(gridDim.x) * MU_NT) {
    const long row = i / words;
    const int col = static_cast<int>(i - row * words) * 8;
    float v[8];
    u.template get<false>(static_cast<size_t>(row) * x.cols + col, min(8, x.cols - col), v);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = static_cast<float>(static_cast<double>(v[e]) * inverse);
    put_halves(x, static_cast<int>(row), col, split_halves(v, scale), true);
  }
}
// (no steps) X as it is
template <class T>
__global__ void __launch_bounds__(MU_NT)
muon_end_kernel(const Planes x, const float unscale, const Apply<T> apply) {
  const long words = x.ld / 8, total = words * x.rows;
  for (long i = static_cast<long>(blockIdx.x) * MU_NT + threadIdx.x; i < total; i += static_cast<long>(gridDim.x) * MU_NT) {
    const long row = i / words;
    const int col = static_cast<int>(i - row * words) * 8;
    const uint16_t *p = x.p + row * x.ld + col;
    float v[8];
    join_halves(*reinterpret_cast<const uint4 *>(p), *reinterpret_cast<const uint4 *>(p + x.plane), unscale, v);
    apply(static_cast<int>(row), col, v);
  }
}

// ------------------------------------------------------------------ the steps
// The scalars of every step, and the powers of two that take the largest X, A and polynomial to fp16's upper end (half of it: what rounding adds
// to a singular value is little).
constexpr int MU_STEPS = 32;
struct MuPlan {
  float alpha[MU_STEPS];   // taken from A's diagonal
  float x_scale, a_scale, b_scale;
};
bool mu_scalars(const tdh_muon &o, int m, MuPlan *p) {
  const double a = o.a, b = o.b, c = o.c;
  if (!std::isfinite(a + b + c)) return false;
  double most = 1.0, worst = 1.0, poly = 0.0, gram = 0.0, flat = 1.0 / std::sqrt(static_cast<double>(m));
  for (int k = 0; k < o.steps; ++k) {
    const double alpha = flat * flat, beta = b * alpha + c * alpha * alpha, top = most * most;
    double next = 0.0;
    auto at = [&](double t) {   // of a singular value whose square is t, up to `top`
      if (!(t >= 0.0 && t <= top)) return;
      const double q = b * t + c * t * t;
      next = std::max(next, std::fabs(std::sqrt(t) * (a + q)));
      poly = std::max(poly, std::fabs(q - beta));
    };
    // the ends, and where a slope is none: a + 3 b t + 5 c t^2 = 0, or b + 2 c t = 0 (a quotient by 0 is beyond `top` or NaN, which at() leaves out)
    const double root = 9.0 * b * b - 20.0 * a * c;
    at(0.0);
    at(top);
    at(-b / (2.0 * c));
    if (root >= 0.0) {   // (a sum of two numbers of one sign: their difference has no figures left where c is small)
      const double q = -0.5 * (3.0 * b + std::copysign(std::sqrt(root), b));
      at(q / (5.0 * c));
      at(a / q);
    }
    if (!(next <= 4.0)) return false;
    gram = std::max(gram, most * most + alpha);
    if (p) p->alpha[k] = static_cast<float>(alpha);
    most  = std::max(next, 1e-30);
    worst = std::max(worst, most);
    flat  = std::fabs(flat * (a + b * alpha + c * alpha * alpha));
  }
  auto scale = [](double most) { return static_cast<float>(std::exp2(std::floor(std::log2(30000.0 / std::max(most, 1e-3))))); };
  if (p) {
    p->x_scale = scale(worst);
    p->a_scale = scale(gram);
    p->b_scale = scale(poly);
  }
  return true;
}

// ------------------------------------------------------------- small matrices
// All of it by one workgroup, in one launch: X in its two parts twice in LDS, along either index, and the Gram matrix, whose place the polynomial takes. A
// wave has 32 x 32 of X, in fp32, from the first step to the last. Three products in either kind. Bound by a chain of barriers and of LDS reads;
// 120 x 84: 45 us, as launches of their own 117.
constexpr int MS_NT = 1024, MS_PAD = 8;   // (rows of LDS of 16 bytes more: 32 of them are read at a time)
struct MuSmall {
  int m, n, mp, np, steps;   // mp, np: in whole blocks of 32
  bool tall;                 // X is the matrix turned round
  double a, b, c, eps;
  MuPlan plan;
};
size_t mu_small_bytes(int mp, int np) {
  return 2 * sizeof(uint16_t) * (static_cast<size_t>(mp) * (np + MS_PAD) + static_cast<size_t>(np) * (mp + MS_PAD) + static_cast<size_t>(mp) * (mp + MS_PAD));
}
constexpr size_t MS_LDS = 156 << 10;
bool mu_small(int rows, int cols) {
  const int mp = ceil_div(std::min(rows, cols), 32) * 32, np = ceil_div(std::max(rows, cols), 32) * 32;
  return static_cast<long>(mp) * np <= 16 * 1024 && mu_small_bytes(mp, np) <= MS_LDS;
}
template <class T, class D>
__global__ void __launch_bounds__(MS_NT)
muon_small_kernel(const Momentum<T> u, const Apply<D> apply, const MuSmall s) {
  extern __shared__ __align__(16) uint16_t small_lds[];
  __shared__ double sums[MS_NT / 64];
  struct Matrix {
    uint16_t *hi, *lo;
    int ld;
    __device__ __forceinline__ void put(const int row, const int col, const float v) const {
      const _Float16 h = static_cast<_Float16>(v), l = static_cast<_Float16>(v - static_cast<float>(h));
      hi[row * ld + col] = __builtin_bit_cast(uint16_t, h);
      lo[row * ld + col] = __builtin_bit_cast(uint16_t, l);
    }
    __device__ __forceinline__ float get(const int row, const int col) const {
      return static_cast<float>(__builtin_bit_cast(_Float16, hi[row * ld + col])) + static_cast<float>(__builtin_bit_cast(_Float16, lo[row * ld + col]));
    }
    // four neighbours of a row, from a multiple of four on
    typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
    __device__ __forceinline__ void put4(const int row, const int col, const float (&v)[4]) const {
      f16x4 h, l;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        h[e] = static_cast<_Float16>(v[e]);
        l[e] = static_cast<_Float16>(v[e] - static_cast<float>(h[e]));
      }
      *reinterpret_cast<f16x4 *>(hi + row * ld + col) = h;
      *reinterpret_cast<f16x4 *>(lo + row * ld + col) = l;
    }
    __device__ __forceinline__ void get4(const int row, const int col, float (&v)[4]) const {
      const f16x4 h = *reinterpret_cast<const f16x4 *>(hi + row * ld + col), l = *reinterpret_cast<const f16x4 *>(lo + row * ld + col);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = static_cast<float>(h[e]) + static_cast<float>(l[e]);
    }
  };
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, l32 = lane & 31;
  Matrix X, Xt, G;
  uint16_t *at = small_lds;
  auto take = [&](Matrix &mat, int rows, int ld) {
    mat = Matrix{at, at + rows * ld, ld};
    at += 2 * rows * ld;
  };
  take(X, s.mp, s.np + MS_PAD);
  take(Xt, s.np, s.mp + MS_PAD);
  take(G, s.mp, s.mp + MS_PAD);
  for (int i = tid; i < (at - small_lds) / 8; i += MS_NT) reinterpret_cast<uint4 *>(small_lds)[i] = make_uint4(0, 0, 0, 0);
  const int total = s.m * s.n, cols = s.tall ? s.m : s.n;
  float held[16];
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    held[i] = tid + i * MS_NT < total ? u.one(tid + i * MS_NT) : 0.0f;
    sum = __builtin_fma(static_cast<double>(held[i]), static_cast<double>(held[i]), sum);
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
  if (lane == 0) sums[wave] = sum;
  __syncthreads();
  sum = 0.0;
#pragma unroll
  for (int w = 0; w < MS_NT / 64; ++w) sum += sums[w];
  const double inverse = 1.0 / (sqrt(sum) + s.eps);
  const float xs = s.plan.x_scale, as = s.plan.a_scale, bs = s.plan.b_scale;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int e = tid + i * MS_NT;
    if (e >= total) break;
    const int row = e / cols, col = e - row * cols, m = s.tall ? col : row, n = s.tall ? row : col;
    const float v = static_cast<float>(static_cast<double>(held[i]) * inverse) * xs;
    X.put(m, n, v);
    Xt.put(n, m, v);
  }
  __syncthreads();
  const int tn = s.np / 32, tg = s.mp / 32, x0 = wave / tn * 32, x1 = wave % tn * 32, g0 = wave / tg * 32, g1 = wave % tg * 32;
  const bool has_x = wave < s.mp / 32 * tn, has_g = wave < tg * tg;
  // the element of this lane's register r, of a block at (row0, col0): row0 + row_of(r), col0 + l32
  auto row_of = [&](int r) { return 8 * (r >> 2) + 4 * half + (r & 3); };
  float x[16];
  if (has_x)
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = X.get(x0 + row_of(r), x1 + l32);
  // a block of A B^T, both along their rows of `len` (a multiple of 32)
  auto product = [&](const Matrix &A, const int a0, const Matrix &B, const int b0, const int len) {
    g16_f32x16 acc{}, more{};
    const int ao = (a0 + l32) * A.ld + 8 * half, bo = (b0 + l32) * B.ld + 8 * half;
    auto part = [](const uint16_t *p) { return *reinterpret_cast<const g16_s16x8 *>(p); };
#pragma unroll 1
    for (int k = 0; k < len; k += 32) {   // (two sums, so that an instruction need not wait for the one before)
      const g16_s16x8 ah = part(A.hi + ao + k), al = part(A.lo + ao + k), bh = part(B.hi + bo + k), bl = part(B.lo + bo + k);
      const g16_s16x8 ch = part(A.hi + ao + k + 16), cl = part(A.lo + ao + k + 16), dh = part(B.hi + bo + k + 16), dl = part(B.lo + bo + k + 16);
      acc  = mfma16(f16(), al, bh, acc);
      more = mfma16(f16(), cl, dh, more);
      acc  = mfma16(f16(), ah, bl, acc);
      more = mfma16(f16(), ch, dl, more);
      acc  = mfma16(f16(), ah, bh, acc);
      more = mfma16(f16(), ch, dh, more);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] += more[r];
    return acc;
  };
#pragma unroll 1
  for (int k = 0; k < s.steps; ++k) {
    // (addresses are made anew in every step: kept from one to the next they take more registers than there are)
    asm volatile("" : "+s"(X.ld), "+s"(Xt.ld), "+s"(G.ld));
    const double alpha = s.plan.alpha[k];
    if (has_g) {
      const g16_f32x16 acc = product(X, g0, X, g1, s.np);
      const float from = 1.0f / (xs * xs), al = static_cast<float>(alpha);
      // (a lane has four neighbours of a column, which are as well four of a row)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int row = g0 + row_of(r), col = g1 + l32;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = row + e < s.m && col < s.m ? (acc[r + e] * from - (row + e == col ? al : 0.0f)) * as : 0.0f;
        G.put4(col, row, v);
      }
    }
    __syncthreads();
    float p[16];
    if (has_g) {
      const g16_f32x16 acc = product(G, g0, G, g1, s.mp);
      const float one = static_cast<float>(s.b + 2.0 * s.c * alpha) / as, square = static_cast<float>(s.c) / (as * as);
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        float v[4];
        G.get4(g1 + l32, g0 + row_of(r), v);
#pragma unroll
        for (int e = 0; e < 4; ++e) p[r + e] = __builtin_fmaf(acc[r + e], square, one * v[e]) * bs;
      }
    }
    __syncthreads();
    asm volatile("" : "+s"(G.ld));
    if (has_g)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const float v[4] = {p[r], p[r + 1], p[r + 2], p[r + 3]};
        G.put4(g1 + l32, g0 + row_of(r), v);
      }
    __syncthreads();
    if (has_x) {
      const g16_f32x16 acc = product(G, x0, Xt, x1, s.mp);
      const float keep = static_cast<float>(s.a + s.b * alpha + s.c * alpha * alpha), part = 1.0f / bs;   // (x is xs times X)
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = __builtin_fmaf(acc[r], part, keep * x[r]);
    }
    __syncthreads();
    if (k + 1 == s.steps) break;
    asm volatile("" : "+s"(X.ld), "+s"(Xt.ld));
    if (has_x)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const float v[4] = {x[r], x[r + 1], x[r + 2], x[r + 3]};
        Xt.put4(x1 + l32, x0 + row_of(r), v);
#pragma unroll
        for (int e = 0; e < 4; ++e) X.put(x0 + row_of(r + e), x1 + l32, v[e]);
      }
    __syncthreads();
  }
  if (!has_x) return;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int m = x0 + row_of(r), n = x1 + l32;
    if (m < s.m && n < s.n) apply.one(s.tall ? n : m, s.tall ? m : n, x[r] / xs);
  }
}

struct MuBuffers {
  Planes x[2], gram, poly;
  double *partial;
};
size_t planes_bytes(int rows, int ld) { return ws_align(4 * static_cast<size_t>(rows) * ld); }
int mu_ld(int cols) { return (cols + 7) & ~7; }
// the largest of what the three products of a step leave in parts
size_t mu_partial_bytes(bool two, int rows, int cols) {
  const int m = std::min(rows, cols);
  return std::max({mu_partial_bytes(two, m, m, rows > cols ? rows : mu_ld(cols), true), mu_partial_bytes(two, m, m, mu_ld(m), true),
                   rows > cols ? mu_partial_bytes(two, rows, m, mu_ld(m), false) : mu_partial_bytes(two, m, cols, m, false)});
}
size_t mu_bytes(bool two, int rows, int cols) {
  const int m = std::min(rows, cols);
  return ws_align(8 * MU_PARTS) + 2 * planes_bytes(rows, mu_ld(cols)) + 2 * planes_bytes(m, mu_ld(m)) + mu_partial_bytes(two, rows, cols);
}
int take_planes(int rows, int cols, Planes *out) {
  const int ld = mu_ld(cols);
  void *p = nullptr;
  TDH_TRY(ws_take(4 * static_cast<size_t>(rows) * ld, &p));
  *out = Planes{static_cast<uint16_t *>(p), static_cast<long>(rows) * ld, rows, cols, ld};
  return TDH_OK;
}

// U by its rows to `apply`
template <class T, class D>
int mu_run(const tdh_muon &o, int rows, int cols, const Momentum<T> &u, const Apply<D> &apply) {
  const int m = std::min(rows, cols);
  const bool tall = rows > cols, two = o.products == TDH_F32;
  MuPlan plan;
  mu_scalars(o, m, &plan);
  if (mu_small(rows, cols)) {
    const int n = std::max(rows, cols), mp = ceil_div(m, 32) * 32, np = ceil_div(n, 32) * 32;
    const MuSmall small{m, n, mp, np, o.steps, tall, o.a, o.b, o.c, o.eps, plan};
    const size_t lds = mu_small_bytes(mp, np);
    ProfScope prof("muon_small", static_cast<double>(o.steps) * (3.0 * m * m * n + 1.0 * m * m * m), WORK_FLOP);
    TDH_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(muon_small_kernel<T, D>), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(MS_LDS)));
    TDH_LAUNCH((muon_small_kernel<T, D>), dim3(1), dim3(MS_NT), lds, ctx().stream, u, apply, small);
    TDH_LAUNCH_CHECK();
    return TDH_OK;
  }
  MuBuffers w;
  TDH_TRY(ws_begin(mu_bytes(two, rows, cols)));
  void *partial = nullptr;
  TDH_TRY(ws_take(8 * MU_PARTS, &partial));
  w.partial = static_cast<double *>(partial);
  for (Planes &x : w.x) TDH_TRY(take_planes(rows, cols, &x));
  TDH_TRY(take_planes(m, m, &w.gram));
  TDH_TRY(take_planes(m, m, &w.poly));
  void *parts_of_tiles = nullptr;
  if (const size_t bytes = mu_partial_bytes(two, rows, cols)) TDH_TRY(ws_take(bytes, &parts_of_tiles));
  float *tp = static_cast<float *>(parts_of_tiles);

  const size_t n  = static_cast<size_t>(rows) * cols;
  const int cus   = std::max(1, ctx().compute_units);
  const int parts = static_cast<int>(std::min<size_t>(MU_PARTS, ceil_div_sz(n, 8 * MU_NT)));
  {
    ProfScope prof("muon_norm", (sizeof(T) + (u.momentum ? 8.0 : 0.0)) * n, WORK_BYTE);
    TDH_LAUNCH((muon_norm_kernel<T>), dim3(parts), dim3(MU_NT), 0, ctx().stream, u, n, w.partial);
    TDH_LAUNCH_CHECK();
  }
  const size_t words  = static_cast<size_t>(rows) * w.x[0].ld / 8;
  const unsigned grid = static_cast<unsigned>(std::min<size_t>(ceil_div_sz(words, MU_NT), 8 * static_cast<size_t>(cus)));
  {
    ProfScope prof("muon_start", (sizeof(T) + (u.momentum ? 8.0 : 4.0)) * n, WORK_BYTE);
    TDH_LAUNCH((muon_start_kernel<T>), dim3(grid), dim3(MU_NT), 0, ctx().stream, u, w.x[0], plan.x_scale, w.partial, parts, static_cast<double>(o.eps));
    TDH_LAUNCH_CHECK();
  }
  if (o.steps == 0) {
    ProfScope prof("muon_end", 8.0 * n, WORK_BYTE);
    TDH_LAUNCH((muon_end_kernel<D>), dim3(grid), dim3(MU_NT), 0, ctx().stream, w.x[0], 1.0f / plan.x_scale, apply);
    TDH_LAUNCH_CHECK();
    return TDH_OK;
  }
  const float xs = plan.x_scale, as = plan.a_scale, bs = plan.b_scale;
  for (int k = 0; k < o.steps; ++k) {
    const Planes &x = w.x[k & 1], &next = w.x[(k + 1) & 1];
    const float alpha = plan.alpha[k];
    const GramFinish gram{w.gram, 1.0f / (xs * xs), alpha, as, two};
    if (tall)
      TDH_TRY((mu_gemm<false, false, true>(two, x, x, gram, m, m, rows, tp, "muon_gram")));
    else
      TDH_TRY((mu_gemm<true, true, true>(two, x, x, gram, m, m, x.ld, tp, "muon_gram")));
    const PolyFinish poly{w.poly, w.gram, (o.b + 2.0f * o.c * alpha) / as, o.c / (as * as), bs, two};
    TDH_TRY((mu_gemm<true, true, true>(two, w.gram, w.gram, poly, m, m, w.gram.ld, tp, "muon_poly")));
    const double a64 = alpha;
    const float keep = static_cast<float>((o.a + o.b * a64 + o.c * a64 * a64) / xs), part = 1.0f / (bs * xs);
    auto step = [&](const auto &finish) {
      return tall ? mu_gemm<true, true, false>(two, x, w.poly, finish, rows, m, w.poly.ld, tp, "muon_step")
                  : mu_gemm<true, false, false>(two, w.poly, x, finish, m, cols, m, tp, "muon_step");
    };
    if (k + 1 < o.steps)
      TDH_TRY(step(StepFinish{x, next, keep, part, xs}));
    else
      TDH_TRY(step(LastFinish<D>{x, keep, part, apply}));
  }
  return TDH_OK;
}

constexpr int MU_SHORT = 16384, MU_LONG = 1 << 20;
int check_muon(const char *who, const tdh_muon *o, int dtype, int rows, int cols) {
  TDH_CHECK_ARG(dtype_known(dtype), "%s: element type %d", who, dtype);
  TDH_CHECK_ARG(o != nullptr, "%s: null descriptor", who);
  TDH_CHECK_ARG(o->products == TDH_F32 || o->products == TDH_F16, "%s: products in type %d", who, o->products);
  TDH_CHECK_ARG(o->steps >= 0 && o->steps <= MU_STEPS, "%s: %d steps", who, o->steps);
  TDH_CHECK_ARG(o->eps >= FLT_MIN && o->eps <= FLT_MAX, "%s: eps %g", who, o->eps);
  TDH_CHECK_ARG(rows >= 0 && cols >= 0, "%s: bad shape %d x %d", who, rows, cols);
  TDH_CHECK_ARG(std::min(rows, cols) <= MU_SHORT && std::max(rows, cols) <= MU_LONG && static_cast<long>(rows) * cols <= (1l << 30),
                "%s: a matrix of %d x %d is beyond 16384 x 2^20 or 2^30 elements", who, rows, cols);
  TDH_CHECK_ARG(mu_scalars(*o, std::max(1, std::min(rows, cols)), nullptr), "%s: coefficients %g, %g, %g take singular values beyond 4", who, o->a, o->b,
                o->c);
  return TDH_OK;
}

}  // namespace
}  // namespace tdh

using namespace tdh;

extern "C" {

void tdh_muon_default(tdh_muon *o) {
  if (!o) return;
  *o = tdh_muon{0.02f, 0.95f, 0.0f, 1.0f, 1, 5, 3.4445f, -4.7750f, 2.0315f, 1e-7f, TDH_F32};
}

int tdh_orthogonalize(const tdh_muon *o, int dtype, int rows, int cols, const void *x, void *y) {
  const char *who = "tdh_orthogonalize";
  TDH_TRY(check_muon(who, o, dtype, rows, cols));
  const size_t n = static_cast<size_t>(rows) * cols, bytes = n * dtype_size(dtype);
  TDH_CHECK_ARG(n == 0 || (x && y), "%s: null tensor", who);
  TDH_CHECK_ARG(((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & (dtype_size(dtype) - 1)) == 0,
                "%s: a tensor that is not aligned to its elements", who);
  if (x != y) TDH_TRY(check_apart(who, {{y, bytes}}, {{x, bytes}}));
  TDH_REQUIRE_INIT();
  if (n == 0) return TDH_OK;
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    return mu_run(*o, rows, cols, Momentum<T>{static_cast<const T *>(x), nullptr, 1.0f, 0.0f, false}, Apply<T>{static_cast<T *>(y), cols, false, 0.0f, 1.0f});
  });
}

int tdh_muon_update(const tdh_muon *o, int dtype, int rows, int cols, const void *merged_grad, float grad_scale, float *w, float *momentum) {
  const char *who = "tdh_muon_update";
  TDH_TRY(check_muon(who, o, dtype, rows, cols));
  const size_t n = static_cast<size_t>(rows) * cols;
  TDH_CHECK_ARG(n == 0 || (merged_grad && w && momentum), "%s: null tensor", who);
  TDH_CHECK_ARG((reinterpret_cast<uintptr_t>(merged_grad) & (dtype_size(dtype) - 1)) == 0 &&
                    ((reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(momentum)) & 3) == 0,
                "%s: a tensor that is not aligned to its elements", who);
  TDH_TRY(check_apart(who, {{w, 4 * n}, {momentum, 4 * n}}, {{merged_grad, n * dtype_size(dtype)}}));
  TDH_REQUIRE_INIT();
  if (n == 0) return TDH_OK;
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    return mu_run(*o, rows, cols, Momentum<T>{static_cast<const T *>(merged_grad), momentum, grad_scale, o->mu, o->nesterov != 0},
                  Apply<float>{w, cols, true, 1.0f - o->alpha * o->lambda, -o->alpha * o->scale});
  });
}

}  // extern "C"
