// gemm_x3.h — the products of gemm16.h for fp32 matrices, in three bf16 parts (split_bf16.h) that lie split in memory.
//
// fc_x3.hip splits its operands on the way into LDS, once for every tile that reads them, which costs more vector
// instructions than there are matrix instructions to hide them behind. Here every element is split once, by a pass of
// its own that writes three planes (10 bytes moved an element, rows padded to whole words), and tiles of 32 reduction indices
// of all three planes go straight into LDS. Worth its pass where an operand is read by many tiles; where few read B, it is split on
// its way into LDS after all (ON_THE_WAY). One operand carries the sign of its step (split_bf16.h: steps take turns between the
// product and its negative).
//
// Tiles of 128 x 128 on four waves, one of them in LDS at a time (48 KB), two workgroups a compute unit that cover each
// other's loads and epilogues: 4096 x 8192 with k of 256 in 102 us, 4096 x 4096 with k of 2048 in 314 (m, n), 351 (k, k)
// and 336 us (k, n), 196 to 219 TFLOP/s. 256 x 128 on eight waves with the next tile on its way in a second buffer,
// one workgroup a compute unit: 128, 339, 359, 346; operands of 16 indices at a time and three workgroups: 99, 347, 382, 367.
// Bound by the matrix cores at the power limit, and in short sums by what a round of workgroups writes.
#pragma once
#include "gemm16.h"
#include "split_bf16.h"

namespace tdh {
namespace {

constexpr int X3P_BK = 32;

// The planes' columns come in one or two halves, `half` apart, of which `used` are in use and have neighbours in the fp32 matrix.
struct X3Span {
  int used, half;
  // where column i of the planes lies in the matrix, or -1
  __device__ __forceinline__ int at(const int i) const { return i < used ? i : i >= half && i - half < used ? i - half + used : -1; }
};
// The fp32 matrices themselves, for sums that come out infinite or NaN: element (m, k) at a[m am + k ak], (k, n) at
// b[k bk + n bn] with k and n in the matrices' own columns; rows and cols of C, in the planes'.
struct X3Source {
  const float *a, *b;
  long am, ak, bk, bn;
  int rows, cols;
  X3Span k, n;
};

// B's tile of Side from the fp32 matrix, split on the way into LDS: what a thread has of it, eight neighbours a chunk.
template <class Side, bool KC, bool PAIR, int NT>
struct X3OnTheWay {
  float v[Side::PER][8];
  uint4 part[Side::PER][X3_PARTS];
  // asks for the tile at k0 (`left`: reduction indices from there), whose first column is `first`
  __device__ __forceinline__ void load(const X3Source &src, const int first, const int k0, const int left, const int tid) {
#pragma unroll
    for (int i = 0; i < Side::PER; ++i) {
      int row, chunk;
      Side::place(tid, i, row, chunk);
      const X3Span &span = KC ? src.k : src.n;   // of the fast index, eight of which lie in one half
      int h, c, slow;
      bool in;
      if (KC) {
        h    = k0 + 8 * chunk >= span.half ? 1 : 0;
        c    = k0 + 8 * chunk - h * span.half;
        slow = first + row;
        in   = slow < src.cols && 8 * chunk < left;
      } else {
        const int col = 8 * chunk;
        h    = PAIR ? (col >> 5) & 1 : first + col >= span.half ? 1 : 0;
        c    = PAIR ? first + (col >> 6) * 32 + (col & 31) : first + col - h * span.half;
        slow = k0 + row;
        in   = row < left;
      }
      const float *p = src.b + slow * (KC ? src.bn : src.bk) + static_cast<long>(h) * span.used + c;
      if (in && c + 8 <= span.used) {
        load8(p, v[i]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = in && c + e < span.used ? p[e] : 0.0f;
      }
    }
  }
  __device__ __forceinline__ void split(const float scale) {
#pragma unroll
    for (int i = 0; i < Side::PER; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t q[X3_PARTS];
        split_pair(scale * v[i][2 * c], scale * v[i][2 * c + 1], q);
#pragma unroll
        for (int x = 0; x < X3_PARTS; ++x) (&part[i][x].x)[c] = q[x];
      }
  }
  __device__ __forceinline__ void put(char *lds, const int tid) const {
#pragma unroll
    for (int x = 0; x < X3_PARTS; ++x)
#pragma unroll
      for (int i = 0; i < Side::PER; ++i) *reinterpret_cast<uint4 *>(lds + x * Side::BYTES + (i * NT + tid) * 16) = part[i][x];
  }
};

// ON_THE_WAY: B is src.b itself, asked for in front of the products of the tile before.
template <bool A_KC, bool B_KC, bool PAIR, bool ON_THE_WAY, class Epi>
__global__ void __launch_bounds__(256, 2)
gemm_x3_kernel(const G16Matrix A, const G16Matrix B, const long a_plane, const long b_plane, const X3Source src, const Epi epi,
               const int tiles_m, const int tiles_n, const int K, const int k_per_split) {
  constexpr int WM = 2, WN = 2, TM = 2, TN = 2, NT = 64 * WM * WN, BM = 32 * TM * WM, BN = 32 * TN * WN;
  using SideA = G16Side<BM, A_KC, false, NT, X3P_BK>;
  using SideB = G16Side<BN, B_KC, PAIR, NT, X3P_BK>;
  constexpr int STAGE = X3_PARTS * (SideA::BYTES + SideB::BYTES);
  __shared__ __align__(1024) char lds[STAGE];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave % WM, wn = wave / WM;
  const int tiles = tiles_m * tiles_n;
  int id = xcd_compact_id(blockIdx.x, gridDim.x);
  const int split = id / tiles;
  id -= split * tiles;
  int tm, tn;
  g16_tile(id, tiles_m, tiles_n, tm, tn);
  const int m0 = tm * BM, n0 = tn * (PAIR ? BN / 2 : BN);
  const int kbeg = split * k_per_split, kend = min(K, kbeg + k_per_split);

  SideA sa;
  SideB sb;
  sa.plan(A, m0, tid);
  if constexpr (!ON_THE_WAY) sb.plan(B, n0, tid);
  floatx16_x3 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = floatx16_x3{};
  int oa[TM], ob[TN];
#pragma unroll
  for (int i = 0; i < TM; ++i) oa[i] = SideA::lane_offset(lane, 32 * (wm * TM + i));
#pragma unroll
  for (int j = 0; j < TN; ++j) ob[j] = X3_PARTS * SideA::BYTES + SideB::lane_offset(lane, 32 * (wn * TN + j));
  auto fetch = [&](int k0) {
#pragma unroll
    for (int p = 0; p < X3_PARTS; ++p) {
      SideA a = sa;
      SideB b = sb;
      a.base += 2 * p * a_plane;
      a.fetch(A, lds + p * SideA::BYTES, k0, kend - k0, tid);
      if constexpr (!ON_THE_WAY) {
        b.base += 2 * p * b_plane;
        b.fetch(B, lds + X3_PARTS * SideA::BYTES + p * SideB::BYTES, k0, kend - k0, tid);
      }
    }
  };
  X3OnTheWay<SideB, B_KC, PAIR, NT> own;
  if constexpr (ON_THE_WAY) own.load(src, n0, kbeg, kend - kbeg, tid);
#pragma unroll 1
  for (int k0 = kbeg; k0 < kend; k0 += X3P_BK) {
    if constexpr (ON_THE_WAY) own.split(k0 / X3P_BK & 1 ? -X3_SCALE : X3_SCALE);
    __syncthreads();   // everyone has read the tile before
    fetch(k0);
    if constexpr (ON_THE_WAY) own.put(lds + X3_PARTS * SideA::BYTES, tid);
    g16_arrived<0>();
    __syncthreads();
    if constexpr (ON_THE_WAY)
      if (k0 + X3P_BK < kend) own.load(src, n0, k0 + X3P_BK, kend - k0 - X3P_BK, tid);
    bf16x8 a[2][TM][X3_PARTS], b[2][TN][X3_PARTS];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int p = 0; p < X3_PARTS; ++p) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
          a[s][i][p] = __builtin_bit_cast(bf16x8, SideA::read(lds + p * SideA::BYTES, oa[i], lane, s));
#pragma unroll
        for (int j = 0; j < TN; ++j)
          b[s][j][p] = __builtin_bit_cast(bf16x8, SideB::read(lds + p * SideB::BYTES, ob[j], lane, s));
      }
    mfma_x3<TM, TN, 2>(acc, a, b, k0 / X3P_BK & 1 ? -1.0f : 1.0f);
  }
  const int mw = m0 + 32 * TM * wm, nw = n0 + (PAIR ? 16 * TN * wn : 32 * TN * wn);
  const int half = lane >> 5, l32 = lane & 31;
  // the infinite and NaN sums once more in fp32: lane l brings row and column l % 32 of the blocks at index k + l / 32
  {
    int col[TN];   // (PAIR: of either half)
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = PAIR ? nw + 32 * (j >> 1) + l32 : nw + 32 * j + l32;
      col[j]      = n >= (PAIR ? src.n.half : src.cols) ? -1 : src.n.at(PAIR ? n + (j & 1) * src.n.half : n);
    }
    x3_redo(reinterpret_cast<floatx16_x3(&)[TM * TN]>(acc), [&](int b, int r) {
      return mw + 32 * (b / TN) + 8 * (r >> 2) + 4 * half + (r & 3) < src.rows && col[b % TN] >= 0;
    }, [&](floatx16_x3 (&sum)[TM * TN]) {
#pragma unroll 1
      for (int k0 = kbeg; k0 < kend; k0 += 8) {
        float av[4][TM], bv[4][TN];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const int kp = k0 + 2 * s + half, k = kp < kend ? src.k.at(kp) : -1;
#pragma unroll
          for (int i = 0; i < TM; ++i) {
            const int m = mw + 32 * i + l32;
            av[s][i] = k >= 0 && m < src.rows ? src.a[m * src.am + k * src.ak] : 0.0f;
          }
#pragma unroll
          for (int j = 0; j < TN; ++j) bv[s][j] = k >= 0 && col[j] >= 0 ? src.b[k * src.bk + col[j] * src.bn] : 0.0f;
        }
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int b = 0; b < TM * TN; ++b) sum[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(av[s][b / TN], bv[s][b % TN], sum[b], 0, 0, 0);
        if (x3_all_nan(sum)) return;
      }
    });
  }
  static_assert(sizeof(lds) >= WM * WN * G16Turn<32 * TN>::BYTES, "");
  __syncthreads();
  epi.template done<TM, TN>(acc, mw, nw, lane, split, reinterpret_cast<float *>(lds + wave * G16Turn<32 * TN>::BYTES));
}

}  // namespace
}  // namespace tdh
