// gemm16.h — products of 16-bit matrices on the matrix cores with fp32 sums, C[m][n] = sum_k A[m][k] B[k][n], for the
// three products of a layer whose matrices differ in their fast index:
//
//   forward  z[b][o]  = x[b][i] w[i][o]     A along k, B along n
//   dX       dx[b][i] = dz[b][o] w[i][o]    both along k
//   dW       dw[i][o] = x[b][i] dz[b][o]    A along m, B along n
//
// A workgroup of WM x WN waves owns 32 TM WM x 32 TN WN elements of C, a wave TM x TN blocks of
// v_mfma_f32_32x32x16. Tiles of 64 reduction indices go from memory straight into LDS (16 bytes a lane), BUFS of
// them in turns: the next ones are on their way while this one is multiplied, one barrier a tile. LDS holds a tile as it
// lies in memory, its 16-byte chunks permuted within each row so that the reads hit different banks (the lanes fetch
// permuted chunks: the way into LDS is linear in the lane):
//   along k      rows of 64 k (128 bytes), chunk c of row r at c ^ (r/2 mod 8) (rows of 32 k: at c ^ (r/4 mod 4)), so that 16 rows in
//                a row fill the 256 bytes that LDS reads at a time (at c ^ (r mod 8) rows r and r + 8 meet: 4 cycles a read, and
//                the product with both operands along k in 662-708 us for 650); a lane's operand, 8 k of its row, is one
//                16-byte read;
//   along m, n   rows of one k each, 64-byte segments permuted by k mod 4; ds_read_b64_tr_b16 hands every lane 4 k of
//                its column out of 4 rows.
//
// Bound by the card's power on large products: 4096 x 24576 x 4096 in bf16, tiles of 256 x 256 by eight waves, random operands
// 1150-1270 TFLOP/s without the gate, all zero 1440-1490 (whose sums no bits toggle). Slower: tiles of 32 indices, four of them in turns 1100-1113; four
// waves of 128 x 128 each 1074-1111.
#pragma once
#include "lm_types.h"

namespace tdh {

// A product's tile shape, and its split along k
struct FfPlan {
  int cfg;       // 0 to 4: 256 x 256 by eight waves, 128 x 128, 64 x 128, 64 x 64 by two waves, 32 x 256; four waves where none are named
  int splits, k_per_split;
};
FfPlan ff_plan(int M, int N, int K, bool pair);   // (gated_ff.hip)

namespace {

typedef __bf16 g16_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 g16_f16x8 __attribute__((ext_vector_type(8)));
typedef short g16_s16x4 __attribute__((ext_vector_type(4)));
typedef short g16_s16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t g16_u32x4 __attribute__((ext_vector_type(4)));
typedef float g16_f32x16 __attribute__((ext_vector_type(16)));

constexpr int G16_BK = 64;

__device__ __forceinline__ g16_f32x16 mfma16(bf16, const g16_s16x8 a, const g16_s16x8 b, const g16_f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(g16_bf16x8, a), __builtin_bit_cast(g16_bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ g16_f32x16 mfma16(f16, const g16_s16x8 a, const g16_s16x8 b, const g16_f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(g16_f16x8, a), __builtin_bit_cast(g16_f16x8, b), c, 0, 0, 0);
}

// Eight-bit integers in pairs, which take the place of 16-bit elements everywhere but in the products; their sums are whole numbers, held in the
// bits of the accumulators.
struct i8x2 {
  int8_t v[2];
};
typedef int g16_i32x4 __attribute__((ext_vector_type(4)));
typedef int g16_i32x16 __attribute__((ext_vector_type(16)));
__device__ __forceinline__ g16_f32x16 mfma16(i8x2, const g16_s16x8 a, const g16_s16x8 b, const g16_f32x16 c) {
  return __builtin_bit_cast(g16_f32x16, __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(g16_i32x4, a), __builtin_bit_cast(g16_i32x4, b),
                                                                             __builtin_bit_cast(g16_i32x16, c), 0, 0, 0));
}

// waits until all but the last LEFT of the wave's loads into LDS have arrived
template <int LEFT>
__device__ __forceinline__ void g16_arrived() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory");
}

// A matrix in memory on a 16-byte boundary, rows `ld` elements apart (a multiple of 8).
struct G16Matrix {
  const void *p;
  long ld;
  int rows, cols;   // both in use; cols is a multiple of 8
};

// One operand's tile of ROWS rows (along m or n) x BK k. KC: the matrix has k as its fast index.
// PAIR (not KC): the ROWS columns are 32 of the first half of the matrix' columns, 32 of the second half, 32 of
// the first, ...
template <int ROWS, bool KC, bool PAIR, int NT, int BK = G16_BK>
struct G16Side {
  static constexpr int BYTES = ROWS * BK * 2;
  static constexpr int PER   = BYTES / (NT * 16);   // 16-byte loads a thread
  static_assert(BYTES % (NT * 16) == 0, "");
  const char *base;   // of the tile's k = 0
  unsigned off[PER];  // bytes from there, by load
  // chunk c of row r lies at c ^ turn(r) (KC): the sixteen lanes that read at a time hit different banks
  __device__ __forceinline__ static int turn(const int row) { return BK == 64 ? (row >> 1) & 7 : (row >> 2) & 3; }
  __device__ __forceinline__ static int swizzle(const int k) { return ROWS >= 128 ? (k & 3) * 4 : ROWS == 64 ? ((k >> 1) & 1) * 4 : 0; }
  // where thread tid's load i lies: row of the tile and 16-byte chunk (of memory) in it
  __device__ __forceinline__ static void place(const int tid, const int i, int &row, int &chunk) {
    const int p = (i * NT + tid) * 16;
    if (KC) {
      row   = p / (BK * 2);
      chunk = ((p >> 4) & (BK / 8 - 1)) ^ turn(row);
    } else {
      row   = p / (ROWS * 2);                        // k
      chunk = ((p / 16) % (ROWS / 8)) ^ swizzle(row);
    }
  }
  __device__ __forceinline__ void plan(const G16Matrix &mat, const int first, const int tid) {
    base = static_cast<const char *>(mat.p);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      int row, chunk;
      place(tid, i, row, chunk);
      if (KC) {
        off[i] = static_cast<unsigned>(min(first + row, mat.rows - 1) - first) * static_cast<unsigned>(2 * mat.ld) + 16u * chunk;
      } else {
        int col = 8 * chunk;
        if (PAIR) {
          const int half = mat.cols >> 1, blk = col >> 5;
          col = min(first + (blk >> 1) * 32 + (col & 31), half - 8) + (blk & 1) * half;
        } else {
          col = min(first + col, mat.cols - 8);
        }
        off[i] = static_cast<unsigned>(row) * static_cast<unsigned>(2 * mat.ld) + 2u * col;
      }
    }
    if (KC) base += static_cast<size_t>(first) * 2 * mat.ld;
  }
  // Asks for the tile that starts at k0; `left`: reduction indices from there. What it asks for has arrived when
  // g16_arrived() returns (the compiler would wait for it before any read of LDS, so it is not told).
  __device__ __forceinline__ void fetch(const G16Matrix &mat, char *lds, const int k0, const int left, const int tid) const {
    const char *at = base + (KC ? 2L * k0 : 2L * k0 * mat.ld);
    if (left >= BK) {
      const uint64_t where = reinterpret_cast<uint64_t>(at);
      const g16_u32x4 desc = {static_cast<uint32_t>(where), static_cast<uint32_t>(where >> 32), 0xffffffffu, 0x00027000u};
      // (a wave's 64 lanes fill 1024 bytes of LDS from an address that is the same for all of them)
      const unsigned to = __builtin_amdgcn_readfirstlane(
          static_cast<unsigned>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char *)lds)) + (tid & ~63) * 16);
      // (m0 holds where the load writes; the compiler keeps that register for itself, and finds it as it was)
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        unsigned was;
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
                     : "=&s"(was)
                     : "s"(to + i * NT * 16), "v"(off[i]), "s"(desc)
                     : "memory");
      }
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        int row, chunk;
        place(tid, i, row, chunk);
        const bool in = KC ? 8 * chunk < left : row < left;
        uint4 v       = make_uint4(0, 0, 0, 0);
        if (in) v = *reinterpret_cast<const uint4 *>(at + off[i]);
        *reinterpret_cast<uint4 *>(lds + (i * NT + tid) * 16) = v;
      }
    }
  }
  // The operand of 32 rows from `row0` (a multiple of 32) and the 16 k of step s: lane l has row l % 32 and k
  // 8 (l / 32) .. + 7. `lane_off` is what lane_offset() gives for row0's 32 rows.
  __device__ __forceinline__ static int lane_offset(const int lane, const int row0) {
    if (KC) return (row0 + (lane & 31)) * BK * 2;
    const int j = lane & 15, g = lane >> 4;
    const int k = 8 * (g >> 1) + (j >> 2), col = row0 + 16 * (g & 1) + 4 * (j & 3);
    return k * ROWS * 2 + (((col >> 3) ^ swizzle(k)) << 4) + (col & 7) * 2;
  }
  __device__ __forceinline__ static g16_s16x8 read(const char *lds, const int lane_off, const int lane, const int s) {
    if constexpr (KC) {
      const int chunk = (2 * s + (lane >> 5)) ^ turn(lane & 31);
      return *reinterpret_cast<const g16_s16x8 *>(lds + lane_off + chunk * 16);
    } else {
      typedef __attribute__((address_space(3))) g16_s16x4 lds_vec;
      const char *p = lds + lane_off + s * 16 * ROWS * 2;
      const g16_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_vec *)p);
      const g16_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_vec *)(p + 4 * ROWS * 2));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
};

// Which tile a workgroup takes: neighbours on one XCD, in groups of GROUP tile rows that go through the tile columns
// together, so that the 32 workgroups of an XCD share a few panels of either operand in its L2.
__device__ __forceinline__ void g16_tile(int id, const int tiles_m, const int tiles_n, int &tm, int &tn) {
  constexpr int GROUP = 8;
  const int per = GROUP * tiles_n, group = id / per, first = group * GROUP, rows = min(GROUP, tiles_m - first);
  id -= group * per;
  tm = first + id % rows;
  tn = id / rows;
}

// All tiles, or those on and below the diagonal of a symmetric product.
struct G16AllTiles {
  __host__ __device__ static int count(const int tiles_m, const int tiles_n) { return tiles_m * tiles_n; }
  __device__ __forceinline__ static void place(const int id, const int tiles_m, const int tiles_n, int &tm, int &tn) { g16_tile(id, tiles_m, tiles_n, tm, tn); }
};
struct G16LowerTiles {
  __host__ __device__ static int count(const int tiles_m, const int) { return tiles_m * (tiles_m + 1) / 2; }
  __device__ __forceinline__ static void place(const int id, const int, const int, int &tm, int &tn) {
    tm = static_cast<int>((sqrtf(8.0f * id + 1.0f) - 1.0f) * 0.5f);   // (up to rounding)
    while ((tm + 1) * (tm + 2) / 2 <= id) ++tm;
    while (tm * (tm + 1) / 2 > id) --tm;
    tn = id - tm * (tm + 1) / 2;
  }
};

// 32 rows of COLS fp32 values that a wave turns in LDS, so that a lane has eight neighbours of one row: put() takes
// block j in the matrix cores' layout, rows() hands out (row, column of the first, values).
template <int COLS>
struct G16Turn {
  static constexpr int STRIDE = COLS + 4, BYTES = 32 * STRIDE * 4;
  float *at;
  template <class F>
  __device__ __forceinline__ void put(const int lane, const int j, const F &value) const {
#pragma unroll
    for (int r = 0; r < 16; ++r) at[(8 * (r >> 2) + 4 * (lane >> 5) + (r & 3)) * STRIDE + 32 * j + (lane & 31)] = value(r);
  }
  template <class F>
  __device__ __forceinline__ void rows(const int lane, const F &take) const {
    constexpr int PER = COLS / 8, ROWS = 64 / PER;   // lanes a row, rows at a time
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int k = 0; k < 32 / ROWS; ++k) {
      const int row = k * ROWS + lane / PER, col = lane % PER * 8;
      const float4 *p = reinterpret_cast<const float4 *>(at + row * STRIDE + col);
      const float4 lo = p[0], hi = p[1];
      const float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      take(row, col, v);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");   // (before the next put)
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
};

// A launch may have a part of a product's tiles: those from epi.first_tile on, epi.tiles_here of them (an Epi without these: all).
template <class Epi>
__device__ __forceinline__ auto g16_first_tile(const Epi &epi, int) -> decltype(epi.first_tile) { return epi.first_tile; }
template <class Epi>
__device__ __forceinline__ int g16_first_tile(const Epi &, long) { return 0; }
template <class Epi>
__device__ __forceinline__ auto g16_tiles_here(const Epi &epi, int, int) -> decltype(epi.tiles_here) { return epi.tiles_here; }
template <class Epi>
__device__ __forceinline__ int g16_tiles_here(const Epi &, const int all, long) { return all; }

// Epi: done(acc, m0, n0, lane, split, lds) with the wave's blocks: register r of lane l of block (i, j) is row
// m0 + 32 i + 8 (r / 4) + 4 (l / 32) + r % 4 and column n0 + 32 j + l % 32 (PAIR: of the tile's column order); lds:
// G16Turn<32 TN>::BYTES of the wave's own.
template <class T, int WM, int WN, int TM, int TN, int BUFS, bool A_KC, bool B_KC, bool PAIR, class Epi, class Tiles = G16AllTiles>
__global__ void __launch_bounds__(64 * WM * WN)
gemm16_kernel(const G16Matrix A, const G16Matrix B, const Epi epi, const int tiles_m, const int tiles_n, const int K,
              const int k_per_split) {
  constexpr int NT = 64 * WM * WN, BM = 32 * TM * WM, BN = 32 * TN * WN;
  using SideA = G16Side<BM, A_KC, false, NT>;
  using SideB = G16Side<BN, B_KC, PAIR, NT>;
  __shared__ __align__(1024) char lds[BUFS][SideA::BYTES + SideB::BYTES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave % WM, wn = wave / WM;
  const int tiles = g16_tiles_here(epi, Tiles::count(tiles_m, tiles_n), 0);
  int id = xcd_compact_id(blockIdx.x, gridDim.x);
  const int split = id / tiles;
  id -= split * tiles;
  int tm, tn;
  Tiles::place(id + g16_first_tile(epi, 0), tiles_m, tiles_n, tm, tn);
  const int m0 = tm * BM, n0 = tn * (PAIR ? BN / 2 : BN);
  const int kbeg = split * k_per_split, kend = min(K, kbeg + k_per_split);

  SideA sa;
  SideB sb;
  sa.plan(A, m0, tid);
  sb.plan(B, n0, tid);
  g16_f32x16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
  int oa[TM], ob[TN];
#pragma unroll
  for (int i = 0; i < TM; ++i) oa[i] = SideA::lane_offset(lane, 32 * (wm * TM + i));
#pragma unroll
  for (int j = 0; j < TN; ++j) ob[j] = SideA::BYTES + SideB::lane_offset(lane, 32 * (wn * TN + j));

  // tile t lies in buffer t % BUFS; BUFS - 1 tiles are on their way or being multiplied
  constexpr int LOADS = SideA::PER + SideB::PER;   // of a tile, by a wave
  const int left = kend - kbeg, ntiles = (left + G16_BK - 1) / G16_BK, nfull = left / G16_BK;   // (a last, shorter one goes through registers)
  auto fetch = [&](int t, int buf) {
    sa.fetch(A, lds[buf], kbeg + t * G16_BK, left - t * G16_BK, tid);
    sb.fetch(B, lds[buf] + SideA::BYTES, kbeg + t * G16_BK, left - t * G16_BK, tid);
  };
#pragma unroll
  for (int t = 0; t < BUFS - 1; ++t)
    if (t < ntiles) fetch(t, t);
  int buf = 0, next = BUFS - 1;
#pragma unroll 1
  for (int t = 0; t < ntiles; ++t) {
    if (t + BUFS - 2 < nfull) g16_arrived<(BUFS - 2) * LOADS>(); else g16_arrived<0>();
    __syncthreads();   // this tile has arrived, and everyone has read the one before
    if (t + BUFS - 1 < ntiles) fetch(t + BUFS - 1, next);
    const char *at = lds[buf];
    // (a step's operands are asked for in front of the products of the step before; left alone, the compiler asks where it
    // needs them, which takes 47 us instead of 38 for 256 tiles of 256 x 256 with k of 1024)
    g16_s16x8 a[2][TM], b[2][TN];
    auto read = [&](int s) {
#pragma unroll
      for (int i = 0; i < TM; ++i) a[s & 1][i] = SideA::read(at, oa[i], lane, s);
#pragma unroll
      for (int j = 0; j < TN; ++j) b[s & 1][j] = SideB::read(at, ob[j], lane, s);
    };
    read(0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if (s < 3) read(s + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = mfma16(T(), a[s & 1][i], b[s & 1][j], acc[i][j]);
      __builtin_amdgcn_sched_barrier(0);
    }
    buf  = buf + 1 == BUFS ? 0 : buf + 1;
    next = next + 1 == BUFS ? 0 : next + 1;
  }
  static_assert(sizeof(lds) >= WM * WN * G16Turn<32 * TN>::BYTES, "");
  __syncthreads();
  epi.template done<TM, TN>(acc, m0 + 32 * TM * wm, n0 + (PAIR ? 16 * TN * wn : 32 * TN * wn), lane, split,
                            reinterpret_cast<float *>(lds[0] + wave * G16Turn<32 * TN>::BYTES));
}

}  // namespace
}  // namespace tdh
