// 8-bit operands: quantizing rows and columns, the RMS norm that ends in one, and back.
// (The products are in fp8_gemm.hip.)
#include "fp8.h"

#include <algorithm>
#include <type_traits>

namespace mesh_moe {

// Pieces of 16 bytes that lie on a T: the hardware takes any address.  (Rows and columns
// of 9000 x 2050 in bf16 take 29 us with them, 53 with a load per value, and 26 at 2048
// columns, where pieces lie on 16 bytes; the norm of 32000 x 2050 124, 267 and 83.)
template <typename T> struct PieceOf;
template <> struct PieceOf<bf16_t> {
  typedef uint32_t type __attribute__((ext_vector_type(4), aligned(2)));
};
template <> struct PieceOf<float> {
  typedef uint32_t type __attribute__((ext_vector_type(4), aligned(4)));
};
template <typename T, bool ONCE>
__device__ __forceinline__ uint4 load_piece(const T* at) {
  typedef typename PieceOf<T>::type piece_t;
  const piece_t* p = reinterpret_cast<const piece_t*>(at);
  const piece_t v = ONCE ? __builtin_nontemporal_load(p) : *p;
  return make_uint4(v[0], v[1], v[2], v[3]);
}
template <typename T>
__device__ __forceinline__ void store_piece(T* at, uint4 v) {
  typedef typename PieceOf<T>::type piece_t;
  __builtin_nontemporal_store(piece_t{v.x, v.y, v.z, v.w}, reinterpret_cast<piece_t*>(at));
}

// 8 neighbouring values of a row from column `at` on, zeros from `end` on.  ALIGNED:
// every row's pieces of 16 bytes lie on 16 bytes, and `end` is a multiple of 8.  ONCE:
// nothing reads them again.  (`at` goes up to 2^31 - 8, so nothing is added to it before
// it is known to be below `end`.)
template <typename T, bool ALIGNED, bool ONCE = true>
__device__ __forceinline__ void load8(const T* row, int at, int end, float (&v)[8]) {
  if (ALIGNED ? at < end : at <= end - 8) {
    if constexpr (sizeof(T) == 2) {
      unpack16(load_piece<T, ONCE>(row + at), v, T());
    } else {
      float lo[4], hi[4];
      unpack16(load_piece<T, ONCE>(row + at), lo, T());
      unpack16(load_piece<T, ONCE>(row + at + 4), hi, T());
#pragma unroll
      for (int j = 0; j < 4; ++j) { v[j] = lo[j]; v[4 + j] = hi[j]; }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = 0.f;
  if constexpr (!ALIGNED)
    if (at < end)
#pragma unroll
      for (int j = 0; j < 7; ++j)
        if (at + j < end) v[j] = load_f32<T>(row + at + j);
}

template <typename T, bool ALIGNED>
__device__ __forceinline__ void store8(T* row, int at, int end, const float (&v)[8]) {
  if (ALIGNED ? at < end : at <= end - 8) {
    if constexpr (sizeof(T) == 2) {
      store_piece(row + at, pack16(v, T()));
    } else {
      const float lo[4] = {v[0], v[1], v[2], v[3]}, hi[4] = {v[4], v[5], v[6], v[7]};
      store_piece(row + at, pack16(lo, T()));
      store_piece(row + at + 4, pack16(hi, T()));
    }
    return;
  }
  if constexpr (!ALIGNED)
#pragma unroll
    for (int j = 0; j < 7; ++j)
      if (at + j < end) store_f32<T>(row + at + j, v[j]);
}

// ---------------------------------------------------------------------------
// Quantizing.  A block of 256 threads has a tile of 128 rows x 128 columns in
// registers, 8 rows x 8 columns a thread: thread t the columns 8 (t % 16) .. and the
// rows 8 (t / 16) ...  A row's block of 128 lies in 16 neighbouring lanes, whose
// largest magnitude four DPP steps find; a column's in four lanes of each of the four
// wavefronts, which meet in LDS.  The rows' bytes leave from the registers (16 lanes
// fill a 128-byte line); the columns' are turned round in 16 KB of LDS, 8 bytes (of a
// thread's rows) at a time, the 8-byte units of a column XOR-ed with its thread's
// column so that the lanes of a write spread over all banks.
//
// Bound by memory: the tensor is read once, whichever forms are wanted.  Both forms of
// 65536 x 4096 in bf16 take 204 to 231 us, 5.3 to 4.7 TB/s (254 with 144 registers and
// three blocks per CU instead of 94 and five), the rows alone 143; pieces that do not lie
// on 16 bytes need the registers.
// ---------------------------------------------------------------------------
constexpr int QT = FP8_BLOCK;     // a tile's rows and columns

// Tile of this block: 4 x 4 tiles share the lines that the scale bytes lie in, and
// follow each other on an XCD (block b runs on XCD b % 8), in whose L2 they meet.  Which
// group of every 8 an XCD takes goes round, 3 on each time: a matrix's last row of groups
// may have few tiles, and would always fall to the same ones (18 us for 32 x 640 x 1024
// with counts, 26 without).
struct TileOrder {
  int tiles_r, tiles_k;
  int groups_k;                   // groups of 4 x 4 along the columns
  int64_t groups;                 // of one expert
  bool by_xcd;
};
__device__ __forceinline__ bool tile_of(const TileOrder& o, int& e, int& tr, int& tk) {
  const int64_t b = blockIdx.x;
  const int64_t logical =
      o.by_xcd ? (b & ~127LL) + (((b & 7) + 3 * (b >> 7)) & 7) * 16 + ((b >> 3) & 15) : b;
  const int64_t group = logical >> 4;
  e = (int)(group / o.groups);
  const int64_t g = group - e * o.groups;
  tr = (int)(g / o.groups_k) * 4 + (int)((logical >> 2) & 3);
  tk = (int)(g % o.groups_k) * 4 + (int)(logical & 3);
  return tr < o.tiles_r && tk < o.tiles_k;
}

template <typename T, bool ALIGNED>
__global__ __launch_bounds__(256, ALIGNED ? 4 : 3) void fp8_quantize_kernel(
    const T* __restrict__ x, const T* __restrict__ relu_mask,
    const int32_t* __restrict__ row_count, uint8_t* __restrict__ row_values,
    uint8_t* __restrict__ row_scales, uint8_t* __restrict__ column_values,
    uint8_t* __restrict__ column_scales, int E, int R, int K, TileOrder order,
    bool only_counted) {
  __shared__ uint32_t tops[4][QT];
  __shared__ __attribute__((aligned(16))) uint2 turned[QT][QT / 8];
  int e, tr, tk;
  if (!tile_of(order, e, tr, tk) || e >= E) return;
  const int t = threadIdx.x, c = t & 15, r = t >> 4;
  const int count =
      row_count != nullptr ? min(max(row_count[e], 0), R) : R;
  // (a weight gradient reads the blocks of rows that there are, but two at least)
  if (only_counted && tr * QT >= max(count, 2 * QT)) return;
  const int row0 = tr * QT + 8 * r, col0 = tk * QT + 8 * c;
  float v[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = row0 + i;
    load8<T, ALIGNED>(x + ((int64_t)e * R + min(row, R - 1)) * K, col0,
                      row < count ? K : 0, v[i]);
  }
  if (relu_mask != nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = row0 + i;
      float m[8];
      load8<T, ALIGNED>(relu_mask + ((int64_t)e * R + min(row, R - 1)) * K, col0,
                        row < count ? K : 0, m);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = m[j] > 0.f ? v[i][j] : 0.f;
    }
  }
  if (row_values != nullptr) {
    const int64_t kp = fp8_row_bytes(K), ks = fp8_scale_bytes(K);
    const int stored = only_counted ? count : R;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, magnitude_bits(v[i][j]));
      const Fp8Scale s = fp8_scale(max16(top));
      const int row = row0 + i;
      if (row >= stored) continue;
      uint2 q;
      q.x = fp8_pack4(v[i][0] * s.factor, v[i][1] * s.factor, v[i][2] * s.factor,
                      v[i][3] * s.factor);
      q.y = fp8_pack4(v[i][4] * s.factor, v[i][5] * s.factor, v[i][6] * s.factor,
                      v[i][7] * s.factor);
      const int64_t at = (int64_t)e * R + row;
      *reinterpret_cast<uint2*>(row_values + at * kp + col0) = q;
      if (c == 0) row_scales[at * ks + tk] = (uint8_t)s.byte;
    }
  }
  if (column_values == nullptr) return;
  uint32_t top[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    top[j] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top[j] = max(top[j], magnitude_bits(v[i][j]));
    top[j] = max(top[j], (uint32_t)__shfl_xor((int)top[j], 16));
    top[j] = max(top[j], (uint32_t)__shfl_xor((int)top[j], 32));
  }
  if ((t & 63) < 16) {
    uint4* to = reinterpret_cast<uint4*>(&tops[t >> 6][8 * c]);
    to[0] = make_uint4(top[0], top[1], top[2], top[3]);
    to[1] = make_uint4(top[4], top[5], top[6], top[7]);
  }
  __syncthreads();
  const int64_t rp = fp8_row_bytes(R), rs = fp8_scale_bytes(R);
  const int64_t first = (int64_t)e * K + tk * QT;       // the tile's first column
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int col = 8 * c + j;
    const Fp8Scale s = fp8_scale(max(max(tops[0][col], tops[1][col]),
                                     max(tops[2][col], tops[3][col])));
    uint2 q;
    q.x = fp8_pack4(v[0][j] * s.factor, v[1][j] * s.factor, v[2][j] * s.factor,
                    v[3][j] * s.factor);
    q.y = fp8_pack4(v[4][j] * s.factor, v[5][j] * s.factor, v[6][j] * s.factor,
                    v[7][j] * s.factor);
    turned[col][r ^ c] = q;
    if (r == 0 && tk * QT + col < K)
      column_scales[(first + col) * rs + tr] = (uint8_t)s.byte;
  }
  __syncthreads();
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const int col = it * 32 + (t >> 3), piece = t & 7, swap = col >> 3;
    if (tk * QT + col >= K) continue;
    uint4 q = *reinterpret_cast<const uint4*>(&turned[col][(2 * piece ^ swap) & ~1]);
    if (swap & 1) q = make_uint4(q.z, q.w, q.x, q.y);
    *reinterpret_cast<uint4*>(column_values + (first + col) * rp + tr * QT +
                              16 * piece) = q;
  }
}

template <typename T>
static int run_quantize(const T* x, const T* relu_mask, const int32_t* row_count,
                        uint8_t* row_values, uint8_t* row_scales,
                        uint8_t* column_values, uint8_t* column_scales, int E, int R,
                        int K, bool only_counted, hipStream_t st) {
  TileOrder o;
  o.tiles_r = (int)(((int64_t)R + QT - 1) / QT);
  o.tiles_k = (int)(((int64_t)K + QT - 1) / QT);
  o.groups_k = (o.tiles_k + 3) / 4;
  o.groups = (int64_t)((o.tiles_r + 3) / 4) * o.groups_k;
  // (in multiples of 128 the limit is one, too; divided, not to pass 64 bits)
  constexpr int64_t most = MAX_THREADS / 256 / 128 * 128;
  MOE_REQUIRE(o.groups <= most / 16 / E, MESH_MOE_E_UNSUPPORTED,
              "fp8_quantize: too many tiles (E=%d R=%d K=%d)", E, R, K);
  int64_t blocks = o.groups * E * 16;
  o.by_xcd = blocks >= 1024;
  if (o.by_xcd) blocks = (blocks + 127) / 128 * 128;
  const bool aligned =
      K % 8 == 0 && ((uintptr_t)x | (uintptr_t)relu_mask) % 16 == 0;
  auto kernel = aligned ? fp8_quantize_kernel<T, true> : fp8_quantize_kernel<T, false>;
  kernel<<<(unsigned)blocks, 256, 0, st>>>(x, relu_mask, row_count, row_values,
                                           row_scales, column_values, column_scales, E,
                                           R, K, o, only_counted);
  MOE_CHECK_LAUNCH("fp8_quantize");
  return 0;
}

int fp8_quantize(const void* x, const void* relu_mask, const int32_t* row_count,
                 void* row_values, uint8_t* row_scales, void* column_values,
                 uint8_t* column_scales, int E, int R, int K, int dtype,
                 bool only_counted, hipStream_t st) {
  if (dtype == MESH_MOE_F32)
    return run_quantize<float>((const float*)x, (const float*)relu_mask, row_count,
                               (uint8_t*)row_values, row_scales,
                               (uint8_t*)column_values, column_scales, E, R, K,
                               only_counted, st);
  return run_quantize<bf16_t>((const bf16_t*)x, (const bf16_t*)relu_mask, row_count,
                              (uint8_t*)row_values, row_scales,
                              (uint8_t*)column_values, column_scales, E, R, K,
                              only_counted, st);
}

// ---------------------------------------------------------------------------
// What an operand stands for.  A thread writes pieces of 16 bytes, the lanes of a
// wavefront neighbouring ones, so that each store fills whole lines.  (With 16 values per
// lane, two or four stores of every second or fourth piece, it took 404 us instead of 143
// for 65536 x 4096 in bf16, 5.6 TB/s, and 1491 instead of 278 in float32.)
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void fp8_dequantize_kernel(
    const uint8_t* __restrict__ values, const uint8_t* __restrict__ scales,
    T* __restrict__ y, int64_t rows, int K, int pieces, int64_t groups) {
  constexpr int V = 16 / sizeof(T), PER = 4;
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  const int64_t kp = fp8_row_bytes(K), ks = fp8_scale_bytes(K);
  for (int64_t group = blockIdx.x; group < groups; group += gridDim.x) {
    const int64_t first = group * (256 * PER), row0 = first / pieces;
    const uint32_t start = (uint32_t)(first - row0 * pieces) + threadIdx.x;
    uint32_t w[PER][V / 4], unit[PER];
    int64_t row[PER];
    int at[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const uint32_t piece = start + 256 * u, down = piece / (uint32_t)pieces;
      row[u] = row0 + down;
      at[u] = (int)(piece - down * (uint32_t)pieces) * V;
      if (row[u] >= rows) continue;
      const uint32_t* from =
          reinterpret_cast<const uint32_t*>(values + row[u] * kp + at[u]);
#pragma unroll
      for (int j = 0; j < V / 4; ++j) w[u][j] = __builtin_nontemporal_load(from + j);
      unit[u] = scales[row[u] * ks + at[u] / FP8_BLOCK];
    }
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      if (row[u] >= rows) continue;
      // (2^-127 is not a normal number)
      const float f = __uint_as_float(unit[u] == 255   ? 0x7fc00000u
                                      : unit[u] == 0 ? 0x00400000u
                                                     : unit[u] << 23);
      float v[V];
#pragma unroll
      for (int j = 0; j < V / 4; ++j) {
        const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[u][j], false);
        const f32x2_t hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[u][j], true);
        v[4 * j] = lo[0] * f;
        v[4 * j + 1] = lo[1] * f;
        v[4 * j + 2] = hi[0] * f;
        v[4 * j + 3] = hi[1] * f;
      }
      T* to = y + row[u] * K + at[u];
      if (at[u] + V <= K) {
        store_piece(to, pack16(v, T()));
      } else {
#pragma unroll
        for (int j = 0; j < V - 1; ++j)
          if (at[u] + j < K) store_f32<T>(to + j, v[j]);
      }
    }
  }
}

template <typename T>
static void run_dequantize(const uint8_t* values, const uint8_t* scales, T* y,
                           int64_t rows, int K, hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const int pieces = (int)(((int64_t)K + V - 1) / V);
  const int64_t groups = (rows * pieces + 1023) / 1024;
  fp8_dequantize_kernel<T><<<(unsigned)(groups < 0x100000 ? groups : 0x100000), 256, 0,
                             st>>>(values, scales, y, rows, K, pieces, groups);
}

// ---------------------------------------------------------------------------
// RMS norm into an 8-bit operand.  WPR wavefronts have a row in registers, 8
// neighbouring values per lane and step, so that the row is read once and a block of
// 128 lies in 16 neighbouring lanes; the scale bytes of a step's four blocks leave as
// one dword.  Rows past ITERS steps (STREAMED) are read again for the second half,
// from the sum that the same threads wrote.  The mean's sum, the root and the product
// are float32; the residual sum is rounded to the tensors' type first, being one.
//
// Bound by memory: 32000 x 4096 in bf16 with a residual 140 us, 6.5 TB/s.  At most 32
// values of a lane's row are in registers: 4000 rows of 16384 take 85 us on 8
// wavefronts, 118 on 4 with 64 values each; 30000 rows of 2048 take 78 us on one
// wavefront with 32, 82 on 4 with 8 (whose barrier the others wait at).
// ---------------------------------------------------------------------------
struct NormArgs {
  const void *x, *residual, *scale, *row_mask;
  void *sum, *norm;
  uint8_t *values, *scales;
  int64_t rows;
  int M;
  float inv_m, epsilon;
};

template <typename T, int WPR, int ITERS, bool ALIGNED, bool STREAMED>
__global__ __launch_bounds__(WPR > 4 ? 64 * WPR : 256) void fp8_rms_norm_kernel(
    NormArgs a) {
  __shared__ float parts[WPR];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = (int64_t)blockIdx.x * (WPR == 1 ? 4 : 1) + wave / WPR;
  const int w = wave % WPR;
  if (WPR == 1 && row >= a.rows) return;
  const int M = a.M;
  const T* x = (const T*)a.x + row * M;
  const T* residual = (const T*)a.residual + row * M;
  T* sum_out = (T*)a.sum + row * M;
  const int64_t mp = fp8_row_bytes(M), ms = fp8_scale_bytes(M);
  const int steps = STREAMED ? (int)((mp / 8 + 64 * WPR - 1) / (64 * WPR)) : ITERS;
  auto column = [&](int it) { return (lane + 64 * (w + WPR * it)) * 8; };
  auto load_row = [&](int it, float (&v)[8]) {
    load8<T, ALIGNED>(x, column(it), M, v);
    if (a.residual != nullptr) {
      float b[8];
      load8<T, ALIGNED>(residual, column(it), M, b);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = round_to<T>(v[j] + b[j]);
    }
  };
  float v[ITERS][8];
  float squares = 0.f;
  auto keep = [&](int it, const float (&u)[8]) {
    if (a.residual != nullptr) store8<T, ALIGNED>(sum_out, column(it), M, u);
#pragma unroll
    for (int j = 0; j < 8; ++j) squares = fmaf(u[j], u[j], squares);
  };
  if constexpr (STREAMED) {
    for (int it = 0; it < steps; ++it) {
      float u[8];
      load_row(it, u);
      keep(it, u);
    }
  } else {
#pragma unroll
    for (int it = 0; it < ITERS; ++it) load8<T, ALIGNED>(x, column(it), M, v[it]);
    if (a.residual != nullptr) {
#pragma unroll
      for (int it = 0; it < ITERS; ++it) {
        float b[8];
        load8<T, ALIGNED>(residual, column(it), M, b);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[it][j] = round_to<T>(v[it][j] + b[j]);
      }
    }
#pragma unroll
    for (int it = 0; it < ITERS; ++it) keep(it, v[it]);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) squares += __shfl_xor(squares, off);
  if constexpr (WPR > 1) {
    if (lane == 0) parts[wave] = squares;
    __syncthreads();
    squares = (parts[0] + parts[1]) + (parts[2] + parts[3]);
    if constexpr (WPR == 8)
      squares += (parts[4] + parts[5]) + (parts[6] + parts[7]);
  }
  const float mask =
      a.row_mask != nullptr ? load_f32<T>((const T*)a.row_mask + row) : 1.f;
  const float r = 1.0f / sqrtf(squares * a.inv_m + a.epsilon);
  auto finish = [&](int it, float (&u)[8]) {
    const int at = column(it);
    if (at - lane * 8 >= mp) return;        // (the same for the wavefront)
    float s[8];
    load8<T, ALIGNED, false>((const T*)a.scale, at, M, s);
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      // (a masked row is zero whatever it holds)
      u[j] = mask != 0.f ? u[j] * r * s[j] * mask : 0.f;
      top = max(top, magnitude_bits(u[j]));
    }
    const Fp8Scale q = fp8_scale(max16(top));
    if (a.norm != nullptr) store8<T, ALIGNED>((T*)a.norm + row * M, at, M, u);
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] *= q.factor;
    if (at < mp)
      *reinterpret_cast<uint2*>(a.values + row * mp + at) =
          make_uint2(fp8_pack4(u[0], u[1], u[2], u[3]),
                     fp8_pack4(u[4], u[5], u[6], u[7]));
    uint32_t bytes = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b)
      bytes |= (uint32_t)__builtin_amdgcn_readlane((int)q.byte, 16 * b) << (8 * b);
    if (lane == 0)
      *reinterpret_cast<uint32_t*>(a.scales + row * ms + at / FP8_BLOCK) = bytes;
  };
  if constexpr (STREAMED) {
    const T* again = a.residual != nullptr ? sum_out : x;
    for (int it = 0; it < steps; ++it) {
      float u[8];
      load8<T, ALIGNED>(again, column(it), M, u);
      finish(it, u);
    }
  } else {
#pragma unroll
    for (int it = 0; it < ITERS; ++it) finish(it, v[it]);
  }
}

// rows `row` .. row + rows - 1 of a norm
template <typename T>
static NormArgs norm_rows(const NormArgs& a, int64_t row, int64_t rows) {
  NormArgs p = a;
  auto skip = [&](auto& at, int64_t bytes) {
    if (at != nullptr) at = (std::remove_reference_t<decltype(at)>)((uint8_t*)at + bytes);
  };
  const int64_t line = row * a.M * (int64_t)sizeof(T);
  skip(p.x, line);
  skip(p.residual, line);
  skip(p.sum, line);
  skip(p.norm, line);
  skip(p.row_mask, row * (int64_t)sizeof(T));
  skip(p.values, row * fp8_row_bytes(a.M));
  skip(p.scales, row * fp8_scale_bytes(a.M));
  p.rows = rows;
  return p;
}

template <typename T, bool ALIGNED>
static void launch_norm(const NormArgs& a, hipStream_t st) {
  const int64_t mp = fp8_row_bytes(a.M);
  // (a launch has MAX_THREADS threads at most: 67 million rows of one wavefront)
  auto launch = [&](auto kernel, int threads, int per_block) {
    const int64_t most = MAX_THREADS / threads * per_block;
    for (int64_t row = 0; row < a.rows; row += most) {
      const NormArgs p = norm_rows<T>(a, row, std::min(most, a.rows - row));
      kernel<<<(unsigned)((p.rows + per_block - 1) / per_block), threads, 0, st>>>(p);
    }
  };
  if (mp <= 1024)
    launch(fp8_rms_norm_kernel<T, 1, 2, ALIGNED, false>, 256, 4);
  else if (mp <= 2048)
    launch(fp8_rms_norm_kernel<T, 1, 4, ALIGNED, false>, 256, 4);
  else if (mp <= 4096)
    launch(fp8_rms_norm_kernel<T, 4, 2, ALIGNED, false>, 256, 1);
  else if (mp <= 8192)
    launch(fp8_rms_norm_kernel<T, 4, 4, ALIGNED, false>, 256, 1);
  else if (mp <= 16384)
    launch(fp8_rms_norm_kernel<T, 8, 4, ALIGNED, false>, 512, 1);
  else
    launch(fp8_rms_norm_kernel<T, 4, 1, ALIGNED, true>, 256, 1);
}

template <typename T>
static void run_norm(const NormArgs& a, hipStream_t st) {
  const bool aligned =
      a.M % 8 == 0 && ((uintptr_t)a.x | (uintptr_t)a.residual | (uintptr_t)a.scale |
                       (uintptr_t)a.sum | (uintptr_t)a.norm) % 16 == 0;
  if (aligned) launch_norm<T, true>(a, st);
  else launch_norm<T, false>(a, st);
}

}  // namespace mesh_moe

using namespace mesh_moe;

extern "C" int mesh_moe_fp8_abi_version(void) { return MESH_MOE_FP8_ABI_VERSION; }

extern "C" int mesh_moe_fp8_quantize(const void* x, const void* relu_mask,
                                     const int32_t* row_count, void* row_values,
                                     uint8_t* row_scales, void* column_values,
                                     uint8_t* column_scales, int E, int R, int K,
                                     int dtype, void* stream) {
  MOE_REQUIRE(x && (row_values != nullptr) == (row_scales != nullptr) &&
                  (column_values != nullptr) == (column_scales != nullptr) &&
                  (row_values || column_values),
              MESH_MOE_E_ARG, "fp8_quantize: null pointer");
  MOE_REQUIRE(valid_dtype(dtype), MESH_MOE_E_ARG, "fp8_quantize: bad dtype %d", dtype);
  MOE_REQUIRE(E >= 1 && R >= 1 && K >= 1 && R <= 0x7fffff00 && K <= 0x7fffff00,
              MESH_MOE_E_ARG, "fp8_quantize: bad sizes E=%d R=%d K=%d", E, R, K);
  MOE_REQUIRE(((uintptr_t)row_values | (uintptr_t)column_values) % 16 == 0 &&
                  ((uintptr_t)x | (uintptr_t)relu_mask) % dtype_size(dtype) == 0,
              MESH_MOE_E_UNSUPPORTED,
              "fp8_quantize: 8-bit values need to lie on 16 bytes");
  return fp8_quantize(x, relu_mask, row_count, row_values, row_scales, column_values,
                      column_scales, E, R, K, dtype, false, (hipStream_t)stream);
}

extern "C" int mesh_moe_fp8_dequantize(const void* values, const uint8_t* scales,
                                       void* y, int64_t rows, int K, int dtype,
                                       void* stream) {
  MOE_REQUIRE(values && scales && y, MESH_MOE_E_ARG, "fp8_dequantize: null pointer");
  MOE_REQUIRE(valid_dtype(dtype), MESH_MOE_E_ARG, "fp8_dequantize: bad dtype %d",
              dtype);
  MOE_REQUIRE(rows >= 1 && K >= 1 && K <= 0x7fffff00, MESH_MOE_E_ARG,
              "fp8_dequantize: bad sizes rows=%lld K=%d", (long long)rows, K);
  MOE_REQUIRE((uintptr_t)values % 16 == 0, MESH_MOE_E_UNSUPPORTED,
              "fp8_dequantize: 8-bit values need to lie on 16 bytes");
  hipStream_t st = (hipStream_t)stream;
  if (dtype == MESH_MOE_F32)
    run_dequantize<float>((const uint8_t*)values, scales, (float*)y, rows, K, st);
  else
    run_dequantize<bf16_t>((const uint8_t*)values, scales, (bf16_t*)y, rows, K, st);
  MOE_CHECK_LAUNCH("fp8_dequantize");
  return 0;
}

extern "C" int mesh_moe_fp8_residual_rms_norm(const void* x, const void* residual,
                                              const void* scale, const void* row_mask,
                                              void* sum, void* norm, void* values,
                                              uint8_t* scales, int64_t rows, int M,
                                              double epsilon, int dtype, void* stream) {
  MOE_REQUIRE(x && scale && values && scales &&
                  (residual == nullptr) == (sum == nullptr),
              MESH_MOE_E_ARG, "fp8_residual_rms_norm: null pointer");
  MOE_REQUIRE(valid_dtype(dtype), MESH_MOE_E_ARG,
              "fp8_residual_rms_norm: bad dtype %d", dtype);
  MOE_REQUIRE(rows >= 1 && rows <= 0x7fffffffLL && M >= 1 && M <= 0x7fffff00,
              MESH_MOE_E_ARG, "fp8_residual_rms_norm: bad sizes rows=%lld M=%d",
              (long long)rows, M);
  MOE_REQUIRE((uintptr_t)values % 16 == 0 && (uintptr_t)scales % 4 == 0,
              MESH_MOE_E_UNSUPPORTED,
              "fp8_residual_rms_norm: 8-bit values need to lie on 16 bytes, scales on 4");
  const NormArgs a = {x, residual, scale, row_mask, sum, norm, (uint8_t*)values,
                      scales, rows, M, (float)(1.0 / (double)M), (float)epsilon};
  if (dtype == MESH_MOE_F32) run_norm<float>(a, (hipStream_t)stream);
  else run_norm<bf16_t>(a, (hipStream_t)stream);
  MOE_CHECK_LAUNCH("fp8_residual_rms_norm");
  return 0;
}
