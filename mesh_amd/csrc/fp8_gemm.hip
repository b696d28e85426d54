// Products of 8-bit operands (see mesh_moe_fp8.h) on the scaled matrix instructions.
//
// The instructions (v_mfma_scale_f32_32x32x64_f8f6f4, _16x16x128_) take a power of two for
// every 32 values of a row, from a byte of a register that each lane has for its row: a
// block of 128 uses the same byte throughout, and the scales cost no instruction of their
// own.  Which 32 values of a block a lane has in a step is free, as long as both operands
// agree.  The weights are the first operand and the tokens the second, so that a lane ends
// up with one token's row: 4 neighbouring columns per group of 4 accumulators.
#include "fp8.h"

#include <type_traits>

namespace mesh_moe {

typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

// The activations as the products apply them to their float32 sums; NaN stays NaN.  All
// but relu are (n0 or v) / (1 + exp(v (k1 + k3 v^2))) + off with constants of the
// activation: 0.5 (1 + tanh u) = 1 / (1 + exp(-2 u)), tanh v = 2 / (1 + exp(-2 v)) - 1,
// the latter by its series where the difference would lose bits.  v^2 is kept finite and
// the numerator chosen: 0 times an infinity would be NaN, where only gelu has a k3 and
// sigmoid and tanh no v.  (gelu and swish of -infinity are NaN, as an infinity divided by
// one is.)  The hardware's exponential and reciprocal are off by 2^-21 or so (relative,
// for arguments that matter; results below 2^-119 may become zeros), far below the
// rounding of the result.
struct Fp8Act {
  float n0, k1, k3, off, near;
  bool times_v;
  __device__ __forceinline__ explicit Fp8Act(int act) {
    const bool tanh = act == MESH_MOE_ACT_TANH, gelu = act == MESH_MOE_ACT_GELU;
    n0 = tanh ? 2.f : 1.f;
    times_v = gelu || act == MESH_MOE_ACT_SWISH;
    k1 = gelu ? -1.5957691216057308f : tanh ? -2.f : -1.f;
    k3 = gelu ? -1.5957691216057308f * 0.044715f : 0.f;
    off = tanh ? -1.f : 0.f;
    near = tanh ? 4e-4f : 0.f;
  }
  __device__ __forceinline__ float operator()(float v) const {
    const float v2 = fminf(v * v, 3e38f);
    const float y = (times_v ? v : n0) *
                        __builtin_amdgcn_rcpf(1.f + __expf(v * (k1 + k3 * v2))) + off;
    const float series = v - v * v2 * 0.33333334f;
    return v2 < near ? series : y;
  }
};
__device__ __forceinline__ float fp8_relu(float v) { return v < 0.f ? 0.f : v; }
__device__ __forceinline__ float fp8_activation(float v, int act) {
  return act == MESH_MOE_ACT_LINEAR ? v
         : act == MESH_MOE_ACT_RELU ? fp8_relu(v) : Fp8Act(act)(v);
}

// rows of expert e that are multiplied
__device__ __forceinline__ int live_rows(const int32_t* row_count, int e, int R) {
  return row_count != nullptr ? min(max(row_count[e], 0), R) : R;
}

struct GemmArgs {
  const uint8_t *a, *a_scales, *w, *w_scales;
  const int32_t* row_count;
  void* y;                  // bf16, float32 or e4m3, see the kernels
  uint8_t* y_scales;
  int E, R, K, N, activation;
  // values of expert e's rows that are not zeros, or null: a kernel may leave the others out
  const int32_t* k_count;
};

// ---------------------------------------------------------------------------
// Few rows: 16 TM rows per block, and 16 columns with the reduction dealt out over the 8
// wavefronts, whose sums meet in LDS (CW = 1), or 8 times 16 columns of a wavefront each
// (CW = 8: for a reduction of one block of 128, and what the tile kernels cannot address).
// Bound by the weights, which are read once, straight from memory into registers: four
// blocks of 128 of a row are requested before the first is multiplied.  One row 4096 ->
// 16384 takes 15.6 us, 4.3 TB/s, with weights from memory, 13.7 from the caches (14.4, and
// 16.0 with requests for 32 bytes of each row instead of 64, when that was chosen).  That leaves time to multiply in bfloat16, which holds an e4m3 number times its
// unit, so that the sums are float32 ones; the instructions for 8 bits cut 8 neighbouring
// products off below 2^-13 of the largest one's power of two.
// TO: bf16_t, float (rows of fp8_row_bytes(N), without the activation: fp8_parts_kernel
// goes on from there) or uint8_t (an 8-bit operand; CW is 8: a block of 128 columns).
// ---------------------------------------------------------------------------
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
// the unit that a scale byte stands for, 255 being NaN
__device__ __forceinline__ float fp8_unit(uint8_t byte) {
  return __uint_as_float(byte == 255 ? 0x7fc00000u : (uint32_t)byte << 23);
}
// 8 numbers times their unit, exact: 2^-9 times the least unit, 2^-117, is normal
__device__ __forceinline__ bf16x8_t fp8_widen(int lo, int hi, float unit) {
  bf16x2_t v[4];
  v[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)lo, unit, false);
  v[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)lo, unit, true);
  v[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)hi, unit, false);
  v[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)hi, unit, true);
  const bf16x4_t a = __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3);
  const bf16x4_t b = __builtin_shufflevector(v[2], v[3], 0, 1, 2, 3);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

template <int TM, int CW, typename TO>
__global__ __launch_bounds__(512) void fp8_few_rows_kernel(GemmArgs g, int tiles_m,
                                                           int tiles_n) {
  constexpr bool EIGHT = std::is_same<TO, uint8_t>::value;
  constexpr int WAVES = 8, KW = WAVES / CW, U = TM == 4 ? 2 : 4;
  static_assert(CW == 1 || CW == 8, "see above");
  static_assert(!EIGHT || CW == 8, "a block of 128 columns");
  __shared__ float parts[KW][TM * 4][64];
  __shared__ uint32_t tops[TM][16][CW];
  const int tile = blockIdx.x / tiles_n, tn = blockIdx.x - tile * tiles_n;
  const int e = tile / tiles_m, row0 = (tile - e * tiles_m) * 16 * TM;
  const int live = live_rows(g.row_count, e, g.R);
  if (row0 >= live) return;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = wave % CW, k = wave / CW;
  const int at = lane & 15, quarter = lane >> 4;
  const int col0 = tn * 16 * CW + 16 * c;
  const int64_t kp = fp8_row_bytes(g.K), ks = fp8_scale_bytes(g.K);
  const uint8_t *a[TM], *as[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int64_t row = (int64_t)e * g.R + min(row0 + 16 * i + at, live - 1);
    a[i] = g.a + row * kp + quarter * 16;
    as[i] = g.a_scales + row * ks;
  }
  const int64_t w_row = (int64_t)e * g.N + min(col0 + at, g.N - 1);
  const uint8_t* w = g.w + w_row * kp + quarter * 16;
  const uint8_t* ws = g.w_scales + w_row * ks;
  // (a lane's chunks of 16 bytes lie 64 apart: a request takes whole halves of lines)
  auto fragment = [](const uint8_t* from) {
    const uint4 lo = reinterpret_cast<const uint4*>(from)[0];
    const uint4 hi = reinterpret_cast<const uint4*>(from)[4];
    return i32x8_t{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w,
                   (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
  };
  f32x4_t acc[TM] = {};
  // `n` blocks from b on, all of them requested before the first is multiplied
  auto step = [&](auto n_tag, int b) __attribute__((always_inline)) {
    constexpr int N = decltype(n_tag)::value;
    i32x8_t vw[N], va[N][TM];
    uint8_t sw[N], sa[N][TM];
#pragma unroll
    for (int u = 0; u < N; ++u) {
      vw[u] = fragment(w + (int64_t)(b + u) * FP8_BLOCK);
      sw[u] = ws[b + u];
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        va[u][i] = fragment(a[i] + (int64_t)(b + u) * FP8_BLOCK);
        sa[u][i] = as[i][b + u];
      }
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const float fw = fp8_unit(sw[u]);
      float fa[TM];
#pragma unroll
      for (int i = 0; i < TM; ++i) fa[i] = fp8_unit(sa[u][i]);
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const bf16x8_t w8 = fp8_widen(vw[u][2 * m], vw[u][2 * m + 1], fw);
#pragma unroll
        for (int i = 0; i < TM; ++i)
          acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              w8, fp8_widen(va[u][i][2 * m], va[u][i][2 * m + 1], fa[i]), acc[i], 0, 0, 0);
      }
    }
  };
  // (runs of whole groups of U where there are that many)
  const int blocks = (int)(kp / FP8_BLOCK);
  int run = (blocks + KW - 1) / KW;
  if (run >= U) run = (run + U - 1) / U * U;
  int b = k * run;
  const int last = min(b + run, blocks);
  for (; b + U <= last; b += U) step(std::integral_constant<int, U>{}, b);
  if (U == 4 && b + 2 <= last) {
    step(std::integral_constant<int, 2>{}, b);
    b += 2;
  }
  if (b < last) step(std::integral_constant<int, 1>{}, b);
  // lane l has token l % 16 and the columns 4 (l / 16) .. + 3
  if constexpr (KW > 1) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) parts[k][4 * i + q][lane] = acc[i][q];
    __syncthreads();
    for (int v = wave; v < 4 * TM; v += WAVES) {
      float sum = 0.f;
#pragma unroll
      for (int p = 0; p < KW; ++p) sum += parts[p][v][lane];
      const int row = row0 + 16 * (v >> 2) + at, col = col0 + 4 * quarter + (v & 3);
      if (row < live && col < g.N) {
        const int64_t to = (int64_t)e * g.R + row;
        if constexpr (std::is_same<TO, float>::value)
          ((float*)g.y)[to * fp8_row_bytes(g.N) + col] = sum;
        else
          ((bf16_t*)g.y)[to * g.N + col] = f32_to_bf16(fp8_activation(sum, g.activation));
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      uint32_t top = 0;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float v = fp8_activation(acc[i][q], g.activation);
        acc[i][q] = col0 + 4 * quarter + q < g.N ? v : 0.f;
        top = max(top, magnitude_bits(acc[i][q]));
      }
      if constexpr (EIGHT) {
        top = max(top, (uint32_t)__shfl_xor((int)top, 16));
        top = max(top, (uint32_t)__shfl_xor((int)top, 32));
        if (quarter == 0) tops[i][at][c] = top;
      }
    }
    if constexpr (EIGHT) __syncthreads();
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int row = row0 + 16 * i + at, col = col0 + 4 * quarter;
      if (row >= live) continue;
      const int64_t to = (int64_t)e * g.R + row;
      if constexpr (EIGHT) {
        uint32_t top = 0;
#pragma unroll
        for (int p = 0; p < CW; ++p) top = max(top, tops[i][at][p]);
        const Fp8Scale s = fp8_scale(top);
        *reinterpret_cast<uint32_t*>((uint8_t*)g.y + to * fp8_row_bytes(g.N) + col) =
            fp8_pack4(acc[i][0] * s.factor, acc[i][1] * s.factor, acc[i][2] * s.factor,
                      acc[i][3] * s.factor);
        if (c == 0 && quarter == 0)
          g.y_scales[to * fp8_scale_bytes(g.N) + tn] = (uint8_t)s.byte;
      } else {
        bf16_t* const y = (bf16_t*)g.y + to * g.N + col;
        if (g.N % 4 == 0 && (uintptr_t)g.y % 8 == 0) {
          if (col < g.N)
            *reinterpret_cast<uint2*>(y) = make_uint2(
                f32x2_to_bf16x2(acc[i][0], acc[i][1]), f32x2_to_bf16x2(acc[i][2], acc[i][3]));
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (col + q < g.N) y[q] = f32_to_bf16(acc[i][q]);
        }
      }
    }
  }
}

// --- what the tile kernels share ------------------------------------------------
typedef __attribute__((address_space(3))) void lds_void_t;
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// what a kernel writes
constexpr int TO_LINES = 0;       // bf16 rows of whole 16-byte pieces on 16 bytes
constexpr int TO_BF16 = 1;        // bf16 rows of any kind
constexpr int TO_FP8 = 2;         // an 8-bit operand
constexpr int TO_PARTS = 3;       // float32 sums of a part of the reduction

struct TileGrid {
  int tiles_m, tiles_n;           // of an expert with all of its rows
  int tiles;                      // of all experts and parts
  int split;                      // parts of the reduction, whole groups of 4 K tiles
};

#define FP8_INLINE __attribute__((always_inline))

// a pointer that all lanes have
__device__ __forceinline__ const uint8_t* uniform(const uint8_t* p) {
  const uint64_t u = (uint64_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)u);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((int)(u >> 32));
  return (const uint8_t*)((uint64_t)hi << 32 | lo);
}

// 16 bytes per lane, from at + skip of the `bytes` at `from` (zeros behind them), to LDS:
// lane after lane from `to` on
__device__ __forceinline__ void load_to_lds(const uint8_t* from, int bytes, uint32_t at,
                                            int skip, unsigned char* to) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(
      __builtin_amdgcn_make_buffer_rsrc((void*)from, 0, bytes, 0x00027000),
      (lds_void_t*)to, 16, at, skip, 0, 0);
}

// 16 bytes per lane, at `at` of the `bytes` at `base`; what lies behind is dropped.  Past
// the caches (the last argument, nt), which the operands need: weight gradients of 32
// experts 4096 x 640 -> 1024 take 90 us instead of 110, 64 experts' 705 rows 1024 -> 4096
// 197 instead of 204.
__device__ __forceinline__ void store_line(u32x4_t v, uint8_t* base, int bytes,
                                           uint32_t at) {
  __builtin_amdgcn_raw_buffer_store_b128(
      v, __builtin_amdgcn_make_buffer_rsrc(base, 0, max(bytes, 0), 0x00027000), at, 0, 2);
}

__device__ __forceinline__ f32x16_t fp8_mfma(i32x8_t w, i32x8_t a, f32x16_t c,
                                             uint32_t w_scale, uint32_t a_scale) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w, a, c, 0, 0, 0, (int)w_scale,
                                                         0, (int)a_scale);
}

// two 16-byte chunks of a row
__device__ __forceinline__ i32x8_t fp8_fragment(const unsigned char* lo,
                                                const unsigned char* hi) {
  const u32x4_t a = *reinterpret_cast<const u32x4_t*>(lo);
  const u32x4_t b = *reinterpret_cast<const u32x4_t*>(hi);
  return __builtin_bit_cast(
      i32x8_t, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// Four 16-byte reads, STEP bytes apart, and the wait for them in one asm, whose outputs
// then hold what the compiler takes them for.
template <int STEP>
__device__ __forceinline__ void lds_read_lines(u32x4_t (&p)[4], uint32_t at) {
  asm volatile("ds_read_b128 %0, %4\n\t"
               "ds_read_b128 %1, %4 offset:%5\n\t"
               "ds_read_b128 %2, %4 offset:%6\n\t"
               "ds_read_b128 %3, %4 offset:%7\n\t"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(p[0]), "=&v"(p[1]), "=&v"(p[2]), "=&v"(p[3])
               : "v"(at), "n"(STEP), "n"(2 * STEP), "n"(3 * STEP)
               : "memory");
}
__device__ __forceinline__ void lds_write_b64(uint32_t at, u32x2_t v) {
  asm volatile("ds_write_b64 %0, %1" :: "v"(at), "v"(v) : "memory");
}
__device__ __forceinline__ void lds_write_b32(uint32_t at, uint32_t v) {
  asm volatile("ds_write_b32 %0, %1" :: "v"(at), "v"(v) : "memory");
}

// s_waitcnt with vmcnt `vm` and, or not, lgkmcnt 0
template <int VM, bool LGKM>
__device__ __forceinline__ void wait_counts() {
  __builtin_amdgcn_s_waitcnt((VM & 15) | (VM >> 4) << 14 | (7 << 4) | (LGKM ? 0 : 15) << 8);
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ void block_barrier() {
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// A tile of a launch: rows row0 .. row0 + valid - 1 and columns from col0 on of expert e,
// over the K tiles k0 .. k0 + nk - 1.
struct Tile {
  int e, row0, col0;
  int valid;                      // 0: there is no such tile
  int part, k0, nk;
};
// Tile number `logical`.  With row counts the tiles are those that hold rows, counted
// through 64 experts at a time: lane l adds up the row tiles of expert l and below.
// PARTS: the reduction is split, all tiles of a part follow each other.
template <int BM, int BN, bool PARTS>
__device__ __forceinline__ Tile find_tile(const GemmArgs& g, const TileGrid& grid,
                                          int k_tiles, int logical, int lane) {
  Tile t = {0, 0, 0, 0, 0, 0, k_tiles};
  int tiles_m = grid.tiles_m, rem = 0;
  if (logical >= grid.tiles) return t;
  if constexpr (PARTS) {
    const int whole = grid.tiles / grid.split;
    t.part = logical / whole;
    logical -= t.part * whole;
    const int groups = (k_tiles + 3) / 4;
    t.k0 = 4 * (groups * t.part / grid.split);
    t.nk = min(4 * (groups * (t.part + 1) / grid.split), k_tiles) - t.k0;
  }
  if (g.row_count == nullptr) {
    const int per = grid.tiles_m * grid.tiles_n;
    t.e = logical / per;
    rem = logical - t.e * per;
    t.valid = g.R;
  } else {
    int before = 0;
    bool found = false;
    for (int e0 = 0; e0 < g.E && !found; e0 += 64) {
      const int live = e0 + lane < g.E ? live_rows(g.row_count, e0 + lane, g.R) : 0;
      int sum = (live + BM - 1) / BM * grid.tiles_n;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int below = __shfl_up(sum, off);
        if (lane >= off) sum += below;
      }
      const uint64_t past = __ballot(before + sum > logical);
      if (past != 0) {
        const int at = __builtin_ctzll(past);
        t.e = e0 + at;
        t.valid = __builtin_amdgcn_readlane(live, at);
        tiles_m = (t.valid + BM - 1) / BM;
        rem = logical - before -
              (__builtin_amdgcn_readlane(sum, at) - tiles_m * grid.tiles_n);
        found = true;
      }
      before += __builtin_amdgcn_readlane(sum, 63);
    }
    if (!found) return t;
  }
  const int band = rem / (8 * grid.tiles_n);
  const int high = min(8, tiles_m - 8 * band);
  const int r = rem - band * 8 * grid.tiles_n;
  const int tn = r / high;
  t.row0 = __builtin_amdgcn_readfirstlane((band * 8 + (r - tn * high)) * BM);
  t.col0 = __builtin_amdgcn_readfirstlane(tn * BN);
  t.e = __builtin_amdgcn_readfirstlane(t.e);
  t.valid = __builtin_amdgcn_readfirstlane(min(BM, t.valid - t.row0));
  if constexpr (!PARTS)
    if (g.k_count != nullptr)       // (two K tiles at least)
      t.nk = max(min((live_rows(g.k_count, t.e, g.K) + FP8_BLOCK - 1) / FP8_BLOCK, k_tiles),
                 2);
  return t;
}
// number of the block's tile of round `round`
__device__ __forceinline__ int tile_number(int round) {
  return (int)(round * gridDim.x + (blockIdx.x & 7) * (gridDim.x >> 3) +
               (blockIdx.x >> 3));
}

// ---------------------------------------------------------------------------
// 256 x 256 tiles.  8 wavefronts, two per SIMD: wavefront (wm, wn) has the rows 32 wm ..
// and 128 + 32 wm .. of a tile and 128 columns from 128 wn on, that is 2 x 4 matrix
// tiles of 32 x 32 in 128 accumulator registers.  (Its rows lie 128 apart so that a
// last row tile keeps all four SIMDs busy, and its columns are one block of 128, so
// that an 8-bit result's scale needs no other wavefront.)
//
// A K tile is one block of 128 values: 256 + 256 rows of 128 bytes, brought to LDS by
// direct loads, 8 rows per instruction and whole 128-byte lines; the 16-byte chunks of
// a row are XOR-ed with its number on the way (on the global side), which spreads the
// fragment reads over all banks.  The 160 KB of LDS hold two token slots and three
// weight slots.  Two steps of 8 matrix instructions per K tile t:
//   step 0   reads the fragments of step 1; weight loads of K tile t + 2
//   barrier  all of tile t's fragments are in registers, tile t + 1 has landed
//            (vmcnt counts in order: only the four weight loads of step 0 may be out)
//   step 1   reads the fragments of tile t + 1's step 0; token loads of tile t + 2,
//            into the slot that the barrier freed
// Blocks are persistent, one per CU, and the K tiles of a block's tiles follow each other:
// the loads of a tile's last two K tiles are the first of the next.  (An only K tile is
// followed by one of zeros: 16384 rows 128 -> 4096 take 28 us, 150 with few-rows blocks.)
// Block b runs on XCD b % 8; the blocks of an XCD hold consecutive tiles, numbered in
// bands of 8 row tiles, so that 32 of them share 8 + 4 operand panels in its L2.
//
// A lane's scales are a dword per row and four K tiles, shifted along as the K tiles go
// by; the next four are requested a K tile or more ahead.
//
// A result is turned round in the weight slot that the last K tile has left, 32 rows of
// 128 bytes at a time, each wavefront in the kilobytes that its own loads fill
// afterwards (so no barrier), and leaves in whole 128-byte lines.
//
// 8192^3 takes 427 us, 2575 TFLOP/s, 1.6 us per K tile; with zeros for operands 349 us:
// the difference is what the socket's power limit takes.  16384 rows 1024 -> 4096 65 us (49).
// ---------------------------------------------------------------------------
struct BigCfg {
  static constexpr int BM = 256, BN = 256, THREADS = 512, WAVES = 8;
  static constexpr int TM = 2, TN = 4;
  static constexpr int SLOT = 256 * FP8_BLOCK;          // 32 KB
  static constexpr int W_BASE = 2 * SLOT;
  static constexpr int LDS_BYTES = 5 * SLOT;
};

// EIGHT: the result is an 8-bit operand; ACT: an activation that is neither linear nor
// relu; WHOLE: rows of a bf16 result are whole pieces of 16 bytes that lie on 16 bytes.
template <bool EIGHT, bool ACT, bool WHOLE>
__global__ __launch_bounds__(BigCfg::THREADS) void fp8_tile256_kernel(GemmArgs g,
                                                                    TileGrid grid) {
  using Cfg = BigCfg;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const int fr = lane & 31, fc = lane >> 5;
  const int64_t kp = fp8_row_bytes(g.K), ks = fp8_scale_bytes(g.K);
  // (an only K tile is followed by one of zeros, with scales that are no NaN)
  const bool single = kp == FP8_BLOCK;
  const int nk = single ? 2 : (int)(kp / FP8_BLOCK);
  const uint32_t scale_mask = single ? 0xffu : ~0u;

  // (What is computed from the lane index outside the K loop is computed from a copy
  // that the compiler cannot see through: made once it would be live across the K loop,
  // which has no registers to spare.)
  auto lane_again = [&]() FP8_INLINE {
    int l = lane;
    asm volatile("" : "+v"(l));
    return l;
  };

  auto tile_at = [&](int round) FP8_INLINE {
    return find_tile<Cfg::BM, Cfg::BN, false>(g, grid, nk, tile_number(round),
                                              lane_again());
  };

  // The tile that is being loaded.  A wavefront's load j fills the rows 8 (wave + 8 j) ..
  // + 7 of an LDS tile through a buffer that ends with the rows there are: what lies
  // behind is not fetched.  (A row's place is the lanes' part of an address, the K tile's
  // the wavefront's: whichever of them the range check looks at, a row that is there
  // passes it and one that is not fails.)
  const uint8_t *a_base, *w_base;
  int a_bytes, w_bytes;
  uint32_t load_at[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    load_at[j] = (uint32_t)((wave + 8 * j) * 8 + (lane >> 3)) * (uint32_t)kp +
                 ((lane & 7) ^ (lane >> 3) ^ (wave & 1)) * 16;
  auto set_loads = [&](const Tile& t) FP8_INLINE {
    a_base = uniform(g.a + ((int64_t)t.e * g.R + t.row0) * kp);
    w_base = uniform(g.w + ((int64_t)t.e * g.N + t.col0) * kp);
    a_bytes = t.valid * (int)kp;
    w_bytes = min(Cfg::BN, g.N - t.col0) * (int)kp;
  };
  auto load_a = [&](int kt, int j, int slot) FP8_INLINE {
    load_to_lds(a_base, single && kt == 1 ? 0 : a_bytes, load_at[j], kt * FP8_BLOCK,
                smem + slot * Cfg::SLOT + (wave + 8 * j) * 1024);
  };
  auto load_w = [&](int kt, int j, int slot) FP8_INLINE {
    load_to_lds(w_base, single && kt == 1 ? 0 : w_bytes, load_at[j], kt * FP8_BLOCK,
                smem + Cfg::W_BASE + slot * Cfg::SLOT + (wave + 8 * j) * 1024);
  };

  // scales of this lane's rows: of the K tiles that are multiplied, and the next four
  uint32_t sa[Cfg::TM], sw[Cfg::TN], sa_next[Cfg::TM], sw_next[Cfg::TN];
  auto load_scales = [&](const Tile& t, int group) FP8_INLINE {
    const int fr = lane_again() & 31;
    const uint8_t* as = g.a_scales + ((int64_t)t.e * g.R + t.row0) * ks + 4 * group;
    const uint8_t* ws = g.w_scales + ((int64_t)t.e * g.N + t.col0) * ks + 4 * group;
#pragma unroll
    for (int i = 0; i < Cfg::TM; ++i)
      sa_next[i] = *reinterpret_cast<const uint32_t*>(
          as + (uint32_t)min(128 * i + 32 * wm + fr, t.valid - 1) * (uint32_t)ks);
#pragma unroll
    for (int j = 0; j < Cfg::TN; ++j)
      sw_next[j] = *reinterpret_cast<const uint32_t*>(
          ws + (uint32_t)min(128 * wn + 32 * j + fr, g.N - 1 - t.col0) * (uint32_t)ks);
  };

  // Fragment chunk c of a row lies at its chunk position c ^ (row % 8) ^ (row / 8 % 2);
  // step s has the chunks 4 s + fc and 4 s + 2 + fc.  (Positions and slots have bits of
  // their own in an address.)
  const int swizzle = (fr & 7) ^ ((fr >> 3) & 1);
  const int frag_at = fr * FP8_BLOCK + (fc ^ swizzle) * 16;
  // (again a copy: one register lives on instead of all sums with constants)
  auto frag_again = [&]() FP8_INLINE {
    int at = frag_at;
    asm volatile("" : "+v"(at));
    return at;
  };
  auto read_a = [&](int frag_at, int slot, int s, int i) FP8_INLINE {
    const int at = frag_at + (slot * Cfg::SLOT + 32 * wm * FP8_BLOCK);
    return fp8_fragment(smem + (at ^ (64 * s)) + i * 128 * FP8_BLOCK,
                        smem + (at ^ (64 * s + 32)) + i * 128 * FP8_BLOCK);
  };
  auto read_w = [&](int frag_at, int slot, int s, int j) FP8_INLINE {
    const int at =
        frag_at + (Cfg::W_BASE + slot * Cfg::SLOT + 128 * wn * FP8_BLOCK);
    return fp8_fragment(smem + (at ^ (64 * s)) + j * 32 * FP8_BLOCK,
                        smem + (at ^ (64 * s + 32)) + j * 32 * FP8_BLOCK);
  };

  f32x16_t acc[Cfg::TM][Cfg::TN];
  i32x8_t fa[2][Cfg::TM], fw[Cfg::TN];
  auto fence = [&]() FP8_INLINE { __builtin_amdgcn_sched_barrier(0); };
  int aslot = 0, wslot = 0;

  auto first_fragments = [&](int as, int ws) FP8_INLINE {
    const int at = frag_again();
#pragma unroll
    for (int i = 0; i < Cfg::TM; ++i) fa[0][i] = read_a(at, as, 0, i);
#pragma unroll
    for (int j = 0; j < Cfg::TN; ++j) fw[j] = read_w(at, ws, 0, j);
  };

  // One K tile; lk: the one that the loads fetch; NA: the wavefront's pieces of 32 rows
  // that hold rows of the tile; FIRST: the sums begin; LAST: the next tile's fragments
  // are read when the result is out of the registers.  No branches inside: the compiler
  // would move matrix instructions past them, behind the barrier.
  constexpr int STORES = EIGHT ? 4 : 8;           // of 16 bytes per lane and piece
  auto k_tile = [&](auto na_tag, auto first_tag, auto last_tag, int lk) FP8_INLINE {
    constexpr int NA = decltype(na_tag)::value;
    constexpr bool FIRST = decltype(first_tag)::value, LAST = decltype(last_tag)::value;
    const int wnext = wslot == 2 ? 0 : wslot + 1, wload = wnext == 2 ? 0 : wnext + 1;
    const int anext = aslot ^ 1;
    const f32x16_t none = {};
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int at = frag_again();
      const int as = s == 0 ? aslot : anext, ws = s == 0 ? wslot : wnext;
      const int to = s ^ 1;
      auto mfma = [&](int m) {
        const int j = m >> 1, i = m & 1;
        if (i >= NA) return;
        acc[i][j] = fp8_mfma(fw[j], fa[s][i], FIRST && s == 0 ? none : acc[i][j], sw[j],
                             sa[i]);
      };
      constexpr bool READ[2] = {NA > 0, NA > 0 && !LAST};
      auto rd_a = [&](int i) { if (READ[s] && i < NA) fa[to][i] = read_a(at, as, to, i); };
      auto rd_w = [&](int j) { if (READ[s]) fw[j] = read_w(at, ws, to, j); };
      // (the weight loads have half a K tile more than the token loads, which go first)
      auto ld = [&](int j, bool here) {
        if (!here) return;
        if (s == 0) load_w(lk, j, wload);
        else load_a(lk, j, aslot);
      };
      fence();
      if (s == 1) {
#pragma unroll
        for (int j = 0; j < 4; ++j) ld(j, true);
        fence();
      }
      rd_a(0);
      mfma(0); fence();
      rd_a(1);
      mfma(1); fence();
      rd_w(0);
      ld(0, s == 0);
      mfma(2); fence();
      mfma(3); fence();
      rd_w(1);
      ld(1, s == 0);
      mfma(4); fence();
      mfma(5); fence();
      rd_w(2);
      ld(2, s == 0);
      mfma(6); fence();
      mfma(7); fence();
      rd_w(3);
      ld(3, s == 0);
      fence();
      if (s == 0) {
        // lgkmcnt 0, and vmcnt: besides the weight loads of step 0 the first K tile leaves
        // out as many of the last tile's stores as every wavefront has at least (see the
        // end of a tile)
        constexpr int OUT = FIRST ? 4 + STORES : 4;
        __builtin_amdgcn_s_waitcnt((OUT & 15) | (OUT >> 4) << 14 | (7 << 4));
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
      }
    }
    aslot = anext;
    wslot = wnext;
  };

  // The result of a tile.  A pass turns 32 rows of 128 bytes round: 64 columns of bf16, or
  // a block of 128 in 8 bits.  Lane l writes 8-byte units of row l % 32 and reads 16
  // bytes of the rows 8 n + l / 8; unit u of a row lies at u ^ 2 (row % 8) ^ (row / 8 %
  // 2).  The stores of whole lines go through a buffer that ends with the tile's rows, so
  // that they leave in any case and the next tile's first wait can count on them.
  auto write_out = [&](const Tile& t, auto na_tag) FP8_INLINE {
    constexpr int NA = decltype(na_tag)::value;
    const int wfree = wslot == 0 ? 2 : wslot - 1;       // of the last K tile
    const int lane = lane_again(), fr = lane & 31, fc = lane >> 5;
    const uint32_t stage = (uint32_t)(size_t)(lds_void_t*)smem + Cfg::W_BASE +
                           wfree * Cfg::SLOT + wave * 1024;
    const uint32_t put_at = stage + (fr >> 3) * 8192 + (fr & 7) * 128 +
                            ((fc ^ ((fr & 7) << 1) ^ ((fr >> 3) & 1)) * 8);
    const int get_row = lane >> 3, get_chunk = lane & 7;
    const uint32_t get_at = stage + get_row * 128 + ((get_chunk ^ get_row) * 16);
    const int col0 = t.col0 + 128 * wn;
    const int64_t first = (int64_t)t.e * g.R + t.row0;
    const int64_t np = fp8_row_bytes(g.N), ns = fp8_scale_bytes(g.N);
    u32x4_t line[4];
    auto chunk_of = [&](int n) {
      u32x4_t v = line[n];
      return n & 1 ? __builtin_shufflevector(v, v, 2, 3, 0, 1) : v;
    };
    const int row_bytes = EIGHT ? (int)np : 2 * g.N;
    // lines from column `col` (in bytes) of the piece's rows
    auto store_lines = [&](int piece, int col) FP8_INLINE {
      const int rows = t.valid - piece;
      uint8_t* const base = (uint8_t*)g.y + (first + piece) * row_bytes + col;
      const uint32_t at = col + 16 * get_chunk < row_bytes
                              ? (uint32_t)(get_row * row_bytes + 16 * get_chunk)
                              : 0x80000000u;      // (past every buffer)
#pragma unroll
      for (int n = 0; n < 4; ++n)
        store_line(chunk_of(n), base + (int64_t)8 * n * row_bytes,
                   max(min(rows - 8 * n, 8), 0) * row_bytes - col, at);
    };
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int piece = 128 * i + 32 * wm;
      f32x16_t(&v)[Cfg::TN] = acc[i];
      if constexpr (ACT) {
        const Fp8Act act(g.activation);
        int columns = g.N - col0 - 4 * fc;
        asm volatile("" : "+v"(columns));      // (not 64 masks kept for the next piece)
#pragma unroll
        for (int j = 0; j < Cfg::TN; ++j)
#pragma unroll
          for (int q = 0; q < 16; ++q) {
            const float u = act(v[j][q]);
            v[j][q] = 32 * j + 8 * (q >> 2) + (q & 3) < columns ? u : 0.f;
          }
      } else if (g.activation == MESH_MOE_ACT_RELU) {
#pragma unroll
        for (int j = 0; j < Cfg::TN; ++j)
#pragma unroll
          for (int q = 0; q < 16; ++q) v[j][q] = fp8_relu(v[j][q]);
      }
      if constexpr (EIGHT) {
        // (columns past N are zeros: the weights' buffer ends there)
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < Cfg::TN; ++j)
#pragma unroll
          for (int q = 0; q < 16; ++q) top = max(top, magnitude_bits(v[j][q]));
        top = max(top, (uint32_t)__shfl_xor((int)top, 32));
        const Fp8Scale s = fp8_scale(top);
#pragma unroll
        for (int j = 0; j < Cfg::TN; ++j)
#pragma unroll
          for (int q = 0; q < 16; q += 8) {
            uint32_t d[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int at = q + 4 * h;
              d[h] = fp8_pack4(v[j][at] * s.factor, v[j][at + 1] * s.factor,
                               v[j][at + 2] * s.factor, v[j][at + 3] * s.factor);
            }
            // a lane has columns 4 fc .. of each 8: trade halves for whole 8s
            const auto w = __builtin_amdgcn_permlane32_swap(d[0], d[1], false, false);
            const int unit = 2 * (2 * j + (q >> 3));    // + fc, which put_at has
            lds_write_b64(put_at ^ (unit * 8), u32x2_t{w[0], w[1]});
          }
        if (fc == 0 && piece + fr < t.valid && col0 < g.N)
          g.y_scales[(first + piece + fr) * ns + col0 / FP8_BLOCK] = (uint8_t)s.byte;
        lds_read_lines<8192>(line, get_at);
        store_lines(piece, col0);
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int j = 2 * h; j < 2 * h + 2; ++j)
#pragma unroll
            for (int q = 0; q < 16; q += 4) {
              const int unit = 2 * ((j & 1) * 4 + (q >> 2));
              lds_write_b64(put_at ^ (unit * 8),
                            u32x2_t{f32x2_to_bf16x2(v[j][q], v[j][q + 1]),
                                    f32x2_to_bf16x2(v[j][q + 2], v[j][q + 3])});
            }
          lds_read_lines<8192>(line, get_at);
          if constexpr (WHOLE) {
            store_lines(piece, 2 * (col0 + 64 * h));
          } else if (col0 + 64 * h + lane < g.N) {
            // rows that do not start on 16 bytes: a column per lane
            bf16_t* const to = (bf16_t*)g.y + (first + piece) * g.N + col0 + 64 * h;
            const int rows = min(32, t.valid - piece);
#pragma unroll 1
            for (int row = 0; row < rows; ++row) {
              const int unit = (lane >> 2) ^ ((row & 7) << 1) ^ ((row >> 3) & 1);
              to[(int64_t)row * g.N + lane] = *reinterpret_cast<const bf16_t*>(
                  smem + Cfg::W_BASE + wfree * Cfg::SLOT + wave * 1024 +
                  (row >> 3) * 8192 + (row & 7) * 128 + unit * 8 + (lane & 3) * 2);
            }
          }
        }
      }
    }
  };

  int round = 0;
  Tile t = tile_at(0);
  if (t.valid == 0) return;
  set_loads(t);
  load_scales(t, 0);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
#pragma unroll
    for (int j = 0; j < 4; ++j) load_a(k, j, k);
#pragma unroll
    for (int j = 0; j < 4; ++j) load_w(k, j, k);
  }
  __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8));             // vmcnt 0
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  for (;;) {
    Tile after = {};
    auto tile_pass = [&](auto na_tag) FP8_INLINE {
      constexpr int NA = decltype(na_tag)::value;
      auto next_scales = [&](int kt) FP8_INLINE {
        if ((kt & 3) == 0) {
#pragma unroll
          for (int i = 0; i < Cfg::TM; ++i) sa[i] = sa_next[i] & scale_mask;
#pragma unroll
          for (int j = 0; j < Cfg::TN; ++j) sw[j] = sw_next[j] & scale_mask;
          if (kt + 4 < t.nk) load_scales(t, kt / 4 + 1);
        } else {
#pragma unroll
          for (int i = 0; i < Cfg::TM; ++i) sa[i] >>= 8;
#pragma unroll
          for (int j = 0; j < Cfg::TN; ++j) sw[j] >>= 8;
        }
      };
      // the last two K tiles load the next tile's first two (without a next one, this
      // one's again, which nobody reads)
      auto advance = [&]() FP8_INLINE {
        after = tile_at(++round);
        set_loads(after.valid != 0 ? after : t);
      };
      if constexpr (NA > 0) first_fragments(aslot, wslot);
      next_scales(0);
      if (t.nk == 2) advance();
      k_tile(na_tag, std::true_type{}, std::false_type{}, t.nk == 2 ? 0 : 2);
      for (int kt = 1; kt < t.nk - 1; ++kt) {
        next_scales(kt);
        if (kt == t.nk - 2) advance();
        k_tile(na_tag, std::false_type{}, std::false_type{}, kt == t.nk - 2 ? 0 : kt + 2);
      }
      next_scales(t.nk - 1);
      if (after.valid != 0) load_scales(after, 0);
      k_tile(na_tag, std::false_type{}, std::true_type{}, 1);
      write_out(t, na_tag);
      // The next first K tile's barrier takes it that STORES stores at least came after
      // the loads that it waits for, or that they have landed.
      if constexpr (NA == 0 || !WHOLE) __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8));
    };
    const int pieces = t.valid > 128 + 32 * wm ? 2 : t.valid > 32 * wm ? 1 : 0;
    if (pieces == 2) tile_pass(std::integral_constant<int, 2>{});
    else if (pieces == 1) tile_pass(std::integral_constant<int, 1>{});
    else tile_pass(std::integral_constant<int, 0>{});
    if (after.valid == 0) break;
    t = after;
  }
  // no direct load may outlive the block
  __builtin_amdgcn_s_waitcnt(0 | (7 << 4) | (15 << 8));
}
// ---------------------------------------------------------------------------
// Tiles of 128 x 128 (TM = 2) and 64 x 128 (TM = 1), for products that have few of the
// 256 x 256 ones: two blocks per CU fill each other's pauses, and a reduction may be split
// over blocks.  4 wavefronts; each has 16 TM rows and all 128 columns as TM x 8 matrix
// tiles of 16 x 16 (v_mfma_scale_f32_16x16x128_f8f6f4, a whole block of 128 at a time):
// pieces of 16 rows 64 apart, so that a last row tile with few rows gives all SIMDs the
// same, and columns that are one block of 128.
//
// K tiles reach LDS as in the kernel above; two token slots and three weight slots.  K
// tile t is multiplied in 8 groups, one per weight fragment j, TM matrix instructions
// each:
//   groups 0 .. 4  read the weight fragments 3 .. 7
//   before group 1 a barrier: everybody has the token fragments of t in registers
//   groups 1 .. 4  token loads of K tile t + 2, into the slot that this freed
//   before group 6 a barrier: everybody has the weight fragments of t, and K tile t + 1
//                  has landed (vmcnt counts in order: the weight loads of t + 2 and the
//                  token loads of t + 2 may be out)
//   groups 6, 7    weight loads of K tile t + 3, into the slot that this freed; the
//                  fragments of t + 1: weights 0 .. 2, and tokens as group 7 is done
//                  with the ones before
// so that token loads have 1.6 and weight loads 2 K tiles' time.  (The same with 4
// wavefronts of 128 x 128 on 256 x 256 tiles, sums in accumulator registers: 2624 against
// 2502 TFLOP/s at 8192^3, but 1803 against 2091 at 16384 rows 1024 -> 4096, where a
// SIMD's one wavefront has nothing to hide a tile's end behind.)
//
// A lane's scales are a dword per row and four K tiles, a byte of it per K tile; the next
// four are requested more than a K tile ahead.  A result is turned round in the weight
// slot that the last K tile has left, each wavefront in the kilobytes that its own loads
// fill afterwards (so no barrier), and leaves in whole lines.
//
// 1024 rows 11080 -> 4096 (256 tiles of 128 x 128, one per CU) take 52 us, 0.60 us per K
// tile, and two blocks on a CU 1.0 together: bound by what the L2s give, 27 bytes per
// clock and CU.
// ---------------------------------------------------------------------------
// TM: 2 or 1
template <int TM_>
struct TileCfg {
  static constexpr int TM = TM_, TN = 8, WM = 4, WAVES = 4, THREADS = 256;
  static constexpr int BM = 16 * TM * WM, BN = 128;
  // of a wavefront per K tile, 8 rows each
  static constexpr int A_LOADS = BM / 8 / WAVES, W_LOADS = BN / 8 / WAVES;
  static constexpr int PIECE_STEP = 1024 * WAVES;   // between its kilobytes of a slot
  static constexpr int A_SLOT = BM * FP8_BLOCK, W_SLOT = BN * FP8_BLOCK;
  static constexpr int W_BASE = 2 * A_SLOT;
  static constexpr int LDS_BYTES = 2 * A_SLOT + 3 * W_SLOT;
};

// ACT: an activation that is neither linear nor relu
template <int TM, int TO, bool ACT>
__global__ __launch_bounds__(256, 2) void fp8_tile_kernel(GemmArgs g, TileGrid grid) {
  using Cfg = TileCfg<TM>;
  constexpr int WM = Cfg::WM, TN = Cfg::TN, BM = Cfg::BM, BN = Cfg::BN;
  constexpr int A_LOADS = Cfg::A_LOADS, W_LOADS = Cfg::W_LOADS;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave;
  const int64_t kp = fp8_row_bytes(g.K), ks = fp8_scale_bytes(g.K);
  // (an only K tile is followed by one of zeros, with scales that are no NaN)
  const bool single = kp == FP8_BLOCK;
  const int k_tiles = single ? 2 : (int)(kp / FP8_BLOCK);
  const uint32_t scale_mask = single ? 0xffu : ~0u;

  // (What is computed from the lane index outside the K loop is computed from a copy
  // that the compiler cannot see through: made once it would be live across the K loop.)
  auto lane_again = [&]() FP8_INLINE {
    int l = lane;
    asm volatile("" : "+v"(l));
    return l;
  };

  // Where a tile's operands lie.  A wavefront's load n fills the rows 8 (wave + WAVES n)
  // .. + 7 of an LDS tile through a buffer that ends with the rows there are: what lies
  // behind is not fetched.  (A row's place is the lanes' part of an address, the K tile's
  // the wavefront's: whichever of them the range check looks at, a row that is there
  // passes it and one that is not fails.)
  struct Operands {
    const uint8_t *a, *w;
    int a_bytes, w_bytes;
  };
  auto operands = [&](const Tile& t) FP8_INLINE {
    Operands o;
    o.a = uniform(g.a + ((int64_t)t.e * g.R + t.row0) * kp + t.k0 * FP8_BLOCK);
    o.w = uniform(g.w + ((int64_t)t.e * g.N + t.col0) * kp + t.k0 * FP8_BLOCK);
    o.a_bytes = t.valid * (int)kp - t.k0 * FP8_BLOCK;
    o.w_bytes = min(BN, g.N - t.col0) * (int)kp - t.k0 * FP8_BLOCK;
    return o;
  };
  constexpr int LOADS = A_LOADS > W_LOADS ? A_LOADS : W_LOADS;
  uint32_t load_at[LOADS];
#pragma unroll
  for (int n = 0; n < LOADS; ++n)
    load_at[n] = (uint32_t)((wave + Cfg::WAVES * n) * 8 + (lane >> 3)) * (uint32_t)kp +
                 ((lane & 7) ^ (lane >> 3)) * 16;
  // where the loads of a K tile read and write
  struct Source {
    const uint8_t* from;
    int bytes, skip, to;
  };
  auto load = [&](const Source& s, int n) FP8_INLINE {
    load_to_lds(s.from, s.bytes, load_at[n], s.skip,
                smem + s.to + wave * 1024 + n * Cfg::PIECE_STEP);
  };

  // scales of this lane's rows: of the K tiles that are multiplied, and the next four
  uint32_t sa[TM], sw[TN], sa_next[TM], sw_next[TN];
  auto load_scales = [&](const Tile& t, int group) FP8_INLINE {
    const int fr = lane_again() & 15;
    const uint8_t* as =
        g.a_scales + ((int64_t)t.e * g.R + t.row0) * ks + t.k0 + 4 * group;
    const uint8_t* ws =
        g.w_scales + ((int64_t)t.e * g.N + t.col0) * ks + t.k0 + 4 * group;
#pragma unroll
    for (int i = 0; i < TM; ++i)
      sa_next[i] = *reinterpret_cast<const uint32_t*>(
          as + (uint32_t)min((i * WM + wm) * 16 + fr, t.valid - 1) * (uint32_t)ks);
#pragma unroll
    for (int j = 0; j < TN; ++j)
      sw_next[j] = *reinterpret_cast<const uint32_t*>(
          ws + (uint32_t)min(16 * j + fr, g.N - 1 - t.col0) * (uint32_t)ks);
  };

  // Chunk c of a row lies at its chunk position c ^ (row % 8); lane l has row l % 16 of a
  // fragment and its chunks l / 16 and l / 16 + 4.  (A read of 64 times 16 bytes is served
  // 256 bytes at a time, lanes 0 .. 3, 12 .. 15, 20 .. 27 together, then 4 .. 11, 16 .. 19,
  // 28 .. 31, and the upper half alike: with this order those lie in different banks.)
  const int frag_at = (lane & 15) * FP8_BLOCK + (((lane >> 4) ^ (lane & 7)) * 16);
  // where the fragments of a slot begin: the lane's first chunk, and its second one
  struct Fragments {
    int lo, hi;
  };
  auto fragments = [&](int slot_at) FP8_INLINE {
    int lo = frag_at + slot_at;
    asm volatile("" : "+v"(lo));  // (one register lives on, not its sums with constants)
    return Fragments{lo, lo ^ 64};
  };
  auto a_fragments = [&](int slot) FP8_INLINE {
    return fragments(slot * Cfg::A_SLOT + wm * 16 * FP8_BLOCK);
  };
  auto w_fragments = [&](int slot) FP8_INLINE {
    return fragments(Cfg::W_BASE + slot * Cfg::W_SLOT);
  };
  auto read_a = [&](const Fragments& f, int i) FP8_INLINE {
    const unsigned char* base = smem + i * WM * 16 * FP8_BLOCK;
    return fp8_fragment(base + f.lo, base + f.hi);
  };
  auto read_w = [&](const Fragments& f, int j) FP8_INLINE {
    const unsigned char* base = smem + j * 16 * FP8_BLOCK;
    return fp8_fragment(base + f.lo, base + f.hi);
  };

  f32x4_t acc[TM][TN];
  i32x8_t fa[TM], fw[4];          // weight fragment j lies in fw[j % 4]
  auto fence = [&]() FP8_INLINE { __builtin_amdgcn_sched_barrier(0); };
  int aslot = 0, wslot = 0;

  // One K tile: number kt of tile t.  NA: how many of the wavefront's TM pieces are
  // multiplied.  FIRST: the sums begin; the weight loads that the tile before left out
  // come here.  LAST: the next tile's fragments are read, and the weight slot is filled,
  // when the result is out.  SCALES: requests the next scales (in LAST: the next tile's).
  // PHASE: the byte of the scales that is kt's, or -1: byte 0, the scales are shifted on.
  // No branches inside: the compiler would move matrix instructions past them, behind
  // the barriers.
  constexpr int STORES =          // of 16 bytes per lane, with half of the pieces
      TO == TO_LINES ? 2 * TM : TO == TO_FP8 ? TM : 0;
  auto k_tile = [&](const Tile& t, const Tile& after, const Operands& here,
                    const Operands& next, int kt, auto na_tag, auto first_tag,
                    auto last_tag, auto scales_tag, auto phase_tag) FP8_INLINE {
    constexpr int PHASE = decltype(phase_tag)::value, BYTE = PHASE < 0 ? 0 : PHASE;
    constexpr int NA = decltype(na_tag)::value;
    constexpr bool FIRST = decltype(first_tag)::value, LAST = decltype(last_tag)::value;
    constexpr bool SCALES = decltype(scales_tag)::value;
    const int wnext = wslot == 2 ? 0 : wslot + 1, anext = aslot ^ 1;
    // the K tiles that are loaded: of this tile, or the next one
    auto a_source = [&](int p) {
      const bool mine = p < t.nk;
      const int at = mine ? p : p - t.nk;
      return Source{mine ? here.a : next.a,
                    single && at == 1 ? 0 : mine ? here.a_bytes : next.a_bytes,
                    at * FP8_BLOCK, aslot * Cfg::A_SLOT};
    };
    auto w_source = [&](int p, int slot) {
      const bool mine = p < t.nk;
      const int at = mine ? p : p - t.nk;
      return Source{mine ? here.w : next.w,
                    single && at == 1 ? 0 : mine ? here.w_bytes : next.w_bytes,
                    at * FP8_BLOCK, Cfg::W_BASE + slot * Cfg::W_SLOT};
    };
    const Fragments w_now = w_fragments(wslot);
    Fragments w_then = {0, 0}, a_then = {0, 0};
    const bool regroup = ((kt + 1) & 3) == 0;
    const f32x4_t none = {};
    Source a_from, w_from;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      if (j == 0 && FIRST) {
        w_from = w_source(2, wnext == 2 ? 0 : wnext + 1);
#pragma unroll
        for (int n = 0; n < W_LOADS; ++n) load(w_from, n);
        fence();
      }
      if (j == 1) {
        fence();
        block_barrier();
        a_from = a_source(kt + 2);
      }
      if (j == 6) {
        fence();
        wait_counts<A_LOADS + W_LOADS + (FIRST ? STORES : 0), true>();
        block_barrier();
        if constexpr (SCALES) {
          if constexpr (LAST) load_scales(after, 0);
          else load_scales(t, min(kt / 4 + 1, (t.nk - 1) / 4));
          fence();
        }
        if (!LAST) {
          w_from = w_source(kt + 3, wslot);
          w_then = w_fragments(wnext);
          a_then = a_fragments(anext);
        }
      }
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        fence();
        if (i < NA)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
              fw[j & 3], fa[i], FIRST ? none : acc[i][j], 0, 0, BYTE, (int)sw[j], BYTE,
              (int)sa[i]);
        fence();
        // what group j does beside piece i
        if (j < 5 && i == 0) fw[(j + 3) & 3] = read_w(w_now, j + 3);
        if (!LAST && i == 0) {
          if (j == 6) fw[0] = read_w(w_then, 0);
          if (j == 7) fw[2] = read_w(w_then, 2);
        }
        if (!LAST && i == TM / 2 && j == 6) fw[1] = read_w(w_then, 1);
        if (!LAST && j == 7 && i < NA) {
          fa[i] = read_a(a_then, i);
          if (PHASE < 0) sa[i] = regroup ? sa_next[i] : sa[i] >> 8;
          else if (PHASE == 3) sa[i] = sa_next[i];
        }
        if (!LAST && i == TM - 1) {
          if (PHASE < 0) sw[j] = regroup ? sw_next[j] : sw[j] >> 8;
          else if (PHASE == 3) sw[j] = sw_next[j];
        }
        if (j >= 1 && j <= 4) {
          constexpr int PER = A_LOADS / 4 > 0 ? A_LOADS / 4 : 1;
#pragma unroll
          for (int n = i * PER / TM; n < (i + 1) * PER / TM; ++n)
            if ((j - 1) * PER + n < A_LOADS) load(a_from, (j - 1) * PER + n);
        }
        if (!LAST && j >= 6) {
          constexpr int PER = W_LOADS / 2;
          static_assert(W_LOADS % 2 == 0, "dealt out over two groups");
#pragma unroll
          for (int n = i * PER / TM; n < (i + 1) * PER / TM; ++n)
            load(w_from, (j - 6) * PER + n);
        }
      }
    }
    fence();
    aslot = anext;
    wslot = wnext;
  };

  // The result of a tile: 32 rows at a time are turned round and leave 16 bytes per lane.
  // Lane l has row l % 16 and the columns 16 j + 4 (l / 16) .. of a piece.  The stores of
  // whole lines go through a buffer that ends with the tile's rows, so that they leave in
  // any case and the next tile's first wait can count on them.  (Rows that are not there
  // count as none before they are multiplied: up to -59 times a row passes 32 bits.)
  auto write_out = [&](const Tile& t, auto na_tag) FP8_INLINE {
    constexpr int NA = decltype(na_tag)::value;
    const int wfree = wslot == 0 ? 2 : wslot - 1;       // of the last K tile
    const int lane = lane_again(), fr = lane & 15, fc = lane >> 4;
    unsigned char* const free_slot = smem + Cfg::W_BASE + wfree * Cfg::W_SLOT + wave * 1024;
    const uint32_t stage = (uint32_t)(size_t)(lds_void_t*)free_slot;
    const int col0 = t.col0;
    const int64_t first = (int64_t)t.e * g.R + t.row0;
    const int64_t ns = fp8_scale_bytes(g.N);
    auto row_of = [&](int i) { return (i * WM + wm) * 16; };
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      if constexpr (ACT) {
        const Fp8Act act(g.activation);
        int columns = g.N - col0 - 4 * fc;
        asm volatile("" : "+v"(columns));      // (not masks kept for the next piece)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float u = act(acc[i][j][q]);
            acc[i][j][q] = 16 * j + q < columns ? u : 0.f;
          }
      } else if (TO != TO_PARTS && g.activation == MESH_MOE_ACT_RELU) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) acc[i][j][q] = fp8_relu(acc[i][j][q]);
      }
    }
    if constexpr (TO == TO_PARTS) {
      // (rows of whole 128s of columns, so that every piece of 16 bytes is there)
      const int64_t np = fp8_row_bytes(g.N);
      float* const parts = (float*)g.y + ((int64_t)t.part * g.E * g.R + first) * np + col0;
      if (col0 < g.N)
#pragma unroll
        for (int i = 0; i < NA; ++i)
          if (row_of(i) + fr < t.valid)
#pragma unroll
            for (int j = 0; j < TN; ++j)
              *reinterpret_cast<f32x4_t*>(parts + (int64_t)(row_of(i) + fr) * np + 16 * j +
                                          4 * fc) = acc[i][j];
      return;
    }
    const int row_bytes = TO == TO_FP8 ? (int)fp8_row_bytes(g.N) : 2 * g.N;
    u32x4_t line[4];
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int64_t row = first + row_of(i);
      const int rows = t.valid - row_of(i);
      if constexpr (TO == TO_FP8) {
        // Rows of 128 bytes, 8 to a kilobyte; chunk j of row r lies at j ^ (r % 8).
        // (columns past N are zeros: the weights' buffer ends there)
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) top = max(top, magnitude_bits(acc[i][j][q]));
        top = max(top, (uint32_t)__shfl_xor((int)top, 16));
        top = max(top, (uint32_t)__shfl_xor((int)top, 32));
        const Fp8Scale s = fp8_scale(top);
        const uint32_t put_at = stage + ((i & 1) * 2 + (fr >> 3)) * Cfg::PIECE_STEP + (fr & 7) * 128 +
                                (fr & 7) * 16 + fc * 4;
#pragma unroll
        for (int j = 0; j < TN; ++j)
          lds_write_b32(put_at ^ (j * 16),
                        fp8_pack4(acc[i][j][0] * s.factor, acc[i][j][1] * s.factor,
                                  acc[i][j][2] * s.factor, acc[i][j][3] * s.factor));
        if (fc == 0 && fr < rows && col0 < g.N)
          g.y_scales[(row + fr) * ns + col0 / FP8_BLOCK] = (uint8_t)s.byte;
        if ((i & 1) == 0 && i + 1 < NA) continue;
        const int lr = lane >> 3, lc = lane & 7;
        lds_read_lines<Cfg::PIECE_STEP>(line, stage + lr * 128 + ((lc ^ lr) * 16));
        const uint32_t at = (uint32_t)(lr * row_bytes + 16 * lc);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          // lines 0, 1 are rows 0 .. 15 of the even piece, 2, 3 of the odd one
          const int p = (i & ~1) + (n >> 1), left = t.valid - row_of(p) - 8 * (n & 1);
          if (p >= NA) continue;
          store_line(line[n],
                     (uint8_t*)g.y + (first + row_of(p) + 8 * (n & 1)) * row_bytes + col0,
                     col0 < g.N ? max(min(left, 8), 0) * row_bytes - col0 : 0, at);
        }
      } else {
        // Rows of 256 bytes, 4 to a kilobyte; the 8 bytes of unit u (4 columns) of row r
        // lie at u ^ 4 (r % 8).
        const uint32_t put_at = stage + (fr >> 2) * Cfg::PIECE_STEP + (fr & 3) * 256 +
                                ((fc ^ ((fr & 7) << 2)) * 8);
#pragma unroll
        for (int j = 0; j < TN; ++j)
          lds_write_b64(put_at ^ (j * 32),
                        u32x2_t{f32x2_to_bf16x2(acc[i][j][0], acc[i][j][1]),
                                f32x2_to_bf16x2(acc[i][j][2], acc[i][j][3])});
        const int lr = lane >> 4, lc = lane & 15;
        if constexpr (TO == TO_LINES) {
          // line n: rows 4 n .. + 3
          uint32_t get_at = stage + lr * 256;
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            // (rows 4 n + lr and 8 + 4 n + lr have the same units)
            const uint32_t from =
                get_at + n * Cfg::PIECE_STEP + ((lc ^ (((4 * n + lr) & 7) << 1)) * 16);
            asm volatile("ds_read_b128 %0, %2\n\t"
                         "ds_read_b128 %1, %2 offset:%3\n\t"
                         "s_waitcnt lgkmcnt(0)"
                         : "=&v"(line[n]), "=&v"(line[n + 2])
                         : "v"(from), "n"(2 * Cfg::PIECE_STEP) : "memory");
          }
          const int col = 2 * col0 + 16 * lc;
          const uint32_t at = col < row_bytes ? (uint32_t)(lr * row_bytes + 16 * lc)
                                              : 0x80000000u;      // (past every buffer)
#pragma unroll
          for (int n = 0; n < 4; ++n)
            store_line(line[n], (uint8_t*)g.y + (row + 4 * n) * row_bytes + 2 * col0,
                       max(min(rows - 4 * n, 4), 0) * row_bytes - 2 * col0, at);
        } else {
          // rows that do not start on 16 bytes: a column per lane
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          const int some = min(16, rows);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int col = col0 + 64 * h + lane, unit = 16 * h + (lane >> 2);
            if (col >= g.N) continue;
            bf16_t* const to = (bf16_t*)g.y + row * g.N + col;
#pragma unroll 4
            for (int r = 0; r < some; ++r)
              to[(int64_t)r * g.N] = *reinterpret_cast<const bf16_t*>(
                  free_slot + (r >> 2) * Cfg::PIECE_STEP + (r & 3) * 256 +
                  (unit ^ ((r & 7) << 2)) * 8 + (lane & 3) * 2);
          }
        }
      }
    }
  };

  int round = 0;
  auto tile_at = [&](int round) FP8_INLINE {
    return find_tile<BM, BN, TO == TO_PARTS>(g, grid, k_tiles, tile_number(round),
                                             lane_again());
  };
  Tile t = tile_at(0);
  if (t.valid == 0) return;
  Operands here = operands(t);
  load_scales(t, 0);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const bool zeros = single && k == 1;
    const Source as = {here.a, zeros ? 0 : here.a_bytes, k * FP8_BLOCK, k * Cfg::A_SLOT};
    const Source ws = {here.w, zeros ? 0 : here.w_bytes, k * FP8_BLOCK,
                       Cfg::W_BASE + k * Cfg::W_SLOT};
#pragma unroll
    for (int n = 0; n < A_LOADS; ++n) load(as, n);
#pragma unroll
    for (int n = 0; n < W_LOADS; ++n) load(ws, n);
  }
  wait_counts<0, false>();
  block_barrier();
  for (;;) {
    Tile after;
    Operands next;
    auto tile_pass = [&](auto na_tag) FP8_INLINE {
      constexpr int NA = decltype(na_tag)::value;
      const std::true_type yes{};
      const std::false_type no{};
      const Fragments a_first = a_fragments(aslot), w_first = w_fragments(wslot);
#pragma unroll
      for (int i = 0; i < NA; ++i) fa[i] = read_a(a_first, i);
#pragma unroll
      for (int j = 0; j < 3; ++j) fw[j] = read_w(w_first, j);
#pragma unroll
      for (int i = 0; i < TM; ++i) sa[i] = sa_next[i] & scale_mask;
#pragma unroll
      for (int j = 0; j < TN; ++j) sw[j] = sw_next[j] & scale_mask;
      // (without a next tile its loads fetch this one again, which nobody reads)
      after = tile_at(++round);
      next = operands(after.valid != 0 ? after : t);
      const std::integral_constant<int, -1> any{};
      k_tile(t, after, here, next, 0, na_tag, yes, no, yes, any);
      int kt = 1;
      for (; kt < min(4, t.nk - 1); ++kt)
        k_tile(t, after, here, next, kt, na_tag, no, no, no, any);
      for (; kt + 3 < t.nk - 1; kt += 4) {
        k_tile(t, after, here, next, kt, na_tag, no, no, yes,
               std::integral_constant<int, 0>{});
        k_tile(t, after, here, next, kt + 1, na_tag, no, no, no,
               std::integral_constant<int, 1>{});
        k_tile(t, after, here, next, kt + 2, na_tag, no, no, no,
               std::integral_constant<int, 2>{});
        k_tile(t, after, here, next, kt + 3, na_tag, no, no, no,
               std::integral_constant<int, 3>{});
      }
      // (what is left of the last four: their scales are there)
      for (; kt < t.nk - 1; ++kt)
        k_tile(t, after, here, next, kt, na_tag, no, no, no, any);
      k_tile(t, after.valid != 0 ? after : t, here, next, t.nk - 1, na_tag, no, yes, yes,
             any);
      write_out(t, na_tag);
      // The next first K tile's barrier takes it that STORES stores at least came after
      // the loads that it waits for, or that they have landed.
      if constexpr (STORES == 0) wait_counts<0, false>();
    };
    if constexpr (TM > 1) {
      if (t.valid <= BM / 2) tile_pass(std::integral_constant<int, TM / 2>{});
      else tile_pass(std::integral_constant<int, TM>{});
    } else {
      tile_pass(std::integral_constant<int, TM>{});
    }
    if (after.valid == 0) break;
    t = after;
    here = next;
  }
  // no direct load may outlive the block
  wait_counts<0, false>();
}
#undef FP8_INLINE

// The parts of a reduction that was split: added up in order, activation, rounding.  16
// lanes have a block of 128 columns of a row.
template <bool EIGHT>
__global__ __launch_bounds__(256) void fp8_parts_kernel(const float* __restrict__ parts,
                                                        GemmArgs g, int split) {
  const int64_t np = fp8_row_bytes(g.N), pieces = np / 8;
  const int64_t total = (int64_t)g.E * g.R * pieces;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;         // (whole rows of 16 lanes)
  const int64_t row = i / pieces;
  const int col = (int)(i - row * pieces) * 8;
  const int e = (int)(row / g.R);
  if (row - (int64_t)e * g.R >= live_rows(g.row_count, e, g.R)) return;
  float v[8] = {};
  const float* from = parts + row * np + col;
#pragma unroll 4
  for (int p = 0; p < split; ++p, from += (int64_t)g.E * g.R * np) {
    const float4 lo = reinterpret_cast<const float4*>(from)[0];
    const float4 hi = reinterpret_cast<const float4*>(from)[1];
    v[0] += lo.x; v[1] += lo.y; v[2] += lo.z; v[3] += lo.w;
    v[4] += hi.x; v[5] += hi.y; v[6] += hi.z; v[7] += hi.w;
  }
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    v[j] = col + j < g.N ? fp8_activation(v[j], g.activation) : 0.f;
    top = max(top, magnitude_bits(v[j]));
  }
  if constexpr (EIGHT) {
    const Fp8Scale s = fp8_scale(max16(top));
    *reinterpret_cast<uint2*>((uint8_t*)g.y + row * np + col) =
        make_uint2(fp8_pack4(v[0] * s.factor, v[1] * s.factor, v[2] * s.factor,
                             v[3] * s.factor),
                   fp8_pack4(v[4] * s.factor, v[5] * s.factor, v[6] * s.factor,
                             v[7] * s.factor));
    if (col % FP8_BLOCK == 0)
      g.y_scales[row * fp8_scale_bytes(g.N) + col / FP8_BLOCK] = (uint8_t)s.byte;
  } else {
    bf16_t* to = (bf16_t*)g.y + row * g.N + col;
    if (g.N % 8 == 0 && (uintptr_t)g.y % 16 == 0) {
      if (col < g.N) *reinterpret_cast<uint4*>(to) = pack16(v, bf16_t());
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (col + j < g.N) to[j] = f32_to_bf16(v[j]);
    }
  }
}

// How a product is run: the kind, and over how many blocks the reduction is split, whose
// estimated time is the least.  The estimates are microseconds on a card with 256 CUs,
// fitted to 94 products between 1 and 64 experts, 1 and 8192 rows, 128 and 16384 columns
// and values; what they choose is 1.1 % slower than the best of all choices in the mean
// (15 % at worst).  Some of what they weigh, measured:
//   rows x K -> N           few rows   64 x 128        128 x 128       256 x 256
//   1, 4096 -> 16384           14.1       21.4
//   16, 4096 -> 1024            6.6       19.3, 10.7 in 8 parts
//   32 x (5, 4096 -> 1024)     29.1       25.9
//   64, 4096 -> 4096           16.0       19.7, 13.4 in 4    20.3
//   512, 4096 -> 4096                     22.6               25.8       46.5
//   2048, 2048 -> 2048                    16.8               14.7       24.6
//   1024, 11080 -> 4096                   74.1               53.7       108.5
//   4096, 4096 -> 4096                    129.9              85.7       60.8
enum ProductKind { ONE_BLOCK, FEW_ROWS, TILES_64, TILES_128, TILES_256 };
struct Plan {
  ProductKind kind = ONE_BLOCK;
  int split = 1;                  // parts of the reduction (TILES_64, TILES_128)
  size_t workspace = 0;           // of the parts, or a few rows' sums
};

static Plan plan_product(int E, int R, int K, int N, bool eight_bit, bool counted) {
  Plan p;
  // (a tile's operand rows and 8 rows of its result are addressed in 31 bits)
  if (K > 1 << 22 || N > 1 << 26) return p;
  const bool single = K <= FP8_BLOCK;
  const int nk = single ? 2 : (int)(fp8_row_bytes(K) / FP8_BLOCK);
  const int64_t np = fp8_row_bytes(N);
  const double weights = (double)E * N * nk * FP8_BLOCK / 1e6;        // MB
  auto over = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  double best = 1e300;
  auto offer = [&](ProductKind kind, int split, double time) {
    if (time < best) {
      best = time;
      p.kind = kind;
      p.split = split;
    }
  };
  if (single) {
    // nothing to deal out over wavefronts, nor to be overlapped with
    const int rows = R <= 16 ? 16 : R <= 32 ? 32 : 64;
    const int64_t blocks = over(N, 128) * over(R, rows) * E;
    offer(ONE_BLOCK, 1, 3.2 + over(blocks, 256) * (rows == 16 ? 1.0 : rows == 32 ? 1.6 : 4.2));
  } else if (R <= 128) {
    // a wavefront's run is nk / 8 blocks: bound by the weights, by the blocks' own reads,
    // or by the time to memory
    const bool one = R <= 16;
    const double blocks = (double)E * over(N, 16) * over(R, one ? 16 : 32);
    const double read = weights / 5.8, run = nk / 8.0 * (one ? 0.56 : 1.5);
    const double work = blocks / 256 * (1.0 + nk / 8.0 * (one ? 0.19 : 1.3));
    offer(FEW_ROWS, 1, 3.2 + (eight_bit ? 1.7 : 0.0) +
                           (read > run ? (read > work ? read : work)
                                       : (run > work ? run : work)));
  }
  // tiles: time per K tile of a block alone on its CU, and of two
  struct { ProductKind kind; int bm; double start, one, two, end; } const kinds[] = {
      {TILES_64, 64, 2.5, 0.67, 0.96, 0.6}, {TILES_128, 128, 4.6, 0.67, 1.0, 0.7}};
  for (const auto& t : kinds)
    for (const int split : {1, 2, 3, 4, 6, 8, 12, 16}) {
      const int64_t groups = over(nk, 4);
      // (parts are whole groups of 4 K tiles, two K tiles at least; with row counts the
      // number of tiles is not known)
      if (split > 1 && (counted || split > groups ||
                        nk - 4 * (groups * (split - 1) / split) < 2))
        continue;
      const int64_t units = over(R, t.bm) * over(N, 128) * E * split;
      const int64_t whole = 4 * over(groups, split), k_tiles = whole < nk ? whole : nk;
      double time = t.start + (units <= 256 ? t.one * k_tiles
                                            : over(units, 512) * (t.two * k_tiles + t.end));
      if (time < 4.8 + weights / 6.9) time = 4.8 + weights / 6.9;
      if (split > 1) time += 3.5 + (double)split * E * R * np * 8 / 4.5e6;
      offer(t.kind, split, time);
    }
  const int64_t units = over(R, 256) * over(N, 256) * E;
  double time = 3.0 + over(units, 256) * (1.25 * nk + 1.8);
  if (time < 4.8 + weights / 6.9) time = 4.8 + weights / 6.9;
  offer(TILES_256, 1, time);
  if (p.split > 1 || (p.kind == FEW_ROWS && eight_bit))
    p.workspace = (size_t)p.split * E * R * np * sizeof(float);
  return p;
}

// The grid of a launch over tiles of `bm` x `bn`, `per_cu` blocks a CU at most.
static int tile_grid(const GemmArgs& g, int bm, int bn, int split, int per_cu,
                     TileGrid* grid, unsigned* blocks) {
  grid->tiles_m = (int)(((int64_t)g.R + bm - 1) / bm);
  grid->tiles_n = (int)(((int64_t)g.N + bn - 1) / bn);
  grid->split = split;
  // (numbers of tiles, those past the end too, are int)
  const int64_t one = (int64_t)grid->tiles_m * grid->tiles_n;
  MOE_REQUIRE(one <= 1 << 30 && one * g.E <= 1 << 30 && one * g.E * split <= 1 << 30,
              MESH_MOE_E_UNSUPPORTED, "fp8_expert_linear: too many tiles (E=%d R=%d N=%d)",
              g.E, g.R, g.N);
  grid->tiles = (int)(one * g.E * split);
  const int cus = compute_units();
  if (cus == 0) return MESH_MOE_E_HIP;
  const int most = cus / 8 * 8 * per_cu, want = (grid->tiles + 7) / 8 * 8;
  *blocks = (unsigned)(want < most ? want : most);
  return 0;
}
static bool is_act(const GemmArgs& g) {
  return g.activation != MESH_MOE_ACT_LINEAR && g.activation != MESH_MOE_ACT_RELU;
}
static bool whole_lines(const GemmArgs& g) {
  return g.N % 8 == 0 && (uintptr_t)g.y % 16 == 0;
}

template <bool EIGHT, bool WHOLE>
static int launch_256(const GemmArgs& g, hipStream_t st) {
  TileGrid grid;
  unsigned blocks;
  const int rc = tile_grid(g, BigCfg::BM, BigCfg::BN, 1, 1, &grid, &blocks);
  if (rc != 0) return rc;
  auto kernel = is_act(g) ? fp8_tile256_kernel<EIGHT, true, WHOLE>
                          : fp8_tile256_kernel<EIGHT, false, WHOLE>;
  MOE_ALLOW_LDS(kernel, BigCfg::LDS_BYTES);
  kernel<<<blocks, BigCfg::THREADS, BigCfg::LDS_BYTES, st>>>(g, grid);
  MOE_CHECK_LAUNCH("fp8_expert_linear");
  return 0;
}

template <int TM, int TO>
static int launch_tiles(const GemmArgs& g, int split, hipStream_t st) {
  using Cfg = TileCfg<TM>;
  TileGrid grid;
  unsigned blocks;
  const int rc = tile_grid(g, Cfg::BM, Cfg::BN, split, 2, &grid, &blocks);
  if (rc != 0) return rc;
  auto kernel = TO != TO_PARTS && is_act(g) ? fp8_tile_kernel<TM, TO, TO != TO_PARTS>
                                            : fp8_tile_kernel<TM, TO, false>;
  MOE_ALLOW_LDS(kernel, Cfg::LDS_BYTES);
  kernel<<<blocks, Cfg::THREADS, Cfg::LDS_BYTES, st>>>(g, grid);
  MOE_CHECK_LAUNCH("fp8_expert_linear");
  return 0;
}

static int add_parts(const GemmArgs& g, const float* parts, int split, hipStream_t st) {
  const int64_t threads = (int64_t)g.E * g.R * (fp8_row_bytes(g.N) / 8);
  const int64_t blocks = (threads + 255) / 256;
  MOE_REQUIRE(blocks <= MAX_THREADS / 256, MESH_MOE_E_UNSUPPORTED,
              "fp8_expert_linear: too many elements (E=%d R=%d N=%d)", g.E, g.R, g.N);
  if (g.y_scales)
    fp8_parts_kernel<true><<<(unsigned)blocks, 256, 0, st>>>(parts, g, split);
  else
    fp8_parts_kernel<false><<<(unsigned)blocks, 256, 0, st>>>(parts, g, split);
  MOE_CHECK_LAUNCH("fp8_expert_linear");
  return 0;
}

template <int TM>
static int run_tiles(const GemmArgs& g, int split, void* workspace, hipStream_t st) {
  if (split > 1) {
    GemmArgs parts = g;
    parts.y = workspace;
    const int rc = launch_tiles<TM, TO_PARTS>(parts, split, st);
    if (rc != 0) return rc;
    return add_parts(g, (const float*)workspace, split, st);
  }
  if (g.y_scales) return launch_tiles<TM, TO_FP8>(g, 1, st);
  return whole_lines(g) ? launch_tiles<TM, TO_LINES>(g, 1, st)
                        : launch_tiles<TM, TO_BF16>(g, 1, st);
}

template <int TM, int CW, typename TO>
static int launch_few_rows(const GemmArgs& g, hipStream_t st) {
  const int64_t tiles_m = ((int64_t)g.R + 16 * TM - 1) / (16 * TM);
  const int64_t tiles_n = ((int64_t)g.N + 16 * CW - 1) / (16 * CW);
  MOE_REQUIRE(tiles_m * tiles_n <= MAX_THREADS / 512 / g.E,
              MESH_MOE_E_UNSUPPORTED, "fp8_expert_linear: too many tiles (E=%d R=%d N=%d)",
              g.E, g.R, g.N);
  fp8_few_rows_kernel<TM, CW, TO>
      <<<(unsigned)(tiles_m * tiles_n * g.E), 512, 0, st>>>(g, (int)tiles_m, (int)tiles_n);
  MOE_CHECK_LAUNCH("fp8_expert_linear");
  return 0;
}
// a block of 128, and nothing to deal out over wavefronts
template <int TM>
static int run_one_block(const GemmArgs& g, hipStream_t st) {
  return g.y_scales ? launch_few_rows<TM, 8, uint8_t>(g, st)
                    : launch_few_rows<TM, 8, bf16_t>(g, st);
}
static int run_product(const GemmArgs& g, void* workspace, hipStream_t st) {
  const Plan p = plan_product(g.E, g.R, g.K, g.N, g.y_scales != nullptr,
                              g.row_count != nullptr);
  switch (p.kind) {
    case TILES_256:
      if (g.y_scales) return launch_256<true, true>(g, st);
      return whole_lines(g) ? launch_256<false, true>(g, st)
                            : launch_256<false, false>(g, st);
    case TILES_128: return run_tiles<2>(g, p.split, workspace, st);
    case TILES_64: return run_tiles<1>(g, p.split, workspace, st);
    default: break;
  }
  if (p.kind == ONE_BLOCK)
    return g.R <= 16 ? run_one_block<1>(g, st)
                     : g.R <= 32 ? run_one_block<2>(g, st) : run_one_block<4>(g, st);
  if (g.y_scales == nullptr)
    return g.R <= 16 ? launch_few_rows<1, 1, bf16_t>(g, st)
                     : launch_few_rows<2, 1, bf16_t>(g, st);
  GemmArgs f = g;
  f.y = workspace;
  const int rc = g.R <= 16 ? launch_few_rows<1, 1, float>(f, st)
                           : launch_few_rows<2, 1, float>(f, st);
  return rc != 0 ? rc : add_parts(g, (const float*)workspace, 1, st);
}

// workspace pieces start on 256 bytes
static size_t piece(size_t bytes) { return (bytes + 255) / 256 * 256; }

}  // namespace mesh_moe

using namespace mesh_moe;

// (a row of an operand, and what a product's sizes are counted in, stay below 2^31)
static bool fp8_sizes(int E, int R, int K, int N) {
  return E >= 1 && R >= 1 && K >= 1 && N >= 1 && R <= 0x7fffff00 && K <= 0x7fffff00 &&
         N <= 0x7fffff00;
}

extern "C" int mesh_moe_fp8_expert_linear_exact(int E, int R, int K, int N,
                                                int eight_bit, int counted) {
  if (!fp8_sizes(E, R, K, N)) return 0;
  const ProductKind kind =
      plan_product(E, R, K, N, eight_bit != 0, counted != 0).kind;
  return kind == ONE_BLOCK || kind == FEW_ROWS ? 1 : 0;
}

extern "C" size_t mesh_moe_fp8_expert_linear_workspace_bytes(int E, int R, int K, int N,
                                                             int eight_bit) {
  if (!fp8_sizes(E, R, K, N)) return 0;
  // (of both kinds of calls)
  const size_t whole = plan_product(E, R, K, N, eight_bit != 0, false).workspace;
  const size_t counted = plan_product(E, R, K, N, eight_bit != 0, true).workspace;
  return whole > counted ? whole : counted;
}

extern "C" int mesh_moe_fp8_expert_linear(const void* a_values, const uint8_t* a_scales,
                                          const void* w_values, const uint8_t* w_scales,
                                          const int32_t* row_count, void* y,
                                          uint8_t* y_scales, int E, int R, int K, int N,
                                          int activation, void* workspace,
                                          size_t workspace_bytes, void* stream) {
  MOE_REQUIRE(a_values && a_scales && w_values && w_scales && y, MESH_MOE_E_ARG,
              "fp8_expert_linear: null pointer");
  MOE_REQUIRE(fp8_sizes(E, R, K, N), MESH_MOE_E_ARG,
              "fp8_expert_linear: bad sizes E=%d R=%d K=%d N=%d", E, R, K, N);
  MOE_REQUIRE(activation >= MESH_MOE_ACT_LINEAR && activation <= MESH_MOE_ACT_SWISH,
              MESH_MOE_E_ARG, "fp8_expert_linear: bad activation %d", activation);
  MOE_REQUIRE(((uintptr_t)a_values | (uintptr_t)w_values | (uintptr_t)workspace |
               (y_scales ? (uintptr_t)y : 0)) % 16 == 0 && (uintptr_t)y % 2 == 0 &&
                  ((uintptr_t)a_scales | (uintptr_t)w_scales | (uintptr_t)y_scales) %
                          4 == 0,
              MESH_MOE_E_UNSUPPORTED,
              "fp8_expert_linear: 8-bit values need to lie on 16 bytes, scales on 4");
  const size_t need =
      plan_product(E, R, K, N, y_scales != nullptr, row_count != nullptr).workspace;
  MOE_REQUIRE(workspace_bytes >= need && (workspace || need == 0), MESH_MOE_E_ARG,
              "fp8_expert_linear: workspace too small (%zu of %zu)", workspace_bytes,
              need);
  const GemmArgs g = {(const uint8_t*)a_values, a_scales, (const uint8_t*)w_values,
                      w_scales, row_count, y, y_scales, E, R, K, N, activation, nullptr};
  return run_product(g, workspace, (hipStream_t)stream);
}

namespace mesh_moe {

// where the parts of the gradients' workspace lie
struct BackwardParts {
  size_t rows, row_scales, columns, column_scales, products, bytes;
};
static BackwardParts backward_parts(int E, int R, int K, int N, bool want_da) {
  BackwardParts p;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += piece(bytes);
    return here;
  };
  p.rows = take(want_da ? (size_t)E * R * fp8_row_bytes(N) : 0);
  p.row_scales = take(want_da ? (size_t)E * R * fp8_scale_bytes(N) : 0);
  p.columns = take((size_t)E * N * fp8_row_bytes(R));
  p.column_scales = take((size_t)E * N * fp8_scale_bytes(R));
  const size_t dw = plan_product(E, K, R, N, false, false).workspace;
  // (bf16 results: with row counts there are no parts, and no workspace)
  const size_t da = want_da ? plan_product(E, R, N, K, false, false).workspace : 0;
  p.products = take(dw > da ? dw : da);
  p.bytes = at;
  return p;
}

}  // namespace mesh_moe

extern "C" size_t mesh_moe_fp8_expert_linear_backward_workspace_bytes(int E, int R,
                                                                      int K, int N,
                                                                      int want_da) {
  if (!fp8_sizes(E, R, K, N)) return 0;
  return backward_parts(E, R, K, N, want_da != 0).bytes;
}

extern "C" int mesh_moe_fp8_expert_linear_backward(
    const void* a_column_values, const uint8_t* a_column_scales, const void* dy,
    const void* relu_mask, const int32_t* row_count, const void* w_row_values,
    const uint8_t* w_row_scales, void* da, void* dw, int E, int R, int K, int N,
    int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  MOE_REQUIRE(a_column_values && a_column_scales && dy && dw && workspace &&
                  (da == nullptr || (w_row_values && w_row_scales)),
              MESH_MOE_E_ARG, "fp8_expert_linear_backward: null pointer");
  MOE_REQUIRE(fp8_sizes(E, R, K, N), MESH_MOE_E_ARG,
              "fp8_expert_linear_backward: bad sizes E=%d R=%d K=%d N=%d", E, R, K, N);
  MOE_REQUIRE(valid_dtype(dtype), MESH_MOE_E_ARG,
              "fp8_expert_linear_backward: bad dtype %d", dtype);
  MOE_REQUIRE(((uintptr_t)a_column_values | (uintptr_t)w_row_values |
               (uintptr_t)workspace) % 16 == 0 &&
                  ((uintptr_t)a_column_scales | (uintptr_t)w_row_scales) % 4 == 0 &&
                  ((uintptr_t)dy | (uintptr_t)relu_mask) % dtype_size(dtype) == 0 &&
                  ((uintptr_t)da | (uintptr_t)dw) % 2 == 0,
              MESH_MOE_E_UNSUPPORTED,
              "fp8_expert_linear_backward: 8-bit values need to lie on 16 bytes, scales "
              "on 4");
  const BackwardParts p = backward_parts(E, R, K, N, da != nullptr);
  MOE_REQUIRE(workspace_bytes >= p.bytes, MESH_MOE_E_ARG,
              "fp8_expert_linear_backward: workspace too small (%zu of %zu)",
              workspace_bytes, p.bytes);
  hipStream_t st = (hipStream_t)stream;
  uint8_t* ws = (uint8_t*)workspace;
  uint8_t* rows = da ? ws + p.rows : nullptr;
  // (tiles read the blocks of rows that an expert has, other kinds and parts all of them;
  // for half of 32 x 640 rows x 1024 the pass takes 26 us instead of 28)
  const Plan dw_plan = plan_product(E, K, R, N, false, false);
  const bool only_counted = row_count != nullptr && dw_plan.kind >= TILES_64 &&
                            dw_plan.split == 1;
  int rc = fp8_quantize(dy, relu_mask, row_count, rows, da ? ws + p.row_scales : nullptr,
                        ws + p.columns, ws + p.column_scales, E, R, N, dtype,
                        only_counted, st);
  if (rc != 0) return rc;
  const GemmArgs weights = {(const uint8_t*)a_column_values, a_column_scales,
                            ws + p.columns, ws + p.column_scales, nullptr, dw, nullptr,
                            E, K, R, N, MESH_MOE_ACT_LINEAR, row_count};
  rc = run_product(weights, ws + p.products, st);
  if (rc != 0 || da == nullptr) return rc;
  const GemmArgs input = {rows, ws + p.row_scales, (const uint8_t*)w_row_values,
                          w_row_scales, row_count, da, nullptr, E, R, N, K,
                          MESH_MOE_ACT_LINEAR, nullptr};
  return run_product(input, ws + p.products, st);
}
