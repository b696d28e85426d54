// Products of 8-bit operands (see mesh_moe_fp8.h) on the scaled matrix instructions.
//
// v_mfma_scale_f32_32x32x64_f8f6f4 takes 64 values of a row per step and a power of two
// for every 32 of them, from a byte of a register that each lane has for its row: a
// block of 128 is two steps with the same byte, and the scales cost no instruction of
// their own.  Which 32 values of a block a lane's half of the wavefront has in a step is
// free, as long as both operands agree: here lane l has row l % 32 and bytes 64 (l / 32)
// + 32 s .. + 31 of a block in step s.  The weights are the first operand and the
// tokens the second, so that a lane ends up with one token's row: 4 neighbouring
// columns per group of 4 accumulators.
#include "fp8.h"

#include <type_traits>

namespace mesh_moe {

typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16_t fp8_mfma(i32x8_t w, i32x8_t a, f32x16_t c,
                                             uint32_t w_scale, uint32_t a_scale) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w, a, c, 0, 0, 0, (int)w_scale,
                                                         0, (int)a_scale);
}

// The activations as the products apply them to their float32 sums; NaN stays NaN.  All
// but relu are (n0 + n1 v) / (1 + exp(v (k1 + k3 v^2))) + off with constants of the
// activation: 0.5 (1 + tanh u) = 1 / (1 + exp(-2 u)), tanh v = 2 / (1 + exp(-2 v)) - 1,
// the latter by its series where the difference would lose bits.  The hardware's
// exponential and reciprocal are off by 2^-21 or so (relative, for arguments that
// matter), far below the rounding of the result.
struct Fp8Act {
  float n0, n1, k1, k3, off, near;
  __device__ __forceinline__ explicit Fp8Act(int act) {
    const bool tanh = act == MESH_MOE_ACT_TANH, gelu = act == MESH_MOE_ACT_GELU;
    n0 = tanh ? 2.f : act == MESH_MOE_ACT_SIGMOID ? 1.f : 0.f;
    n1 = gelu || act == MESH_MOE_ACT_SWISH ? 1.f : 0.f;
    k1 = gelu ? -1.5957691216057308f : tanh ? -2.f : -1.f;
    k3 = gelu ? -1.5957691216057308f * 0.044715f : 0.f;
    off = tanh ? -1.f : 0.f;
    near = tanh ? 4e-4f : 0.f;
  }
  __device__ __forceinline__ float operator()(float v) const {
    const float v2 = v * v;
    const float y = (n0 + n1 * v) *
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
};

// ---------------------------------------------------------------------------
// 32 rows x 32 columns per block, the reduction dealt out over WAVES wavefronts, whose
// sums meet in LDS.  Operands come straight from memory: a lane reads 64 bytes of its
// row per block of 128.
// ---------------------------------------------------------------------------
template <int WAVES, typename TO>
__global__ __launch_bounds__(WAVES * 64) void fp8_few_rows_kernel(GemmArgs g) {
  __shared__ float parts[WAVES][16][64];
  const int e = blockIdx.z, row0 = blockIdx.y * 32, col0 = blockIdx.x * 32;
  const int live = live_rows(g.row_count, e, g.R);
  if (row0 >= live) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int at = lane & 31, half = lane >> 5;
  const int64_t kp = fp8_row_bytes(g.K), ks = fp8_scale_bytes(g.K);
  const int64_t a_row = (int64_t)e * g.R + min(row0 + at, live - 1);
  const int64_t w_row = (int64_t)e * g.N + min(col0 + at, g.N - 1);
  const uint8_t* a = g.a + a_row * kp + half * 64;
  const uint8_t* w = g.w + w_row * kp + half * 64;
  const uint8_t* as = g.a_scales + a_row * ks;
  const uint8_t* ws = g.w_scales + w_row * ks;
  f32x16_t acc = {};
  const int blocks = (int)(kp / FP8_BLOCK);
  for (int b = wave; b < blocks; b += WAVES) {
    i32x8_t va[2], vw[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint4* pa = reinterpret_cast<const uint4*>(a + (int64_t)b * FP8_BLOCK) + 2 * s;
      const uint4* pw = reinterpret_cast<const uint4*>(w + (int64_t)b * FP8_BLOCK) + 2 * s;
      const uint4 a0 = pa[0], a1 = pa[1], w0 = pw[0], w1 = pw[1];
      va[s] = i32x8_t{(int)a0.x, (int)a0.y, (int)a0.z, (int)a0.w,
                      (int)a1.x, (int)a1.y, (int)a1.z, (int)a1.w};
      vw[s] = i32x8_t{(int)w0.x, (int)w0.y, (int)w0.z, (int)w0.w,
                      (int)w1.x, (int)w1.y, (int)w1.z, (int)w1.w};
    }
    const uint32_t sa = as[b], sw = ws[b];
    acc = fp8_mfma(vw[0], va[0], acc, sw, sa);
    acc = fp8_mfma(vw[1], va[1], acc, sw, sa);
  }
#pragma unroll
  for (int q = 0; q < 16; ++q) parts[wave][q][lane] = acc[q];
  __syncthreads();
  const int row = row0 + at;
  for (int q = wave; q < 16; q += WAVES) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) sum += parts[i][q][lane];
    const int col = col0 + 8 * (q >> 2) + 4 * half + (q & 3);
    if (row < live && col < g.N)
      store_f32<TO>((TO*)g.y + ((int64_t)e * g.R + row) * g.N + col,
                    fp8_activation(sum, g.activation));
  }
}

// ---------------------------------------------------------------------------
// Tiles.  4 wavefronts, one per SIMD; each has 16 TM rows and 128 columns of the tile as
// TM x 8 matrix tiles of 16 x 16 (v_mfma_scale_f32_16x16x128_f8f6f4: a whole block of
// 128 per instruction; of the two shapes the one that draws less power: 4.3 against 4.0
// PFLOP/s of random operands, nothing else running).  The wavefronts lie WM down and 4 /
// WM across.  A wavefront's row pieces of 16 lie 16 WM apart, so that a last row tile
// with few rows gives all SIMDs the same, and its columns are one block of 128, so that
// an 8-bit result's scale needs no other wavefront.
//
// A K tile is one block of 128 values: rows of 128 bytes, brought to LDS by direct loads,
// 8 rows per instruction and whole 128-byte lines; the 16-byte chunks of a row are
// XOR-ed with its number on the way (on the global side), which spreads the fragment
// reads over all banks.  There are two token slots and three weight slots.  K tile t is
// multiplied in 8 groups, one per weight fragment j, TM matrix instructions each:
//   groups 0 .. 4  read the weight fragments 3 .. 7
//   before group 1 a barrier: everybody has the token fragments of t in registers
//   groups 1 .. 4  token loads of K tile t + 2, into the slot that this freed
//   before group 6 a barrier: everybody has the weight fragments of t, and K tile t + 1
//                  has landed (vmcnt counts in order: the weight loads of t + 2 and the
//                  token loads of t + 2 may be out)
//   groups 6, 7    weight loads of K tile t + 3, into the slot that this freed; the
//                  fragments of t + 1: weights 0 .. 2, and tokens as group 7 is done
//                  with the ones before
// so that token loads have 1.6 and weight loads 2 K tiles' time.  Blocks are persistent,
// and the K tiles of a block's tiles follow each other: what a tile's last two K tiles
// load belongs to the next one.  Needs two K tiles.  Block b runs on XCD b % 8; the
// blocks of an XCD hold consecutive tiles, numbered in bands of 8 row tiles, so that 32
// of them share 8 + 4 operand panels in its L2.
//
// A lane's scales are a dword per row and four K tiles, shifted along as the K tiles go
// by; the next four are requested more than a K tile ahead.
//
// A result is turned round in the weight slot that the last K tile has left, each
// wavefront in the kilobytes that its own loads fill afterwards (so no barrier), and
// leaves in whole lines.
// ---------------------------------------------------------------------------
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void_t;
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

template <int TM_, int WM_, int WN_>
struct TileCfg {
  static constexpr int TM = TM_, TN = 8, WM = WM_, WN = WN_;
  static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
  static constexpr int BM = 16 * TM * WM, BN = 128 * WN;
  // of a wavefront per K tile, 8 rows each
  static constexpr int A_LOADS = BM / 8 / WAVES, W_LOADS = BN / 8 / WAVES;
  static constexpr int PIECE_STEP = 1024 * WAVES;   // between its kilobytes of a slot
  static_assert(WAVES % 2 == 0 && A_LOADS > 0 && W_LOADS >= 4, "loads and staging");
  static constexpr int A_SLOT = BM * FP8_BLOCK, W_SLOT = BN * FP8_BLOCK;
  static constexpr int W_BASE = 2 * A_SLOT;
  static constexpr int LDS_BYTES = 2 * A_SLOT + 3 * W_SLOT;
};

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

// 16 bytes per lane, at `at` of the `bytes` at `base`; what lies behind is dropped
__device__ __forceinline__ void store_line(u32x4_t v, uint8_t* base, int bytes,
                                           uint32_t at) {
  __builtin_amdgcn_raw_buffer_store_b128(
      v, __builtin_amdgcn_make_buffer_rsrc(base, 0, max(bytes, 0), 0x00027000), at, 0, 0);
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

// acc (+)= w . a of a matrix tile, with the byte BYTE of both scales.  ASM: as written, the
// sums in place in accumulator registers: with 64 matrix tiles of them the compiler's
// own form copies them between the two halves of the register file (100 copies per K
// tile).  What it knows of hazards is then the caller's: the operands come from LDS,
// scales are written several matrix instructions ahead, sums are read after mfma_drain.
template <bool ASM, bool FIRST, int BYTE>
__device__ __forceinline__ void fp8_mfma16(f32x4_t& acc, i32x8_t w, i32x8_t a,
                                           uint32_t w_scale, uint32_t a_scale) {
  if constexpr (!ASM) {
    const f32x4_t none = {};
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
        w, a, FIRST ? none : acc, 0, 0, BYTE, (int)w_scale, BYTE, (int)a_scale);
  } else if constexpr (FIRST) {
    static_assert(BYTE == 0, "a tile begins with whole scales");
    asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, 0, %3, %4 "
                 "op_sel_hi:[0,0,0]"
                 : "=a"(acc) : "v"(w), "v"(a), "v"(w_scale), "v"(a_scale));
  } else {
#define FP8_MFMA16(SEL)                                                            \
  asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 " SEL     \
               : "+a"(acc) : "v"(w), "v"(a), "v"(w_scale), "v"(a_scale))
    if constexpr (BYTE == 0) FP8_MFMA16("op_sel_hi:[0,0,0]");
    else if constexpr (BYTE == 1) FP8_MFMA16("op_sel:[1,1,0] op_sel_hi:[0,0,0]");
    else if constexpr (BYTE == 2) FP8_MFMA16("op_sel_hi:[1,1,0]");
    else FP8_MFMA16("op_sel:[1,1,0] op_sel_hi:[1,1,0]");
#undef FP8_MFMA16
  }
}
// the last matrix instructions' results can be read after it
__device__ __forceinline__ void mfma_drain() {
  asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
}

// ACT: an activation that is neither linear nor relu
template <int TM, int WM, int WN, int TO, bool ACT>
__global__ __launch_bounds__(64 * WM * WN, TM > 2 && WM * WN == 4 ? 1 : 2)
void fp8_tile_kernel(GemmArgs g, TileGrid grid) {
  using Cfg = TileCfg<TM, WM, WN>;
  constexpr int TN = Cfg::TN, BM = Cfg::BM, BN = Cfg::BN;
  constexpr int A_LOADS = Cfg::A_LOADS, W_LOADS = Cfg::W_LOADS;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM;
  const int64_t kp = fp8_row_bytes(g.K), ks = fp8_scale_bytes(g.K);
  const int k_tiles = (int)(kp / FP8_BLOCK);

  // (What is computed from the lane index outside the K loop is computed from a copy
  // that the compiler cannot see through: made once it would be live across the K loop.)
  auto lane_again = [&]() FP8_INLINE {
    int l = lane;
    asm volatile("" : "+v"(l));
    return l;
  };

  struct Tile {
    int e, row0, col0;
    int valid;                    // its rows (0: there is no such tile)
    int part, k0, nk;             // K tiles k0 .. k0 + nk - 1
  };
  // Tile number `logical`.  With row counts the tiles are those that hold rows, counted
  // through 64 experts at a time: lane l adds up the row tiles of expert l and below.
  auto tile_at = [&](int logical) FP8_INLINE {
    Tile t = {0, 0, 0, 0, 0, 0, k_tiles};
    int tiles_m = grid.tiles_m, rem = 0;
    if (logical >= grid.tiles) return t;
    if constexpr (TO == TO_PARTS) {
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
      const int lane = lane_again();
      int before = 0;
      bool found = false;
      for (int e0 = 0; e0 < g.E && !found; e0 += 64) {
        const int live =
            e0 + lane < g.E ? live_rows(g.row_count, e0 + lane, g.R) : 0;
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
    return t;
  };
  // the block's tile of round `round`
  auto number = [&](int round) FP8_INLINE {
    return (int)(round * gridDim.x + (blockIdx.x & 7) * (gridDim.x >> 3) +
                 (blockIdx.x >> 3));
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
          ws + (uint32_t)min(128 * wn + 16 * j + fr, g.N - 1 - t.col0) * (uint32_t)ks);
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
    return fragments(Cfg::W_BASE + slot * Cfg::W_SLOT + wn * 128 * FP8_BLOCK);
  };
  auto read_a = [&](const Fragments& f, int i) FP8_INLINE {
    const unsigned char* base = smem + i * WM * 16 * FP8_BLOCK;
    return fp8_fragment(base + f.lo, base + f.hi);
  };
  auto read_w = [&](const Fragments& f, int j) FP8_INLINE {
    const unsigned char* base = smem + j * 16 * FP8_BLOCK;
    return fp8_fragment(base + f.lo, base + f.hi);
  };

  constexpr bool IN_PLACE = TM == 8 || (TM == 4 && WM * WN == 8);
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
      return Source{mine ? here.a : next.a, mine ? here.a_bytes : next.a_bytes,
                    (mine ? p : p - t.nk) * FP8_BLOCK, aslot * Cfg::A_SLOT};
    };
    auto w_source = [&](int p, int slot) {
      const bool mine = p < t.nk;
      return Source{mine ? here.w : next.w, mine ? here.w_bytes : next.w_bytes,
                    (mine ? p : p - t.nk) * FP8_BLOCK,
                    Cfg::W_BASE + slot * Cfg::W_SLOT};
    };
    const Fragments w_now = w_fragments(wslot);
    Fragments w_then = {0, 0}, a_then = {0, 0};
    const bool regroup = ((kt + 1) & 3) == 0;
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
          fp8_mfma16<IN_PLACE, FIRST, BYTE>(acc[i][j], fw[j & 3], fa[i], sw[j], sa[i]);
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
  // any case and the next tile's first wait can count on them.
  auto write_out = [&](const Tile& t, auto na_tag) FP8_INLINE {
    constexpr int NA = decltype(na_tag)::value;
    const int wfree = wslot == 0 ? 2 : wslot - 1;       // of the last K tile
    const int lane = lane_again(), fr = lane & 15, fc = lane >> 4;
    unsigned char* const free_slot = smem + Cfg::W_BASE + wfree * Cfg::W_SLOT + wave * 1024;
    const uint32_t stage = (uint32_t)(size_t)(lds_void_t*)free_slot;
    const int col0 = t.col0 + 128 * wn;
    const int64_t first = (int64_t)t.e * g.R + t.row0;
    const int64_t ns = fp8_scale_bytes(g.N);
    auto row_of = [&](int i) { return (i * WM + wm) * 16; };
    if constexpr (IN_PLACE) mfma_drain();
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
                     col0 < g.N ? min(left, 8) * row_bytes - col0 : 0, at);
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
                       min(rows - 4 * n, 4) * row_bytes - 2 * col0, at);
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
  Tile t = tile_at(number(0));
  if (t.valid == 0) return;
  Operands here = operands(t);
  load_scales(t, 0);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const Source as = {here.a, here.a_bytes, k * FP8_BLOCK, k * Cfg::A_SLOT};
    const Source ws = {here.w, here.w_bytes, k * FP8_BLOCK, Cfg::W_BASE + k * Cfg::W_SLOT};
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
      for (int i = 0; i < TM; ++i) sa[i] = sa_next[i];
#pragma unroll
      for (int j = 0; j < TN; ++j) sw[j] = sw_next[j];
      // (without a next tile its loads fetch this one again, which nobody reads)
      after = tile_at(number(++round));
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

// How a product is run.
struct Plan {
  int kind = 0;                   // TILES: 256 x 256, 128 x 256, 128 x 128, 64 x 128
  int split = 1;
  size_t workspace = 0;
};
enum { FEW_ROWS, TILES_256, TILES_128_256, TILES_128, TILES_64 };

static Plan plan_product(int E, int R, int K, int N, bool eight_bit, bool counted) {
  Plan p;
  // (a tile's operand rows and 8 rows of its result are addressed in 31 bits)
  if (K <= FP8_BLOCK || K > 1 << 22 || N > 1 << 26) {
    p.kind = FEW_ROWS;
    p.workspace = eight_bit ? (size_t)E * R * N * sizeof(float) : 0;
    return p;
  }
  p.kind = R <= 64 ? TILES_64 : R <= 128 ? TILES_128 : TILES_256;
  return p;
}

template <int TM, int WM, int WN, int TO>
static int launch_tiles(const GemmArgs& g, int split, hipStream_t st) {
  using Cfg = TileCfg<TM, WM, WN>;
  TileGrid grid;
  grid.tiles_m = (int)(((int64_t)g.R + Cfg::BM - 1) / Cfg::BM);
  grid.tiles_n = (g.N + Cfg::BN - 1) / Cfg::BN;
  grid.split = split;
  // (numbers of tiles, those past the end too, are int)
  const int64_t one = (int64_t)grid.tiles_m * grid.tiles_n;
  MOE_REQUIRE(one <= 1 << 30 && one * g.E <= 1 << 30 && one * g.E * split <= 1 << 30,
              MESH_MOE_E_UNSUPPORTED, "fp8_expert_linear: too many tiles (E=%d R=%d N=%d)",
              g.E, g.R, g.N);
  grid.tiles = (int)(one * g.E * split);
  const int cus = compute_units();
  if (cus == 0) return MESH_MOE_E_HIP;
  const int most = cus / 8 * 8 * (160 * 1024 / Cfg::LDS_BYTES);
  const int want = (grid.tiles + 7) / 8 * 8;
  const bool act = TO != TO_PARTS && g.activation != MESH_MOE_ACT_LINEAR &&
                   g.activation != MESH_MOE_ACT_RELU;
  auto kernel = act ? fp8_tile_kernel<TM, WM, WN, TO, TO != TO_PARTS>
                    : fp8_tile_kernel<TM, WM, WN, TO, false>;
  MOE_ALLOW_LDS(kernel, Cfg::LDS_BYTES);
  kernel<<<(unsigned)(want < most ? want : most), Cfg::THREADS, Cfg::LDS_BYTES, st>>>(
      g, grid);
  MOE_CHECK_LAUNCH("fp8_expert_linear");
  return 0;
}

template <int TM, int WM, int WN>
static int run_tiles(const GemmArgs& g, int split, void* workspace, hipStream_t st) {
  if (split > 1) {
    GemmArgs parts = g;
    parts.y = workspace;
    const int rc = launch_tiles<TM, WM, WN, TO_PARTS>(parts, split, st);
    if (rc != 0) return rc;
    const int64_t threads = (int64_t)g.E * g.R * (fp8_row_bytes(g.N) / 8);
    const unsigned blocks = (unsigned)((threads + 255) / 256);
    if (g.y_scales)
      fp8_parts_kernel<true><<<blocks, 256, 0, st>>>((const float*)workspace, g, split);
    else
      fp8_parts_kernel<false><<<blocks, 256, 0, st>>>((const float*)workspace, g, split);
    MOE_CHECK_LAUNCH("fp8_expert_linear");
    return 0;
  }
  if (g.y_scales) return launch_tiles<TM, WM, WN, TO_FP8>(g, 1, st);
  if (g.N % 8 == 0 && (uintptr_t)g.y % 16 == 0)
    return launch_tiles<TM, WM, WN, TO_LINES>(g, 1, st);
  return launch_tiles<TM, WM, WN, TO_BF16>(g, 1, st);
}

static int run_product(const GemmArgs& g, void* workspace, hipStream_t st) {
  const Plan p = plan_product(g.E, g.R, g.K, g.N, g.y_scales != nullptr,
                              g.row_count != nullptr);
  switch (p.kind) {
    case TILES_256: return run_tiles<8, 2, 2>(g, p.split, workspace, st);
    case TILES_128_256: return run_tiles<4, 2, 2>(g, p.split, workspace, st);
    case TILES_128: return run_tiles<2, 4, 1>(g, p.split, workspace, st);
    case TILES_64: return run_tiles<1, 4, 1>(g, p.split, workspace, st);
    default: break;
  }
  const dim3 grid((g.N + 31) / 32, (g.R + 31) / 32, g.E);
  MOE_REQUIRE(grid.y <= 65535 && grid.z <= 65535, MESH_MOE_E_UNSUPPORTED,
              "fp8_expert_linear: too many rows or experts (E=%d R=%d)", g.E, g.R);
  if (g.y_scales == nullptr) {
    fp8_few_rows_kernel<4, bf16_t><<<grid, 256, 0, st>>>(g);
    MOE_CHECK_LAUNCH("fp8_expert_linear");
    return 0;
  }
  GemmArgs f = g;
  f.y = workspace;
  fp8_few_rows_kernel<4, float><<<grid, 256, 0, st>>>(f);
  MOE_CHECK_LAUNCH("fp8_expert_linear");
  return fp8_quantize(workspace, nullptr, g.row_count, g.y, g.y_scales, nullptr, nullptr,
                      g.E, g.R, g.N, MESH_MOE_F32, true, st);
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

extern "C" size_t mesh_moe_fp8_expert_linear_workspace_bytes(int E, int R, int K, int N,
                                                             int eight_bit) {
  if (!fp8_sizes(E, R, K, N)) return 0;
  return plan_product(E, R, K, N, eight_bit != 0, false).workspace;
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
                      w_scales, row_count, y, y_scales, E, R, K, N, activation};
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
  int rc = fp8_quantize(dy, relu_mask, row_count, rows, da ? ws + p.row_scales : nullptr,
                        ws + p.columns, ws + p.column_scales, E, R, N, dtype, false, st);
  if (rc != 0) return rc;
  const GemmArgs weights = {(const uint8_t*)a_column_values, a_column_scales,
                            ws + p.columns, ws + p.column_scales, nullptr, dw, nullptr,
                            E, K, R, N, MESH_MOE_ACT_LINEAR};
  rc = run_product(weights, ws + p.products, st);
  if (rc != 0 || da == nullptr) return rc;
  const GemmArgs input = {rows, ws + p.row_scales, (const uint8_t*)w_row_values,
                          w_row_scales, row_count, da, nullptr, E, R, N, K,
                          MESH_MOE_ACT_LINEAR};
  return run_product(input, ws + p.products, st);
}
