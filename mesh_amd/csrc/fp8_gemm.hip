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
// the loads of a tile's last two K tiles are the first of the next.  Needs two K tiles.
// Block b runs on XCD b % 8; the blocks of an XCD hold consecutive tiles, numbered in
// bands of 8 row tiles, so that 32 of them share 8 + 4 operand panels in its L2.
//
// A lane's scales are a dword per row and four K tiles, shifted along as the K tiles go
// by; the next four are requested a K tile or more ahead.
//
// A result is turned round in the weight slot that the last K tile has left, 32 rows of
// 128 bytes at a time, each wavefront in the kilobytes that its own loads fill
// afterwards (so no barrier), and leaves in whole 128-byte lines.
// ---------------------------------------------------------------------------
typedef __attribute__((address_space(3))) void lds_void_t;
typedef const __attribute__((address_space(1))) void glb_void_t;
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

struct TileCfg {
  static constexpr int BM = 256, BN = 256, THREADS = 512, WAVES = 8;
  static constexpr int TM = 2, TN = 4;
  static constexpr int SLOT = 256 * FP8_BLOCK;          // 32 KB
  static constexpr int W_BASE = 2 * SLOT;
  static constexpr int LDS_BYTES = 5 * SLOT;
};

struct TileGrid {
  int tiles_m, tiles_n;           // of an expert with all of its rows
  int tiles;                      // of all experts
};

#define FP8_INLINE __attribute__((always_inline))

// a pointer that all lanes have
__device__ __forceinline__ const uint8_t* uniform(const uint8_t* p) {
  const uint64_t u = (uint64_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)u);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((int)(u >> 32));
  return (const uint8_t*)((uint64_t)hi << 32 | lo);
}

// 16 bytes per lane, from `at` of the `bytes` at `from` (zeros behind them), to LDS: lane
// after lane from `to` on
__device__ __forceinline__ void load_to_lds(const uint8_t* from, int bytes, uint32_t at,
                                            unsigned char* to) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(
      __builtin_amdgcn_make_buffer_rsrc((void*)from, 0, max(bytes, 0), 0x00027000),
      (lds_void_t*)to, 16, at, 0, 0, 0);
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

// Four 16-byte reads, 8192 bytes apart, and the wait for them in one asm, whose outputs
// then hold what the compiler takes them for.
__device__ __forceinline__ void lds_read_lines(u32x4_t (&p)[4], uint32_t at) {
  asm volatile("ds_read_b128 %0, %4\n\t"
               "ds_read_b128 %1, %4 offset:8192\n\t"
               "ds_read_b128 %2, %4 offset:16384\n\t"
               "ds_read_b128 %3, %4 offset:24576\n\t"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(p[0]), "=&v"(p[1]), "=&v"(p[2]), "=&v"(p[3])
               : "v"(at)
               : "memory");
}
__device__ __forceinline__ void lds_write_b64(uint32_t at, u32x2_t v) {
  asm volatile("ds_write_b64 %0, %1" :: "v"(at), "v"(v) : "memory");
}

// EIGHT: the result is an 8-bit operand; ACT: an activation that is neither linear nor
// relu; WHOLE: rows of a bf16 result are whole pieces of 16 bytes that lie on 16 bytes.
template <bool EIGHT, bool ACT, bool WHOLE>
__global__ __launch_bounds__(TileCfg::THREADS) void fp8_tile_kernel(GemmArgs g,
                                                                    TileGrid grid) {
  using Cfg = TileCfg;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const int fr = lane & 31, fc = lane >> 5;
  const int64_t kp = fp8_row_bytes(g.K), ks = fp8_scale_bytes(g.K);
  const int nk = (int)(kp / FP8_BLOCK);

  // (What is computed from the lane index outside the K loop is computed from a copy
  // that the compiler cannot see through: made once it would be live across the K loop,
  // which has no registers to spare.)
  auto lane_again = [&]() FP8_INLINE {
    int l = lane;
    asm volatile("" : "+v"(l));
    return l;
  };

  struct Tile {
    int e, row0, col0;
    int valid;                    // its rows (0: there is no such tile)
  };
  // Tile number `logical`.  With row counts the tiles are those that hold rows, counted
  // through 64 experts at a time: lane l adds up the row tiles of expert l and below.
  auto tile_at = [&](int logical) FP8_INLINE {
    Tile t = {0, 0, 0, 0};
    int tiles_m = grid.tiles_m, rem = 0;
    if (g.row_count == nullptr) {
      if (logical >= grid.tiles) return t;
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
        int sum = (live + Cfg::BM - 1) / Cfg::BM * grid.tiles_n;
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
          tiles_m = (t.valid + Cfg::BM - 1) / Cfg::BM;
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
    t.row0 = __builtin_amdgcn_readfirstlane((band * 8 + (r - tn * high)) * Cfg::BM);
    t.col0 = __builtin_amdgcn_readfirstlane(tn * Cfg::BN);
    t.e = __builtin_amdgcn_readfirstlane(t.e);
    t.valid = __builtin_amdgcn_readfirstlane(min(Cfg::BM, t.valid - t.row0));
    return t;
  };
  // the block's tile of round `round`
  auto number = [&](int round) FP8_INLINE {
    return (int)(round * gridDim.x + (blockIdx.x & 7) * (gridDim.x >> 3) +
                 (blockIdx.x >> 3));
  };

  // The tile that is being loaded.  A wavefront's load j fills the rows 8 (wave + 8 j) ..
  // + 7 of an LDS tile through a buffer that ends with the rows there are: what lies
  // behind is not fetched.
  const uint8_t *a_base, *w_base;
  int a_bytes, w_bytes;
  const uint32_t load_at = (uint32_t)(wave * 8 + (lane >> 3)) * (uint32_t)kp +
                           ((lane & 7) ^ (lane >> 3) ^ (wave & 1)) * 16;
  const int load_step = 64 * (int)kp;
  auto set_loads = [&](const Tile& t) FP8_INLINE {
    a_base = uniform(g.a + ((int64_t)t.e * g.R + t.row0) * kp);
    w_base = uniform(g.w + ((int64_t)t.e * g.N + t.col0) * kp);
    a_bytes = t.valid * (int)kp;
    w_bytes = min(Cfg::BN, g.N - t.col0) * (int)kp;
  };
  // where the next load of a K tile reads (the loads follow each other by load_step)
  struct Source {
    const uint8_t* from;
    int bytes;
  };
  auto load = [&](Source& s, int j, int at) FP8_INLINE {
    load_to_lds(s.from, s.bytes, load_at, smem + at + (wave + 8 * j) * 1024);
    s.from += load_step;
    s.bytes -= load_step;
  };
  auto a_source = [&](int kt) FP8_INLINE {
    return Source{a_base + kt * FP8_BLOCK, a_bytes - kt * FP8_BLOCK};
  };
  auto w_source = [&](int kt) FP8_INLINE {
    return Source{w_base + kt * FP8_BLOCK, w_bytes - kt * FP8_BLOCK};
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
      Source from = s == 0 ? w_source(lk) : a_source(lk);
      const int into = s == 0 ? Cfg::W_BASE + wload * Cfg::SLOT : aslot * Cfg::SLOT;
      constexpr bool READ[2] = {NA > 0, NA > 0 && !LAST};
      auto rd_a = [&](int i) { if (READ[s] && i < NA) fa[to][i] = read_a(at, as, to, i); };
      auto rd_w = [&](int j) { if (READ[s]) fw[j] = read_w(at, ws, to, j); };
      // (the weight loads have half a K tile more than the token loads, which go first)
      auto ld = [&](int j, bool here) { if (here) load(from, j, into); };
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
        lds_read_lines(line, get_at);
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
          lds_read_lines(line, get_at);
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
  Tile t = tile_at(number(0));
  if (t.valid == 0) return;
  set_loads(t);
  load_scales(t, 0);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    Source as = a_source(k), ws = w_source(k);
#pragma unroll
    for (int j = 0; j < 4; ++j) load(as, j, k * Cfg::SLOT);
#pragma unroll
    for (int j = 0; j < 4; ++j) load(ws, j, Cfg::W_BASE + k * Cfg::SLOT);
  }
  __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8));             // vmcnt 0
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  for (;;) {
    Tile after = {0, 0, 0, 0};
    auto tile_pass = [&](auto na_tag) FP8_INLINE {
      constexpr int NA = decltype(na_tag)::value;
      auto next_scales = [&](int kt) FP8_INLINE {
        if ((kt & 3) == 0) {
#pragma unroll
          for (int i = 0; i < Cfg::TM; ++i) sa[i] = sa_next[i];
#pragma unroll
          for (int j = 0; j < Cfg::TN; ++j) sw[j] = sw_next[j];
          if (kt + 4 < nk) load_scales(t, kt / 4 + 1);
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
        after = tile_at(number(++round));
        set_loads(after.valid != 0 ? after : t);
      };
      if constexpr (NA > 0) first_fragments(aslot, wslot);
      next_scales(0);
      if (nk == 2) advance();
      k_tile(na_tag, std::true_type{}, std::false_type{}, nk == 2 ? 0 : 2);
      for (int kt = 1; kt < nk - 1; ++kt) {
        next_scales(kt);
        if (kt == nk - 2) advance();
        k_tile(na_tag, std::false_type{}, std::false_type{}, kt == nk - 2 ? 0 : kt + 2);
      }
      next_scales(nk - 1);
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
#undef FP8_INLINE

// bytes of scratch one product needs
// (a tile's operand rows and 8 rows of its result are addressed in 31 bits)
static bool tiles_apply(int R, int K, int N) {
  return R > 64 && K > FP8_BLOCK && K <= 1 << 22 && N <= 1 << 26;
}
static size_t product_workspace(int E, int R, int K, int N, bool eight_bit) {
  return eight_bit && !tiles_apply(R, K, N) ? (size_t)E * R * N * sizeof(float) : 0;
}

template <bool EIGHT>
static int run_tiles(const GemmArgs& g, hipStream_t st) {
  TileGrid grid;
  grid.tiles_m = (g.R + TileCfg::BM - 1) / TileCfg::BM;
  grid.tiles_n = (g.N + TileCfg::BN - 1) / TileCfg::BN;
  const int64_t tiles = (int64_t)grid.tiles_m * grid.tiles_n * g.E;
  // (numbers of tiles, those past the end too, are int)
  MOE_REQUIRE((int64_t)grid.tiles_m * grid.tiles_n <= 1 << 30 && tiles <= 1 << 30,
              MESH_MOE_E_UNSUPPORTED, "fp8_expert_linear: too many tiles (E=%d R=%d N=%d)",
              g.E, g.R, g.N);
  grid.tiles = (int)tiles;
  const int cus = compute_units();
  if (cus == 0) return MESH_MOE_E_HIP;
  const int most = cus / 8 * 8, want = (grid.tiles + 7) / 8 * 8;
  const bool act =
      g.activation != MESH_MOE_ACT_LINEAR && g.activation != MESH_MOE_ACT_RELU;
  const bool whole = EIGHT || (g.N % 8 == 0 && (uintptr_t)g.y % 16 == 0);
  auto kernel = whole ? act ? fp8_tile_kernel<EIGHT, true, true>
                            : fp8_tile_kernel<EIGHT, false, true>
                : act ? fp8_tile_kernel<EIGHT, true, EIGHT>
                      : fp8_tile_kernel<EIGHT, false, EIGHT>;
  MOE_ALLOW_LDS(kernel, TileCfg::LDS_BYTES);
  kernel<<<(unsigned)(want < most ? want : most), TileCfg::THREADS,
                           TileCfg::LDS_BYTES, st>>>(g, grid);
  MOE_CHECK_LAUNCH("fp8_expert_linear");
  return 0;
}

static int run_product(const GemmArgs& g, void* workspace, hipStream_t st) {
  if (tiles_apply(g.R, g.K, g.N))
    return g.y_scales ? run_tiles<true>(g, st) : run_tiles<false>(g, st);
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
  return product_workspace(E, R, K, N, eight_bit != 0);
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
  const size_t need = product_workspace(E, R, K, N, y_scales != nullptr);
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
  const size_t dw = product_workspace(E, K, R, N, false);
  const size_t da = want_da ? product_workspace(E, R, N, K, false) : 0;
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
