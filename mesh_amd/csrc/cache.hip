// The paged cache: rows of keys and values into pages and back, and attention of one new
// token over them.
#include "../../include/mesh_moe_cache.h"
#include "fp8.h"

#include <algorithm>
#include <type_traits>

namespace mesh_moe {

typedef float f32x2_t __attribute__((ext_vector_type(2)));

constexpr int MAX_WIDTH = 256;                  // D
constexpr int TILES_FROM = 16;                  // D of the kernels on matrix cores
constexpr int MAX_HEADS = 1 << 16;              // HK
constexpr int MAX_POSITIONS = 1 << 30;          // P * S
constexpr int64_t MAX_BLOCKS = MAX_THREADS / 256;   // of 256 threads

// Where a cache's rows lie.
struct Pages {
  const int32_t* table;           // [B][P]
  int N, P, shift;                // pages, table columns, log2 of a page's rows
  int HK, D, DB;                  // heads, values and blocks of 128 of a row
  // Row number (of all pages' rows, of head 0) of position p of sequence b, -1: not there.
  __device__ __forceinline__ int64_t row(int b, int64_t p) const {
    if (p < 0 || (p >> shift) >= P) return -1;
    const int page = table[(int64_t)b * P + (p >> shift)];
    if ((unsigned)page >= (unsigned)N) return -1;
    return (((int64_t)page * HK) << shift) + (p & ((1 << shift) - 1));
  }
  // ... of head h
  __device__ __forceinline__ int64_t head(int64_t row, int h) const {
    return row + ((int64_t)h << shift);
  }
};

// What nothing in a launch writes, from an address that is the same for all lanes: a load
// through the scalar cache, which does not wait for the vector loads before it.
__device__ __forceinline__ int32_t scalar_load(const int32_t* p) {
  typedef const __attribute__((address_space(4))) int32_t* constant_t;
  return *reinterpret_cast<constant_t>(reinterpret_cast<uintptr_t>(p));
}

// What a scale byte stands for (2^-127 is not a normal number).
__device__ __forceinline__ float unit_of(uint32_t byte) {
  return __uint_as_float(byte == 255 ? 0x7fc00000u
                         : byte == 0 ? 0x00400000u
                                     : byte << 23);
}

// The largest of a group of `lanes` (a power of two up to 16) neighbouring lanes.
__device__ __forceinline__ uint32_t max_of_lanes(uint32_t v, int lanes) {
  if (lanes >= 2) v = max(v, dpp<0xb1>(v));     // quad_perm [1,0,3,2]
  if (lanes >= 4) v = max(v, dpp<0x4e>(v));     // quad_perm [2,3,0,1]
  if (lanes >= 8) v = max(v, dpp<0x141>(v));    // row_half_mirror
  if (lanes >= 16) v = max(v, dpp<0x140>(v));   // row_mirror
  return v;
}

template <int BYTES> struct Words;                 // of any address
template <> struct Words<4> { typedef uint32_t type __attribute__((aligned(1))); };
template <> struct Words<8> {
  typedef uint32_t type __attribute__((ext_vector_type(2), aligned(1)));
};
template <> struct Words<16> {
  typedef uint32_t type __attribute__((ext_vector_type(4), aligned(1)));
};
template <int BYTES>
__device__ __forceinline__ void load_words(const uint8_t* at, uint32_t* to) {
  typedef typename Words<BYTES>::type words_t;
  const words_t v = *reinterpret_cast<const words_t*>(at);
  if constexpr (BYTES == 4) {
    to[0] = v;
  } else {
#pragma unroll
    for (int i = 0; i < BYTES / 4; ++i) to[i] = v[i];
  }
}

// 8 values of 8 bits of a row of D from value `at` on, zeros behind the row, and back.
template <bool ALIGNED>
__device__ __forceinline__ void load_eight(const uint8_t* row, int at, int D,
                                           uint32_t (&w)[2]) {
  if (ALIGNED || at + 8 <= D) {
    load_words<8>(row + at, w);
    return;
  }
#pragma unroll
  for (int j = 0; j < 7; ++j)
    if (at + j < D) w[j / 4] |= (uint32_t)row[at + j] << 8 * (j & 3);
}
template <bool ALIGNED>
__device__ __forceinline__ void store_eight(uint8_t* row, int at, int D, uint32_t lo,
                                            uint32_t hi) {
  if (ALIGNED || at + 8 <= D) {
    *reinterpret_cast<Words<8>::type*>(row + at) = Words<8>::type{lo, hi};
    return;
  }
#pragma unroll
  for (int j = 0; j < 7; ++j)
    if (at + j < D) row[at + j] = (uint8_t)((j < 4 ? lo : hi) >> 8 * (j & 3));
}

// ---------------------------------------------------------------------------
// Rows into pages and back.  A wavefront has R rows of keys or of values (blockIdx.z) that
// follow each other in a sequence (blockIdx.y), so that loads of R rows are on their way at
// once; wide rows are shared by two or four wavefronts.  A lane has 8 values of each, and a
// head's lanes are a power of two (16 for each block of 128 where it has more than one), so
// that a block's largest magnitude is found by DPP steps among neighbours.
// Nothing is used twice: bound by the memory, but for writes of narrow heads.  16 sequences
// of up to 4096 rows of 16 x 64 bfloat16 keys and values into 8 bits move 215 MB in 48 us,
// 4.4 TB/s where a copy of 1 GiB reaches 5.2 (probably: a row of 64 bytes is half a line, a
// wavefront's store goes to all heads' pages, and scale bytes are stored one by one).  The way
// back moves 341 MB in 46, 7.5 TB/s, as the pages are in the last level's cache still (of the
// 268 MB that it stores, 5.9 where a fill reaches 6.7); 4 x 16384 rows 404 MB in 60 when
// repeated on the same pages, 75 on others (5.4 TB/s).
// ---------------------------------------------------------------------------
struct RowsOf {
  Pages pages;
  const int32_t* position;        // [B]
  const int32_t* count;           // [B] or null
  int B, T;
  int lanes;                      // of a head, log2
  int sharing;                    // wavefronts that share a row (1, 2 or 4), log2
};
// Rows of a wavefront, where there are many: 4 x 16384 rows of 1024 values out of an 8-bit
// cache take 84 us by one, 82 by two, 70 by four (recorded calls); 23 x 1000 of 480 out of a
// bfloat16 one 24 by one, 18 by two, 21 by four.
template <typename T, bool EIGHT> constexpr int ROWS = EIGHT && sizeof(T) == 2 ? 4 : 2;

// Where piece `piece` of a head's row begins: a piece that would end behind the row begins as
// much earlier, if that is in its block of 128 (EIGHT) or row, and the values that two lanes
// have then are the same.  D for a piece that the row does not have.
template <bool EIGHT, bool ALIGNED>
__device__ __forceinline__ int piece_at(int piece, int D) {
  const int at = min(piece * 8, D);
  if (ALIGNED || at == D || at + 8 <= D) return at;
  return D - (EIGHT ? at / FP8_BLOCK * FP8_BLOCK : 0) >= 8 ? D - 8 : at;
}

// Calls f(b, t0, rows, from, piece, step): rows t0 .. of sequence b, which lie (from) in
// rows of the pages or nowhere (-1), of which this lane has the pieces piece, piece + step,
// ...  `rows` of them are before the count.
template <int R, typename F>
__device__ __forceinline__ void for_rows(const RowsOf& r, F f) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int groups = (r.T + R - 1) / R;
  for (int b = blockIdx.y; b < r.B; b += gridDim.y) {
    const int count = r.count ? min(max(scalar_load(r.count + b), 0), r.T) : r.T;
    const int position = scalar_load(r.position + b);
    const int32_t* table = r.pages.table + (int64_t)b * r.pages.P;
    for (int64_t g = ((int64_t)blockIdx.x * 4 + wave) >> r.sharing; g < groups;
         g += (int64_t)gridDim.x * 4 >> r.sharing) {
      const int t0 = (int)g * R;
      int64_t rows[R];
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int64_t p = (int64_t)position + t0 + i;
        rows[i] = -1;
        if (t0 + i >= count || p < 0 || (p >> r.pages.shift) >= r.pages.P) continue;
        const int page = scalar_load(table + (p >> r.pages.shift));
        if ((unsigned)page < (unsigned)r.pages.N)
          rows[i] = (((int64_t)page * r.pages.HK) << r.pages.shift) +
                    (p & ((1 << r.pages.shift) - 1));
      }
      f(b, t0, min(r.T - t0, R), rows, (wave & (1 << r.sharing) - 1) * 64 + lane,
        64 << r.sharing);
    }
  }
}

template <typename T, bool EIGHT, bool ALIGNED, int R>
__global__ __launch_bounds__(256) void cache_write_kernel(
    RowsOf r, const T* __restrict__ k, const T* __restrict__ v, void* k_pages,
    void* v_pages, uint8_t* k_scales, uint8_t* v_scales) {
  const bool is_v = blockIdx.z != 0;
  const T* x = is_v ? v : k;
  uint8_t* values = static_cast<uint8_t*>(is_v ? v_pages : k_pages);
  uint8_t* scales = is_v ? v_scales : k_scales;
  const int D = r.pages.D, HK = r.pages.HK;
  const int pieces = HK << r.lanes, group = min(1 << r.lanes, 16);
  for_rows<R>(r, [&](int b, int t0, int, const int64_t (&to)[R], int first, int step) {
    const T* from = x + ((int64_t)b * r.T + t0) * HK * D;
    // (whole wavefronts, as the maxima take them)
    for (int piece = first; piece < (pieces + 63) / 64 * 64; piece += step) {
      const int h = piece >> r.lanes;
      const int at =
          h < HK ? piece_at<EIGHT, ALIGNED>(piece & ((1 << r.lanes) - 1), D) : D;
      float f[R][8];
#pragma unroll
      for (int i = 0; i < R; ++i)
        load8<T, ALIGNED>(from + ((int64_t)i * HK + min(h, HK - 1)) * D,
                          to[i] < 0 ? D : at, D, f[i]);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if (to[i] < 0) continue;
        const int64_t row = r.pages.head(to[i], h);
        if constexpr (EIGHT) {
          uint32_t top = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) top = max(top, magnitude_bits(f[i][j]));
          const Fp8Scale s = fp8_scale(max_of_lanes(top, group));
          if (at >= D) continue;
#pragma unroll
          for (int j = 0; j < 8; ++j) f[i][j] *= s.factor;
          const uint32_t lo = fp8_pack4(f[i][0], f[i][1], f[i][2], f[i][3]);
          const uint32_t hi = fp8_pack4(f[i][4], f[i][5], f[i][6], f[i][7]);
          store_eight<ALIGNED>(values + row * D, at, D, lo, hi);
          if ((piece & (group - 1)) == 0)
            scales[row * r.pages.DB + at / FP8_BLOCK] = (uint8_t)s.byte;
        } else {
          if (at < D)
            store8<T, ALIGNED>(reinterpret_cast<T*>(values) + row * D, at, D, f[i]);
        }
      }
    }
  });
}

template <typename T, bool EIGHT, bool ALIGNED, int R>
__global__ __launch_bounds__(256) void cache_read_kernel(
    RowsOf r, const void* __restrict__ k_pages, const void* __restrict__ v_pages,
    const uint8_t* __restrict__ k_scales, const uint8_t* __restrict__ v_scales,
    T* __restrict__ k, T* __restrict__ v) {
  const bool is_v = blockIdx.z != 0;
  T* y = is_v ? v : k;
  const uint8_t* values = static_cast<const uint8_t*>(is_v ? v_pages : k_pages);
  const uint8_t* scales = is_v ? v_scales : k_scales;
  const int D = r.pages.D, HK = r.pages.HK;
  const int pieces = HK << r.lanes;
  for_rows<R>(r, [&](int b, int t0, int n, const int64_t (&from)[R], int first, int step) {
    T* to = y + ((int64_t)b * r.T + t0) * HK * D;
    for (int piece = first; piece < pieces; piece += step) {
      const int h = piece >> r.lanes;
      const int at = piece_at<EIGHT, ALIGNED>(piece & ((1 << r.lanes) - 1), D);
      if (at >= D) continue;
      float f[R][8];
      uint32_t w[R][2], byte[R];
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int64_t row = r.pages.head(from[i], h);
        w[i][0] = w[i][1] = 0;
        byte[i] = FP8_UNIT;
        if constexpr (!EIGHT) {
          load8<T, ALIGNED>(reinterpret_cast<const T*>(values) + row * D,
                            from[i] < 0 ? D : at, D, f[i]);
        } else if (from[i] >= 0) {
          load_eight<ALIGNED>(values + row * D, at, D, w[i]);
          byte[i] = scales[row * r.pages.DB + at / FP8_BLOCK];
        }
      }
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if (i >= n) continue;
        if constexpr (EIGHT) {
          const float unit = unit_of(byte[i]);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i][j], false);
            const f32x2_t hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i][j], true);
            f[i][4 * j] = lo[0] * unit;
            f[i][4 * j + 1] = lo[1] * unit;
            f[i][4 * j + 2] = hi[0] * unit;
            f[i][4 * j + 3] = hi[1] * unit;
          }
        }
        store8<T, ALIGNED>(to + ((int64_t)i * HK + h) * D, at, D, f[i]);
      }
    }
  });
}

// ---------------------------------------------------------------------------
// Attention of one token over a cache: with m the largest logit so far, l the sum of
// exp(logit - m) and o the sum of exp(logit - m) v, another position's logit x and value v
// turn them into
//   m' = max(m, x)   l' = l e^(m - m') + e^(x - m')   o' = o e^(m - m') + e^(x - m') v
// and two such triples of different positions are joined the same way; o / l is the
// result.
//
// The kernel for rows of fewer than 16 values, which the matrix cores' tiles (below) do not
// take: a block has a query head of a sequence, and a lane every 256th position, with sums
// of its own.  Bound by the latency of one turn after the other, as a long sequence has no
// more blocks than a short one: 1 sequence of 16384, 8 heads of 8, bfloat16 takes 122 us
// (2863 with a wavefront for a position), 64 of 500 take 10.
// ---------------------------------------------------------------------------
struct Attention {
  Pages pages;
  const void *q, *k_pages, *v_pages;
  const uint8_t *k_scales, *v_scales;
  const void *k_new, *v_new;      // the step's own row, which goes into the pages, or null
  const int32_t* position;        // [B]
  const void* rel_values;         // [H][NB] or null
  const int32_t* rel_bucket;      // [2 * reach - 1]
  int NB, reach;
  void* out;
  int B, H, G;                    // G query heads share a key / value head
};

// visible positions of a sequence whose query is at `position`
__device__ __forceinline__ int seen_from(const Attention& a, int position) {
  const int64_t all = (int64_t)a.pages.P << a.pages.shift;
  return (int)min(max((int64_t)position + 1, (int64_t)0), all);
}
__device__ __forceinline__ int seen_of(const Attention& a, int b) {
  return seen_from(a, a.position[b]);
}

// the bucket of a position `distance` (0 or less) from the query's
__device__ __forceinline__ int bucket_of(const Attention& a, int distance) {
  const int bucket = a.rel_bucket[max(distance, 1 - a.reach) + a.reach - 1];
  return min(max(bucket, 0), a.NB - 1);
}

// e^(x - m) with m >= x; 0 for x = -infinity.  (The difference first: it is exact where it
// matters, and what is lost of a larger one is lost of a small weight.)
__device__ __forceinline__ float weight_of(float x, float m) {
  return x == -INFINITY ? 0.f
                        : __builtin_amdgcn_exp2f((x - m) * 1.4426950408889634f);
}

// a row's values, 0 from D on
template <typename T, bool EIGHT>
__device__ __forceinline__ void few_values(const void* pages, const uint8_t* scales,
                                           int64_t row, int D, float (&f)[TILES_FROM]) {
  uint32_t code[TILES_FROM];
  float unit = 1.f;
  if constexpr (EIGHT) unit = unit_of(scales[row]);
#pragma unroll
  for (int d = 0; d < TILES_FROM; ++d) {
    f[d] = 0.f;
    if (d >= D) continue;
    if constexpr (EIGHT) code[d] = static_cast<const uint8_t*>(pages)[row * D + d];
    else f[d] = load_f32<T>(static_cast<const T*>(pages) + row * D + d);
  }
  if constexpr (EIGHT)
#pragma unroll
    for (int d = 0; d < TILES_FROM; ++d)
      if (d < D) f[d] = __builtin_amdgcn_cvt_f32_fp8((int)code[d], 0) * unit;
}

template <typename T, bool EIGHT>
__global__ __launch_bounds__(256) void cache_attention_kernel(Attention a) {
  __shared__ float part_o[4][TILES_FROM], part_m[4], part_l[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int b = (int)(blockIdx.x / a.H), h = (int)(blockIdx.x - (int64_t)b * a.H);
  const int D = a.pages.D, last = scalar_load(a.position + b), seen = seen_from(a, last);
  const int64_t at = ((int64_t)b * a.H + h) * D;
  float q[TILES_FROM], o[TILES_FROM], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int d = 0; d < TILES_FROM; ++d) {
    q[d] = d < D ? load_f32<T>(static_cast<const T*>(a.q) + at + d) : 0.f;
    o[d] = 0.f;
  }
  for (int j = threadIdx.x; j < seen; j += 256) {
    int64_t row = a.pages.row(b, j);
    if (row < 0) continue;
    row = a.pages.head(row, h / a.G);
    float k[TILES_FROM], v[TILES_FROM];
    few_values<T, EIGHT>(a.k_pages, a.k_scales, row, D, k);
    few_values<T, EIGHT>(a.v_pages, a.v_scales, row, D, v);
    float x = 0.f;
#pragma unroll
    for (int d = 0; d < TILES_FROM; ++d)
      if (d < D) x = fmaf(q[d], k[d], x);
    if (a.rel_values)
      x += load_f32<T>(static_cast<const T*>(a.rel_values) + (int64_t)h * a.NB +
                       bucket_of(a, j - last));
    const float top = fmaxf(m, x), was = weight_of(m, top);
    const float w = round_to<T>(weight_of(x, top));
    m = top;
    l = l * was + w;
#pragma unroll
    for (int d = 0; d < TILES_FROM; ++d)
      if (d < D) o[d] = fmaf(w, v[d], o[d] * was);
  }
  // ---- the lanes' triples, then the wavefronts'
  float top = m;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
  const float factor = weight_of(m, top);
  l *= factor;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) l += __shfl_xor(l, off, 64);
#pragma unroll
  for (int d = 0; d < TILES_FROM; ++d) {
    if (d >= D) continue;
    o[d] *= factor;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) o[d] += __shfl_xor(o[d], off, 64);
    if (lane == 0) part_o[wave][d] = o[d];
  }
  if (lane == 0) {
    part_m[wave] = top;
    part_l[wave] = l;
  }
  __syncthreads();
  if ((int)threadIdx.x >= D) return;
  const int d = threadIdx.x;
  top = part_m[0];
  for (int w = 1; w < 4; ++w) top = fmaxf(top, part_m[w]);
  float sum = 0.f, all = 0.f;
  for (int w = 0; w < 4; ++w) {
    const float of_wave = weight_of(part_m[w], top);
    sum += part_o[w][d] * of_wave;
    all += part_l[w] * of_wave;
  }
  // (nothing seen: 0)
  store_f32<T>(static_cast<T*>(a.out) + at + d, all == 0.f ? 0.f : sum / all);
}

// ---------------------------------------------------------------------------
// The same on the matrix cores, for rows of 16 values and more.
//
// The query heads that share a key / value head are a tile of 16 columns (a group has
// several where it is larger, empty columns where it is smaller), 16 positions the tile's
// rows: logits^T [position][head] = K . q^T, out^T [value][head] = V^T . w^T.  The first
// product leaves lane 16 j + c with the logits of head c for positions 4 j .. 4 j + 3,
// which is where the second one wants the weights of its reduction index, so that nothing
// but two steps of a maximum crosses lanes.  Keys and values go from memory to registers in
// the forms that the products take:
//   keys    lane 16 j + c the pieces j, j + 4, .. of 16 bytes of position c (reductions
//           take the pieces in whatever order the queries have them, too)
//   values  lane 16 j + c the values of chunk c of positions 4 j .. 4 j + 3, so that 16
//           lanes read a whole row; pairs of positions are put together (bfloat16) by
//           v_perm, and a lane's results are neighbours in the output
// Bound by the memory: a position costs 2 D values of traffic for 4 D operations a head,
// and the products of 16 columns take a twentieth of the matrix cores' time.  Four
// wavefronts take turns with groups of NS x 16 positions, without barriers; what they have
// in flight at once is what hides the memory's latency.  One sequence of 131072 positions,
// 8 key / value heads of 128, 8 bits: 42 us, 6.4 TB/s when repeated, as some of the 270 MB
// stay in the last level's cache; 128 of up to 16384 in bfloat16: 715 us, 6.05 TB/s (a kernel
// that only reads reaches 6.3).  A wavefront's next group is not loaded ahead of the one in
// use: the registers for it cost the second block of a CU, and two blocks take turns as well
// (64 sequences of up to 8192: 121 us with, 118 without; rows of 256, 87 and 71).
//
// The work is dealt out evenly to one to three blocks a CU (at_once), by what the sequences'
// lengths turn out to be on the device (run_of).  Where a unit's positions fall
// to several blocks, their triples go to the workspace, and cache_attention_join_kernel
// puts them together.  (In the same launch, by the block of a unit that is done last, a
// join costs its block round trips to a memory that is busy with the others' streams: 64
// sequences of up to 8192, 130 us instead of 125.)  Where there are many units and all are
// short, every wavefront has units of its own.
// ---------------------------------------------------------------------------
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

// two 8-bit values of a word, times their unit, in bfloat16 (exact)
template <bool HIGH>
__device__ __forceinline__ uint32_t widened(uint32_t word, float unit) {
  return __builtin_bit_cast(
      uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, unit, HIGH));
}

// ... the four of a word in float32
__device__ __forceinline__ void four_floats(uint32_t word, float unit, float (&f)[4]) {
  const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)word, false);
  const f32x2_t hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)word, true);
  f[0] = lo[0] * unit;
  f[1] = lo[1] * unit;
  f[2] = hi[0] * unit;
  f[3] = hi[1] * unit;
}

constexpr int HEADS = 16;                          // columns of a tile

// N values (a multiple of 4) to neighbouring places, but for the first `skip`.
template <typename T, int N>
__device__ __forceinline__ void store_some(T* to, const float (&f)[N], int skip) {
  if (skip != 0) {
#pragma unroll
    for (int u = 0; u < N; ++u)
      if (u >= skip) store_f32<T>(to + u, f[u]);
    return;
  }
#pragma unroll
  for (int u = 0; u < N; u += 4) {
    if constexpr (sizeof(T) == 2)
      *reinterpret_cast<Words<8>::type*>(to + u) = Words<8>::type{
          f32x2_to_bf16x2(f[u], f[u + 1]), f32x2_to_bf16x2(f[u + 2], f[u + 3])};
    else
      *reinterpret_cast<Words<16>::type*>(to + u) =
          Words<16>::type{__float_as_uint(f[u]), __float_as_uint(f[u + 1]),
                          __float_as_uint(f[u + 2]), __float_as_uint(f[u + 3])};
  }
}

template <typename T, bool EIGHT, int DP>
struct TileOf {
  static constexpr int SIZE = EIGHT ? 1 : (int)sizeof(T);      // of a value in a page
  static constexpr int KV = 16 / SIZE;                         // values of a key's piece
  static constexpr int KC = DP / (4 * KV);                     // a lane's pieces of a key
  static constexpr int VD = DP / 16;                           // a lane's values of a row,
  static constexpr int VB = VD * SIZE < 16 ? VD * SIZE : 16;   // in pieces of VB bytes
  static constexpr int VP = VD * SIZE / VB;
  static constexpr int VE = VB / SIZE;                         // values of a piece
  static constexpr bool WIDE = sizeof(T) == 4;                 // float32 products
  // Groups of 16 positions that a wavefront has in registers at once: as many as leave the
  // blocks below their registers.  (8 bits, 128 values, 64 sequences of up to 8192: 125 us
  // by 2, 115 by 4; bfloat16, 64 values, by 4 with two blocks 18.5, by 2 with three 17.4.
  // Padded 8-bit rows of 65 to 127 values do not have the registers for 4 in pages of 4 and 8
  // rows, where 28 bytes a lane go to scratch memory, and of 1 and 2, where it is 84; 2 has
  // not been timed there.)
  static constexpr int NS =
      WIDE ? (EIGHT ? (DP == 256 ? 1 : 2) : (DP == 64 ? 2 : 1))
           : (EIGHT && DP < 256 ? 4 : 2);
  static constexpr int GRAIN = 4 * 16 * NS;                    // positions of four wavefronts
  // Blocks that divided work counts on in a CU, and that the registers are kept below for.
  // (Rows of 256, 16 sequences of 16384, 8 bits: 79 us by one, 72 by two; bfloat16, where two
  // do not have the registers for it, 100 and 125.)  Some kernels without padding come out
  // with registers for more, which has not been timed: 8-bit rows of 64 (153 of them) and
  // float32 ones (155) for three, 8-bit ones under float32 for four (119; of 128, 157, for
  // three), bfloat16 ones of 64 (117) for four.
  template <bool PADDED>
  static constexpr int at_once() {
    return DP == 256 && !(EIGHT && !PADDED) ? 1 : DP == 64 && !EIGHT && !WIDE ? 3 : 2;
  }
  // grains that are not divided among blocks (see divide)
  static constexpr int WHOLE = DP == 64 && !EIGHT && !WIDE ? 8 : 4;
  // positions of a wavefront's own units (see divide): eight turns
  static constexpr int ALONE = 8 * 16 * NS;
};

// How the work is divided.  A unit is a key / value head of a sequence with a tile of its
// query heads; its positions come in grains of Tile::GRAIN (one at least).  The grains of
// all units, sequence by sequence, are dealt out in runs of equal length, a block each.
struct Shares {
  int units;                      // of a sequence
  int grain;
  int blocks;                     // at most; 0: a block for every unit
  // Where no sequence has more than `alone` positions, every wavefront takes units of its
  // own instead; blocks = 0: whether that is so (not 0) is known from the table's size.
  int alone;
};
// A unit's first positions take their block about as long to begin with and to put away as
// a grain of them to go through: units count as that much longer.  (64 sequences of up to
// 8192: 125 us without it, 115 with one grain, 118 with two.)
constexpr int AHEAD = 1;

// grains of a unit, those ahead of the first included
__device__ __forceinline__ int grains_of(int seen, int grain) {
  return max((seen + grain - 1) / grain, 1) + AHEAD;
}

// Sums over the lanes up to each, in six steps without LDS.
__device__ __forceinline__ int sums_up_to(int v) {
#define STEP(ctrl, rows)                                                              \
  v += __builtin_amdgcn_update_dpp(0, v, ctrl, rows, 0xf, false)
  STEP(0x111, 0xf);               // row_shr by 1, 2, 4, 8
  STEP(0x112, 0xf);
  STEP(0x114, 0xf);
  STEP(0x118, 0xf);
  STEP(0x142, 0xa);               // a row's last lane to the next row
  STEP(0x143, 0xc);               // ... to the next two
#undef STEP
  return v;
}

// A block's run of grains, and where the first one is.
struct Run {
  int first, count;               // of all grains
  int b, unit, grain;             // sequence, unit and grain of that
  int of_unit;                    // grains of that unit
  int of_all;                     // ... and of all units
};
struct Runs {
  int blocks, each, longer;       // `longer` of the blocks have one grain more than `each`
  __device__ __forceinline__ Runs(const Shares& s, int grains) {
    blocks = min(s.blocks, grains);
    each = grains / blocks;
    longer = grains - each * blocks;
  }
  __device__ __forceinline__ int first(int block) const {
    return block * each + min(block, longer);
  }
  __device__ __forceinline__ int block_of(int grain) const {
    const int more = longer * (each + 1);
    return grain < more ? grain / (each + 1) : longer + (grain - more) / each;
  }
};

// false for a block without work; *alone: every wavefront takes units of its own, and there
// is no run (MANY: s.alone may be set).  The same for all lanes of a wavefront.
template <bool MANY>
__device__ __forceinline__ bool run_of(const Attention& a, const Shares& s, int block,
                                       Run* run, bool* alone) {
  const int lane = threadIdx.x & 63;
  run->count = 0;
  *alone = MANY && s.blocks == 0 && s.alone != 0;
  if (*alone) return true;
  if (s.blocks == 0) {
    run->b = block / s.units;
    run->unit = block - run->b * s.units;
    run->first = run->grain = 0;
    run->count = run->of_unit = grains_of(seen_of(a, run->b), s.grain);
    return true;
  }
  bool longer = false;
  auto grains = [&](int b) {
    const int seen = seen_of(a, min(b, a.B - 1));    // (no branch around the load)
    longer = longer || seen > s.alone;
    return b < a.B ? grains_of(seen, s.grain) : 0;
  };
  const int of_lane = grains(lane);
  int up_to = sums_up_to(of_lane), all = __builtin_amdgcn_readlane(up_to, 63);
  if (a.B > 64) {
    int rest = 0;
    for (int b = 64; b < a.B; b += 256) {
#pragma unroll
      for (int i = 0; i < 4; ++i) rest += grains(b + 64 * i + lane);
    }
    all += __builtin_amdgcn_readlane(sums_up_to(rest), 63);
  }
  *alone = MANY && s.alone != 0 && !__any(longer);
  if (*alone) return true;
  run->of_all = all * s.units;
  const Runs runs(s, run->of_all);
  if (block >= runs.blocks) return false;
  run->first = runs.first(block);
  run->count = runs.each + (block < runs.longer ? 1 : 0);
  int before = 0, count = of_lane;                   // grains of units of one kind
  for (int b = 0;; b += 64) {
    const uint64_t behind =
        __ballot((int64_t)(before + up_to) * s.units > (int64_t)run->first);
    if (behind) {
      const int at = __builtin_ctzll(behind);
      run->b = b + at;
      run->of_unit = __builtin_amdgcn_readlane(count, at);
      const int in = run->first - (before + __builtin_amdgcn_readlane(up_to, at) -
                                   run->of_unit) * s.units;
      run->unit = in / run->of_unit;
      run->grain = in - run->unit * run->of_unit;
      return true;
    }
    before += __builtin_amdgcn_readlane(up_to, 63);
    if (b + 64 >= a.B) return false;                 // (not reached)
    count = grains(b + 64 + lane);
    up_to = sums_up_to(count);
  }
}

// A wavefront keeps the step's key (of = 0) or value: in `row` and `units`, and in the page
// where `writes` says so.
template <typename T, bool EIGHT>
__device__ __forceinline__ void keep_row(const Attention& a, int of, int b, int kv_head,
                                         int64_t to, bool writes, uint8_t* row,
                                         uint8_t* units) {
  const int lane = threadIdx.x & 63, D = a.pages.D, at = lane * 8;
  const bool own = of == 0 || a.v_new != nullptr;    // (else the key is the value)
  const T* x = static_cast<const T*>(of && own ? a.v_new : a.k_new) +
               ((int64_t)b * a.pages.HK + kv_head) * D;
  void* pages = const_cast<void*>(of ? a.v_pages : a.k_pages);
  uint8_t* scales = const_cast<uint8_t*>(of ? a.v_scales : a.k_scales);
  float f[8];
  load8<T, false>(x, at, D, f);
  if constexpr (EIGHT) {
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, magnitude_bits(f[e]));
    const Fp8Scale s = fp8_scale(max_of_lanes(top, 16));
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] *= s.factor;
    const uint32_t lo = fp8_pack4(f[0], f[1], f[2], f[3]);
    const uint32_t hi = fp8_pack4(f[4], f[5], f[6], f[7]);
    if (at < D) {
      store_eight<false>(row, at, D, lo, hi);
      if (writes && own)
        store_eight<false>(static_cast<uint8_t*>(pages) + to * D, at, D, lo, hi);
    }
    if (at < D && lane % 16 == 0) {
      units[lane / 16] = (uint8_t)s.byte;
      if (writes && own) scales[to * a.pages.DB + lane / 16] = (uint8_t)s.byte;
    }
  } else {
    if (at < D) {
      T* kept = reinterpret_cast<T*>(row);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (at + e < D) store_f32<T>(kept + at + e, f[e]);
      if (writes && own) store8<T, false>(static_cast<T*>(pages) + to * D, at, D, f);
    }
  }
}

// Units that fall to several blocks.  A block has a place in the workspace for the triple
// of the unit it begins with (if that began before) and one for the unit it ends with.
struct Part {                     // a unit's parts are those of blocks from, from + 1, ..
  int b, unit, from, parts;       // (1: it is whole, 0: there is none)
};
struct Joins {
  float2* tops;                   // [places][columns]: largest logit, sum of weights
  float2* sums;                   // [places][columns][(D + 1) / 2]: two values each
  // For the launch that joins them, null if there is none: of every unit, or (where blocks
  // are fewer) of every block the unit that others go on with.
  Part* parts;
  bool of_units;
};
// the place of part `part` of a unit whose first block is `from`
__device__ __forceinline__ int64_t place_of(int from, int part) {
  return 2 * (int64_t)(from + part) + (part == 0 ? 1 : 0);
}

// What a wavefront has of NS x 16 positions: words of keys and values as the products take
// them, their scale bytes, and which of the pages are there.  SMALL: 0 for pages of
// 16 rows and more, 1 of 4 or 8, 2 of 1 or 2.
template <typename T, bool EIGHT, int DP, int SMALL>
struct Group {
  typedef TileOf<T, EIGHT, DP> Tile;
  static constexpr int NS = Tile::NS, BLOCKS = DP == 256 ? 2 : 1;
  uint32_t k[NS][Tile::KC][4], v[NS][4][Tile::VP][Tile::VB / 4];
  uint32_t k_units[NS];                      // a byte for each block of the lane's key
  static constexpr int PAGES = SMALL == 2 ? 4 : 1;   // of a lane's values
  uint32_t v_units[NS][SMALL == 2 ? 4 : BLOCKS];     // [4 rows][blocks] bytes, of each row
  bool there[NS][PAGES];                     // the values' pages
};

// What a scale byte (bits 8 n .. of the word) stands for.
__device__ __forceinline__ float unit_in(uint32_t word, int n) {
  return __uint_as_float((n < 3 ? word << (23 - 8 * n) : word >> 1) & 0x7f800000u);
}

// PADDED: rows of fewer than DP values, or on any address.  MANY: wavefronts may take units
// of their own; without it there is less code, which every block of a short launch waits for
// (one sequence of 1600, 8 heads of 128: 10.2 us with, 9.8 without).
template <typename T, bool EIGHT, int DP, bool PADDED, int SMALL, bool MANY>
__global__ __launch_bounds__(256, (TileOf<T, EIGHT, DP>::template at_once<PADDED>()))
void cache_attention_tiles_kernel(Attention a, Shares shares, Joins joins) {
  typedef TileOf<T, EIGHT, DP> Tile;
  typedef Group<T, EIGHT, DP, SMALL> Group;
  constexpr int NS = Tile::NS, KC = Tile::KC, KV = Tile::KV, SIZE = Tile::SIZE;
  constexpr int VD = Tile::VD, VP = Tile::VP, VE = Tile::VE, VB = Tile::VB;
  constexpr int VW = VB / 4;                         // words of a value's piece
  constexpr int PAGES = Group::PAGES, PER_PAGE = 4 / PAGES;
  extern __shared__ __attribute__((aligned(16))) float joined[];
  __shared__ __attribute__((aligned(16))) uint8_t fresh_of[4][2][DP * SIZE];
  __shared__ uint8_t fresh_units_of[4][2][2];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (joins.parts && !joins.of_units && threadIdx.x == 0)
    joins.parts[blockIdx.x] = Part{0, 0, 0, 0};
  Run run;
  bool alone;
  if (!run_of<MANY>(a, shares, (int)blockIdx.x, &run, &alone)) return;
  auto& fresh_rows = fresh_of[alone ? wave : 0];
  auto& fresh_units = fresh_units_of[alone ? wave : 0];
  const int c = lane & 15, j = lane >> 4;
  const int D = PADDED ? a.pages.D : DP, S = 1 << a.pages.shift;
  const int DB = DP == 256 ? 2 : 1;
  const int tiles = (a.G + HEADS - 1) / HEADS, columns = min(a.G, HEADS);
  const uint8_t* k_pages = static_cast<const uint8_t*>(a.k_pages);
  const uint8_t* v_pages = static_cast<const uint8_t*>(a.v_pages);

  // Where a lane's pieces of a row begin.  A piece that would end behind the row begins
  // as much earlier; its first `extra` values are another piece's.
  int k_at[KC], v_at[VP], k_extra[KC], v_extra[VP];
#pragma unroll
  for (int i = 0; i < KC; ++i) {
    const int at = (j + 4 * i) * KV;
    k_at[i] = PADDED ? min(at, D - KV) : at;
    k_extra[i] = at - k_at[i];
  }
#pragma unroll
  for (int p = 0; p < VP; ++p) {
    const int at = p * 16 * VE + c * VE;
    v_at[p] = PADDED ? min(at, D - VE) : at;
    v_extra[p] = at - v_at[p];
  }

  int left = run.count, id = (int)blockIdx.x * 4 + wave;   // (id: of the unit of this wavefront)
  while (alone ? id < a.B * shares.units : left > 0) {
    // ---- the next unit, or what of it falls to this block
    if (alone) {
      run.b = id / shares.units;
      run.unit = id - run.b * shares.units;
      run.grain = 0;
      run.of_unit = left = 1 << 30;                  // (all of it)
      id += (int)gridDim.x * 4;
    }
    const int b = __builtin_amdgcn_readfirstlane(run.b);
    const int unit = __builtin_amdgcn_readfirstlane(run.unit);
    const int taken = min(left, run.of_unit - run.grain);
    const int from_grain = max(run.grain - AHEAD, 0), to_grain = run.grain + taken - AHEAD;
    const bool begins = from_grain == 0, ends = run.grain + taken == run.of_unit;
    left -= taken;
    if (to_grain <= 0 || b >= a.B) break;            // (only what is ahead: the run's end)
    const int kv_head = unit / tiles, head0 = (unit - kv_head * tiles) * HEADS;
    const int heads = min(a.G - head0, HEADS);       // columns in use
    const int64_t first_head = (int64_t)kv_head * a.G + head0;
    const int last = scalar_load(a.position + b), seen = seen_from(a, last);
    const int first = from_grain * Tile::GRAIN;
    const int end = (int)min((int64_t)to_grain * Tile::GRAIN, (int64_t)seen);
    const int32_t* table = a.pages.table + (int64_t)b * a.pages.P;
    const int step = alone ? 16 * NS : Tile::GRAIN;
    const int start = alone ? 0 : first + wave * (16 * NS);

    // The pages of the 16 positions from t0 + 16 s on, SMALL: of the lane's key and values;
    // behind the end, that of the last one.
    struct Looked { int k, v[PAGES]; };
    auto look_up = [&](int t0, Looked (&page)[NS]) {
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const int t = t0 + 16 * s, most = max(end - 1, 0);
        if constexpr (SMALL) {
          page[s].k = table[min(t + c, most) >> a.pages.shift];
#pragma unroll
          for (int n = 0; n < PAGES; ++n)
            page[s].v[n] = table[min(t + 4 * j + n, most) >> a.pages.shift];
        } else {
          page[s].k = page[s].v[0] = scalar_load(table + (min(t, most) >> a.pages.shift));
        }
      }
    };
    // Loads positions t0 .. t0 + 16 NS - 1; what of them is not there, or not before the end,
    // is read from rows that are, and left out when it is used.
    auto load = [&](int t0, const Looked (&page)[NS], Group& g) {
      // row number of position t in a page, 0 for a page that is not there
      auto row_in = [&](int page, int t) {
        const int there = (unsigned)page < (unsigned)a.pages.N ? page : 0;
        return (((int64_t)there * a.pages.HK + kv_head) << a.pages.shift) + (t & (S - 1));
      };
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        // (not SMALL: of the 16 positions' first)
        const int64_t row =
            row_in(page[s].k, SMALL ? t0 + 16 * s + c : min(t0 + 16 * s, end - 1) & ~15);
        const uint8_t* from = k_pages + row * D * SIZE;
#pragma unroll
        for (int i = 0; i < KC; ++i)
          if (!PADDED || k_extra[i] < KV)
            load_words<16>(from + (uint32_t)(((SMALL ? 0 : c * D) + k_at[i]) * SIZE),
                           g.k[s][i]);
        if constexpr (EIGHT) {
          const uint8_t* units = a.k_scales + row * DB + (SMALL ? 0 : c * DB);
          g.k_units[s] = DB == 2 ? units[0] | (uint32_t)units[1] << 8 : units[0];
        }
      }
#pragma unroll
      for (int s = 0; s < NS; ++s) {
#pragma unroll
        for (int n = 0; n < PAGES; ++n) {
          const int64_t row = row_in(page[s].v[n], SMALL ? t0 + 16 * s + 4 * j + n
                                                         : min(t0 + 16 * s, end - 1) & ~15);
          const uint8_t* from = v_pages + row * D * SIZE;
          g.there[s][n] = (unsigned)page[s].v[n] < (unsigned)a.pages.N;
#pragma unroll
          for (int r = 0; r < PER_PAGE; ++r)
#pragma unroll
            for (int p = 0; p < VP; ++p)
              if (!PADDED || v_extra[p] < VE)
                load_words<VB>(from + r * D * SIZE +
                                   (uint32_t)(((SMALL ? 0 : 4 * j * D) + v_at[p]) * SIZE),
                               g.v[s][n + r][p]);
          if constexpr (EIGHT && SMALL == 2) {
            const uint8_t* units = a.v_scales + row * DB;
            g.v_units[s][n] = DB == 2 ? units[0] | (uint32_t)units[1] << 8 : units[0];
          } else if constexpr (EIGHT) {
            load_words<4 * Group::BLOCKS>(
                a.v_scales + row * DB + (SMALL ? 0 : 4 * j * DB), g.v_units[s]);
          }
        }
      }
    };

    // zeros for the first bytes of a piece: another's values do not count twice
    auto without_first = [](int bytes, uint32_t (&w)[4]) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int bits = min(max(bytes * 8 - 32 * e, 0), 32);
        w[e] &= bits == 32 ? 0u : ~0u << bits;
      }
    };

    // ---- the queries, as the second operand of the first product; 0 where there is no head
    Looked page[NS];
    look_up(start, page);
    constexpr int QN = Tile::WIDE ? KC * KV : KC * KV / 8;
    typedef std::conditional_t<Tile::WIDE, float, bf16x8_t> query_t;
    query_t q[QN];
    {
      const T* row = static_cast<const T*>(a.q) +
                     ((int64_t)b * a.H + first_head + min(c, heads - 1)) * D;
      constexpr int PER = 16 / sizeof(T);            // values of 16 bytes of q
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        const bool there = c < heads && (!PADDED || k_extra[i] < KV);
#pragma unroll
        for (int u = 0; u < KV / PER; ++u) {
          uint32_t w[4] = {0, 0, 0, 0};
          if (there)
            load_words<16>(reinterpret_cast<const uint8_t*>(row + k_at[i] + u * PER), w);
          if constexpr (PADDED) without_first((k_extra[i] - u * PER) * (int)sizeof(T), w);
          if constexpr (Tile::WIDE) {
#pragma unroll
            for (int e = 0; e < 4; ++e) q[i * KV + u * 4 + e] = __uint_as_float(w[e]);
          } else {
            q[i * (KV / 8) + u] =
                __builtin_bit_cast(bf16x8_t, make_uint4(w[0], w[1], w[2], w[3]));
          }
        }
      }
    }

    // The step's own row: written by the block that ends its unit (of the head's first
    // tile), which reads it from LDS.
    bool fresh = false;
    if (a.k_new && ends && last >= 0) {
      const int64_t to = a.pages.row(b, last);
      fresh = to >= 0;
      if (fresh) {
        auto wait = [&] {
          if (alone) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          else __syncthreads();
        };
        wait();                                      // (the unit before is done with them)
#pragma unroll 1
        for (int of = alone ? 0 : wave; of < 2; of += alone ? 1 : 2)
          keep_row<T, EIGHT>(a, of, b, kv_head, a.pages.head(to, kv_head), head0 == 0,
                             fresh_rows[of], fresh_units[of]);
        wait();
      }
    }

    // the relative biases of the lane's head, and that of all positions far away
    const T* rel_row = nullptr;
    float far_bias = 0.f;
    if (a.rel_values) {
      rel_row = static_cast<const T*>(a.rel_values) +
                (first_head + min(c, heads - 1)) * a.NB;
      far_bias = load_f32<T>(rel_row + bucket_of(a, 1 - a.reach));
    }

    f32x4_t o[VD];
#pragma unroll
    for (int t = 0; t < VD; ++t) o[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;

    // the scale bytes of the values of a lane's row r
    auto set_units = [&](Group& g, int s, int r, uint32_t units) {
      if constexpr (SMALL == 2) {
        g.v_units[s][r] = units;
      } else {
        const int bits = 8 * DB * (r % (4 / DB));
        uint32_t& word = g.v_units[s][r * DB / 4];
        word = (word & ~((DB == 2 ? 0xffffu : 0xffu) << bits)) |
               (DB == 2 ? units : units & 0xffu) << bits;
      }
    };

    // ---- a group's positions into m, l and o
    auto use = [&](int t0, Group& g) {
      if (PADDED) {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
#pragma unroll
          for (int i = 0; i < KC; ++i)
            if (k_extra[i] >= KV)
#pragma unroll
              for (int w = 0; w < 4; ++w) g.k[s][i][w] = 0;
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int p = 0; p < VP; ++p)
              if (v_extra[p] >= VE)
#pragma unroll
                for (int w = 0; w < VW; ++w) g.v[s][r][p][w] = 0;
        }
      }
      if (fresh && t0 <= last && last < t0 + 16 * NS) {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          if (t0 + 16 * s + c == last) {
#pragma unroll
            for (int i = 0; i < KC; ++i)
              if (!PADDED || k_extra[i] < KV)
                load_words<16>(fresh_rows[0] + k_at[i] * SIZE, g.k[s][i]);
            if (EIGHT) g.k_units[s] = fresh_units[0][0] | (uint32_t)fresh_units[0][1] << 8;
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (t0 + 16 * s + 4 * j + r != last) continue;
#pragma unroll
            for (int p = 0; p < VP; ++p)
              if (!PADDED || v_extra[p] < VE)
                load_words<VB>(fresh_rows[1] + v_at[p] * SIZE, g.v[s][r][p]);
            if constexpr (EIGHT)
              set_units(g, s, r, fresh_units[1][0] | (uint32_t)fresh_units[1][1] << 8);
          }
        }
      }
      // -- logits
      float x[NS][4];
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < KC; ++i) {
          uint32_t* w = g.k[s][i];
          if constexpr (PADDED) without_first(k_extra[i] * SIZE, g.k[s][i]);
          if constexpr (EIGHT) {
            const float unit = unit_in(g.k_units[s], DP == 256 ? i / 2 : 0);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              if constexpr (Tile::WIDE) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  float f[4];
                  four_floats(w[2 * half + e], unit, f);
#pragma unroll
                  for (int u = 0; u < 4; ++u)
                    sum = __builtin_amdgcn_mfma_f32_16x16x4f32(
                        f[u], q[i * KV + 8 * half + 4 * e + u], sum, 0, 0, 0);
                }
              } else {
                uint4 wide;
                wide.x = widened<false>(w[2 * half], unit);
                wide.y = widened<true>(w[2 * half], unit);
                wide.z = widened<false>(w[2 * half + 1], unit);
                wide.w = widened<true>(w[2 * half + 1], unit);
                sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    __builtin_bit_cast(bf16x8_t, wide), q[i * 2 + half], sum, 0, 0, 0);
              }
            }
          } else if constexpr (Tile::WIDE) {
#pragma unroll
            for (int u = 0; u < 4; ++u)
              sum = __builtin_amdgcn_mfma_f32_16x16x4f32(
                  __uint_as_float(w[u]), q[i * KV + u], sum, 0, 0, 0);
          } else {
            sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                __builtin_bit_cast(bf16x8_t, make_uint4(w[0], w[1], w[2], w[3])), q[i], sum,
                0, 0, 0);
          }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) x[s][r] = sum[r];
      }
      if (a.rel_values) {
        if (last - (t0 + 16 * NS - 1) >= a.reach - 1) {
#pragma unroll
          for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int r = 0; r < 4; ++r) x[s][r] += far_bias;
        } else {
          // (all loads of a kind at once)
          int bucket[NS][4];
#pragma unroll
          for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              bucket[s][r] = bucket_of(a, min(t0 + 16 * s + 4 * j + r, end - 1) - last);
          float bias[NS][4];
#pragma unroll
          for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int r = 0; r < 4; ++r) bias[s][r] = load_f32<T>(rel_row + bucket[s][r]);
#pragma unroll
          for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int r = 0; r < 4; ++r) x[s][r] += bias[s][r];
        }
      }
      bool whole = t0 + 16 * NS <= end;
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int n = 0; n < PAGES; ++n) whole = whole && g.there[s][n];
      if (SMALL ? !__all(whole) : !whole) {
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (g.there[s][r / PER_PAGE] && t0 + 16 * s + 4 * j + r < end) continue;
            x[s][r] = -INFINITY;
#pragma unroll
            for (int p = 0; p < VP; ++p)
#pragma unroll
              for (int w = 0; w < VW; ++w) g.v[s][r][p][w] = 0;
            if constexpr (EIGHT) set_units(g, s, r, 0);   // (255 times 0 is NaN)
          }
      }
      // -- weights
      float top = m;
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, x[s][r]);
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      if (__any(top > m)) {
        const float was = weight_of(m, top);
        l *= was;
#pragma unroll
        for (int t = 0; t < VD; ++t) o[t] *= was;
        m = top;
      }
      uint32_t pairs[NS][2];                         // of weights (bfloat16)
#pragma unroll
      for (int s = 0; s < NS; ++s) {
#pragma unroll
        for (int r = 0; r < 4; ++r) x[s][r] = weight_of(x[s][r], m);
        if constexpr (!Tile::WIDE) {
          pairs[s][0] = f32x2_to_bf16x2(x[s][0], x[s][1]);
          pairs[s][1] = f32x2_to_bf16x2(x[s][2], x[s][3]);
          // (Rounded, as the products of bfloat16 values on the matrix cores take them; the
          // sum is of what is multiplied, so that weights add up to 1.  Against 64 bits, 128
          // sequences of up to 16384 are off by 0.0017 of the result's norm, with weights
          // in float32 by 0.0016: the result's own rounding is most of both.)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            l += __uint_as_float(pairs[s][e] << 16) +
                 __uint_as_float(pairs[s][e] & 0xffff0000u);
        } else {
          l += (x[s][0] + x[s][1]) + (x[s][2] + x[s][3]);
        }
      }
      // -- sums of values
      auto v_unit = [&](int s, int r) {
        if constexpr (!EIGHT) return 1.f;
        else if constexpr (SMALL == 2)
          return DB == 2 && c >= 8 ? unit_in(g.v_units[s][r], 1) : unit_in(g.v_units[s][r], 0);
        else if constexpr (DB == 2)
          return c >= 8 ? unit_in(g.v_units[s][r / 2], r % 2 * 2 + 1)
                        : unit_in(g.v_units[s][r / 2], r % 2 * 2);
        else
          return unit_in(g.v_units[s][0], r);
      };
      if constexpr (Tile::WIDE) {
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float unit = v_unit(s, r);
#pragma unroll
            for (int p = 0; p < VP; ++p)
#pragma unroll
              for (int w = 0; w < VW; ++w) {
                const uint32_t word = g.v[s][r][p][w];
                if constexpr (EIGHT) {
                  float f[4];
                  four_floats(word, unit, f);
#pragma unroll
                  for (int u = 0; u < 4; ++u)
                    o[p * VE + 4 * w + u] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                        f[u], x[s][r], o[p * VE + 4 * w + u], 0, 0, 0);
                } else {
                  o[p * VE + w] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                      __uint_as_float(word), x[s][r], o[p * VE + w], 0, 0, 0);
                }
              }
          }
      } else {
#pragma unroll
        for (int s = 0; s < NS; s += 2) {
          const bf16x8_t w = __builtin_bit_cast(
              bf16x8_t,
              make_uint4(pairs[s][0], pairs[s][1], pairs[s + 1][0], pairs[s + 1][1]));
          float unit[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) unit[e] = v_unit(s + e / 4, e % 4);
#pragma unroll
          for (int p = 0; p < VP; ++p)
#pragma unroll
            for (int pair = 0; pair < VE / 2; ++pair) {
              uint32_t two[8];                       // values 2 pair, 2 pair + 1 of 8 positions
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const uint32_t* words = g.v[s + e / 4][e % 4][p];
                if constexpr (EIGHT)
                  two[e] = pair & 1 ? widened<true>(words[pair / 2], unit[e])
                                    : widened<false>(words[pair / 2], unit[e]);
                else
                  two[e] = words[pair];
              }
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                constexpr uint32_t PICK[2] = {0x05040100u, 0x07060302u};
                uint4 v;
                v.x = __builtin_amdgcn_perm(two[1], two[0], PICK[u]);
                v.y = __builtin_amdgcn_perm(two[3], two[2], PICK[u]);
                v.z = __builtin_amdgcn_perm(two[5], two[4], PICK[u]);
                v.w = __builtin_amdgcn_perm(two[7], two[6], PICK[u]);
                f32x4_t& sum = o[p * VE + 2 * pair + u];
                sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    __builtin_bit_cast(bf16x8_t, v), w, sum, 0, 0, 0);
              }
            }
        }
      }
    };

    // (the pages of the next group are looked up while this one is used)
    for (int t0 = start; t0 < end; t0 += step) {
      Group g;
      load(t0, page, g);
      look_up(t0 + step, page);
      use(t0, g);
    }

    // ---- the result, or the four wavefronts' triples
    // (known again only now, so that the places below are not computed ahead of the
    // positions and held in registers meanwhile)
    int column = c, rows = 4 * j;
    asm volatile("" : "+v"(column), "+v"(rows));
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    T* out = static_cast<T*>(a.out) + ((int64_t)b * a.H + first_head) * D;
    if (alone) {
      if (column < heads) {
        const float of_all = 1.f / l;
#pragma unroll
        for (int p = 0; p < VP; ++p)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            // (row 4 j + r of the product is what lane c = 4 j + r read)
            const int at = p * 16 * VE + (rows + r) * VE;
            if (PADDED && at >= D) continue;
            const int from = PADDED ? min(at, D - VE) : at;
            float f[VE];
#pragma unroll
            for (int u = 0; u < VE; ++u)             // (nothing seen: 0)
              f[u] = l == 0.f ? 0.f : o[p * VE + u][r] * of_all;
            store_some<T, VE>(out + (int64_t)column * D + from, f, at - from);
          }
      }
      continue;
    }
    float* ms = joined;                              // [4][HEADS]
    float* ls = ms + 4 * HEADS;                      // [4][HEADS]
    float* os = ls + 4 * HEADS;                      // [4][heads][D]
    __syncthreads();                                 // (the unit before is done with them)
    if (lane < HEADS) {
      ms[wave * HEADS + lane] = m;
      ls[wave * HEADS + lane] = l;
    }
    if (column < heads) {
      float* to = os + (wave * heads + column) * D;
#pragma unroll
      for (int p = 0; p < VP; ++p)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          // (row 4 j + r of the product is what lane c = 4 j + r read)
          const int at = p * 16 * VE + (rows + r) * VE;
          if (!PADDED || D % VE == 0) {
            if (!PADDED || at < D)
#pragma unroll
              for (int u = 0; u < VE; ++u) to[at + u] = o[p * VE + u][r];
          } else {
            const int from = min(at, D - VE);
#pragma unroll
            for (int u = 0; u < VE; ++u)
              if (from + u >= at && at < D) to[from + u] = o[p * VE + u][r];
          }
        }
    }
    __syncthreads();
    const bool whole_unit = begins && ends;
    const int64_t place = 2 * (int64_t)blockIdx.x + (begins ? 1 : 0);
    if (joins.parts && begins && (!ends || joins.of_units) && threadIdx.x == 0) {
      // (the unit's last grain, of all)
      const int to = run.first + run.count - left - taken - run.grain + run.of_unit - 1;
      const int from = (int)blockIdx.x;
      joins.parts[joins.of_units ? b * shares.units + unit : from] =
          Part{b, unit, from, ends ? 1 : Runs(shares, run.of_all).block_of(to) - from + 1};
    }
    // (two values a thread, as they go to the workspace)
    const int halves = (D + 1) / 2;
    for (int i = threadIdx.x; i < heads * halves; i += 256) {
      const int h = i / halves, d = 2 * (i - h * halves);
      float top = ms[h];
#pragma unroll
      for (int w = 1; w < 4; ++w) top = fmaxf(top, ms[w * HEADS + h]);
      float sum[2] = {0.f, 0.f}, all = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float factor = weight_of(ms[w * HEADS + h], top);
        const float* from = os + (w * heads + h) * D + d;
        sum[0] += from[0] * factor;
        if (!PADDED || d + 1 < D) sum[1] += from[1] * factor;
        all += ls[w * HEADS + h] * factor;
      }
      if (whole_unit) {
        // (nothing seen: 0)
        store_f32<T>(out + (int64_t)h * D + d, all == 0.f ? 0.f : sum[0] / all);
        if (!PADDED || d + 1 < D)
          store_f32<T>(out + (int64_t)h * D + d + 1, all == 0.f ? 0.f : sum[1] / all);
      } else {
        joins.sums[(place * columns + h) * halves + d / 2] = make_float2(sum[0], sum[1]);
        if (d == 0) joins.tops[place * columns + h] = make_float2(top, all);
      }
    }
    run.grain = 0;
    run.unit = unit + 1;
    if (run.unit == shares.units) {
      run.unit = 0;
      run.b = b + 1;
      if (left > 0)
        run.of_unit = grains_of(seen_from(a, scalar_load(a.position + b + 1)), shares.grain);
    }
  }
}

// Puts the parts of a unit together.  Block (x, y): the unit of joins.parts[x], `per` (a power
// of two) of its heads' pairs of values; 256 / per groups of threads take every so many-th
// part.
template <typename T>
__global__ __launch_bounds__(256) void cache_attention_join_kernel(Attention a, Joins joins,
                                                                   int per) {
  constexpr int IN_FLIGHT = 16;
  __shared__ float tops[256], alls[256], sums[2][256];
  const int32_t* part = reinterpret_cast<const int32_t*>(joins.parts + blockIdx.x);
  const int b = scalar_load(part), unit = scalar_load(part + 1);
  const int from = scalar_load(part + 2), parts = scalar_load(part + 3);
  if (parts <= 1) return;
  const int D = a.pages.D, halves = (D + 1) / 2;
  const int tiles = (a.G + HEADS - 1) / HEADS, columns = min(a.G, HEADS);
  const int kv_head = unit / tiles, head0 = (unit - kv_head * tiles) * HEADS;
  const int items = min(a.G - head0, HEADS) * halves;
  const int lane_item = threadIdx.x & (per - 1), group = threadIdx.x / per;
  const int groups = 256 / per;
  const int item = min((int)blockIdx.y * per + lane_item, items - 1);
  const int h = item / halves, d = item - h * halves;
  float top = -INFINITY, all = 0.f, sum[2] = {0.f, 0.f};
  for (int i0 = group; i0 < parts; i0 += IN_FLIGHT * groups) {
    float2 ml[IN_FLIGHT], o[IN_FLIGHT];
#pragma unroll
    for (int u = 0; u < IN_FLIGHT; ++u) {
      const int i = i0 + u * groups;
      ml[u] = make_float2(-INFINITY, 0.f);
      o[u] = make_float2(0.f, 0.f);
      if (i >= parts) continue;
      const int64_t at = place_of(from, i) * columns + h;
      ml[u] = joins.tops[at];
      o[u] = joins.sums[at * halves + d];
    }
    float most = top;
#pragma unroll
    for (int u = 0; u < IN_FLIGHT; ++u) most = fmaxf(most, ml[u].x);
    const float was = weight_of(top, most);
    top = most;
    all *= was;
    sum[0] *= was;
    sum[1] *= was;
#pragma unroll
    for (int u = 0; u < IN_FLIGHT; ++u) {
      const float factor = weight_of(ml[u].x, top);
      all += ml[u].y * factor;
      sum[0] += o[u].x * factor;
      sum[1] += o[u].y * factor;
    }
  }
  tops[threadIdx.x] = top;
  alls[threadIdx.x] = all;
  sums[0][threadIdx.x] = sum[0];
  sums[1][threadIdx.x] = sum[1];
  __syncthreads();
  if (group != 0 || (int)blockIdx.y * per + lane_item >= items) return;
  for (int g = 1; g < groups; ++g) top = fmaxf(top, tops[lane_item + g * per]);
  all = sum[0] = sum[1] = 0.f;
  for (int g = 0; g < groups; ++g) {
    const int at = lane_item + g * per;
    const float factor = weight_of(tops[at], top);
    all += alls[at] * factor;
    sum[0] += sums[0][at] * factor;
    sum[1] += sums[1][at] * factor;
  }
  T* out = static_cast<T*>(a.out) +
           ((int64_t)b * a.H + (int64_t)kv_head * a.G + head0 + h) * D + 2 * d;
  // (no weights: 0)
  store_f32<T>(out, all == 0.f ? 0.f : sum[0] / all);
  if (2 * d + 1 < D) store_f32<T>(out + 1, all == 0.f ? 0.f : sum[1] / all);
}

// ---------------------------------------------------------------------------
// the host's side
// ---------------------------------------------------------------------------
static bool on_16_bytes(std::initializer_list<const void*> all) {
  uintptr_t bits = 0;
  for (const void* p : all) bits |= reinterpret_cast<uintptr_t>(p);
  return bits % 16 == 0;
}

// Checks the sizes of a cache and describes it.
static int pages_of(const char* what, const int32_t* table, int B, int HK, int D, int N,
                    int S, int P, Pages* pages) {
  MOE_REQUIRE(B >= 1 && HK >= 1 && D >= 1 && N >= 1 && S >= 1 && P >= 1, MESH_MOE_E_ARG,
              "%s: bad sizes B=%d HK=%d D=%d N=%d S=%d P=%d", what, B, HK, D, N, S, P);
  MOE_REQUIRE(HK <= MAX_HEADS, MESH_MOE_E_UNSUPPORTED,
              "%s: %d key / value heads, up to %d", what, HK, MAX_HEADS);
  MOE_REQUIRE((S & (S - 1)) == 0, MESH_MOE_E_UNSUPPORTED,
              "%s: pages of %d rows, not a power of two", what, S);
  MOE_REQUIRE(D <= MAX_WIDTH, MESH_MOE_E_UNSUPPORTED, "%s: heads of %d values, up to %d",
              what, D, MAX_WIDTH);
  MOE_REQUIRE((int64_t)P * S <= MAX_POSITIONS, MESH_MOE_E_UNSUPPORTED,
              "%s: %d pages of %d rows a sequence, up to 2^30 positions", what, P, S);
  int shift = 0;
  while ((1 << shift) < S) ++shift;
  *pages = Pages{table, N, P, shift, HK, D, (D + FP8_BLOCK - 1) / FP8_BLOCK};
  return 0;
}

// the lanes of a head, log2: a power of two, of 8 values each
static int lanes_of(int D) {
  int n = 0;
  while ((8 << n) < D) ++n;
  return n;
}

// Sets the wavefronts that share a row; true if a wavefront is to have one row at a time.
// Few rows: as many wavefronts as there can be (writing 2 x 400 rows of 2048 values in 8
// bits and reading them 22 us with rows by four and a wavefront each, 9 so; at 4000 rows
// they are even).  Many: rows that fill four wavefronts to three quarters, or two (16 x 1000
// rows of 2048 in 8 bits 41 us and 31, of 480 in bfloat16 18 and 20).  Float32 rows of a
// wavefront and more take their registers one by one, too (16 x 1000 of 1024 116 us by two,
// 103; of 64 values 15 and 19).  One shape lost by it: 3 x 1000 rows of 4096 8-bit values
// back into float32, whose results stay in the last level's cache, took 30 us by two and
// unshared and take 36 (4 x 1000 53 and 48, 16 x 1000 238 and 198).  Float32 rows that come
// out of 8 bits are stored at 2.6 to 3.1 TB/s: a lane's eight values are two stores of 16
// bytes, each of them every other piece of a line.
static bool few_rows(RowsOf& r, bool wide_type) {
  const int64_t pieces = (int64_t)r.pages.HK << r.lanes;
  const bool few = r.T == 1 || (int64_t)r.B * r.T <= 2048;
  if (few) r.sharing = pieces <= 64 ? 0 : pieces <= 128 ? 1 : 2;
  else r.sharing = pieces < 128 ? 0 : pieces < 192 ? 1 : 2;
  return few || (wide_type && pieces >= 64);
}

// the grid of the kernels that have rows, of `rows` a wavefront
static dim3 row_grid(const RowsOf& r, int rows, bool v) {
  const int64_t groups = ((int64_t)r.T + rows - 1) / rows;
  const int of_block = 4 >> r.sharing;
  return dim3((unsigned)std::min<int64_t>((groups + of_block - 1) / of_block, 1 << 14),
              (unsigned)std::min(r.B, 1 << 14), v ? 2 : 1);
}

template <typename T, bool EIGHT>
static void run_write(RowsOf r, const void* k, const void* v, void* k_pages,
                      void* v_pages, uint8_t* k_scales, uint8_t* v_scales,
                      hipStream_t st) {
  const bool aligned = r.pages.D % 8 == 0 && on_16_bytes({k, v, k_pages, v_pages});
  const bool one = few_rows(r, sizeof(T) == 4);
  auto kern = aligned ? (one ? cache_write_kernel<T, EIGHT, true, 1>
                             : cache_write_kernel<T, EIGHT, true, ROWS<T, EIGHT>>)
                      : (one ? cache_write_kernel<T, EIGHT, false, 1>
                             : cache_write_kernel<T, EIGHT, false, ROWS<T, EIGHT>>);
  kern<<<row_grid(r, one ? 1 : ROWS<T, EIGHT>, v != nullptr), 256, 0, st>>>(
      r, static_cast<const T*>(k), static_cast<const T*>(v), k_pages, v_pages, k_scales,
      v_scales);
}

template <typename T, bool EIGHT>
static void run_read(RowsOf r, const void* k_pages, const void* v_pages,
                     const uint8_t* k_scales, const uint8_t* v_scales, void* k, void* v,
                     hipStream_t st) {
  const bool aligned = r.pages.D % 8 == 0 && on_16_bytes({k, v, k_pages, v_pages});
  const bool one = few_rows(r, sizeof(T) == 4);
  auto kern = aligned ? (one ? cache_read_kernel<T, EIGHT, true, 1>
                             : cache_read_kernel<T, EIGHT, true, ROWS<T, EIGHT>>)
                      : (one ? cache_read_kernel<T, EIGHT, false, 1>
                             : cache_read_kernel<T, EIGHT, false, ROWS<T, EIGHT>>);
  kern<<<row_grid(r, one ? 1 : ROWS<T, EIGHT>, v != nullptr), 256, 0, st>>>(
      r, k_pages, v_pages, k_scales, v_scales, static_cast<T*>(k), static_cast<T*>(v));
}

constexpr int CUS = 256;
// How the tiles' kernel divides its work and its workspace.
struct Division {
  Shares shares;
  int64_t blocks;
  bool joins;                     // whether a unit can fall to several blocks
  size_t sums, parts, bytes;      // of the workspace: tops, sums, parts
  bool fits;                      // all grains can be counted
};

template <typename T, bool EIGHT, int DP>
static Shares shares_of(bool padded, int* whole) {
  typedef TileOf<T, EIGHT, DP> Tile;
  *whole = Tile::WHOLE;
  return Shares{0, Tile::GRAIN,
                CUS * (padded ? Tile::template at_once<true>()
                              : Tile::template at_once<false>()),
                Tile::ALONE};
}
template <typename T, bool EIGHT>
static Shares shares_of(int D, bool padded, int* whole) {
  return D <= 64    ? shares_of<T, EIGHT, 64>(padded, whole)
         : D <= 128 ? shares_of<T, EIGHT, 128>(padded, whole)
                    : shares_of<T, EIGHT, 256>(padded, whole);
}

static Division divide(int B, int H, int HK, int D, int S, int P, int dtype, bool eight,
                       bool padded) {
  Division v = {};
  int whole = 0;
  v.shares = dtype == MESH_MOE_BF16
                 ? (eight ? shares_of<bf16_t, true>(D, padded, &whole)
                          : shares_of<bf16_t, false>(D, padded, &whole))
                 : (eight ? shares_of<float, true>(D, padded, &whole)
                          : shares_of<float, false>(D, padded, &whole));
  const int G = H / HK;
  const int64_t most = ((int64_t)P * S + v.shares.grain - 1) / v.shares.grain;
  const int64_t each = most + AHEAD;
  const int64_t units = (int64_t)HK * ((G + HEADS - 1) / HEADS);
  v.fits = units <= 0x7fffffff / each / B && units * B <= MAX_BLOCKS;
  if (!v.fits) return v;
  v.shares.units = (int)units;
  // Units that are this short are not divided, with as many of them as CUs twice as long
  // ones: 64 sequences of 1024, 8 heads of 128 (8 grains) take 49 us whole, 52 divided; one
  // of 2001, 1 head of 128 in 8 bits (8 grains) 19 whole, 12 divided; one of 700, 16 heads
  // of 64 (6 grains) 8.4 whole, 10.3 divided.
  v.joins = most > (units * B >= CUS ? 2 * whole : whole);
  // Of many short units each is a wavefront's, from beginning to end: no barriers, no sums
  // of four, and four times as many units under way.  512 sequences of 20, 8 heads of 128
  // in tables of 8192: 35 us by blocks, 19 alone; of up to 250 77 and 72; of up to 500 in 8
  // bits (8 turns) 88 and 78.  192 of up to 500 in bfloat16 (16 turns) take 52 us by blocks,
  // 60 alone, and with no more units than blocks (64 of 250, 8 bits) it is 14 and 16.
  if (2 * units * B < 3 * v.shares.blocks || (!v.joins && (int64_t)P * S > v.shares.alone))
    v.shares.alone = 0;
  if (!v.joins) v.shares.blocks = 0;
  v.blocks = v.joins          ? std::min<int64_t>(v.shares.blocks, units * each * B)
             : v.shares.alone ? (units * B + 3) / 4
                              : units * B;
  if (v.joins) {
    const size_t rows = 2 * (size_t)v.blocks * std::min(G, HEADS);
    v.sums = sizeof(float2) * rows;
    v.parts = v.sums + sizeof(float2) * rows * ((D + 1) / 2);
    v.bytes = v.parts + sizeof(Part) * v.blocks + 8;
  }
  return v;
}

template <typename T, bool EIGHT, int DP, bool PADDED, int SMALL, bool MANY>
static int run_tiles(const Attention& a, const Division& v, char* workspace,
                     hipStream_t st) {
  auto kern = cache_attention_tiles_kernel<T, EIGHT, DP, PADDED, SMALL, MANY>;
  const int heads = std::min(a.G, HEADS);
  const size_t lds = v.shares.blocks == 0 && v.shares.alone
                         ? 0
                         : sizeof(float) * 4 * (2 * HEADS + (size_t)heads * a.pages.D);
  MOE_ALLOW_LDS(kern, lds);
  Joins joins = {};
  joins.tops = reinterpret_cast<float2*>(workspace);
  joins.sums = reinterpret_cast<float2*>(workspace + v.sums);
  joins.parts = v.joins ? reinterpret_cast<Part*>(workspace + v.parts) : nullptr;
  joins.of_units = (int64_t)a.B * v.shares.units <= v.blocks;
  kern<<<(unsigned)v.blocks, 256, lds, st>>>(a, v.shares, joins);
  MOE_CHECK_LAUNCH("cache_attention");
  if (v.joins) {
    // (blocks for every CU twice, as far as there are pairs of values)
    const int64_t units = joins.of_units ? (int64_t)a.B * v.shares.units : v.blocks;
    const int items = heads * ((a.pages.D + 1) / 2);
    int per = 256;
    while (per > 32 && (per >= 2 * items || units * ((items + per - 1) / per) < 2 * CUS))
      per /= 2;
    cache_attention_join_kernel<T>
        <<<dim3((unsigned)units, (items + per - 1) / per), 256, 0, st>>>(a, joins, per);
    MOE_CHECK_LAUNCH("cache_attention");
  }
  return 0;
}

// whether the tiles' kernel takes its PADDED form
static bool rows_padded(const Attention& a) {
  const int D = a.pages.D;
  return a.pages.shift < 2 || (D != 64 && D != 128 && D != 256) ||
         !on_16_bytes({a.q, a.k_pages, a.v_pages});
}

template <typename T, bool EIGHT>
static int run_attention(const Attention& a, const Division& v, bool padded,
                         char* workspace, hipStream_t st) {
  const int D = a.pages.D;
  if (D < TILES_FROM) {
    cache_attention_kernel<T, EIGHT><<<(unsigned)((int64_t)a.B * a.H), 256, 0, st>>>(a);
    MOE_CHECK_LAUNCH("cache_attention");
    return 0;
  }
  const int small = a.pages.shift >= 4 ? 0 : a.pages.shift >= 2 ? 1 : 2;
#define TILES(dp, padded)                                                             \
  (v.shares.alone ? run_tiles<T, EIGHT, dp, padded, 0, true>                          \
                  : run_tiles<T, EIGHT, dp, padded, 0, false>)
#define TILES_OF(dp)                                                                  \
  (small == 2   ? run_tiles<T, EIGHT, dp, true, 2, true>                              \
   : small == 1 ? (padded ? run_tiles<T, EIGHT, dp, true, 1, true>                    \
                          : run_tiles<T, EIGHT, dp, false, 1, true>)                  \
                : (padded ? TILES(dp, true) : TILES(dp, false)))
  auto run = D <= 64 ? TILES_OF(64) : D <= 128 ? TILES_OF(128) : TILES_OF(256);
#undef TILES_OF
#undef TILES
  return run(a, v, workspace, st);
}

}  // namespace mesh_moe

using namespace mesh_moe;

extern "C" int mesh_moe_cache_abi_version(void) { return MESH_MOE_CACHE_ABI_VERSION; }

// (a cache's buffers: values always with keys, scales for both or none)
#define CACHE_REQUIRE_PAGES(what, k, v)                                                \
  MOE_REQUIRE((k) && k_pages && table && position, MESH_MOE_E_ARG, what                \
              ": null pointer");                                                       \
  MOE_REQUIRE(((v) != nullptr) == (v_pages != nullptr), MESH_MOE_E_ARG, what           \
              ": values and v_pages go together");                                     \
  MOE_REQUIRE((v_scales != nullptr) == (k_scales && v_pages), MESH_MOE_E_ARG, what     \
              ": scales go with the pages of keys and of values");                     \
  MOE_REQUIRE(valid_dtype(dtype), MESH_MOE_E_ARG, what ": bad dtype %d", dtype)

extern "C" int mesh_moe_cache_write(const void* k, const void* v, const int32_t* table,
                                    const int32_t* position, const int32_t* count,
                                    void* k_pages, void* v_pages, uint8_t* k_scales,
                                    uint8_t* v_scales, int B, int T, int HK, int D, int N,
                                    int S, int P, int dtype, void* stream) {
  CACHE_REQUIRE_PAGES("cache_write", k, v);
  RowsOf r = {};
  if (int rc = pages_of("cache_write", table, B, HK, D, N, S, P, &r.pages)) return rc;
  MOE_REQUIRE(T >= 1, MESH_MOE_E_ARG, "cache_write: bad sizes T=%d", T);
  MOE_REQUIRE(T <= MAX_POSITIONS, MESH_MOE_E_UNSUPPORTED, "cache_write: %d rows, up to 2^30", T);
  r.position = position;
  r.count = count;
  r.B = B;
  r.T = T;
  r.lanes = lanes_of(D);
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto run = dtype == MESH_MOE_BF16
                 ? (k_scales ? run_write<bf16_t, true> : run_write<bf16_t, false>)
                 : (k_scales ? run_write<float, true> : run_write<float, false>);
  run(r, k, v, k_pages, v_pages, k_scales, v_scales, st);
  MOE_CHECK_LAUNCH("cache_write");
  return 0;
}

extern "C" int mesh_moe_cache_read(const void* k_pages, const void* v_pages,
                                   const uint8_t* k_scales, const uint8_t* v_scales,
                                   const int32_t* table, const int32_t* position,
                                   const int32_t* count, void* k, void* v, int B, int T,
                                   int HK, int D, int N, int S, int P, int dtype,
                                   void* stream) {
  CACHE_REQUIRE_PAGES("cache_read", k, v);
  RowsOf r = {};
  if (int rc = pages_of("cache_read", table, B, HK, D, N, S, P, &r.pages)) return rc;
  MOE_REQUIRE(T >= 1, MESH_MOE_E_ARG, "cache_read: bad sizes T=%d", T);
  MOE_REQUIRE(T <= MAX_POSITIONS, MESH_MOE_E_UNSUPPORTED, "cache_read: %d rows, up to 2^30", T);
  r.position = position;
  r.count = count;
  r.B = B;
  r.T = T;
  r.lanes = lanes_of(D);
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto run = dtype == MESH_MOE_BF16
                 ? (k_scales ? run_read<bf16_t, true> : run_read<bf16_t, false>)
                 : (k_scales ? run_read<float, true> : run_read<float, false>);
  run(r, k_pages, v_pages, k_scales, v_scales, k, v, st);
  MOE_CHECK_LAUNCH("cache_read");
  return 0;
}

extern "C" size_t mesh_moe_cache_attention_workspace_bytes(int B, int H, int HK, int D,
                                                           int S, int P, int dtype,
                                                           int eight_bit) {
  if (B < 1 || H < 1 || HK < 1 || H % HK || D < TILES_FROM || D > MAX_WIDTH || S < 1 || P < 1 ||
      !valid_dtype(dtype))
    return 0;
  // (the form with more blocks, wherever the operands lie)
  return divide(B, H, HK, D, S, P, dtype, eight_bit != 0, false).bytes;
}

extern "C" int mesh_moe_cache_attention(
    const void* q, const void* k_new, const void* v_new, void* k_pages, void* v_pages,
    uint8_t* k_scales, uint8_t* v_scales, const int32_t* table, const int32_t* position,
    const void* rel_values, const int32_t* rel_bucket, int num_buckets, int reach,
    void* out, int B, int H, int HK, int D, int N, int S, int P, int dtype,
    void* workspace, size_t workspace_bytes, void* stream) {
  CACHE_REQUIRE_PAGES("cache_attention", q && out, v_pages);
  Attention a = {};
  if (int rc = pages_of("cache_attention", table, B, HK, D, N, S, P, &a.pages)) return rc;
  MOE_REQUIRE(H >= 1 && H % HK == 0, MESH_MOE_E_ARG,
              "cache_attention: %d query heads for %d key / value heads", H, HK);
  MOE_REQUIRE(k_new ? (v_new != nullptr) == (v_pages != nullptr) : !v_new,
              MESH_MOE_E_ARG, "cache_attention: k_new, v_new and v_pages go together");
  MOE_REQUIRE((rel_values != nullptr) == (rel_bucket != nullptr) &&
                  (!rel_values || (num_buckets >= 1 && reach >= 1)),
              MESH_MOE_E_ARG, "cache_attention: rel_values, rel_bucket, num_buckets and "
              "reach go together");
  a.q = q;
  a.k_pages = k_pages;
  a.v_pages = v_pages ? v_pages : k_pages;
  a.k_scales = k_scales;
  a.v_scales = v_pages ? v_scales : k_scales;
  const bool tiles = D >= TILES_FROM;
  a.k_new = tiles ? k_new : nullptr;
  a.v_new = tiles ? v_new : nullptr;
  a.position = position;
  a.rel_values = rel_values;
  a.rel_bucket = rel_bucket;
  a.NB = num_buckets;
  a.reach = reach;
  a.out = out;
  a.B = B;
  a.H = H;
  a.G = H / HK;
  const bool padded = rows_padded(a);
  const Division v = tiles ? divide(B, H, HK, D, S, P, dtype, k_scales != nullptr, padded)
                           : Division{};
  MOE_REQUIRE(tiles ? v.fits : (int64_t)B * H <= MAX_BLOCKS, MESH_MOE_E_UNSUPPORTED,
              "cache_attention: %d sequences of %d heads and %d pages are more than a "
              "launch has", B, H, P);
  MOE_REQUIRE(!tiles || v.bytes == 0 || (workspace && workspace_bytes >= v.bytes),
              MESH_MOE_E_ARG, "cache_attention: workspace too small");
  if (k_new && !tiles) {
    if (int rc = mesh_moe_cache_write(k_new, v_new, table, position, nullptr, k_pages,
                                      v_pages, k_scales, v_scales, B, 1, HK, D, N, S, P,
                                      dtype, stream))
      return rc;
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  char* at = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(workspace) + 7) &
                                     ~(uintptr_t)7);
  auto run = dtype == MESH_MOE_BF16
                 ? (k_scales ? run_attention<bf16_t, true> : run_attention<bf16_t, false>)
                 : (k_scales ? run_attention<float, true> : run_attention<float, false>);
  return run(a, v, padded, at, st);
}
