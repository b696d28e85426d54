// The paged cache: rows of keys and values into pages and back, and attention of one new
// token over them.
#include "../../include/mesh_moe_cache.h"
#include "fp8.h"

#include <algorithm>

namespace mesh_moe {

constexpr int MAX_WIDTH = 256;                  // D
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

// ---------------------------------------------------------------------------
// Rows into pages and back.  A wavefront has a row of keys or of values (blockIdx.y),
// whose page is the same for all its lanes; a lane has 8 values, and a head's lanes are a
// power of two (16 for each block of 128 where it has more than one), so that a block's
// largest magnitude is found by DPP steps among neighbours.
// ---------------------------------------------------------------------------
struct RowsOf {
  Pages pages;
  const int32_t* position;        // [B]
  const int32_t* count;           // [B] or null
  int B, T;
  int lanes;                      // of a head, log2
};

template <typename T, bool EIGHT, bool ALIGNED>
__global__ __launch_bounds__(256) void cache_write_kernel(
    RowsOf r, const T* __restrict__ k, const T* __restrict__ v, void* k_pages,
    void* v_pages, uint8_t* k_scales, uint8_t* v_scales) {
  const bool is_v = blockIdx.y != 0;
  const T* x = is_v ? v : k;
  uint8_t* values = static_cast<uint8_t*>(is_v ? v_pages : k_pages);
  uint8_t* scales = is_v ? v_scales : k_scales;
  const int lane = threadIdx.x & 63, D = r.pages.D, HK = r.pages.HK;
  const int pieces = HK << r.lanes, group = min(1 << r.lanes, 16);
  const int64_t rows = (int64_t)r.B * r.T;
  for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < rows;
       i += (int64_t)gridDim.x * 4) {
    const int b = (int)(i / r.T), t = (int)(i - (int64_t)b * r.T);
    if (r.count && t >= r.count[b]) continue;
    const int64_t to = r.pages.row(b, (int64_t)r.position[b] + t);
    if (to < 0) continue;
    const T* from = x + i * HK * D;
    for (int piece = lane; piece < (pieces + 63) / 64 * 64; piece += 64) {
      const int h = piece >> r.lanes;
      const int at = h < HK ? (piece & ((1 << r.lanes) - 1)) * 8 : D;
      float f[8];
      load8<T, ALIGNED>(from + (int64_t)min(h, HK - 1) * D, at, D, f);
      const int64_t row = r.pages.head(to, h);
      if constexpr (EIGHT) {
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, magnitude_bits(f[j]));
        const Fp8Scale s = fp8_scale(max_of_lanes(top, group));
        if (at >= D) continue;
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] *= s.factor;
        const uint32_t lo = fp8_pack4(f[0], f[1], f[2], f[3]);
        const uint32_t hi = fp8_pack4(f[4], f[5], f[6], f[7]);
        uint8_t* q = values + row * D + at;
        if (ALIGNED) {
          *reinterpret_cast<uint2*>(q) = make_uint2(lo, hi);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (at + j < D) q[j] = (uint8_t)((j < 4 ? lo : hi) >> 8 * (j & 3));
        }
        if ((piece & (group - 1)) == 0)
          scales[row * r.pages.DB + at / FP8_BLOCK] = (uint8_t)s.byte;
      } else {
        if (at < D)
          store8<T, ALIGNED>(reinterpret_cast<T*>(values) + row * D, at, D, f);
      }
    }
  }
}

template <typename T, bool EIGHT, bool ALIGNED>
__global__ __launch_bounds__(256) void cache_read_kernel(
    RowsOf r, const void* __restrict__ k_pages, const void* __restrict__ v_pages,
    const uint8_t* __restrict__ k_scales, const uint8_t* __restrict__ v_scales,
    T* __restrict__ k, T* __restrict__ v) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  const bool is_v = blockIdx.y != 0;
  T* y = is_v ? v : k;
  const uint8_t* values = static_cast<const uint8_t*>(is_v ? v_pages : k_pages);
  const uint8_t* scales = is_v ? v_scales : k_scales;
  const int lane = threadIdx.x & 63, D = r.pages.D, HK = r.pages.HK;
  const int pieces = HK << r.lanes;
  const int64_t rows = (int64_t)r.B * r.T;
  for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < rows;
       i += (int64_t)gridDim.x * 4) {
    const int b = (int)(i / r.T), t = (int)(i - (int64_t)b * r.T);
    const int64_t from = r.count && t >= r.count[b]
                             ? -1 : r.pages.row(b, (int64_t)r.position[b] + t);
    T* to = y + i * HK * D;
    for (int piece = lane; piece < pieces; piece += 64) {
      const int h = piece >> r.lanes, at = (piece & ((1 << r.lanes) - 1)) * 8;
      if (at >= D) continue;
      const int64_t row = r.pages.head(from, h);
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = 0.f;
      if (from >= 0) {
        if constexpr (EIGHT) {
          const uint8_t* q = values + row * D + at;
          uint32_t w[2] = {0, 0};
          if (ALIGNED) {
            const uint2 both = *reinterpret_cast<const uint2*>(q);
            w[0] = both.x;
            w[1] = both.y;
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (at + j < D) w[j / 4] |= (uint32_t)q[j] << 8 * (j & 3);
          }
          const float unit = unit_of(scales[row * r.pages.DB + at / FP8_BLOCK]);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[j], false);
            const f32x2_t hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[j], true);
            f[4 * j] = lo[0] * unit;
            f[4 * j + 1] = lo[1] * unit;
            f[4 * j + 2] = hi[0] * unit;
            f[4 * j + 3] = hi[1] * unit;
          }
        } else {
          load8<T, ALIGNED>(reinterpret_cast<const T*>(values) + row * D, at, D, f);
        }
      }
      store8<T, ALIGNED>(to + (int64_t)h * D, at, D, f);
    }
  }
}

// ---------------------------------------------------------------------------
// Attention of one token over a cache: with m the largest logit so far, l the sum of
// exp(logit - m) and o the sum of exp(logit - m) v, another position's logit x and value v
// turn them into
//   m' = max(m, x)   l' = l e^(m - m') + e^(x - m')   o' = o e^(m - m') + e^(x - m') v
// and two such triples of different positions are joined the same way; o / l is the
// result.  A block has a query head of a sequence, its four wavefronts every fourth
// position each.
// ---------------------------------------------------------------------------
struct Attention {
  Pages pages;
  const void *q, *k_pages, *v_pages;
  const uint8_t *k_scales, *v_scales;
  const int32_t* position;        // [B]
  const void* rel_values;         // [H][NB] or null
  const int32_t* rel_bucket;      // [2 * reach - 1]
  int NB, reach;
  void* out;
  int B, H, G;                    // G query heads share a key / value head
};

// visible positions of sequence b
__device__ __forceinline__ int seen_of(const Attention& a, int b) {
  const int64_t all = (int64_t)a.pages.P << a.pages.shift;
  return (int)min(max((int64_t)a.position[b] + 1, (int64_t)0), all);
}

// the relative bias of head h for position j, `last` being the query's
template <typename T>
__device__ __forceinline__ float bias_of(const Attention& a, int h, int j, int last) {
  const int back = max(j - last, 1 - a.reach);
  const int bucket = a.rel_bucket[back + a.reach - 1];
  return load_f32<T>(static_cast<const T*>(a.rel_values) + (int64_t)h * a.NB +
                     min(max(bucket, 0), a.NB - 1));
}

// e^(x - m) with m >= x; 0 for x = -infinity
__device__ __forceinline__ float weight_of(float x, float m) {
  return x == -INFINITY ? 0.f : expf(x - m);
}

template <typename T, bool EIGHT>
__device__ __forceinline__ float page_value(const void* pages, const uint8_t* scales,
                                            int64_t row, int d, int D, int DB) {
  if constexpr (EIGHT) {
    const uint32_t byte = static_cast<const uint8_t*>(pages)[row * D + d];
    return __builtin_amdgcn_cvt_f32_fp8((int)byte, 0) *
           unit_of(scales[row * DB + d / FP8_BLOCK]);
  } else {
    return load_f32<T>(static_cast<const T*>(pages) + row * D + d);
  }
}

template <typename T, bool EIGHT>
__global__ __launch_bounds__(256) void cache_attention_kernel(Attention a) {
  constexpr int NI = MAX_WIDTH / 64;            // values of a row per lane
  __shared__ float part_o[4][MAX_WIDTH], part_m[4], part_l[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int b = (int)(blockIdx.x / a.H), h = (int)(blockIdx.x - (int64_t)b * a.H);
  const int D = a.pages.D, seen = seen_of(a, b), last = a.position[b];
  const int64_t at = ((int64_t)b * a.H + h) * D;
  float q[NI], o[NI], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int d = lane + 64 * i;
    q[i] = d < D ? load_f32<T>(static_cast<const T*>(a.q) + at + d) : 0.f;
    o[i] = 0.f;
  }
  for (int j = wave; j < seen; j += 4) {
    int64_t row = a.pages.row(b, j);
    if (row < 0) continue;
    row = a.pages.head(row, h / a.G);
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < NI; ++i)
      if (lane + 64 * i < D)
        x = fmaf(q[i], page_value<T, EIGHT>(a.k_pages, a.k_scales, row, lane + 64 * i, D,
                                            a.pages.DB), x);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
    if (a.rel_values) x += bias_of<T>(a, h, j, last);
    const float top = fmaxf(m, x), was = weight_of(m, top);
    const float w = round_to<T>(weight_of(x, top));
    m = top;
    l = l * was + w;
#pragma unroll
    for (int i = 0; i < NI; ++i)
      if (lane + 64 * i < D)
        o[i] = fmaf(w, page_value<T, EIGHT>(a.v_pages, a.v_scales, row, lane + 64 * i, D,
                                            a.pages.DB), o[i] * was);
  }
#pragma unroll
  for (int i = 0; i < NI; ++i) part_o[wave][lane + 64 * i] = o[i];
  if (lane == 0) {
    part_m[wave] = m;
    part_l[wave] = l;
  }
  __syncthreads();
  float top = part_m[0];
  for (int w = 1; w < 4; ++w) top = fmaxf(top, part_m[w]);
  for (int d = threadIdx.x; d < D; d += 256) {
    float sum = 0.f, all = 0.f;
    for (int w = 0; w < 4; ++w) {
      const float factor = weight_of(part_m[w], top);
      sum += part_o[w][d] * factor;
      all += part_l[w] * factor;
    }
    // (nothing seen: 0)
    store_f32<T>(static_cast<T*>(a.out) + at + d, all == 0.f ? 0.f : sum / all);
  }
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

// blocks of the kernels that have a wavefront per row
static unsigned row_blocks(int64_t rows) {
  return (unsigned)std::min<int64_t>((rows + 3) / 4, 1 << 20);
}

template <typename T, bool EIGHT>
static void run_write(const RowsOf& r, const void* k, const void* v, void* k_pages,
                      void* v_pages, uint8_t* k_scales, uint8_t* v_scales,
                      hipStream_t st) {
  const dim3 grid(row_blocks((int64_t)r.B * r.T), v ? 2 : 1);
  auto kern = r.pages.D % 8 == 0 && on_16_bytes({k, v, k_pages, v_pages})
                  ? cache_write_kernel<T, EIGHT, true>
                  : cache_write_kernel<T, EIGHT, false>;
  kern<<<grid, 256, 0, st>>>(r, static_cast<const T*>(k), static_cast<const T*>(v),
                             k_pages, v_pages, k_scales, v_scales);
}

template <typename T, bool EIGHT>
static void run_read(const RowsOf& r, const void* k_pages, const void* v_pages,
                     const uint8_t* k_scales, const uint8_t* v_scales, void* k, void* v,
                     hipStream_t st) {
  const dim3 grid(row_blocks((int64_t)r.B * r.T), v ? 2 : 1);
  auto kern = r.pages.D % 8 == 0 && on_16_bytes({k, v, k_pages, v_pages})
                  ? cache_read_kernel<T, EIGHT, true>
                  : cache_read_kernel<T, EIGHT, false>;
  kern<<<grid, 256, 0, st>>>(r, k_pages, v_pages, k_scales, v_scales,
                             static_cast<T*>(k), static_cast<T*>(v));
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
                                                           int S, int P) {
  (void)B, (void)H, (void)HK, (void)D, (void)S, (void)P;
  return 0;
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
  MOE_REQUIRE((int64_t)B * H <= MAX_BLOCKS, MESH_MOE_E_UNSUPPORTED,
              "cache_attention: %d sequences of %d heads are more than a launch has", B, H);
  MOE_REQUIRE(workspace_bytes >=
                  mesh_moe_cache_attention_workspace_bytes(B, H, HK, D, S, P),
              MESH_MOE_E_ARG, "cache_attention: workspace too small");
  (void)workspace;
  if (k_new) {
    if (int rc = mesh_moe_cache_write(k_new, v_new, table, position, nullptr, k_pages,
                                      v_pages, k_scales, v_scales, B, 1, HK, D, N, S, P,
                                      dtype, stream))
      return rc;
  }
  a.q = q;
  a.k_pages = k_pages;
  a.v_pages = v_pages ? v_pages : k_pages;
  a.k_scales = k_scales;
  a.v_scales = v_pages ? v_scales : k_scales;
  a.position = position;
  a.rel_values = rel_values;
  a.rel_bucket = rel_bucket;
  a.NB = num_buckets;
  a.reach = reach;
  a.out = out;
  a.B = B;
  a.H = H;
  a.G = H / HK;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const unsigned grid = (unsigned)((int64_t)B * H);
  auto kern = dtype == MESH_MOE_BF16
                  ? (k_scales ? cache_attention_kernel<bf16_t, true>
                              : cache_attention_kernel<bf16_t, false>)
                  : (k_scales ? cache_attention_kernel<float, true>
                              : cache_attention_kernel<float, false>);
  kern<<<grid, 256, 0, st>>>(a);
  MOE_CHECK_LAUNCH("cache_attention");
  return 0;
}
