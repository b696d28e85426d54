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

namespace mesh_moe {

typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16_t fp8_mfma(i32x8_t w, i32x8_t a, f32x16_t c,
                                             uint32_t w_scale, uint32_t a_scale) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w, a, c, 0, 0, 0, (int)w_scale,
                                                         0, (int)a_scale);
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
                    apply_activation(sum, g.activation));
  }
}

// bytes of scratch one product needs
static size_t product_workspace(int E, int R, int N, bool eight_bit) {
  return eight_bit ? (size_t)E * R * N * sizeof(float) : 0;
}

static int run_product(const GemmArgs& g, void* workspace, hipStream_t st) {
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
  return product_workspace(E, R, N, eight_bit != 0);
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
  const size_t need = product_workspace(E, R, N, y_scales != nullptr);
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
  const size_t dw = product_workspace(E, K, N, false);
  const size_t da = want_da ? product_workspace(E, R, K, false) : 0;
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
