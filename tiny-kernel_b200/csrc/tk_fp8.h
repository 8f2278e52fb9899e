// tk_fp8.h -- 8-bit floating point: e4m3 codes with an f32 scale for each block of 128 values of k, and the
// launchers of the operators on them (tk_fp8.cu, tk_fp8_matmul.cu).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace tk {

constexpr int kFp8Block = 128;
constexpr int kFp8MaxDim = 32768;  // of a row that is normalised

// Rows of `dim` values, strides in elements; scales [rows][ceil(dim / 128)].
struct Fp8RowsParams {
  const void* x;
  const void* residual;  // null: none
  const float* weight;   // null: ones
  void* sum;             // x + residual, null: not written
  uint8_t* codes;
  float* scales;
  long long x_stride, residual_stride, sum_stride, codes_stride;
  int rows, dim;
  float eps;
};
cudaError_t launch_add_rmsnorm_fp8(const Fp8RowsParams& p, int dtype, int sm_count, cudaStream_t st);
// Without the norm; block_rows 1, or 128: scales [ceil(rows / 128)][ceil(dim / 128)].
cudaError_t launch_fp8_quantize(const Fp8RowsParams& p, int block_rows, int dtype, cudaStream_t st);

// out[m][n] = sum over blocks b of k of a_scales[m][b] w_scales[n / 128][b] sum of a[m][k] w[n][k].
struct Fp8MatmulParams {
  const float* a_scales;
  const float* w_scales;
  void* out;
  long long out_stride;
  int m, k, n, dtype;
  unsigned* err;  // the device's error word, and how long a wait of a kernel may take
  unsigned long long timeout_ns;
};
// How a call's work is cut: rows of a and of w that a tile takes, CTAs of a cluster that share a tile's k; and the
// boxes of 128 bytes x box_a, box_w rows, 128-byte swizzle, that a_map and w_map, of codes [rows][k], are made of.
struct Fp8MatmulPlan {
  int rows, cols, split;
  int box_a() const { return rows < 128 ? rows : 128; }
  int box_w() const { return rows == 128 ? cols : 128; }
};
Fp8MatmulPlan fp8_matmul_plan(int m, int k, int n, int sm_count);
// Parts of tiles that are worked on at once, by a CTA each (a pair, of 256 rows): the others follow.
int fp8_matmul_places(const Fp8MatmulPlan& plan, int m, int n, int sm_count);
cudaError_t launch_fp8_matmul(const Fp8MatmulParams& p, const Fp8MatmulPlan& plan, const CUtensorMap& a_map,
                              const CUtensorMap& w_map, int sm_count, cudaStream_t st);

}  // namespace tk
