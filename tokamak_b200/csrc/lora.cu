// lora.cu -- low-rank adapters of many requests beside a shared projection.
#include "tkb_common.cuh"
#include "../../include/tkm_b200.h"

namespace tkb {

struct LoraPlanParams {
  const int32_t* adapter;
  const int32_t* row_start;
  int32_t* of_row;
  int B, rows, n_adapters;
};

// The adapter of every row: -1 none, -2 a row of no sequence.
__global__ void lora_plan_kernel(const __grid_constant__ LoraPlanParams p) {
  grid_wait();
  if (p.row_start && blockIdx.x == 0)
    for (int b = threadIdx.x; b < p.B; b += blockDim.x)
      if (p.row_start[b] < 0 || p.row_start[b + 1] < p.row_start[b] || p.row_start[b + 1] > p.rows)
        atomicOr(&g_device_error, ERR_BAD_INDEX);
  for (int row = blockIdx.x * blockDim.x + threadIdx.x; row < p.rows; row += gridDim.x * blockDim.x) {
    int b = row;
    bool has = true;
    if (p.row_start) {
      int lo = 0, hi = p.B - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p.row_start[mid] <= row) lo = mid;
        else hi = mid - 1;
      }
      b = lo;
      has = p.row_start[b] <= row && row < p.row_start[b + 1];
    }
    int a = p.adapter[b];
    if (a < -1 || a >= p.n_adapters) {
      atomicOr(&g_device_error, ERR_BAD_INDEX);
      a = -1;
    }
    p.of_row[row] = has ? a : -2;
  }
}

struct LoraParams {
  const int32_t* of_row;
  const void *x, *a, *b, *y;
  void* out;
  const float* scale;
  float* t;  // [rows][R]: scale * x A
  long long x_stride, y_stride, out_stride;
  int rows, K, N, R;
};

template <typename T>
__global__ void __launch_bounds__(256) lora_down_kernel(const __grid_constant__ LoraParams p) {
  grid_wait();
  const int row = blockIdx.x, a = p.of_row[row];
  if (a < 0) return;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
  const T* A = static_cast<const T*>(p.a) + static_cast<long long>(a) * p.K * p.R;
  for (int r = warp_id(); r < p.R; r += 8) {
    float s = 0.f;
    for (int k = lane_id(); k < p.K; k += 32) s = fmaf(static_cast<float>(x[k]), static_cast<float>(A[static_cast<long long>(k) * p.R + r]), s);
    s = warp_sum(s);
    if (lane_id() == 0) p.t[static_cast<long long>(row) * p.R + r] = s * (p.scale ? p.scale[a] : 1.f);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) lora_up_kernel(const __grid_constant__ LoraParams p) {
  grid_wait();
  const int row = blockIdx.x, a = p.of_row[row];
  if (a == -2) return;
  const T* y = static_cast<const T*>(p.y) + row * p.y_stride;
  T* out = static_cast<T*>(p.out) + row * p.out_stride;
  const T* Bm = static_cast<const T*>(p.b) + static_cast<long long>(max(a, 0)) * p.R * p.N;
  for (int n = threadIdx.x; n < p.N; n += 256) {
    float s = static_cast<float>(y[n]);
    if (a >= 0)
      for (int r = 0; r < p.R; ++r)
        s = fmaf(p.t[static_cast<long long>(row) * p.R + r], static_cast<float>(Bm[static_cast<long long>(r) * p.N + n]), s);
    out[n] = static_cast<T>(s);
  }
}

template <typename T>
static cudaError_t lora_add_t(const LoraParams& p, cudaStream_t st) {
  cudaError_t e = launch_early(lora_down_kernel<T>, dim3(p.rows), 256, 0, st, p);
  if (e != cudaSuccess) return e;
  return launch_early(lora_up_kernel<T>, dim3(p.rows), 256, 0, st, p);
}

}  // namespace tkb
