// A head with low-rank adapters beside it (carbon_rec.h, crec_adapters_logits): frame f of line i,
//   z[f][c] = sum_k x[f][k] W[c][k] + b[c] + scale_a * sum_j h[f][j] B_a[c][j]
//   h[f][j] = sum_k x[f][k] A_a[j][k],  a = adapter[i]
#pragma once

#include <cuda_fp16.h>

#include <cstdint>

#include "sm100.cuh"

namespace crec {

constexpr int kMaxRank = 64;
constexpr int kMaxHeadK = 512;

struct AdapterParams {
  const __half* x;  // [rows][k], rows x_pitch apart
  long long x_pitch;
  int rows, lines, k, classes;
  const int32_t* line_at;
  const int32_t* adapter;  // null: the head alone
  const __half* w;         // [classes][k]
  const float* bias;       // [classes]
  int adapters, rank;      // rank: the widest, what A and B are padded to
  const __half* a;         // [adapters][rank][k]
  const __half* b;         // [adapters][classes][rank]
  const float* scale;      // [adapters]
  void* z;
  int half;
  long long pitch;
};

// The line of row r, or -1 outside [line_at[0], line_at[lines]).
__device__ __forceinline__ int line_of_row(const int32_t* line_at, int lines, int r) {
  if (lines <= 0 || r < line_at[0] || r >= line_at[lines]) return -1;
  int lo = 0, hi = lines;
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2;
    if (line_at[mid] <= r) lo = mid;
    else hi = mid;
  }
  return lo;
}

constexpr int kHeadRows = 16;

// A block 16 frames x 256 classes: the frames and their adapters' inner sums in shared memory as
// float32, a thread a class, its weights read once for the 16 frames.
__global__ void __launch_bounds__(256) adapter_head_kernel(const __grid_constant__ AdapterParams p) {
  __shared__ float xs[kHeadRows][kMaxHeadK];
  __shared__ float h[kHeadRows][kMaxRank];
  __shared__ int which[kHeadRows];  // the frame's adapter, -1 none, -2 not a line's frame
  const int r0 = blockIdx.x * kHeadRows, n = min(kHeadRows, p.rows - r0);
  if (threadIdx.x < kHeadRows) {
    const int line = static_cast<int>(threadIdx.x) < n ? line_of_row(p.line_at, p.lines, r0 + threadIdx.x) : -1;
    const int a = line < 0 || !p.adapter ? -1 : p.adapter[line];
    which[threadIdx.x] = line < 0 ? -2 : a >= 0 && a < p.adapters ? a : -1;
  }
  for (int i = threadIdx.x; i < n * p.k; i += blockDim.x)
    xs[i / p.k][i % p.k] = __half2float(p.x[(r0 + i / p.k) * p.x_pitch + i % p.k]);
  __syncthreads();
  for (int i = threadIdx.x; i < n * p.rank; i += blockDim.x) {
    const int f = i / p.rank, j = i % p.rank, a = which[f];
    float s = 0.0f;
    if (a >= 0) {
      const __half* row = p.a + (static_cast<long long>(a) * p.rank + j) * p.k;
      for (int k = 0; k < p.k; ++k) s = __fmaf_rn(xs[f][k], __half2float(row[k]), s);
      s = __fmul_rn(s, p.scale[a]);
    }
    h[f][j] = s;
  }
  __syncthreads();
  const int c = blockIdx.y * 256 + threadIdx.x;
  if (c >= p.classes) return;
  float acc[kHeadRows];
  for (int f = 0; f < kHeadRows; ++f) acc[f] = 0.0f;
  for (int k = 0; k < p.k; ++k) {
    const float w = __half2float(p.w[static_cast<long long>(c) * p.k + k]);
#pragma unroll
    for (int f = 0; f < kHeadRows; ++f) acc[f] = __fmaf_rn(xs[f][k], w, acc[f]);
  }
  for (int f = 0; f < n; ++f) {
    if (which[f] == -2) continue;
    float v = __fadd_rn(acc[f], p.bias[c]);
    if (which[f] >= 0) {
      const __half* row = p.b + (static_cast<long long>(which[f]) * p.classes + c) * p.rank;
      float s = 0.0f;
      for (int j = 0; j < p.rank; ++j) s = __fmaf_rn(h[f][j], __half2float(row[j]), s);
      v = __fadd_rn(v, s);
    }
    const long long o = (r0 + f) * p.pitch + c;
    if (p.half) static_cast<__half*>(p.z)[o] = __float2half_rn(v);
    else static_cast<float*>(p.z)[o] = v;
  }
}

}  // namespace crec
