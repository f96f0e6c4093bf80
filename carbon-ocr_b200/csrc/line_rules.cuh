// The logits of packed lines under their lines' rules (carbon_rec.h, crec_rules): the ruled
// logits written out, greedy CTC, and the beam's candidates.
//
// A frame's ruled logit of class c, each operation rounded to float32 on its own so that every
// kernel (and any restatement) takes the same decisions:
//   n = c's count in the line's history
//   n > 0:  z = (z > 0 ? z / repeat : z * repeat) - (n * frequency + presence)
//   z += bias;  z = -inf where the line's set leaves c out
// then best = max_c z, p_c = exp(z_c - best) / sum_c exp(z_c - best).
#pragma once

#include <cuda_fp16.h>

#include <cstdint>

#include "sm100.cuh"

namespace crec {

struct LineParams {
  const void* z;  // [rows][classes], rows `pitch` elements apart
  long long pitch;
  int classes, rows, lines;
  const int32_t* line_at;
  // rules (null: none)
  const int32_t *history, *history_at;
  const float *repeat, *presence, *frequency;
  const float* bias;
  const int32_t* bias_of;
  const uint32_t* allowed;
  const int32_t* set_of;
  int biases, sets, words;
  // outputs
  void* out;  // the ruled logits
  int out_half;
  long long out_pitch;
  int32_t* counts;  // greedy
  int32_t* ids;
  int32_t* starts;
  float* probs;  // greedy: probabilities; candidates: log-probabilities
  float* blank;
  int topk;
};

constexpr int kOpRules = 0, kOpGreedy = 1, kOpCandidates = 2;

// One line's rules.
struct LineRule {
  int first, end;  // its rows
  const int32_t* had;
  int n_had;
  float repeat, presence, frequency;
  const float* bias;        // its table's row, or null
  const uint32_t* allowed;  // its set's words, or null
};

// The line of row r: the last i with line_at[i] <= r, found by a whole warp probing 32 places a
// step (two dependent loads for 1,000 lines instead of a bisection's ten); false where r lies
// outside [line_at[0], line_at[lines]).
__device__ __forceinline__ bool find_line(const LineParams& p, int r, int lane, LineRule& l) {
  if (p.lines <= 0 || r < p.line_at[0] || r >= p.line_at[p.lines]) return false;
  int lo = 0, hi = p.lines;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, at = lo + (lane + 1) * step;
    const unsigned le = __ballot_sync(0xffffffffu, at < hi && p.line_at[at] <= r);
    const int k = __ffs(~le) - 1;  // le's leading ones (at least one 0: the last place is at or past hi)
    lo += k * step;
    hi = min(hi, lo + step);
  }
  l.first = p.line_at[lo];
  l.end = p.line_at[lo + 1];
  if (r < l.first || r >= l.end) return false;  // a line_at that does not ascend
  l.had = nullptr;
  l.n_had = 0;
  if (p.history) {
    l.had = p.history + p.history_at[lo];
    l.n_had = p.history_at[lo + 1] - p.history_at[lo];
  }
  l.repeat = p.repeat ? p.repeat[lo] : 1.0f;
  l.presence = p.presence ? p.presence[lo] : 0.0f;
  l.frequency = p.frequency ? p.frequency[lo] : 0.0f;
  const int b = p.bias_of ? p.bias_of[lo] : 0, s = p.set_of ? p.set_of[lo] : 0;
  l.bias = p.bias && b >= 0 && b < p.biases ? p.bias + static_cast<long long>(b) * p.classes : nullptr;
  l.allowed = p.allowed && s >= 0 && s < p.sets ? p.allowed + static_cast<long long>(s) * p.words : nullptr;
  return true;
}

// z of a class that is n times in the line's history.
__device__ __forceinline__ float penalised(float z, int n, const LineRule& l) {
  const float v = z > 0.0f ? __fdiv_rn(z, l.repeat) : __fmul_rn(z, l.repeat);
  return __fsub_rn(v, __fadd_rn(__fmul_rn(static_cast<float>(n), l.frequency), l.presence));
}

__device__ __forceinline__ float load_logit(const float* z) { return *z; }
__device__ __forceinline__ float load_logit(const __half* z) { return __half2float(*z); }

// The lowest class of the highest logit in a key that a maximum finds: the float's order above
// (-0 made +0, its equal), the class's reverse order below.
__device__ __forceinline__ uint32_t float_order(float v) {
  const uint32_t b = __float_as_uint(__fadd_rn(v, 0.0f));
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float order_float(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ unsigned long long class_key(float v, int c) {
  return static_cast<unsigned long long>(float_order(v)) << 32 | (0xffffffffu - static_cast<uint32_t>(c));
}

constexpr int kRowThreads = 256;

__device__ __forceinline__ unsigned long long block_max(unsigned long long v, unsigned long long* sh) {
  for (int o = 16; o; o >>= 1) {
    const unsigned long long u = __shfl_xor_sync(0xffffffffu, v, o);
    v = u > v ? u : v;
  }
  __syncthreads();
  if (threadIdx.x % 32 == 0) sh[threadIdx.x / 32] = v;
  __syncthreads();
  v = sh[0];
  for (int w = 1; w < kRowThreads / 32; ++w) v = sh[w] > v ? sh[w] : v;
  return v;
}

__device__ __forceinline__ float block_sum(float v, float* sh) {
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if (threadIdx.x % 32 == 0) sh[threadIdx.x / 32] = v;
  __syncthreads();
  v = 0.0f;
  for (int w = 0; w < kRowThreads / 32; ++w) v += sh[w];
  return v;
}

// A block a row: the history's counts in shared memory, then the row.
template <int kOp, typename T>
__global__ void __launch_bounds__(kRowThreads) line_rows_kernel(const __grid_constant__ LineParams p) {
  extern __shared__ int32_t count[];  // [classes]
  __shared__ unsigned long long sh_key[kRowThreads / 32];
  __shared__ float sh_sum[kRowThreads / 32];
  const int r = blockIdx.x;
  LineRule l;
  if (!find_line(p, r, threadIdx.x % 32, l)) return;
  const bool had = l.n_had > 0;
  if (had) {
    for (int c = threadIdx.x; c < p.classes; c += kRowThreads) count[c] = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < l.n_had; j += kRowThreads) {
      const int c = l.had[j];
      if (c >= 0 && c < p.classes) atomicAdd(&count[c], 1);
    }
    __syncthreads();
  }
  const T* z = static_cast<const T*>(p.z) + r * p.pitch;
  auto ruled = [&](int c) {
    float v = load_logit(z + c);
    if (had && count[c] > 0) v = penalised(v, count[c], l);
    if (l.bias) {
      const float b = l.bias[c];
      v = b == -INFINITY ? -INFINITY : __fadd_rn(v, b);
    }
    if (l.allowed && !(l.allowed[c / 32] >> (c % 32) & 1)) v = -INFINITY;
    return v;
  };
  if constexpr (kOp == kOpRules) {
    for (int c = threadIdx.x; c < p.classes; c += kRowThreads) {
      const float v = ruled(c);
      if (p.out_half) static_cast<__half*>(p.out)[r * p.out_pitch + c] = __float2half_rn(v);
      else static_cast<float*>(p.out)[r * p.out_pitch + c] = v;
    }
  } else {
    unsigned long long key = 0;
    for (int c = threadIdx.x; c < p.classes; c += kRowThreads) {
      const float v = ruled(c);
      const unsigned long long k = v == v ? class_key(v, c) : 0ull;
      key = k > key ? k : key;
    }
    key = block_max(key, sh_key);
    const float best = key ? order_float(static_cast<uint32_t>(key >> 32)) : -INFINITY;
    const bool some = best > -INFINITY;
    float sum = 0.0f;
    for (int c = threadIdx.x; c < p.classes; c += kRowThreads) sum += expf(__fsub_rn(ruled(c), some ? best : 0.0f));
    sum = block_sum(sum, sh_sum);
    if constexpr (kOp == kOpGreedy) {
      if (threadIdx.x == 0) {
        p.ids[r] = some ? static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(key)) : 0;
        p.probs[r] = some ? __fdiv_rn(1.0f, sum) : sum == sum ? 0.0f : sum;
      }
    } else {
      const float base = some ? best : 0.0f, ln = some ? logf(sum) : sum == sum ? 0.0f : sum;
      if (threadIdx.x == 0) p.blank[r] = __fsub_rn(__fsub_rn(ruled(0), base), ln);
      unsigned long long above = ~0ull;
      for (int q = 0; q < p.topk; ++q) {
        key = 0;
        for (int c = 1 + threadIdx.x; c < p.classes; c += kRowThreads) {
          const float v = ruled(c);
          const unsigned long long k = v > -INFINITY ? class_key(v, c) : 0ull;
          if (k < above && k > key) key = k;
        }
        key = block_max(key, sh_key);
        if (threadIdx.x == 0) {
          const size_t o = static_cast<size_t>(r) * p.topk + q;
          p.ids[o] = key ? static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(key)) : -1;
          p.probs[o] = key ? __fsub_rn(__fsub_rn(order_float(static_cast<uint32_t>(key >> 32)), base), ln) : -INFINITY;
        }
        above = key;
      }
    }
  }
}

// Greedy CTC's second half, a warp a line, in place: ids and probs hold each frame's class and
// probability; the characters go to the front of the line's places (never past the frames already
// read), the rest is filled.
__global__ void __launch_bounds__(128) collapse_lines_kernel(const __grid_constant__ LineParams p) {
  const int i = blockIdx.x * 4 + threadIdx.x / 32, lane = threadIdx.x % 32;
  if (i >= p.lines) return;
  const int first = min(max(p.line_at[i], 0), p.rows), end = min(max(p.line_at[i + 1], first), p.rows);
  int prev = 0;       // the class of the frame before
  int k = 0;          // characters so far
  float carry = 0.0f;  // the last character's highest probability, where it may go on
  for (int t0 = first; t0 < end; t0 += 32) {
    const int t = t0 + lane;
    const int id = t < end ? p.ids[t] : 0;
    float pr = t < end ? p.probs[t] : 0.0f;
    int before = __shfl_up_sync(0xffffffffu, id, 1);
    if (lane == 0) before = prev;
    const bool goes_on = id != 0 && id == before;
    const unsigned begins = __ballot_sync(0xffffffffu, id != 0 && id != before);
    // the highest probability up to this frame of the frames of its character
    for (int o = 1; o < 32; o <<= 1) {
      const float up = __shfl_up_sync(0xffffffffu, pr, o);
      const unsigned between = lane >= o ? begins & (0xffffffffu >> (31 - lane)) & ~(0xffffffffu >> (31 - (lane - o))) : 1u;
      const int uid = __shfl_up_sync(0xffffffffu, id, o);
      if (lane >= o && between == 0 && uid == id) pr = up > pr ? up : pr;
    }
    const unsigned mine = begins & (0xffffffffu >> (31 - lane));
    const bool from_before = goes_on && mine == 0;
    if (from_before) pr = carry > pr ? carry : pr;
    const int after = __shfl_down_sync(0xffffffffu, id, 1);
    const bool last = id != 0 && (lane == 31 || after != id);
    const int nth = k + __popc(mine) - 1;
    __syncwarp();
    if (last) {
      p.ids[first + nth] = id;
      p.probs[first + nth] = pr;
    }
    if (begins >> lane & 1) p.starts[first + nth] = t - first;
    k += __popc(begins);
    prev = __shfl_sync(0xffffffffu, id, 31);
    carry = __shfl_sync(0xffffffffu, pr, 31);
    __syncwarp();
  }
  for (int t = first + k + lane; t < end; t += 32) {
    p.ids[t] = -1;
    p.starts[t] = -1;
    p.probs[t] = 0.0f;
  }
  if (lane == 0) p.counts[i] = k;
}

}  // namespace crec
