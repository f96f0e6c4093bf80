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
#include <cstring>

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
  long long out_pitch;
  int32_t* counts;  // greedy
  int32_t* ids;
  int32_t* starts;
  float* probs;  // greedy: probabilities; candidates: log-probabilities
  float* blank;
  int topk;
  // how the rows are shared out (line_ops.cu)
  int warps;      // of a team
  int span;       // classes a warp holds at once, a multiple of 32 * V
  int chunks;     // passes over the classes a row takes
  int slots;      // chunks * warps
  int team_rows;  // rows a team takes
  int bias_wide;  // the bias tables' rows may be read 16 bytes at a time
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

// z of a class of the line's history; less: n * frequency + presence.
__device__ __forceinline__ float penalised(float z, float less, float repeat) {
  return __fsub_rn(z > 0.0f ? __fdiv_rn(z, repeat) : __fmul_rn(z, repeat), less);
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

// ---------------------------------------------------------------- the rows
//
// A team of `p.warps` warps takes rows one after another, each warp `p.span` (at most 1,024) of the
// classes, a lane up to 32 of them in registers: V consecutive ones every 32 * V.  What a line's
// rules add to those classes (its bias, -inf for what its set leaves out) stays in registers too, from
// row to row until the line changes.  The classes of the line's history are taken out of that dense
// pass (-inf, a bit in `gone`) and go through a list of their own, so that the division costs a few
// lanes' work once a row and not every class a branch.
//
// A row is read once and held while its maximum is found and its sum of exp(z - best) taken; the
// next row's loads are in flight meanwhile.

constexpr int kLaneClasses = 32;
constexpr int kWarpClasses = 32 * kLaneClasses;
constexpr int kMaxTeam = 16;                        // warps
constexpr int kMaxClasses = 4 * kMaxTeam * kWarpClasses;
constexpr int kMaxSlots = 4 * kMaxTeam;             // a row's partial results
constexpr int kMaxTop = 16;
constexpr int kShortList = 64;  // candidates of a warp ranked at once
constexpr float kLog2e = 1.44269504088896341f;

// A warp's part of shared memory where there are histories: 10 bytes a class of its span.
struct HadList {
  uint32_t* count;  // [span] a class's count, then n * frequency + presence (its bits)
  float* add;       // [span] an entry's bias, -inf where the set leaves it out
  uint16_t* at;     // [span] the entries' classes within the span
  int n;
};

template <typename T, int V>
struct Raw;
template <>
struct Raw<float, 4> {
  float4 r;
  __device__ __forceinline__ void zero() { r = make_float4(0.0f, 0.0f, 0.0f, 0.0f); }
  __device__ __forceinline__ void load(const float* z) { r = *reinterpret_cast<const float4*>(z); }
  __device__ __forceinline__ void part(const float* z, int n) {
    r = make_float4(z[0], n > 1 ? z[1] : 0.0f, n > 2 ? z[2] : 0.0f, 0.0f);
  }
  __device__ __forceinline__ void get(float* v) const {
    v[0] = r.x;
    v[1] = r.y;
    v[2] = r.z;
    v[3] = r.w;
  }
};
template <>
struct Raw<__half, 8> {
  uint4 r;
  __device__ __forceinline__ void zero() { r = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void load(const __half* z) { r = *reinterpret_cast<const uint4*>(z); }
  __device__ __forceinline__ void part(const __half* z, int n) {
    const unsigned short* u = reinterpret_cast<const unsigned short*>(z);
    auto two = [&](int i) { return (i < n ? static_cast<uint32_t>(u[i]) : 0u) | (i + 1 < n ? static_cast<uint32_t>(u[i + 1]) << 16 : 0u); };
    r = make_uint4(two(0), two(2), two(4), two(6));
  }
  __device__ __forceinline__ void get(float* v) const {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __half2 h;
      memcpy(&h, &w[i], 4);
      const float2 f = __half22float2(h);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
};
template <typename T>
struct Raw<T, 1> {
  T r;
  __device__ __forceinline__ void zero() { memset(&r, 0, sizeof r); }
  __device__ __forceinline__ void load(const T* z) { r = *z; }
  __device__ __forceinline__ void part(const T* z, int) { r = *z; }
  __device__ __forceinline__ void get(float* v) const { v[0] = load_logit(&r); }
};

// V ruled logits written at o, those in `gone` (a bit each) left to the list.
template <typename O, int V>
__device__ __forceinline__ void store_ruled(O* o, const float* v, uint32_t gone, int n) {
  if (V > 1 && gone == 0 && n >= V) {
    if constexpr (sizeof(O) == 2) {
      uint32_t w[V / 2 > 0 ? V / 2 : 1];
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        memcpy(&w[i], &h, 4);
      }
      if constexpr (V == 8) __stcs(reinterpret_cast<uint4*>(o), make_uint4(w[0], w[1], w[2], w[3]));
      if constexpr (V == 4) __stcs(reinterpret_cast<uint2*>(o), make_uint2(w[0], w[1]));
    } else {
#pragma unroll
      for (int i = 0; i < V / 4; ++i)
        __stcs(reinterpret_cast<float4*>(o) + i, make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]));
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (i < n && !(gone >> i & 1)) {
      if constexpr (sizeof(O) == 2) o[i] = __float2half_rn(v[i]);
      else o[i] = v[i];
    }
}

__device__ __forceinline__ float warp_max(float v) {
  float m;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ unsigned long long warp_max_key(unsigned long long k) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(k >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(k >> 32) == hi ? static_cast<uint32_t>(k) : 0u);
  return static_cast<unsigned long long>(hi) << 32 | lo;
}
__device__ __forceinline__ float exp_less(float v, float best) { return ex2_approx(__fmul_rn(__fsub_rn(v, best), kLog2e)); }

// A row's partial results, one a (chunk, warp) slot, two rows' worth (the next row's are written
// while a warp joins this one's).
struct RowSlots {
  float best[2][kMaxSlots];
  float sum[2][kMaxSlots];
  int32_t arg[2][kMaxSlots];  // greedy: the lowest class of the slot's best
  float blank[2];
};

// A warp's topk highest of its classes (v, the lanes' registers) and its n entries, as keys at
// top[0, topk), highest first, 0 where nothing is left (-inf never is one).  The k-th highest of the
// lanes' own maxima is at most the k-th highest of all, so only what reaches it is ranked: k keys
// and a few more, unless many classes tie.
template <int V, typename Entry>
__device__ __forceinline__ void warp_top(int topk, int nv, const float (&v)[kLaneClasses], int n, Entry entry, int base,
                                         int lane, unsigned long long* list, unsigned long long* top) {
  constexpr int NV = kLaneClasses / V;
  if (topk == 0) return;
  float high = -INFINITY;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (j >= nv) break;
#pragma unroll
    for (int i = 0; i < V; ++i) high = fmaxf(high, v[j * V + i]);
  }
  for (int e = lane; e < n; e += 32) {
    int c;
    high = fmaxf(high, entry(e, c));
  }
  float s = high;  // sorted over the lanes, highest first
#pragma unroll
  for (int k = 2; k <= 32; k *= 2)
#pragma unroll
    for (int o = k / 2; o > 0; o /= 2) {
      const float u = __shfl_xor_sync(0xffffffffu, s, o);
      s = ((lane & o) == 0) == ((lane & k) == 0) ? fmaxf(s, u) : fminf(s, u);
    }
  const float reach = fmaxf(__shfl_sync(0xffffffffu, s, topk - 1), -3.402823466e38f);
  int mine = 0;
  if (high >= reach) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (j >= nv) break;
#pragma unroll
      for (int i = 0; i < V; ++i) mine += v[j * V + i] >= reach;
    }
    for (int e = lane; e < n; e += 32) {
      int c;
      mine += entry(e, c) >= reach;
    }
  }
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int u = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += u;
  }
  const int all = __shfl_sync(0xffffffffu, upto, 31);
  if (all <= kShortList) {
    if (mine) {
      int at = upto - mine;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (j >= nv) break;
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (v[j * V + i] >= reach) list[at++] = class_key(v[j * V + i], base + (j * 32 + lane) * V + i);
      }
      for (int e = lane; e < n; e += 32) {
        int c;
        const float x = entry(e, c);
        if (x >= reach) list[at++] = class_key(x, c);
      }
    }
    __syncwarp();
    const unsigned long long a = lane < all ? list[lane] : 0ull, b = lane + 32 < all ? list[lane + 32] : 0ull;
    int ra = 0, rb = 0;
    for (int i = 0; i < all; ++i) {
      const unsigned long long k = list[i];
      ra += k > a;
      rb += k > b;
    }
    if (a && ra < topk) top[ra] = a;
    if (b && rb < topk) top[rb] = b;
    for (int q = all + lane; q < topk; q += 32) top[q] = 0ull;
    __syncwarp();
    return;
  }
  // many alike: the highest key below the last one found, topk times
  unsigned long long below = ~0ull;
  for (int q = 0; q < topk; ++q) {
    unsigned long long k = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (j >= nv) break;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const unsigned long long u = v[j * V + i] >= reach ? class_key(v[j * V + i], base + (j * 32 + lane) * V + i) : 0ull;
        if (u < below && u > k) k = u;
      }
    }
    for (int e = lane; e < n; e += 32) {
      int c;
      const float x = entry(e, c);
      const unsigned long long u = x >= reach ? class_key(x, c) : 0ull;
      if (u < below && u > k) k = u;
    }
    below = warp_max_key(k);
    if (lane == 0) top[q] = below;
  }
  __syncwarp();
}

// A row's slots joined by one warp, and the row's results written.
template <int kOp>
__device__ __forceinline__ void join_slots(const LineParams& p, int r, int lane, const RowSlots& s, int parity,
                                           const unsigned long long* tops) {
  static_assert(kMaxSlots == 64, "two slots a lane");
  const bool one = lane < p.slots, two = lane + 32 < p.slots;
  const float b0 = one ? s.best[parity][lane] : -INFINITY, b1 = two ? s.best[parity][lane + 32] : -INFINITY;
  const float best = warp_max(fmaxf(b0, b1));
  const bool some = best > -INFINITY;
  const float from = some ? best : 0.0f;
  const float s0 = one ? s.sum[parity][lane] : 0.0f, s1 = two ? s.sum[parity][lane + 32] : 0.0f;
  const float sum = warp_sum((b0 == -INFINITY ? s0 : s0 * exp_less(b0, from)) + (b1 == -INFINITY ? s1 : s1 * exp_less(b1, from)));
  if constexpr (kOp == kOpGreedy) {
    uint32_t c = one && b0 == best ? static_cast<uint32_t>(s.arg[parity][lane]) : 0x7fffffffu;
    if (two && b1 == best) c = min(c, static_cast<uint32_t>(s.arg[parity][lane + 32]));
    c = __reduce_min_sync(0xffffffffu, c);
    if (lane == 0) {
      p.ids[r] = some ? static_cast<int32_t>(c) : 0;
      p.probs[r] = some ? __fdiv_rn(1.0f, sum) : sum;  // nothing left: 0 (NaN where one is allowed)
    }
  } else {
    const float ln = some ? logf(sum) : sum;
    unsigned long long mine = 0;
    if (p.slots == 1) {
      if (lane < p.topk) mine = tops[lane];
    } else {
      int at0 = 0, at1 = 0;
      unsigned long long h0 = one && p.topk ? tops[lane * kMaxTop] : 0ull, h1 = two && p.topk ? tops[(lane + 32) * kMaxTop] : 0ull;
      for (int q = 0; q < p.topk; ++q) {
        const unsigned long long k = warp_max_key(h0 > h1 ? h0 : h1);
        if (lane == q) mine = k;
        if (k == 0) break;
        if (h0 == k) h0 = ++at0 < p.topk ? tops[lane * kMaxTop + at0] : 0ull;
        else if (h1 == k) h1 = ++at1 < p.topk ? tops[(lane + 32) * kMaxTop + at1] : 0ull;
      }
    }
    if (lane < p.topk) {
      const size_t o = static_cast<size_t>(r) * p.topk + lane;
      p.ids[o] = mine ? static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(mine)) : -1;
      p.probs[o] = mine ? __fsub_rn(__fsub_rn(order_float(static_cast<uint32_t>(mine >> 32)), from), ln) : -INFINITY;
    }
    if (lane == 0) p.blank[r] = __fsub_rn(__fsub_rn(s.blank[parity], from), ln);
  }
}

template <int kOp, typename T, typename O, int V>
__global__ void __launch_bounds__(512, 1) line_rows_kernel(const __grid_constant__ LineParams p) {
  constexpr int NV = kLaneClasses / V;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int team = warp / p.warps, w = warp % p.warps, teams = blockDim.x / 32 / p.warps;
  const int nv = p.span / (32 * V);
  // shared memory: the teams' slots, the warps' candidate lists, the warps' history lists
  RowSlots* slots = reinterpret_cast<RowSlots*>(smem) + team;
  unsigned long long* tops = reinterpret_cast<unsigned long long*>(smem + teams * sizeof(RowSlots)) +
                             static_cast<size_t>(team) * 2 * p.slots * kMaxTop;  // [2][slots][kMaxTop]
  uint8_t* after = smem + teams * sizeof(RowSlots) +
                   (kOp == kOpCandidates ? static_cast<size_t>(teams) * 2 * p.slots * kMaxTop * 8 : 0);
  unsigned long long* shortlist = reinterpret_cast<unsigned long long*>(after) + warp * kShortList;
  if (kOp == kOpCandidates) after += static_cast<size_t>(blockDim.x / 32) * kShortList * 8;
  HadList had;
  had.n = 0;
  had.count = reinterpret_cast<uint32_t*>(after + static_cast<size_t>(warp) * p.span * 10);
  had.add = reinterpret_cast<float*>(had.count + p.span);
  had.at = reinterpret_cast<uint16_t*>(had.add + p.span);
  if (p.history) {
    for (int i = lane; i < p.span; i += 32) had.count[i] = 0;
    __syncwarp();
  }

  const long long r0 = (static_cast<long long>(blockIdx.x) * teams + team) * p.team_rows;
  const int r1 = static_cast<int>(min(static_cast<long long>(p.rows), r0 + p.team_rows));
  if (r0 >= r1) return;

  LineRule l;
  l.first = l.end = 0;
  float add[kLaneClasses];
  uint32_t gone = 0;  // bit j * V + i: the class is in the line's history
  Raw<T, V> raw[NV];
  auto load = [&](int r, int base) {
    const T* z = static_cast<const T*>(p.z) + r * p.pitch + base;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (j >= nv) break;
      const int c = (j * 32 + lane) * V, left = p.classes - base - c;
      if (left >= V) raw[j].load(z + c);
      else if (left > 0) raw[j].part(z + c, left);
      else raw[j].zero();
    }
  };
  // the line's rules on this warp's classes [base, base + span)
  auto set_rules = [&](int base) {
    for (int e = lane; e < had.n; e += 32) had.count[had.at[e]] = 0;
    __syncwarp();
    had.n = 0;
    gone = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (j >= nv) break;
      const int c = base + (j * 32 + lane) * V;
      const uint32_t keep = l.allowed && c < p.classes ? l.allowed[c >> 5] >> (c & 31) : ~0u;
      float b[V];
      if (V > 1 && p.bias_wide && l.bias && c + V <= p.classes) {
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
          const float4 f = *reinterpret_cast<const float4*>(l.bias + c + 4 * i);
          b[4 * i] = f.x;
          b[4 * i + 1] = f.y;
          b[4 * i + 2] = f.z;
          b[4 * i + 3] = f.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) b[i] = l.bias && c + i < p.classes ? l.bias[c + i] : 0.0f;
      }
#pragma unroll
      for (int i = 0; i < V; ++i) add[j * V + i] = c + i < p.classes && (keep >> i & 1) ? b[i] : -INFINITY;
    }
    if (l.n_had <= 0) return;
    for (int k0 = 0; k0 < l.n_had; k0 += 32) {
      const int k = k0 + lane, c = k < l.n_had ? l.had[k] - base : -1;
      const bool mine = c >= 0 && c < p.span && base + c < p.classes;
      const bool first = mine && atomicAdd(&had.count[c], 1u) == 0;
      const unsigned m = __ballot_sync(0xffffffffu, first);
      if (first) had.at[had.n + __popc(m & ((1u << lane) - 1))] = static_cast<uint16_t>(c);
      had.n += __popc(m);
    }
    if (had.n == 0) return;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (j >= nv) break;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (had.count[(j * 32 + lane) * V + i]) {
          gone |= 1u << (j * V + i);
          add[j * V + i] = -INFINITY;
        }
    }
    __syncwarp();
    for (int e = lane; e < had.n; e += 32) {
      const int c = had.at[e];
      const float n = static_cast<float>(had.count[c]);
      had.count[c] = __float_as_uint(__fadd_rn(__fmul_rn(n, l.frequency), l.presence));
      const bool keep = !l.allowed || (l.allowed[(base + c) >> 5] >> ((base + c) & 31) & 1);
      had.add[e] = keep ? (l.bias ? l.bias[base + c] : 0.0f) : -INFINITY;
    }
    __syncwarp();
  };
  // entry e of the line's history in a row (z: its classes from `base`)
  auto entry = [&](const T* z, int e) {
    const int c = had.at[e];
    const float a = had.add[e];
    const float v = penalised(load_logit(z + c), __uint_as_float(had.count[c]), l.repeat);
    return a == -INFINITY ? a : __fadd_rn(v, a);
  };

  int parity = 0;
  const int base0 = w * p.span;
  if (p.chunks == 1) load(static_cast<int>(r0), base0);
  for (int r = static_cast<int>(r0); r < r1; ++r) {
    bool fresh = false;
    if (r < l.first || r >= l.end) {
      fresh = true;
      if (!find_line(p, r, lane, l)) {
        l.first = l.end = 0;
        if (p.chunks == 1 && r + 1 < r1) load(r + 1, base0);
        continue;  // no line's row (every warp of the team finds the same)
      }
    }
    for (int chunk = 0; chunk < p.chunks; ++chunk) {
      const int base = (chunk * p.warps + w) * p.span;
      const T* z = static_cast<const T*>(p.z) + r * p.pitch + base;
      if (p.chunks > 1) load(r, base);
      if (fresh || p.chunks > 1) set_rules(base);
      float v[kLaneClasses];
      auto ruled = [&](bool careful) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          if (j >= nv) break;
          float u[V];
          raw[j].get(u);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float a = add[j * V + i], s = __fadd_rn(u[i], a);
            v[j * V + i] = careful && a == -INFINITY ? a : s;
          }
        }
      };
      if constexpr (kOp == kOpRules) {
        ruled(true);
        if (p.chunks == 1 && r + 1 < r1) load(r + 1, base0);
        O* o = static_cast<O*>(p.out) + r * p.out_pitch + base;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          if (j >= nv) break;
          const int c = (j * 32 + lane) * V;
          if (base + c < p.classes)
            store_ruled<O, V>(o + c, v + j * V, gone >> (j * V) & ((1u << V) - 1), p.classes - base - c);
        }
        for (int e = lane; e < had.n; e += 32) {
          const float x = entry(z, e);
          if constexpr (sizeof(O) == 2) o[had.at[e]] = __float2half_rn(x);
          else o[had.at[e]] = x;
        }
      } else {
        // this warp's best, the sum of exp(z - best) and what else the row wants, into its slot
        const int slot = chunk * p.warps + w;
        float best, sum;
        float m[NV];
        float xm, xs;  // the entries': highest, and the sum of exp(x - xm)
        int arg = 0;   // greedy: the lowest class of the best
        for (bool careful = false;; careful = true) {
          ruled(careful);
          if (p.chunks == 1 && r + 1 < r1) load(r + 1, base0);
#pragma unroll
          for (int j = 0; j < NV; ++j) {
            m[j] = -INFINITY;
            if (j >= nv) continue;
#pragma unroll
            for (int i = 0; i < V; ++i) m[j] = fmaxf(m[j], v[j * V + i]);
          }
#pragma unroll
          for (int s = NV / 2; s > 0; s /= 2)
#pragma unroll
            for (int j = 0; j < s; ++j) m[j] = fmaxf(m[j], m[j + s]);
          xm = -INFINITY;
          xs = 0.0f;
          int xc = 0x7fffffff;
          for (int e = lane; e < had.n; e += 32) {
            const float x = entry(z, e);
            if (x > xm) {
              xs = __fadd_rn(xm == -INFINITY ? xs : __fmul_rn(xs, exp_less(xm, x)), 1.0f);
              xm = x;
              xc = base + had.at[e];
            } else if (x != -INFINITY) {
              if (x == xm) xc = min(xc, base + had.at[e]);
              xs = __fadd_rn(xs, exp_less(x, xm));
            }
          }
          best = warp_max(fmaxf(m[0], xm));
          const float from = best == -INFINITY ? 0.0f : best;
          float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int j = 0; j < NV; ++j) {
            if (j >= nv) break;
#pragma unroll
            for (int i = 0; i < V; ++i) s[(j * V + i) % 4] += exp_less(v[j * V + i], from);
          }
          sum = (s[0] + s[1]) + (s[2] + s[3]);
          if (had.n) sum += xm == -INFINITY ? xs : xs * exp_less(xm, from);
          sum = warp_sum(sum);
          if constexpr (kOp == kOpGreedy) {
            int c = xm == best ? xc : 0x7fffffff;
            if (m[0] == best) {
#pragma unroll
              for (int j = NV - 1; j >= 0; --j) {
                if (j >= nv) continue;
#pragma unroll
                for (int i = V - 1; i >= 0; --i)
                  if (v[j * V + i] == best) c = min(c, base + (j * 32 + lane) * V + i);
              }
            }
            arg = static_cast<int>(__reduce_min_sync(0xffffffffu, static_cast<uint32_t>(c)));
          }
          // a NaN or +inf met a -inf (or is allowed): once more, choosing instead of adding
          if (careful || sum == sum) break;
          load(r, base);
        }
        if (lane == 0) {
          slots->best[parity][slot] = best;
          slots->sum[parity][slot] = sum;
          slots->arg[parity][slot] = arg;
        }
        if constexpr (kOp == kOpCandidates) {
          if (base == 0) {  // the blank: noted, and out of the candidates
            if (lane == 0) {
              slots->blank[parity] = v[0];
              v[0] = -INFINITY;
            }
            __syncwarp();
            for (int e = lane; e < had.n; e += 32)
              if (had.at[e] == 0) slots->blank[parity] = entry(z, e);
            __syncwarp();
          }
          warp_top<V>(p.topk, nv, v, had.n, [&](int e, int& c) {
            c = base + had.at[e];
            return c == 0 ? -INFINITY : entry(z, e);
          }, base, lane, shortlist, tops + (static_cast<size_t>(parity) * p.slots + slot) * kMaxTop);
        }
      }
    }
    if constexpr (kOp != kOpRules) {
      if (p.warps > 1) named_bar(1 + team, p.warps * 32);
      else __syncwarp();
      if (r % p.warps == w) join_slots<kOp>(p, r, lane, *slots, parity, tops + static_cast<size_t>(parity) * p.slots * kMaxTop);
      parity ^= 1;
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
