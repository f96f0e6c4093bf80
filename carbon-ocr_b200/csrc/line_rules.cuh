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
  const void* z_end;  // past the last row's last class
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
  int warps;      // of a team, a power of two
  int chunks;     // rules: the spans that a row takes
  int team_rows;  // rows a team takes
  int bias_wide;  // the bias tables' rows may be read 16 bytes at a time
};

constexpr int kOpGreedy = 1, kOpCandidates = 2;

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
// A warp holds a span of a row's classes in registers, a lane V consecutive ones every 32 * V.  What
// the line's rules add to them (its bias, -inf for what its set leaves out) lies in the warp's shared
// memory from row to row until the line changes (in registers beside the row it spilled: 206 us against
// 94 for greedy decoding of 65,536 frames of 800 classes).  The classes of the line's history are taken
// out of that dense pass (-inf) and go through a list of their own, so that the division costs a few
// lanes' work once a row and not every class a branch.  The next row is copied to shared memory while
// a row is worked on.
//
// Bounds, at 65,536 x 800 float32 (210 MB read): greedy 60 us, 3.5 TB/s, by instructions (400 a frame;
// half the issue slots of 16 warps an SM, each waiting on its own results); the ruled logits 84 us,
// 5.0 TB/s read and written, near what 32 warps' copies in flight bring from HBM.

constexpr int kDecodeLane = 32;  // classes a lane holds in the decoders: 128 registers, 16 warps an SM
constexpr int kDecodeEntries = 256;  // of a span in the decoders; a line with more goes the slow way
constexpr int kRulesLane = 16;   // and where the ruled logits are written
constexpr int kMaxTeam = 16;     // warps that share a row
constexpr int kMaxClasses = 65536;
constexpr int kMaxTop = 16;
constexpr int kShortList = 64;  // a row's candidates ranked at once
constexpr float kLog2e = 1.44269504088896341f;

// 16 bytes (both ends aligned to them) to shared memory without waiting; past `valid` bytes zeros.
__device__ __forceinline__ void copy_async(void* shared, const void* global, int valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(shared)), "l"(global), "r"(valid) : "memory");
}
// n logits from any address to shared memory without waiting, by a whole warp, in the 16-byte pieces that
// hold them: they begin at shared[returned], what comes with them on either side is of no use.  A
// piece that reaches past the array itself (its first or its last) goes logit by logit.
template <typename T>
__device__ __forceinline__ int copy_row(const LineParams& p, T* shared, const T* z, int n, int lane) {
  const uintptr_t first = reinterpret_cast<uintptr_t>(z), end = first + static_cast<uintptr_t>(max(n, 0)) * sizeof(T), low = first & ~uintptr_t(15);
  for (uintptr_t q = low + 16 * lane; q < end; q += 512) {
    T* s = shared + (q - low) / sizeof(T);
    if (q >= reinterpret_cast<uintptr_t>(p.z) && q + 16 <= reinterpret_cast<uintptr_t>(p.z_end)) {
      copy_async(s, reinterpret_cast<const void*>(q), 16);
    } else {
      for (int i = 0; i < 16 / static_cast<int>(sizeof(T)); ++i) {
        const uintptr_t at = q + i * sizeof(T);
        if (at >= first && at < end) s[i] = *reinterpret_cast<const T*>(at);
      }
    }
  }
  return static_cast<int>((first - low) / sizeof(T));
}
__device__ __forceinline__ void copy_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// V logits from shared memory as float32.
template <int V>
__device__ __forceinline__ void get_logits(const float* z, float* v) {
  if constexpr (V == 4) {
    const float4 f = *reinterpret_cast<const float4*>(z);
    v[0] = f.x;
    v[1] = f.y;
    v[2] = f.z;
    v[3] = f.w;
  } else {
    v[0] = z[0];
  }
}
template <int V>
__device__ __forceinline__ void get_logits(const __half* z, float* v) {
  if constexpr (V == 8) {
    const uint4 r = *reinterpret_cast<const uint4*>(z);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __half2 h;
      memcpy(&h, &w[i], 4);
      const float2 f = __half22float2(h);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  } else {
    v[0] = __half2float(z[0]);
  }
}

// V ruled logits (n of them classes) written at o.
template <typename O, int V>
__device__ __forceinline__ void store_ruled(O* o, const float* v, int n) {
  if (V > 1 && n >= V) {
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
    if (i < n) {
      if constexpr (sizeof(O) == 2) o[i] = __float2half_rn(v[i]);
      else o[i] = v[i];
    }
}

// Programmatic dependent launch: a kernel queued to start early waits here for the one before it to
// be done; that one says, once all its blocks run, that the next may start.
__device__ __forceinline__ void launch_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

__device__ __forceinline__ float warp_max(float v) {
  float m;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}
// The maximum, NaN where one of them is.
__device__ __forceinline__ float warp_max_nan(float v) {
  float m;
  asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}
// The same of two.
__device__ __forceinline__ float max_nan(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
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
// exp(v - best) times a factor near 1 that is the same for all of a row's classes: 2^(v log2 e - c), c
// the rounded best * log2 e, in one fused step.  What is made of a row's sums is divided by best's own
// exp_less, which takes the factor out again, and with it the rounding of c.  ex2.approx is within 2^-22:
// greedy's probabilities are 7.1e-8 of their norm from 64 bits where exp's in float32 are 6.2e-8 (65,536
// frames of 800 classes), log-probabilities 3.9e-8 where those are 3.6e-8 (4,096 of 12,000).
__device__ __forceinline__ float exp_less(float v, float c) { return ex2_approx(__fmaf_rn(v, kLog2e, -c)); }

// A row's best (0 where nothing is left) and what its sums are taken against.
struct RowBase {
  float best, c;
  bool fits;  // c's rounding is below 2^-4; else (|best| past 7e5) the difference is taken first
  __device__ __forceinline__ explicit RowBase(float b) {
    best = b == -INFINITY ? 0.0f : b;
    c = __fmul_rn(best, kLog2e);
    fits = fabsf(c) < 1048576.0f;
  }
  __device__ __forceinline__ float term(float v) const { return fits ? exp_less(v, c) : ex2_approx(__fmul_rn(__fsub_rn(v, best), kLog2e)); }
};

// Two at a time on the packed FP32 pipe, each half rounded on its own.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n .reg .b64 a, b, c, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n"
      " fma.rn.f32x2 d, a, b, c;\n mov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}

// A warp's part of shared memory: add, what the rules add to each class of its span in the dense pass,
// -inf for what the set leaves out, for the history's classes and past the last class (while a
// line's rules are set, the history's counts); then the entries, the history's classes that are
// allowed: n * frequency + presence, and places within the span; at most kCap are kept.
template <int kSpan, int kCap>
struct SpanRules {
  float* add;
  float* less;
  uint16_t* at;
  __device__ __forceinline__ explicit SpanRules(uint8_t* shared) {
    add = reinterpret_cast<float*>(shared);
    less = add + kSpan;
    at = reinterpret_cast<uint16_t*>(less + kCap);
  }
  static constexpr int kBytes = kSpan * 4 + kCap * 6;
};

// A line's rules on the classes [base, base + 32 * V * NV) into a warp's SpanRules; the number of
// entries (past kCap they are counted, not kept).  Once a line: not inlined, its code out of the
// rows' way.
template <int V, int NV, int kCap>
__device__ __noinline__ int set_rules(uint8_t* shared, int classes, int base, const int32_t* had, int n_had, float presence,
                                      float frequency, const float* bias, bool bias_wide, const uint32_t* allowed) {
  constexpr int kSpan = 32 * V * NV;
  const SpanRules<kSpan, kCap> s(shared);
  const int lane = threadIdx.x % 32;
  uint32_t* count = reinterpret_cast<uint32_t*>(s.add);
  int n = 0;
  __syncwarp();
  if (n_had > 0) {
    for (int i = lane; i < kSpan; i += 32) count[i] = 0;
    __syncwarp();
    for (int k = lane; k < n_had; k += 32) {
      const int c = had[k] - base;
      if (c >= 0 && c < kSpan) atomicAdd(&count[c], 1u);
    }
    __syncwarp();
    // each class once, by the first lane that has it of the first step that does: the entries' order,
    // and with it the order of every sum over them, is the history's
    for (int k0 = 0; k0 < n_had; k0 += 32) {
      const int c = k0 + lane < n_had ? had[k0 + lane] - base : -1;
      const unsigned same = __match_any_sync(0xffffffffu, c);
      const bool takes = c >= 0 && c < kSpan && (same & ((1u << lane) - 1)) == 0;
      const uint32_t times = takes ? count[c] : 0u;
      __syncwarp();
      if (takes) count[c] = 0;
      __syncwarp();
      const bool left_out = times && (base + c >= classes || (allowed && !(allowed[(base + c) >> 5] >> ((base + c) & 31) & 1)) ||
                                      (bias && bias[base + c] == -INFINITY));
      const unsigned m = __ballot_sync(0xffffffffu, times && !left_out);
      const int e = n + __popc(m & ((1u << lane) - 1));
      if ((m >> lane & 1) && e < kCap) {
        s.at[e] = static_cast<uint16_t>(c);
        s.less[e] = __fadd_rn(__fmul_rn(static_cast<float>(times), frequency), presence);
      }
      n += __popc(m);
    }
    __syncwarp();
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int k = (j * 32 + lane) * V, c = base + k;
    const uint32_t keep = allowed && c < classes ? allowed[c >> 5] >> (c & 31) : ~0u;
    float b[V];
    if (V > 1 && bias_wide && bias && c + V <= classes) {
#pragma unroll
      for (int i = 0; i < V / 4; ++i) {
        const float4 f = *reinterpret_cast<const float4*>(bias + c + 4 * i);
        b[4 * i] = f.x;
        b[4 * i + 1] = f.y;
        b[4 * i + 2] = f.z;
        b[4 * i + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) b[i] = bias && c + i < classes ? bias[c + i] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) s.add[k + i] = c + i < classes && (keep >> i & 1) ? b[i] : -INFINITY;
  }
  __syncwarp();
  for (int e = lane; e < min(n, kCap); e += 32) s.add[s.at[e]] = -INFINITY;
  __syncwarp();
  return n;
}

// Entry e of the span's rules in the row at z (its classes from `base`).
template <typename T>
__device__ __noinline__ float far_entry(const T* z, const float* less, const uint16_t* at, int e, float repeat, const float* bias,
                                        int base) {
  const int k = at[e];
  return __fadd_rn(penalised(load_logit(z + k), less[e], repeat), bias ? bias[base + k] : 0.0f);
}

// A warp's span of a row, and its line's rules on it.  Rows come through a place in shared memory:
// while one is worked on, in registers, the next is on its way there.
template <typename T, int V, int NV, int kMaxEntries>
struct WarpRow {
  static constexpr int kLane = NV * V, kSpan = 32 * kLane;  // classes of a lane, of the warp
  static constexpr int kCap = kSpan < kMaxEntries ? kSpan : kMaxEntries;
  using Rules = SpanRules<kSpan, kCap>;
  static constexpr int kRules = Rules::kBytes, kShared = kRules + kSpan * sizeof(T) + (V == 1 ? 32 : 0);
  int lane, base;  // the span's first class
  LineRule l;
  uint8_t* shared;  // SpanRules, then the rows
  int shift;  // V = 1: where in its place the row begins
  int n;  // entries
  // The first 64 entries, two a lane, in registers: place, less, bias
  int at[2];
  float less[2], plus[2];

  __device__ __forceinline__ void start(const LineParams& p, int base_, uint8_t* shared_) {
    lane = threadIdx.x % 32;
    base = base_;
    shared = shared_;
    l.first = l.end = 0;
    n = 0;
    shift = 0;
    // places past the last class stay 0 (their add is -inf)
    if (V > 1)
      for (int k = max(0, p.classes - base) + lane; k < kSpan; k += 32) place()[k] = T(0.0f);
    __syncwarp();
  }
  __device__ __forceinline__ const T* row(const LineParams& p, int r) const {
    return static_cast<const T*>(p.z) + r * p.pitch + base;
  }
  __device__ __forceinline__ T* place() const { return reinterpret_cast<T*>(shared + kRules) + (V == 1 ? shift : 0); }
  // Row r (where r < r1) on its way.
  __device__ __forceinline__ void fetch(const LineParams& p, int r, int r1) {
    if (r >= r1) return;
    const T* z = row(p, r);
    if constexpr (V == 1) {
      shift = copy_row(p, reinterpret_cast<T*>(shared + kRules), z, min(kSpan, p.classes - base), lane);
    } else {
      z += lane * V;
      T* s = place() + lane * V;
      const int left = p.classes - base - lane * V;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (j * 32 * V < left) copy_async(s + j * 32 * V, z + j * 32 * V, min(V, left - j * 32 * V) * static_cast<int>(sizeof(T)));
    }
  }
  __device__ __forceinline__ void arrived() const {
    copy_wait_all();
    __syncwarp();
  }
  // The rules of the line that the row lies in.
  __device__ __forceinline__ void rules(const LineParams& p) {
    n = set_rules<V, NV, kCap>(shared, p.classes, base, l.had, l.n_had, l.presence, l.frequency, l.bias, p.bias_wide, l.allowed);
    const Rules s(shared);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (lane + 32 * i >= n) continue;
      at[i] = s.at[lane + 32 * i];
      less[i] = s.less[lane + 32 * i];
      plus[i] = l.bias ? l.bias[base + at[i]] : 0.0f;
    }
  }
  // The dense pass.  Where a forbidden class holds NaN or +inf the sum with -inf is NaN; kCareful
  // chooses instead of adding.
  template <bool kCareful>
  __device__ __forceinline__ void ruled(const LineParams& p, float (&v)[kLane]) const {
    const float* t = reinterpret_cast<const float*>(shared) + lane * V;
    const T* z = place() + lane * V;
    const int left = p.classes - base - lane;  // V = 1: beyond are no logits
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float u[V], a[V];
      if constexpr (V == 1) u[0] = j * 32 < left ? load_logit(z + j * 32) : 0.0f;
      else get_logits<V>(z + j * 32 * V, u);
      if constexpr (V == 1) {
        a[0] = t[j * 32];
      } else {
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
          const float4 f = *reinterpret_cast<const float4*>(t + j * 32 * V + 4 * i);
          a[4 * i] = f.x;
          a[4 * i + 1] = f.y;
          a[4 * i + 2] = f.z;
          a[4 * i + 3] = f.w;
        }
      }
      if constexpr (V == 1 || kCareful) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float s = __fadd_rn(u[i], a[i]);
          v[j * V + i] = kCareful && a[i] == -INFINITY ? a[i] : s;
        }
      } else {
#pragma unroll
        for (int i = 0; i < V; i += 2) {
          const float2 s = fadd2_rn(make_float2(u[i], u[i + 1]), make_float2(a[i], a[i + 1]));
          v[j * V + i] = s.x;
          v[j * V + i + 1] = s.y;
        }
      }
    }
  }
  // The ruled logits of this lane's first entries (-inf: none).
  __device__ __forceinline__ void pair(float (&x)[2]) const {
    x[0] = x[1] = -INFINITY;
    if (n == 0) return;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (lane + 32 * i < n) x[i] = __fadd_rn(penalised(load_logit(place() + at[i]), less[i], l.repeat), plus[i]);
  }
  // f(ruled logit, class) for each of this lane's entries in the row at z, x the first.
  template <typename F>
  __device__ __forceinline__ void entries(const T* z, const float (&x)[2], F f) const {
    if (n == 0) return;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (lane + 32 * i < n) f(x[i], base + at[i]);
    if (n <= 64) return;
    const Rules s(shared);
#pragma unroll 1
    for (int e = lane + 64; e < n; e += 32) f(far_entry(z, s.less, s.at, e, l.repeat, l.bias, base), base + s.at[e]);
  }
};

// ---------------------------------------------------------------- the ruled logits

constexpr int kRulesThreads = 128;

// A warp takes `team_rows` rows of one span (of p.chunks); neighbouring warps the same rows' next span.
// 512 classes a span and 32 warps an SM: bytes in flight are what this kernel lives on.
template <typename T, typename O, int V, int NV>
__global__ void __launch_bounds__(kRulesThreads, 8) logit_rules_kernel(const __grid_constant__ LineParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x / 32;
  const long long unit = static_cast<long long>(blockIdx.x) * (kRulesThreads / 32) + warp;
  const long long r0 = unit / p.chunks * p.team_rows;
  const int r1 = static_cast<int>(min(static_cast<long long>(p.rows), r0 + p.team_rows));
  if (r0 >= r1) return;
  using Row = WarpRow<T, V, NV, 32 * V * NV>;  // every class may be an entry
  Row row;
  row.start(p, static_cast<int>(unit % p.chunks) * Row::kSpan, smem + static_cast<size_t>(warp) * Row::kShared);
  row.fetch(p, static_cast<int>(r0), r1);
  for (int r = static_cast<int>(r0); r < r1; ++r) {
    bool some = true;
    if (r < row.l.first || r >= row.l.end) {
      some = find_line(p, r, row.lane, row.l);
      if (some) row.rules(p);
      else row.l.first = row.l.end = 0;
    }
    float v[Row::kLane], x[2];
    row.arrived();
    row.template ruled<true>(p, v);
    row.pair(x);
    __syncwarp();
    const bool early = row.n <= 64;  // entries past the registers' are read from the row's place below
    if (early) row.fetch(p, r + 1, r1);
    if (some) {
      O* o = static_cast<O*>(p.out) + r * p.out_pitch;
      const int c = row.base + row.lane * V;
#pragma unroll
      for (int j = 0; j < NV; ++j) store_ruled<O, V>(o + c + j * 32 * V, v + j * V, p.classes - c - j * 32 * V);
      if (row.n) {  // the entries over what the dense pass wrote
        __syncwarp();
        row.entries(row.place(), x, [&](float y, int k) {
          if constexpr (sizeof(O) == 2) o[k] = __float2half_rn(y);
          else o[k] = y;
        });
        __syncwarp();
      }
    }
    if (!early) row.fetch(p, r + 1, r1);
  }
}

// ---------------------------------------------------------------- the decoders
//
// A team takes rows one after another, a warp a span of each: a warp alone (kTeam false), or a block of
// p.warps of them (a named barrier for each of several teams a block would cost every block all 16 of
// the hardware's, and with them occupancy).  First the maximum: each lane's, then 32 groups' of lanes,
// then the team's best.  Then, against that best, the sums of
// exp(z - best), joined in a fixed order.  Where the blank wins, the greedy decoder asks nothing more
// of a row.

// What a team's warps tell one another of a row, two rows' worth (a warp may be a row ahead).
struct TeamRow {
  float group[2][32];  // the highest of each group of lanes
  float sum[2][kMaxTeam];
  uint32_t arg[2][kMaxTeam];  // greedy: each warp's lowest class of the best
  float blank[2];
  int32_t listed[2];  // candidates: keys in the list
  unsigned long long list[2][kShortList];
  unsigned long long top[kMaxTeam];
};

// A span's classes but the blank in row z (its classes from `base`), from memory: what is seldom
// needed, by whole warps.  f(ruled logit, class); a forbidden class is -inf whatever it holds.
template <int kSpan, int kCap, typename T, typename F>
__device__ __forceinline__ void span_classes(const T* z, uint8_t* shared, int base, int classes, int n, float repeat,
                                             const float* bias, F f) {
  const int lane = threadIdx.x % 32;
  const SpanRules<kSpan, kCap> s(shared);
#pragma unroll 1
  for (int k = lane; k < kSpan && base + k < classes; k += 32) {
    const float a = s.add[k];
    if (base + k != 0 && a != -INFINITY) f(__fadd_rn(load_logit(z + k), a), base + k);
  }
#pragma unroll 1
  for (int e = lane; e < n; e += 32)
    if (base + s.at[e] != 0) f(far_entry(z, s.less, s.at, e, repeat, bias, base), base + s.at[e]);
}

// The lane's sum of exp(z - best) where the dense pass met a NaN.
template <int kSpan, int kCap, typename T>
__device__ __noinline__ float careful_sum(const T* z, uint8_t* shared, int base, int classes, int n, float repeat,
                                          const float* bias, float best) {
  const RowBase from(best);
  float sum = 0.0f;
  span_classes<kSpan, kCap>(z, shared, base, classes, n, repeat, bias, [&](float y, int) { sum += from.term(y); });
  return sum;
}

// The warp's highest key below `below` (0: none).
template <int kSpan, int kCap, typename T>
__device__ __noinline__ unsigned long long key_below(const T* z, uint8_t* shared, int base, int classes, int n,
                                                     float repeat, const float* bias, unsigned long long below) {
  unsigned long long k = 0;
  span_classes<kSpan, kCap>(z, shared, base, classes, n, repeat, bias, [&](float y, int c) {
    const unsigned long long u = y > -INFINITY ? class_key(y, c) : 0ull;
    if (u < below && u > k) k = u;
  });
  return warp_max_key(k);
}

// The k-th highest of 32 groups' maxima, one a lane: at most the k-th highest of all, so what reaches
// it is k keys and a few more, unless many classes tie.  Never -inf.
__device__ __forceinline__ float kth_group(float g, int k, int lane) {
#pragma unroll
  for (int m = 2; m <= 32; m *= 2)  // sorted over the lanes, highest first
#pragma unroll
    for (int o = m / 2; o > 0; o /= 2) {
      const float u = __shfl_xor_sync(0xffffffffu, g, o);
      g = ((lane & o) == 0) == ((lane & m) == 0) ? fmaxf(g, u) : fminf(g, u);
    }
  return fmaxf(__shfl_sync(0xffffffffu, g, k - 1), -3.402823466e38f);
}

__device__ __forceinline__ void list_key(TeamRow& t, int parity, float y, int c) {
  const int at = atomicAdd(&t.listed[parity], 1);
  if (at < kShortList) t.list[parity][at] = class_key(y, c);
}

// A row's candidates, by one warp: the listed keys ranked, the list emptied.  sum: the terms of all
// classes.
__device__ __forceinline__ void write_candidates(const LineParams& p, int r, int lane, TeamRow& t, int parity, float blank,
                                                 const RowBase& from, bool some, float sum) {
  const float ln = some ? logf(__fdiv_rn(sum, from.term(from.best))) : sum;
  const int all = t.listed[parity];
  const unsigned long long a = lane < all ? t.list[parity][lane] : 0ull, b = lane + 32 < all ? t.list[parity][lane + 32] : 0ull;
  int ra = 0, rb = 0;
#pragma unroll 1
  for (int i = 0; i < all; ++i) {
    const unsigned long long k = t.list[parity][i];
    ra += k > a;
    rb += k > b;
  }
  const size_t o = static_cast<size_t>(r) * p.topk;
  auto put = [&](unsigned long long k, int q) {
    p.ids[o + q] = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(k));
    p.probs[o + q] = __fsub_rn(__fsub_rn(order_float(static_cast<uint32_t>(k >> 32)), from.best), ln);
  };
  if (a && ra < p.topk) put(a, ra);
  if (b && rb < p.topk) put(b, rb);
  if (lane >= all && lane < p.topk) {
    p.ids[o + lane] = -1;
    p.probs[o + lane] = -INFINITY;
  }
  if (lane == 0) p.blank[r] = __fsub_rn(__fsub_rn(blank, from.best), ln);
  __syncwarp();
  if (lane == 0) t.listed[parity] = 0;
  __syncwarp();
}

// ---------------------------------------------------------------- rows that no team's registers hold
//
// More classes than a team's registers hold (kRegisterClasses), or a line whose history names more
// classes of a span than its list keeps: a team takes the row in spans of kSlowSpan, each read from
// memory as often as the row asks and its rules set anew.  Right, not fast.

constexpr int kSlowSpan = 256;  // a list holds them all

template <int kOp, typename T, bool kTeam>
__device__ __noinline__ void slow_row(const LineParams& p, int r, LineRule l, TeamRow& t, uint8_t* shared, int w, int warps) {
  const int lane = threadIdx.x % 32;
  const T* z = static_cast<const T*>(p.z) + r * p.pitch;
  auto sync = [&]() {
    if constexpr (kTeam) __syncthreads();
    else __syncwarp();
  };
  // f(ruled logit, class) for this warp's classes but the blank
  auto classes = [&](auto f) {
#pragma unroll 1
    for (int base = w * kSlowSpan; base < p.classes; base += warps * kSlowSpan) {
      const int n = set_rules<1, kSlowSpan / 32, kSlowSpan>(shared, p.classes, base, l.had, l.n_had, l.presence, l.frequency, l.bias,
                                                            false, l.allowed);
      span_classes<kSlowSpan, kSlowSpan>(z + base, shared, base, p.classes, n, l.repeat, l.bias, f);
      __syncwarp();
    }
  };
  sync();
  if (w == 0 && lane == 0) t.listed[0] = 0;
  float high = -INFINITY;
  classes([&](float y, int) { high = fmaxf(high, y); });
  const int groups = 32 / warps;
  for (int o = 16; o >= groups; o /= 2) high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
  if (lane < groups) t.group[0][w * groups + lane] = high;
  if (w == 0 && lane == 0) {  // the blank
    int times = 0;
    for (int k = 0; k < l.n_had; ++k) times += l.had[k] == 0;
    float y = load_logit(z);
    if (times) y = penalised(y, __fadd_rn(__fmul_rn(static_cast<float>(times), l.frequency), l.presence), l.repeat);
    if (l.bias) y = l.bias[0] == -INFINITY ? -INFINITY : __fadd_rn(y, l.bias[0]);
    t.blank[0] = l.allowed && !(l.allowed[0] & 1u) ? -INFINITY : y;
  }
  sync();
  const float blank = t.blank[0], others = warp_max(t.group[0][lane]), best = fmaxf(others, blank);
  const bool some = best > -INFINITY;
  const RowBase from(best);
  if (kOp == kOpGreedy && blank >= others) {
    if (w == 0 && lane == 0) {
      p.ids[r] = 0;
      p.probs[r] = 0.0f;
    }
    sync();
    return;
  }
  float sum = 0.0f;
  uint32_t arg = 0xffffffffu;
  const float reach = kOp == kOpCandidates && p.topk > 0 ? kth_group(t.group[0][lane], p.topk, lane) : INFINITY;
  classes([&](float y, int c) {
    sum += from.term(y);
    if constexpr (kOp == kOpGreedy) arg = y == best ? min(arg, static_cast<uint32_t>(c)) : arg;
    else if (y >= reach && p.topk > 0) list_key(t, 0, y, c);
  });
  sum = warp_sum(sum);
  arg = __reduce_min_sync(0xffffffffu, arg);
  if (lane == 0) {
    t.sum[0][w] = sum;
    t.arg[0][w] = arg;
  }
  sync();
  if (kOp == kOpCandidates && t.listed[0] > kShortList) {
    unsigned long long below = ~0ull;
#pragma unroll 1
    for (int q = 0; q < p.topk; ++q) {
      unsigned long long k = 0;
      classes([&](float y, int c) {
        const unsigned long long u = y > -INFINITY ? class_key(y, c) : 0ull;
        if (u < below && u > k) k = u;
      });
      k = warp_max_key(k);
      if (lane == 0) t.top[w] = k;
      sync();
      below = warp_max_key(lane < warps ? t.top[lane] : 0ull);
      sync();
      if (w == 0 && lane == 0) {
        t.list[0][q] = below;
        t.listed[0] = q + 1;
      }
    }
    sync();
  }
  if (w == 0) {
    sum = warp_sum(lane < warps ? t.sum[0][lane] : 0.0f) + from.term(blank);
    if constexpr (kOp == kOpGreedy) {
      arg = __reduce_min_sync(0xffffffffu, lane < warps ? t.arg[0][lane] : 0xffffffffu);
      if (lane == 0) {
        p.ids[r] = some ? static_cast<int32_t>(arg) : 0;  // nothing left but a NaN that the blank holds: blank
        p.probs[r] = __fdiv_rn(from.term(best), sum);
      }
    } else {
      write_candidates(p, r, lane, t, 0, blank, from, some, sum);
    }
  }
  sync();
}

constexpr int kAloneWarps = 2;  // of a block whose warps take rows alone
constexpr int kDecodeWarps = 16;  // an SM's, at 128 registers (20 at 96 spill: 79 us against 64 at 65,536 x 800)

template <int kOp, typename T, int V, int NV, bool kTeam>
__global__ void __launch_bounds__(32 * kMaxTeam, 1) line_rows_kernel(const __grid_constant__ LineParams p) {
  using Row = WarpRow<T, V, NV, kDecodeEntries>;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int w = kTeam ? warp : 0, warps = kTeam ? p.warps : 1;
  if (kOp == kOpGreedy) launch_next();
  constexpr bool kMayCrowd = Row::kSpan > Row::kCap;
  constexpr int kTeamRow = kTeam || kOp == kOpCandidates || kMayCrowd ? sizeof(TeamRow) : 0;
  static_assert(!kMayCrowd || Row::kRules >= SpanRules<kSlowSpan, kSlowSpan>::kBytes, "");
  const long long team = kTeam ? blockIdx.x : static_cast<long long>(blockIdx.x) * (blockDim.x / 32) + warp;
  TeamRow& t = *reinterpret_cast<TeamRow*>(smem + (kTeam ? 0 : warp * (kTeamRow + Row::kShared)));
  const long long r0 = team * p.team_rows;
  const int r1 = static_cast<int>(min(static_cast<long long>(p.rows), r0 + p.team_rows));
  if (r0 >= r1) return;
  auto team_sync = [&]() {
    if constexpr (kTeam) __syncthreads();
    else __syncwarp();
  };
  if (kOp == kOpCandidates && w == 0 && lane < 2) t.listed[lane] = 0;  // seen by the other warps after a row's first barrier
  Row row;
  row.start(p, w * Row::kSpan, reinterpret_cast<uint8_t*>(&t) + kTeamRow + w * Row::kShared);
  row.fetch(p, static_cast<int>(r0), r1);
  int parity = 0;
  bool crowded = false;  // the line's entries do not fit some warp's list
#pragma unroll 1
  for (int r = static_cast<int>(r0); r < r1; ++r) {
    bool found = true;
    if (r < row.l.first || r >= row.l.end) {
      found = find_line(p, r, lane, row.l);  // the same for every warp of the team
      if (found) row.rules(p);
      else row.l.first = row.l.end = 0;
      if constexpr (kMayCrowd) {
        crowded = found && row.n > Row::kCap;
        if constexpr (kTeam) crowded = __syncthreads_or(crowded);
        if (crowded) row.n = 0;
      }
    }
    if constexpr (kMayCrowd) {
      if (crowded) {
        row.arrived();
        row.fetch(p, r + 1, r1);
        slow_row<kOp, T, kTeam>(p, r, row.l, t, row.shared, w, warps);
        continue;
      }
    }
    float v[Row::kLane], x[2];
    row.arrived();
    row.template ruled<false>(p, v);
    row.pair(x);
    __syncwarp();
    row.fetch(p, r + 1, r1);
    if (!found) continue;

    // the maximum; the blank (class 0) is kept out of it and told apart
    float blank = -INFINITY;
    if (row.base == 0 && lane == 0) {
      blank = reinterpret_cast<const float*>(row.shared)[0] == -INFINITY ? -INFINITY : v[0];
      v[0] = -INFINITY;
    }
    float high;
    {
      float m[NV];
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        m[j] = v[j * V];
#pragma unroll
        for (int i = 1; i < V; ++i) m[j] = fmaxf(m[j], v[j * V + i]);
      }
#pragma unroll
      for (int s = 1; s < NV; s *= 2)
#pragma unroll
        for (int j = 0; j + s < NV; j += 2 * s) m[j] = fmaxf(m[j], m[j + s]);
      high = fmaxf(m[0], -INFINITY);
    }
    row.entries(row.row(p, r), x, [&](float y, int c) {
      if (c == 0) blank = y;
      else high = fmaxf(high, y);
    });
    float best;
    if constexpr (!kTeam) {
      best = warp_max(high);
      blank = warp_max_nan(blank);
    } else {
      const int groups = 32 / warps;  // of each warp
      float g = high;
      for (int o = 16; o >= groups; o /= 2) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
      if (lane < groups) t.group[parity][w * groups + lane] = g;
      if (w == 0) {
        blank = warp_max_nan(blank);
        if (lane == 0) t.blank[parity] = blank;
      }
      team_sync();
      best = warp_max(t.group[parity][lane]);
      blank = t.blank[parity];
    }
    if (kOp == kOpGreedy && blank >= best) {  // a tie is the lower class's
      if (w == 0 && lane == 0) {
        p.ids[r] = 0;
        p.probs[r] = 0.0f;
      }
      parity ^= 1;
      continue;
    }
    best = fmaxf(best, blank);
    const bool some = best > -INFINITY;
    const RowBase from(best);

    // the sum, and the lowest class of the best or what may be a candidate
    float2 s[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
    for (int i = 0; i < Row::kLane; i += 2) {
      const float2 d = fma2(make_float2(v[i], v[i + 1]), make_float2(kLog2e, kLog2e), make_float2(-from.c, -from.c));
      s[i / 2 % 2] = fadd2_rn(s[i / 2 % 2], make_float2(ex2_approx(d.x), ex2_approx(d.y)));
    }
    row.entries(row.row(p, r), x, [&](float y, int c) {
      if (c != 0) s[0].x += exp_less(y, from.c);
    });
    float sum = warp_sum((s[0].x + s[0].y) + (s[1].x + s[1].y));
    if (sum != sum || !from.fits)  // a NaN or +inf met a -inf (or one is allowed), or c overflowed
      sum = warp_sum(careful_sum<Row::kSpan, Row::kCap>(row.row(p, r), row.shared, row.base, p.classes, row.n, row.l.repeat, row.l.bias, best));
    uint32_t arg = 0xffffffffu;
    if constexpr (kOp == kOpGreedy) {
      if (high == best) {
        uint32_t c = 0xffffffffu;  // the place of the lane's lowest class of the best
#pragma unroll
        for (int j = NV - 1; j >= 0; --j)
#pragma unroll
          for (int i = V - 1; i >= 0; --i) c = v[j * V + i] == best ? j * 32 * V + i : c;
        if (c != 0xffffffffu) arg = row.base + lane * V + c;
        row.entries(row.row(p, r), x, [&](float y, int k) {
          if (y == best && k != 0) arg = min(arg, static_cast<uint32_t>(k));
        });
      }
      arg = __reduce_min_sync(0xffffffffu, arg);
      if constexpr (kTeam) {
        if (lane == 0) {
          t.sum[parity][w] = sum;
          t.arg[parity][w] = arg;
        }
        team_sync();
      }
      if (!kTeam || (r & (warps - 1)) == w) {  // joined by one warp, another each row
        if constexpr (kTeam) {
          sum = warp_sum(lane < warps ? t.sum[parity][lane] : 0.0f);
          arg = __reduce_min_sync(0xffffffffu, lane < warps ? t.arg[parity][lane] : 0xffffffffu);
        }
        if (lane == 0) {
          p.ids[r] = static_cast<int32_t>(arg);  // (0 where nothing is left: the blank's own place holds -inf)
          p.probs[r] = __fdiv_rn(from.term(best), sum + from.term(blank));
        }
      }
    } else {
      if (p.topk > 0) {
        const float reach = kth_group(!kTeam ? high : t.group[parity][lane], p.topk, lane);
        if (high >= reach) {
          uint32_t m = 0;
#pragma unroll
          for (int i = 0; i < Row::kLane; ++i) m |= static_cast<uint32_t>(v[i] >= reach) << i;
          while (m) {  // few: the logit read again rather than kept where an index can reach it
            const int i = __ffs(m) - 1, k = (i / V * 32 + lane) * V + i % V;
            m &= m - 1;
            list_key(t, parity, __fadd_rn(load_logit(row.row(p, r) + k), reinterpret_cast<const float*>(row.shared)[k]), row.base + k);
          }
          row.entries(row.row(p, r), x, [&](float y, int k) {
            if (y >= reach && k != 0) list_key(t, parity, y, k);
          });
        }
      }
      if (lane == 0) t.sum[parity][w] = sum;
      team_sync();
      if (t.listed[parity] > kShortList) {  // many alike: the highest key below the last one found, topk times
        unsigned long long below = ~0ull;
#pragma unroll 1
        for (int q = 0; q < p.topk; ++q) {
          unsigned long long k =
              key_below<Row::kSpan, Row::kCap>(row.row(p, r), row.shared, row.base, p.classes, row.n, row.l.repeat, row.l.bias, below);
          if constexpr (kTeam) {
            if (lane == 0) t.top[w] = k;
            team_sync();
            k = warp_max_key(lane < warps ? t.top[lane] : 0ull);
            team_sync();
          }
          below = k;
          if (w == 0 && lane == 0) {
            t.list[parity][q] = k;
            t.listed[parity] = q + 1;
          }
        }
        team_sync();
      }
      if (!kTeam || (r & (warps - 1)) == w) {
        sum = warp_sum(lane < warps ? t.sum[parity][lane] : 0.0f) + from.term(blank);
        write_candidates(p, r, lane, t, parity, blank, from, some, sum);
      }
    }
    parity ^= 1;
  }
}

// ---------------------------------------------------------------- long rows
//
// More than 2,048 classes and 16 frames a line (kLongClasses, kLongLines): a warp a row all the same, a block
// of 8 or 16 warps a line's rows.  The line's rules on all classes lie in shared memory once for the block; a row comes through
// its warp in chunks, three places deep, with the maximum and the sum of exp(z - base) kept as it goes
// (the base, one for the warp, rises with the maximum, and the sum is scaled by the bases' exact
// difference).  No barrier a row: teams of 16 warps that meet twice a row took 3 times as long
// (4,096 x 12,000 float16: 127 us).  Candidates are listed as they reach what the lanes' maxima so far
// promise of the k-th highest; a full list is cut to its k highest, and nothing below those comes in.

constexpr int kLongEntries = 256;  // of a line; one with more goes the slow way
constexpr int kLongList = 128;     // keys of a row
constexpr int kLongPlaces = 3;

template <typename T, int V>
struct LongRow {
  static constexpr int NV = V == 1 ? 16 : 4, kLane = NV * V, kChunk = 32 * kLane;
  static constexpr int kPlace = kChunk + (V == 1 ? 32 / static_cast<int>(sizeof(T)) : 0);  // logits a place holds
  static constexpr int kWarp = kLongPlaces * kPlace * static_cast<int>(sizeof(T)) + kLongList * 8;  // shared bytes of a warp
};

// A warp's listed keys but the k highest dropped, those put in order at the front; the k-th (0 where
// there are fewer).  All of them are at most kLongList.
__device__ __noinline__ unsigned long long keep_highest(unsigned long long* list, int listed, int k) {
  const int lane = threadIdx.x % 32;
  __syncwarp();
  unsigned long long key[kLongList / 32];
  int rank[kLongList / 32];
#pragma unroll
  for (int i = 0; i < kLongList / 32; ++i) {
    key[i] = 32 * i + lane < listed ? list[32 * i + lane] : 0ull;
    rank[i] = 0;
  }
#pragma unroll 4
  for (int u = 0; u < listed; ++u) {
    const unsigned long long other = list[u];
#pragma unroll
    for (int i = 0; i < kLongList / 32; ++i) rank[i] += other > key[i];
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < kLongList / 32; ++i)
    if (key[i] && rank[i] < k) list[rank[i]] = key[i];
  __syncwarp();
  return listed >= k ? list[k - 1] : 0ull;
}

template <int kOp, typename T, int V>
__global__ void __launch_bounds__(32 * kMaxTeam, 1) long_rows_kernel(const __grid_constant__ LineParams p) {
  using L = LongRow<T, V>;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int s_n;
  const int w = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (kOp == kOpGreedy) launch_next();
  const int chunks = (p.classes + L::kChunk - 1) / L::kChunk;
  TeamRow& t = *reinterpret_cast<TeamRow*>(smem);
  float* less = reinterpret_cast<float*>(smem + sizeof(TeamRow));  // the entries
  float* plus = less + kLongEntries;
  uint16_t* at = reinterpret_cast<uint16_t*>(plus + kLongEntries);
  float* add = reinterpret_cast<float*>(at + kLongEntries);  // [chunks * kChunk]
  uint8_t* mine = reinterpret_cast<uint8_t*>(add + chunks * L::kChunk) + w * L::kWarp;
  T* places = reinterpret_cast<T*>(mine);
  unsigned long long* list = reinterpret_cast<unsigned long long*>(mine + kLongPlaces * L::kPlace * sizeof(T));
  auto clear = [&]() {  // past the last class: 0 (its add is -inf)
    for (int k = lane; k < kLongPlaces * L::kPlace; k += 32) places[k] = T(0.0f);
    __syncwarp();
  };
  clear();
  const int b0 = static_cast<int>(min(static_cast<long long>(p.rows), static_cast<long long>(blockIdx.x) * p.team_rows));
  const int b1 = static_cast<int>(min(static_cast<long long>(p.rows), static_cast<long long>(b0) + p.team_rows));
  int r = b0;
  while (r < b1) {
    LineRule l;
    if (!find_line(p, r, lane, l)) {  // the same for every warp
      ++r;
      continue;
    }
    const int end = min(l.end, b1);
    // the fetches run ahead of the rows: (f_row, f_chunk) next
    int f_row = r + w, f_chunk = 0, f_place = 0;
    auto fetch = [&]() {
      if (f_row < end) {
        const int c = f_chunk * L::kChunk;
        const T* z = static_cast<const T*>(p.z) + f_row * p.pitch + c;
        T* s = places + f_place * L::kPlace;
        if constexpr (V == 1) {
          copy_row(p, s, z, min(L::kChunk, p.classes - c), lane);
        } else {
          const int left = p.classes - c - lane * V;
#pragma unroll
          for (int j = 0; j < L::NV; ++j)
            if (j * 32 * V < left)
              copy_async(s + (j * 32 + lane) * V, z + (j * 32 + lane) * V, min(V, left - j * 32 * V) * static_cast<int>(sizeof(T)));
        }
        if (++f_chunk == chunks) {
          f_chunk = 0;
          f_row += p.warps;
        }
      }
      f_place = f_place + 1 == kLongPlaces ? 0 : f_place + 1;
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int k = 0; k < kLongPlaces; ++k) fetch();
    // the line's rules
    __syncthreads();  // the rows before are done with the last line's
    uint32_t* count = reinterpret_cast<uint32_t*>(add);
    int n = 0;
    if (l.n_had > 0) {
      for (int c = threadIdx.x; c < p.classes; c += blockDim.x) count[c] = 0;
      __syncthreads();
      for (int k = threadIdx.x; k < l.n_had; k += blockDim.x) {
        const int c = l.had[k];
        if (c >= 0 && c < p.classes) atomicAdd(&count[c], 1u);
      }
      __syncthreads();
      if (w == 0) {
        for (int k0 = 0; k0 < l.n_had; k0 += 32) {
          const int c = k0 + lane < l.n_had ? l.had[k0 + lane] : -1;
          const unsigned same = __match_any_sync(0xffffffffu, c);
          const bool takes = c >= 0 && c < p.classes && (same & ((1u << lane) - 1)) == 0;
          const uint32_t times = takes ? count[c] : 0u;
          __syncwarp();
          if (takes) count[c] = 0;
          __syncwarp();
          const float b = times && l.bias ? l.bias[c] : 0.0f;
          const bool keeps = times && b != -INFINITY && (!l.allowed || (l.allowed[c >> 5] >> (c & 31) & 1));
          const unsigned m = __ballot_sync(0xffffffffu, keeps);
          const int e = n + __popc(m & ((1u << lane) - 1));
          if (keeps && e < kLongEntries) {
            at[e] = static_cast<uint16_t>(c);
            less[e] = __fadd_rn(__fmul_rn(static_cast<float>(times), l.frequency), l.presence);
            plus[e] = b;
          }
          n += __popc(m);
        }
        if (lane == 0) s_n = n;
      }
      __syncthreads();
      n = s_n;
    }
    for (int c = threadIdx.x; c < chunks * L::kChunk; c += blockDim.x)
      add[c] = c < p.classes && (!l.allowed || (l.allowed[c >> 5] >> (c & 31) & 1)) ? (l.bias ? l.bias[c] : 0.0f) : -INFINITY;
    __syncthreads();
    if (n <= kLongEntries) {
      for (int e = threadIdx.x; e < n; e += blockDim.x) add[at[e]] = -INFINITY;
    }
    __syncthreads();
    if (n > kLongEntries) {
      copy_wait_all();
      __syncthreads();
      for (; r < end; ++r) slow_row<kOp, T, true>(p, r, l, t, reinterpret_cast<uint8_t*>(add) + w * SpanRules<kSlowSpan, kSlowSpan>::kBytes, w, p.warps);
      clear();  // (slow rows work in the table and in what follows it)
      continue;
    }

    int place = 0;
#pragma unroll 1
    for (int row = r + w; row < end; row += p.warps) {
      const T* z = static_cast<const T*>(p.z) + row * p.pitch;
      // the entries first (at most 8 a lane); the blank apart
      float blank = -INFINITY, high = -INFINITY, x[kLongEntries / 32];
#pragma unroll
      for (int i = 0; i < kLongEntries / 32; ++i) {
        x[i] = -INFINITY;
        if (32 * i >= n) continue;
        const int e = 32 * i + lane;
        if (e >= n) continue;
        x[i] = __fadd_rn(penalised(load_logit(z + at[e]), less[e], l.repeat), plus[e]);
        if (at[e] == 0) {
          blank = x[i];
          x[i] = -INFINITY;
        }
        high = fmaxf(high, x[i]);
      }
      float best = warp_max(high), reach = INFINITY;
      uint32_t arg = 0xffffffffu;
      int listed = 0;
      float2 s[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
      float c = __fmul_rn(best == -INFINITY ? 0.0f : best, kLog2e);
      bool based = best > -INFINITY;  // c belongs to a logit
      unsigned long long least = 0;  // k keys are above it
      auto push = [&](bool takes, float y, int k) {  // by whole warps
        const unsigned long long key = class_key(y, k);
        unsigned m = __ballot_sync(0xffffffffu, takes && key > least);
        if (listed + __popc(m) > kLongList) {
          least = keep_highest(list, listed, p.topk);
          listed = min(listed, p.topk);
          m = __ballot_sync(0xffffffffu, takes && key > least);
        }
        if (m >> lane & 1) list[listed + __popc(m & ((1u << lane) - 1))] = key;
        listed += __popc(m);
      };
#pragma unroll
      for (int i = 0; i < kLongEntries / 32; ++i) {
        if (32 * i >= n) continue;
        s[0].x += exp_less(x[i], c);
        if constexpr (kOp == kOpGreedy) {
          if (x[i] == best && best > -INFINITY) arg = min(arg, static_cast<uint32_t>(at[32 * i + lane]));
        }
      }
      if constexpr (kOp == kOpGreedy) arg = __reduce_min_sync(0xffffffffu, arg);
#pragma unroll 1
      for (int chunk = 0; chunk < chunks; ++chunk) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kLongPlaces - 1) : "memory");
        __syncwarp();
        float v[L::kLane];
        const float* a = add + chunk * L::kChunk + lane * V;
        const int shift = V == 1 ? static_cast<int>(reinterpret_cast<uintptr_t>(z) % 16 / sizeof(T)) : 0;  // as copy_row leaves it
        const T* q = places + place * L::kPlace + shift + lane * V;
        const int left = p.classes - chunk * L::kChunk - lane;
#pragma unroll
        for (int j = 0; j < L::NV; ++j) {
          float u[V];
          if constexpr (V == 1) u[0] = j * 32 < left ? load_logit(q + j * 32) : 0.0f;
          else get_logits<V>(q + j * 32 * V, u);
          if constexpr (V == 1) {
            v[j] = __fadd_rn(u[0], a[j * 32]);
          } else {
#pragma unroll
            for (int i = 0; i < V; i += 4) {
              const float4 f = *reinterpret_cast<const float4*>(a + j * 32 * V + i);
              const float2 d0 = fadd2_rn(make_float2(u[i], u[i + 1]), make_float2(f.x, f.y));
              const float2 d1 = fadd2_rn(make_float2(u[i + 2], u[i + 3]), make_float2(f.z, f.w));
              v[j * V + i] = d0.x;
              v[j * V + i + 1] = d0.y;
              v[j * V + i + 2] = d1.x;
              v[j * V + i + 3] = d1.y;
            }
          }
        }
        if (chunk == 0 && lane == 0) {
          if (add[0] != -INFINITY) blank = v[0];
          v[0] = -INFINITY;
        }
        float m = v[0];
#pragma unroll
        for (int i = 1; i < L::kLane; ++i) m = fmaxf(m, v[i]);
        high = fmaxf(high, m);
        const float top = warp_max(m);
        if (top > best) {
          if constexpr (kOp == kOpGreedy) {
            uint32_t k = 0xffffffffu;
            if (m == top) {
#pragma unroll
              for (int j = L::NV - 1; j >= 0; --j)
#pragma unroll
                for (int i = V - 1; i >= 0; --i) k = v[j * V + i] == top ? chunk * L::kChunk + (j * 32 + lane) * V + i : k;
            }
            arg = __reduce_min_sync(0xffffffffu, k);
          }
          best = top;
          const float c2 = __fmul_rn(best, kLog2e);
          const float f = based ? ex2_approx(__fsub_rn(c, c2)) : 0.0f;
          s[0].x = based ? s[0].x * f : s[0].x;
          s[0].y = based ? s[0].y * f : s[0].y;
          s[1].x = based ? s[1].x * f : s[1].x;
          s[1].y = based ? s[1].y * f : s[1].y;
          c = c2;
          based = true;
        } else if (kOp == kOpGreedy && top == best && top > -INFINITY) {
          // an entry's class may lie behind an equal one of the dense pass
          uint32_t k = 0xffffffffu;
#pragma unroll
          for (int j = L::NV - 1; j >= 0; --j)
#pragma unroll
            for (int i = V - 1; i >= 0; --i) k = v[j * V + i] == top ? chunk * L::kChunk + (j * 32 + lane) * V + i : k;
          arg = min(arg, __reduce_min_sync(0xffffffffu, k));
        }
#pragma unroll
        for (int i = 0; i < L::kLane; i += 2) {
          const float2 d = fma2(make_float2(v[i], v[i + 1]), make_float2(kLog2e, kLog2e), make_float2(-c, -c));
          s[i / 2 % 2] = fadd2_rn(s[i / 2 % 2], make_float2(ex2_approx(d.x), ex2_approx(d.y)));
        }
        if (kOp == kOpCandidates && p.topk > 0) {
          if ((chunk & (chunk + 1)) == 0) reach = kth_group(high, p.topk, lane);  // chunks 0, 1, 3, 7, ...
          if (__any_sync(0xffffffffu, m >= reach)) {
            uint32_t bits = 0;
            if (m >= reach) {
#pragma unroll
              for (int i = 0; i < L::kLane; ++i) bits |= static_cast<uint32_t>(v[i] >= reach) << i;
            }
            while (__any_sync(0xffffffffu, bits != 0)) {  // a lane's lowest at a time, read again from its place
              const int i = max(__ffs(bits) - 1, 0), k = (i / V * 32 + lane) * V + i % V;
              push(bits != 0, __fadd_rn(load_logit(places + place * L::kPlace + shift + k), add[chunk * L::kChunk + k]), chunk * L::kChunk + k);
              bits &= bits - 1;
            }
          }
        }
        __syncwarp();
        place = place + 1 == kLongPlaces ? 0 : place + 1;
        fetch();
      }
      blank = warp_max_nan(blank);
      if (kOp == kOpGreedy && blank >= best) {
        if (lane == 0) {
          p.ids[row] = 0;
          p.probs[row] = 0.0f;
        }
        continue;
      }
      const float all = fmaxf(best, blank);
      const bool some = all > -INFINITY;
      const RowBase from(all);
      float sum = warp_sum((s[0].x + s[0].y) + (s[1].x + s[1].y));
      if (sum != sum || !from.fits || !(fabsf(c) < 1048576.0f)) {
        // a NaN or +inf met a -inf (or is allowed), or a base was too large: from memory, by differences
        sum = 0.0f;
#pragma unroll 1
        for (int k = lane; k < p.classes; k += 32)
          if (k != 0 && add[k] != -INFINITY) sum += from.term(__fadd_rn(load_logit(z + k), add[k]));
#pragma unroll
        for (int i = 0; i < kLongEntries / 32; ++i) sum += from.term(x[i]);
        sum = warp_sum(sum);
      } else if (best > -INFINITY) {
        sum *= ex2_approx(__fsub_rn(c, from.c));  // from the highest of the others to the row's base
      }
      sum += from.term(blank);
      if constexpr (kOp == kOpGreedy) {
        if (lane == 0) {
          p.ids[row] = some ? static_cast<int32_t>(arg) : 0;  // as slow_row
          p.probs[row] = __fdiv_rn(from.term(all), sum);
        }
      } else {
        const float ln = some ? logf(__fdiv_rn(sum, from.term(from.best))) : sum;
        const size_t o = static_cast<size_t>(row) * p.topk;
        if (p.topk > 0) {
          reach = kth_group(high, p.topk, lane);
#pragma unroll
          for (int i = 0; i < kLongEntries / 32; ++i)
            if (32 * i < n) push(x[i] >= reach, x[i], 32 * i + lane < n ? at[32 * i + lane] : 0);
          keep_highest(list, listed, p.topk);
          if (lane < p.topk) {
            const unsigned long long key = lane < listed ? list[lane] : 0ull;
            p.ids[o + lane] = key ? static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(key)) : -1;
            p.probs[o + lane] = key ? __fsub_rn(__fsub_rn(order_float(static_cast<uint32_t>(key >> 32)), from.best), ln) : -INFINITY;
          }
          __syncwarp();
        }
        if (lane == 0) p.blank[row] = __fsub_rn(__fsub_rn(blank, from.best), ln);
      }
    }
    copy_wait_all();
    r = end;
  }
}

constexpr int kRegisterClasses = kMaxTeam * 32 * kDecodeLane;

template <int kOp, typename T>
__global__ void __launch_bounds__(32 * kMaxTeam) wide_rows_kernel(const __grid_constant__ LineParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int w = threadIdx.x / 32;
  LineRule l;
  if (kOp == kOpGreedy) launch_next();
  if (!find_line(p, blockIdx.x, threadIdx.x % 32, l)) return;
  slow_row<kOp, T, true>(p, blockIdx.x, l, *reinterpret_cast<TeamRow*>(smem),
                         smem + sizeof(TeamRow) + w * SpanRules<kSlowSpan, kSlowSpan>::kBytes, w, kMaxTeam);
}

// Greedy CTC's second half, a warp a line, in place: ids and probs hold each frame's class and
// probability; the characters go to the front of the line's places (never past the frames already
// read), the rest is filled.  The frames of four steps are read at once: their latency, not their
// bytes, is what this kernel takes.  A NaN among a character's frames stays its maximum, whatever the
// order that the frames are joined in.
__global__ void __launch_bounds__(128) collapse_lines_kernel(const __grid_constant__ LineParams p) {
  const int i = blockIdx.x * 4 + threadIdx.x / 32, lane = threadIdx.x % 32;
  int first = 0, end = 0;
  if (i < p.lines) {
    first = min(max(p.line_at[i], 0), p.rows);
    end = min(max(p.line_at[i + 1], first), p.rows);
  }
  launch_wait();  // the frames' kernel is done
  if (i >= p.lines) return;
  constexpr int kSteps = 4;
  const uint32_t upto = 0xffffffffu >> (31 - lane);
  int prev = 0;        // the class of the frame before
  int k = 0;           // characters so far
  float carry = 0.0f;  // the last character's highest probability, where it may go on
  for (int t0 = first; t0 < end; t0 += 32 * kSteps) {
    int ids[kSteps];
    float prs[kSteps];
#pragma unroll
    for (int u = 0; u < kSteps; ++u) {
      const int t = t0 + 32 * u + lane;
      ids[u] = t < end ? p.ids[t] : 0;
      prs[u] = t < end ? p.probs[t] : 0.0f;
    }
    __syncwarp();
#pragma unroll
    for (int u = 0; u < kSteps; ++u) {
      if (t0 + 32 * u >= end) break;
      const int id = ids[u];
      float pr = prs[u];
      int before = __shfl_up_sync(0xffffffffu, id, 1);
      if (lane == 0) before = prev;
      const unsigned begins = __ballot_sync(0xffffffffu, id != 0 && id != before);
      const unsigned mine = begins & upto;
      if (__any_sync(0xffffffffu, id != 0 && id == before)) {
        // the highest probability up to this frame of the frames of its character
        for (int o = 1; o < 32; o <<= 1) {
          const float up = __shfl_up_sync(0xffffffffu, pr, o);
          const int uid = __shfl_up_sync(0xffffffffu, id, o);
          if (lane >= o && uid == id && (mine & ~(upto >> o)) == 0) pr = max_nan(up, pr);
        }
        if (id != 0 && id == before && mine == 0) pr = max_nan(carry, pr);
      }
      const int after = __shfl_down_sync(0xffffffffu, id, 1);
      const bool last = id != 0 && (lane == 31 || after != id);
      const int nth = k + __popc(mine) - 1;
      if (last) {
        p.ids[first + nth] = id;
        p.probs[first + nth] = pr;
      }
      if (begins >> lane & 1) p.starts[first + nth] = t0 + 32 * u + lane - first;
      k += __popc(begins);
      prev = __shfl_sync(0xffffffffu, id, 31);
      carry = __shfl_sync(0xffffffffu, pr, 31);
      __syncwarp();
    }
  }
  for (int t = first + k + lane; t < end; t += 32) {
    p.ids[t] = -1;
    p.starts[t] = -1;
    p.probs[t] = 0.0f;
  }
  if (lane == 0) p.counts[i] = k;
}

}  // namespace crec
