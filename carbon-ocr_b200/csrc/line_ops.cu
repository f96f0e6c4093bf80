// The C ABI's calls on the logits of packed lines (rules, greedy CTC, candidates) and the head
// with adapters: arguments checked, parameters filled, kernels queued.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <initializer_list>
#include <memory>
#include <new>
#include <string>
#include <utility>
#include <vector>

#include "../../include/carbon_rec.h"
#include "adapters.cuh"
#include "line_rules.cuh"

using namespace crec;

namespace {

struct Errors {
  char* text;
  size_t size;
  int operator()(int code, const char* msg) const {
    if (text && size) std::snprintf(text, size, "%s", msg);
    return code;
  }
  int cuda(cudaError_t e, const char* what) const {
    cudaGetLastError();  // told here: not the next call's
    char msg[256];
    std::snprintf(msg, sizeof msg, "%s: %s", what, cudaGetErrorString(e));
    return (*this)(e == cudaErrorMemoryAllocation ? CREC_E_NOMEM : CREC_E_CUDA, msg);
  }
};

// The current device for a call's duration: the one that holds `array`, the caller's after it.
class OnDeviceOf {
 public:
  cudaError_t enter(const void* array) {
    cudaPointerAttributes a{};
    cudaError_t e = cudaPointerGetAttributes(&a, array);
    if (e != cudaSuccess) {
      cudaGetLastError();
      return e;
    }
    if (a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged) return cudaErrorInvalidDevicePointer;
    return to(a.device);
  }
  cudaError_t to(int device) {
    int cur = 0;
    cudaError_t e = cudaGetDevice(&cur);
    if (e != cudaSuccess || cur == device) return e;
    if ((e = cudaSetDevice(device)) == cudaSuccess) back_ = cur;
    return e;
  }
  ~OnDeviceOf() {
    if (back_ >= 0) cudaSetDevice(back_);
  }

 private:
  int back_ = -1;
};

size_t type_bytes(int type) { return type == CREC_FP16 ? 2 : 4; }
bool is_logits_type(int type) { return type == CREC_FP32 || type == CREC_FP16; }
constexpr int64_t kMaxRows = 0x7fffff00;  // a tile past them still counts in 32 bits
constexpr int kMaxLines = 0x7fffff00;     // and a step of the lines' search

// Whether an array of `rows` rows has such a pitch (its bytes far within 64 bits).
bool fits_pitch(int64_t pitch, int64_t least, int64_t rows) {
  return pitch >= least && pitch <= (int64_t{1} << 40) && pitch <= (int64_t{1} << 60) / std::max<int64_t>(rows, 1);
}
// Whether every array is one of 4-byte values by its address (null ones too).
bool aligned4(std::initializer_list<const void*> arrays) {
  uintptr_t bits = 0;
  for (const void* a : arrays) bits |= reinterpret_cast<uintptr_t>(a);
  return bits % 4 == 0;
}

// What every call on packed lines checks; null where it passes.
const char* lines_fault(const crec_line_logits* z) {
  if (!z) return "no logits";
  if (!is_logits_type(z->type)) return "the logits' type";
  if (z->classes < 1 || z->classes > kMaxClasses) return "classes";
  if (z->rows < 0 || z->rows > kMaxRows || z->lines < 0 || z->lines > kMaxLines) return "rows or lines";
  if (!fits_pitch(z->pitch, z->classes, z->rows)) return "pitch";
  if (!aligned4({z->line_at})) return "line_at's alignment";
  if (z->lines > 0 && !z->line_at) return "no line_at";
  if (z->lines > 0 && z->rows > 0 && !z->logits) return "no logits";
  if (reinterpret_cast<uintptr_t>(z->logits) % type_bytes(z->type)) return "the logits' alignment";
  return nullptr;
}

const char* rules_fault(const crec_rules* r) {
  if (!r) return nullptr;
  if ((r->history != nullptr) != (r->history_at != nullptr)) return "history and history_at go together";
  if (!r->history && (r->repeat || r->presence || r->frequency)) return "penalties without a history";
  if (r->bias ? r->biases < 1 : r->bias_of != nullptr) return "bias tables";
  if (r->allowed ? r->sets < 1 : r->set_of != nullptr) return "allowed sets";
  if (!aligned4({r->history, r->history_at, r->repeat, r->presence, r->frequency, r->bias, r->bias_of, r->allowed, r->set_of}))
    return "the rules' alignment";
  return nullptr;
}

LineParams line_params(const crec_line_logits* z, const crec_rules* r) {
  LineParams p{};
  p.z = z->logits;
  p.z_end = static_cast<const uint8_t*>(z->logits) + (z->rows > 0 ? ((z->rows - 1) * z->pitch + z->classes) * type_bytes(z->type) : 0);
  p.pitch = z->pitch;
  p.classes = z->classes;
  p.rows = static_cast<int>(z->rows);
  p.lines = z->lines;
  p.line_at = z->line_at;
  p.words = static_cast<int>((static_cast<int64_t>(z->classes) + 31) / 32);
  if (r) {
    p.history = r->history;
    p.history_at = r->history_at;
    p.repeat = r->repeat;
    p.presence = r->presence;
    p.frequency = r->frequency;
    p.bias = r->bias;
    p.bias_of = r->bias_of;
    p.biases = r->biases;
    p.allowed = r->allowed;
    p.set_of = r->set_of;
    p.sets = r->sets;
  }
  return p;
}

// The number of SMs of the current device, asked once a device.
cudaError_t sm_count(int* out) {
  static std::atomic<int> known[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  int n = dev < 64 ? known[dev].load(std::memory_order_relaxed) : 0;
  if (n == 0) {
    e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return e;
    if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
  }
  *out = n;
  return cudaSuccess;
}

// A block's largest dynamic shared memory is an attribute of the kernel, on its device, for every thread
// of the program: each call sets the same value, the most that any of these launches may take (227 KB
// less 1 KB for static variables), so that none lowers it between another's setting and launch.
constexpr int kMostShared = 232448 - 1024;

template <typename K>
cudaError_t launch_on(K* k, const LineParams& p, long long blocks, int threads, size_t smem, cudaStream_t s) {
  if (smem > 48 << 10) {
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared);
    if (e != cudaSuccess) return e;
  }
  k<<<static_cast<unsigned>(blocks), threads, smem, s>>>(p);
  return cudaGetLastError();
}

// Blocks that an SM holds at once: 228 KB of shared memory, 1 KB of it each block's own, and as many
// warps as the kernel's registers leave.
int blocks_an_sm(size_t smem, int warps, int most_warps) {
  return std::max(1, std::min(static_cast<int>((228 << 10) / (smem + 1024)), most_warps / warps));
}

// The launches with NV vectors of V classes a lane, NV the fewest in a list that hold `classes` in a
// team's registers.
template <int kOp, typename T, int V, int NV, bool kTeam>
cudaError_t decode_rows(LineParams& p, int sms, cudaStream_t s) {
  using Row = WarpRow<T, V, NV, kDecodeEntries>;
  constexpr size_t kTeamRow = kTeam || kOp == kOpCandidates || Row::kSpan > Row::kCap ? sizeof(TeamRow) : 0;
  const int warps = kTeam ? p.warps : kAloneWarps, teams = kTeam ? 1 : warps;
  const size_t smem = teams * kTeamRow + static_cast<size_t>(warps) * Row::kShared;
  const long long resident = blocks_an_sm(smem, warps, kDecodeWarps) * static_cast<long long>(teams) * sms;
  p.team_rows = static_cast<int>(std::max(1ll, (p.rows + resident - 1) / resident));
  const long long per_block = static_cast<long long>(p.team_rows) * teams;
  return launch_on(line_rows_kernel<kOp, T, V, NV, kTeam>, p, (p.rows + per_block - 1) / per_block, warps * 32, smem, s);
}

template <int kOp, typename T, int V, int... NV>
cudaError_t decode_fit(LineParams& p, int need, int sms, cudaStream_t s, std::integer_sequence<int, NV...>) {
  cudaError_t e = cudaErrorInvalidValue;
  bool done = false;
  ((!done && need <= NV ? (done = true, e = p.warps > 1 ? decode_rows<kOp, T, V, NV, true>(p, sms, s) : decode_rows<kOp, T, V, NV, false>(p, sms, s), 0) : 0), ...);
  return e;
}

template <int kOp, typename T, int V>
cudaError_t decode(LineParams& p, cudaStream_t s) {
  int sms = 0;
  const cudaError_t e = sm_count(&sms);
  if (e != cudaSuccess) return e;
  // a team wide enough to hold a row; wider where the rows alone leave SMs without warps
  int w = 1;
  while (w < kMaxTeam && p.classes > w * 32 * kDecodeLane) w *= 2;
  while (w < 8 && static_cast<long long>(p.rows) * w < 8ll * sms && p.classes > 64 * w) w *= 2;
  p.warps = w;
  const int need = (p.classes + w * 32 * V - 1) / (w * 32 * V);
  if constexpr (V == 4) return decode_fit<kOp, T, V>(p, need, sms, s, std::integer_sequence<int, 1, 2, 3, 4, 5, 6, 7, 8>{});
  else if constexpr (V == 8) return decode_fit<kOp, T, V>(p, need, sms, s, std::integer_sequence<int, 1, 2, 3, 4>{});
  else return decode_fit<kOp, T, V>(p, need, sms, s, std::integer_sequence<int, 4, 16, 32>{});
}

// Long rows where lines are long too: a block sets a line's rules for 8 or 16 warps, so from 16 frames a
// line on average (candidates of 4,096 x 12,000 float16: 118 us against a team's 134 at 16 frames a line,
// 161 against 140 at 8), and from 2,048 classes (75 frames a line, as many logits: 1,504 classes 126 us
// against 124, 2,900 132 against 140, 12,000 85 against 128).
constexpr int kLongLines = 16, kLongClasses = 2048;

template <int kOp, typename T, int V>
cudaError_t decode_long(LineParams& p, cudaStream_t s) {
  using L = LongRow<T, V>;
  int sms = 0;
  const cudaError_t e = sm_count(&sms);
  if (e != cudaSuccess) return e;
  const int chunks = (p.classes + L::kChunk - 1) / L::kChunk;
  const size_t rules = sizeof(TeamRow) + kLongEntries * 10 + static_cast<size_t>(chunks) * L::kChunk * 4;
  // Two blocks of 8 warps an SM, one at work while the other sets rules, or one of 16, whose rules serve
  // twice the rows: the first up to 5,000 classes.  Candidates (k = 16, 75 frames a line, 98 MB), 8 against
  // 16 warps: float16 2,904 classes 100 us against 105, 4,096 89 against 94, 6,000 93 against 89, 12,000 107
  // against 89; float32 2,904 73 against 78, 4,096 73 against 80, 6,000 76 against 68, 12,000 95 against 78;
  // rows of any address (float16) 2,901 134 against 141, 6,001 123 against 123, 9,001 134 against 123.
  p.warps = p.classes <= 5000 ? kMaxTeam / 2 : kMaxTeam;
  const long long blocks = sms * (kMaxTeam / p.warps);
  p.team_rows = static_cast<int>((p.rows + blocks - 1) / blocks);
  return launch_on(long_rows_kernel<kOp, T, V>, p, (static_cast<long long>(p.rows) + p.team_rows - 1) / p.team_rows, 32 * p.warps, rules + p.warps * L::kWarp, s);
}

template <int kOp, typename T>
cudaError_t decode_wide(LineParams& p, cudaStream_t s) {
  return launch_on(wide_rows_kernel<kOp, T>, p, p.rows, 32 * kMaxTeam,
                   sizeof(TeamRow) + static_cast<size_t>(kMaxTeam) * SpanRules<kSlowSpan, kSlowSpan>::kBytes, s);
}

template <typename T, typename O, int V, int NV>
cudaError_t write_rows(LineParams& p, int sms, cudaStream_t s) {
  using Row = WarpRow<T, V, NV, 32 * V * NV>;
  constexpr int kWarps = kRulesThreads / 32;
  p.chunks = (p.classes + Row::kSpan - 1) / Row::kSpan;
  const size_t smem = static_cast<size_t>(kWarps) * Row::kShared;
  const long long resident = blocks_an_sm(smem, kWarps, 32) * static_cast<long long>(kWarps) * sms;
  p.team_rows = static_cast<int>(std::max(1ll, (static_cast<long long>(p.rows) * p.chunks + resident - 1) / resident));
  const long long units = (static_cast<long long>(p.rows) + p.team_rows - 1) / p.team_rows * p.chunks;
  return launch_on(logit_rules_kernel<T, O, V, NV>, p, (units + kWarps - 1) / kWarps, kRulesThreads, smem, s);
}

template <typename T, typename O, int V>
cudaError_t write_rules(LineParams& p, cudaStream_t s) {
  int sms = 0;
  const cudaError_t e = sm_count(&sms);
  if (e != cudaSuccess) return e;
  return write_rows<T, O, V, kRulesLane / V>(p, sms, s);
}

// Whether rows may be read or written `bytes` at a time.
bool wide(const void* a, int64_t pitch, size_t element, size_t bytes) {
  return reinterpret_cast<uintptr_t>(a) % bytes == 0 && pitch * element % bytes == 0;
}

void bias_reads(LineParams& p) { p.bias_wide = p.classes % 4 == 0 && reinterpret_cast<uintptr_t>(p.bias) % 16 == 0; }

template <int kOp>
cudaError_t launch_decode(LineParams& p, int type, cudaStream_t s) {
  bias_reads(p);
  if (p.classes > kRegisterClasses) return type == CREC_FP16 ? decode_wide<kOp, __half>(p, s) : decode_wide<kOp, float>(p, s);
  if (p.classes > kLongClasses && p.rows / p.lines >= kLongLines) {
    if (type == CREC_FP16) return wide(p.z, p.pitch, 2, 16) ? decode_long<kOp, __half, 8>(p, s) : decode_long<kOp, __half, 1>(p, s);
    return wide(p.z, p.pitch, 4, 16) ? decode_long<kOp, float, 4>(p, s) : decode_long<kOp, float, 1>(p, s);
  }
  if (type == CREC_FP16)
    return wide(p.z, p.pitch, 2, 16) ? decode<kOp, __half, 8>(p, s) : decode<kOp, __half, 1>(p, s);
  return wide(p.z, p.pitch, 4, 16) ? decode<kOp, float, 4>(p, s) : decode<kOp, float, 1>(p, s);
}

cudaError_t launch_rules(LineParams& p, int type, int out_type, cudaStream_t s) {
  bias_reads(p);
  const bool w = wide(p.z, p.pitch, type_bytes(type), 16);
  if (type == CREC_FP16) {
    if (out_type == CREC_FP16)
      return w && wide(p.out, p.out_pitch, 2, 16) ? write_rules<__half, __half, 8>(p, s) : write_rules<__half, __half, 1>(p, s);
    return w && wide(p.out, p.out_pitch, 4, 16) ? write_rules<__half, float, 8>(p, s) : write_rules<__half, float, 1>(p, s);
  }
  if (out_type == CREC_FP16)
    return w && wide(p.out, p.out_pitch, 2, 8) ? write_rules<float, __half, 4>(p, s) : write_rules<float, __half, 1>(p, s);
  return w && wide(p.out, p.out_pitch, 4, 16) ? write_rules<float, float, 4>(p, s) : write_rules<float, float, 1>(p, s);
}

// Whether the ruled logits may be written there: apart from the logits, exactly on them, or
// beside them in rows of the same byte pitch.
bool output_fits(const crec_line_logits* z, const void* out, int out_type, int64_t out_pitch) {
  if (z->rows == 0) return true;
  const auto a = reinterpret_cast<uintptr_t>(z->logits), b = reinterpret_cast<uintptr_t>(out);
  const uint64_t ea = type_bytes(z->type), eb = type_bytes(out_type);
  const uint64_t row_a = z->classes * ea, row_b = z->classes * eb, pa = z->pitch * ea, pb = out_pitch * eb;
  const uint64_t end_a = a + (z->rows - 1) * pa + row_a, end_b = b + (z->rows - 1) * pb + row_b;
  if (end_a <= b || end_b <= a) return true;
  if (a == b) return z->type == out_type && (z->pitch == out_pitch || z->rows == 1);
  if (pa != pb) return false;
  const uint64_t d = (b > a ? (b - a) % pa : (pa - (a - b) % pa) % pa);  // out's place within the logits' rows
  return d >= row_a && d + row_b <= pa;
}

}  // namespace

struct crec_adapters {
  int device = 0, sms = 0;
  int classes = 0, k = 0, adapters = 0, rank = 0, r16 = 0;
  __half* w = nullptr;   // [classes][k]
  float* bias = nullptr;  // [classes], then 256 zeros
  __half* a = nullptr;   // [adapters][r16][k]
  float* b = nullptr;    // [adapters][classes][rank]
  float* scale = nullptr;
  int32_t* own = nullptr;  // [adapters] ranks before they are padded
  std::atomic<bool> inject{false};  // the next launch's waits run out (crec_adapters_inject)
  int* err = nullptr;  // pinned, written by a launch whose bounded wait ran out
};

namespace {

// The last layer of a float model blob (CRECMDL1; carbon_rec/netdef.py to_blob): its weights
// [classes][k] as float16 bits and its bias; null where it is a head, else what is wrong.
const char* blob_head(const uint8_t* blob, size_t bytes, int* classes, int* k, std::vector<uint16_t>* w,
                      std::vector<float>* bias) {
  if (!blob || bytes < 40 || std::memcmp(blob, "CRECMDL1", 8) != 0) return "not a CRECMDL1 model blob";
  uint32_t head[8];
  std::memcpy(head, blob + 8, sizeof head);  // version, kind, values, layers, in, out, height, 0
  if (head[0] != 1) return "model blob version";
  if (head[1] != 1) return "a float recognizer's blob is wanted";
  const uint64_t nv = head[2], nl = head[3];
  if (nv > 4096 || nl > 4096 || nl == 0) return "model blob sizes";
  uint64_t at = 40 + nv * 24;
  for (uint64_t i = 0; i < nl; ++i) {
    if (at + 80 > bytes) return "model blob truncated";
    int32_t f[20];  // kind, in, out, residual, kh, kw, sh, sw, pt, pl, pb, pr, cin, cout, relu, ...
    std::memcpy(f, blob + at, sizeof f);
    at += 80;
    if (f[0] == 2) {  // a Resize has no weights
      if (i + 1 == nl) return "the last layer is no head";
      continue;
    }
    if (f[4] < 1 || f[5] < 1 || f[4] > 64 || f[5] > 64 || f[12] < 1 || f[13] < 1 || f[12] > 1 << 20 || f[13] > 1 << 20 || f[19])
      return "a layer of the model blob";
    const uint64_t cells = static_cast<uint64_t>(f[13]) * (f[0] == 1 ? 1 : f[12]) * f[4] * f[5];
    if (cells > bytes || at + 4 * cells + 4ull * f[13] > bytes) return "model blob truncated";
    if (i + 1 == nl) {
      if (f[0] != 0 || f[3] >= 0 || f[4] != 1 || f[5] != 1 || f[6] != 1 || f[7] != 1 || f[8] || f[9] || f[10] || f[11] || f[14])
        return "the last layer is no 1x1 head";
      *classes = f[13];
      *k = f[12];
      w->resize(cells);
      for (uint64_t j = 0; j < cells; ++j) {
        float v;
        std::memcpy(&v, blob + at + 4 * j, 4);
        const __half hv = __float2half_rn(v);
        std::memcpy(&(*w)[j], &hv, 2);
      }
      bias->resize(f[13]);
      std::memcpy(bias->data(), blob + at + 4 * cells, 4ull * f[13]);
    }
    at += 4 * cells + 4ull * f[13];
  }
  return at == bytes ? nullptr : "model blob has trailing bytes";
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encoder() {
  static std::atomic<EncodeTiled> known{nullptr};
  EncodeTiled f = known.load(std::memory_order_relaxed);
  if (f) return f;
  void* fn = nullptr;
  cudaDriverEntryPointQueryResult q{};
  if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) {
    cudaGetLastError();
    return nullptr;
  }
  f = reinterpret_cast<EncodeTiled>(fn);
  known.store(f, std::memory_order_relaxed);
  return f;
}

// [outer][rows][row] elements, rows `pitch` elements apart, in boxes of `box` x box_rows, the box's
// bytes a row the swizzle's width (32, 64 or 128).
bool encode(CUtensorMap* m, const void* base, bool half, uint64_t row, uint64_t rows, uint64_t outer, uint64_t pitch, uint32_t box,
            uint32_t box_rows) {
  const EncodeTiled f = encoder();
  const uint64_t e = half ? 2 : 4;
  const cuuint64_t dims[3] = {row, rows, outer}, strides[2] = {pitch * e, pitch * e * rows};
  const cuuint32_t boxes[3] = {box, box_rows, 1}, steps[3] = {1, 1, 1};
  const CUtensorMapSwizzle sw = box * e == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                                : box * e == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                                : CU_TENSOR_MAP_SWIZZLE_32B;
  return f && f(m, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<void*>(base), dims, strides,
                boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, sw, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// How a head's product is cut: frames a tile, classes a chunk, stages of the ring, a tile's parts.
void plan_adapters(const crec_adapters* h, AdapterParams* p) {
  constexpr int kSmem = 232448;
  p->nkb = (h->k + 63) / 64;
  p->last_steps = (h->k - (p->nkb - 1) * 64 + 15) / 16;
  p->rank = h->rank;
  p->r16 = h->r16;
  p->rank_row = std::min(h->rank, 32) * 4;
  p->h_bytes = h->rank <= 32 ? 128 * p->rank_row : 2 * 16384;
  int room = kSmem - 1024 - static_cast<int>(sizeof(AdapterShared)) - p->nkb * 16384 - 2 * static_cast<int>(p->h_bytes);
  const int unit = p->half ? 64 : 32;  // a box's classes
  p->boxes = p->width >= 16 && room - kBoxBytes >= 3 * 8192;
  if (p->boxes) room -= kBoxBytes;
  p->clipped = h->classes * (p->half ? 2ll : 4ll) % 16 == 0;
  // Of tiles of 128 frames or fewer, chunks of kAdapterChunk classes or fewer and a tile's chunks in one
  // part, two, or as many as fill the SMs once, twice or three times, the cheapest: rounds of SMs times
  // what a part takes, in 0.1 us as measured (K = 256, 160 classes a chunk): 4 us for its frames and h,
  // 0.4 us a block of 64 channels a chunk, 0.5 us an adapter a chunk, and not less than its logits take
  // at an SM's share of HBM.  Fewer frames a tile mean fewer adapters in it, whose MMAs come one after
  // another.
  double least = 0;
  for (int rows = 128; rows >= 16; rows /= 2) {
    const int tiles = (p->rows + rows - 1) / rows;
    const double lines = std::min<double>(rows, 1.0 + static_cast<double>(p->lines) * rows / p->rows);  // that a tile meets
    const double slots = p->adapter ? std::min<double>(lines, h->adapters) : 0.0;
    int last_n = 0;
    for (const int wide : {224, 160, 96, 64, 32}) {
      const int most = std::max(unit, wide / unit * unit), chunks = (h->classes + most - 1) / most;
      const int n = ((h->classes + chunks - 1) / chunks + unit - 1) / unit * unit;
      const int stage = std::max(n * 128, 8192), stages = std::min(kAdapterStages, room / stage);
      if (stages < 2 || (stages < 3 && n > unit) || n == last_n) continue;
      last_n = n;
      const double chunk = std::max(p->nkb * (2.0 + n / 80.0) + slots * (2.0 + n / 60.0) * ((p->rank + 15) / 16),
                                    static_cast<double>(rows) * n * (p->half ? 2 : 4) / 4300.0);
      int before = 0;
      for (const int fill : {1, 2, h->sms / tiles, 2 * h->sms / tiles, 3 * h->sms / tiles}) {
        const int s = std::min(fill, chunks);
        if (s <= before) continue;
        before = s;
        const int per = (chunks + s - 1) / s, parts = (chunks + per - 1) / per;
        const int rounds = (tiles * parts + h->sms - 1) / h->sms;  // (2 parts of 2^27 tiles at most)
        const double cost = rounds * (40.0 + slots * p->nkb * 0.5 + per * chunk);
        if (least != 0 && cost >= least) continue;
        least = cost;
        p->tile_rows = rows;
        p->chunks = chunks;
        p->n = n;
        p->stage_bytes = stage;
        p->stages = stages;
        p->splits = parts;
        p->chunks_per = per;
        p->items = tiles * parts;
      }
    }
  }
  p->a_stage_blocks = std::min(p->nkb, static_cast<int>(p->stage_bytes) / 8192);
}

void free_adapters(crec_adapters* h) {
  OnDeviceOf on;
  if (on.to(h->device) == cudaSuccess) {
    for (void* p : {static_cast<void*>(h->w), static_cast<void*>(h->bias), static_cast<void*>(h->a),
                    static_cast<void*>(h->b), static_cast<void*>(h->scale), static_cast<void*>(h->own)})
      cudaFree(p);
    cudaFreeHost(h->err);
  }
  delete h;
}

template <class T>
cudaError_t to_device(T** d, const void* host, size_t count) {
  cudaError_t e = cudaMalloc(reinterpret_cast<void**>(d), std::max<size_t>(count, 1) * sizeof(T));
  if (e == cudaSuccess && count) e = cudaMemcpy(*d, host, count * sizeof(T), cudaMemcpyHostToDevice);
  return e;
}

int open_adapters(int device, const void* model, size_t model_bytes, int n, const int32_t* ranks, const uint16_t* a,
                  const uint16_t* b, const float* scales, crec_adapters** out, const Errors& fail) {
  std::vector<uint16_t> w;
  std::vector<float> bias;
  int classes = 0, k = 0;
  if (const char* m = blob_head(static_cast<const uint8_t*>(model), model_bytes, &classes, &k, &w, &bias))
    return fail(CREC_E_MODEL, m);
  if (k % 8 || k > kMaxHeadK) return fail(CREC_E_MODEL, "adapters_open: a head of K channels, a multiple of 8, at most 512");
  int rank = 0;
  for (int i = 0; i < n; ++i) {
    if (ranks[i] < 1 || ranks[i] > kMaxRank) return fail(CREC_E_RANGE, "adapters_open: a rank of 1 to 64");
    rank = std::max(rank, static_cast<int>(ranks[i]));
  }
  rank = rank <= 8 ? 8 : rank <= 16 ? 16 : rank <= 32 ? 32 : 64;
  const int r16 = std::max(16, rank);
  // A [n][r16][k] and B [n][classes][rank], the rows past an adapter's own rank 0
  const size_t na = static_cast<size_t>(n) * r16 * k, nb = static_cast<size_t>(n) * classes * rank;
  std::vector<uint16_t> pa(na, 0);
  std::vector<float> pb(nb, 0.0f);
  for (int i = 0; i < n; ++i) {
    const size_t r = static_cast<size_t>(ranks[i]);
    std::memcpy(pa.data() + static_cast<size_t>(i) * r16 * k, a, r * k * 2);
    a += r * k;
    float* o = pb.data() + static_cast<size_t>(i) * classes * rank;
    for (int c = 0; c < classes; ++c, o += rank, b += r)
      for (size_t j = 0; j < r; ++j) {
        __half_raw v;
        v.x = b[j];
        o[j] = __half2float(__half(v));
      }
  }
  bias.resize(bias.size() + 256, 0.0f);  // (the last chunk's are read whole)
  OnDeviceOf on;
  cudaError_t e = on.to(device);
  if (e != cudaSuccess) {
    return fail.cuda(e, "adapters_open");
  }
  int major = 0;
  e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device);
  if (e == cudaSuccess && major != 10) return fail(CREC_E_INVALID, "adapters_open: this build runs on sm_100 (B200)");
  std::unique_ptr<crec_adapters, void (*)(crec_adapters*)> h(new crec_adapters(), free_adapters);
  h->device = device;
  h->classes = classes;
  h->k = k;
  h->adapters = n;
  h->rank = rank;
  h->r16 = r16;
  if (e == cudaSuccess) e = sm_count(&h->sms);
  if (e == cudaSuccess) e = to_device(&h->w, w.data(), w.size());
  if (e == cudaSuccess) e = to_device(&h->bias, bias.data(), bias.size());
  if (e == cudaSuccess) e = to_device(&h->a, pa.data(), na);
  if (e == cudaSuccess) e = to_device(&h->b, pb.data(), nb);
  if (e == cudaSuccess) e = to_device(&h->scale, scales, static_cast<size_t>(n));
  if (e == cudaSuccess) e = to_device(&h->own, ranks, static_cast<size_t>(n));
  if (e == cudaSuccess) e = cudaHostAlloc(reinterpret_cast<void**>(&h->err), sizeof(int), cudaHostAllocMapped);
  if (e == cudaSuccess) *h->err = 0;
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(adapter_head_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448);
  if (e != cudaSuccess) {
    return fail.cuda(e, "adapters_open");
  }
  *out = h.release();
  return CREC_OK;
}

}  // namespace

extern "C" {

int crec_logit_rules(const crec_line_logits* z, const crec_rules* rules, void* out, int out_type, int64_t out_pitch,
                     void* stream, char* error, size_t error_size) {
  const Errors fail{error, error_size};
  if (const char* m = lines_fault(z)) return fail(CREC_E_INVALID, m);
  if (const char* m = rules_fault(rules)) return fail(CREC_E_INVALID, m);
  if (!is_logits_type(out_type)) return fail(CREC_E_INVALID, "logit_rules: the output's type");
  if (!fits_pitch(out_pitch, z->classes, z->rows)) return fail(CREC_E_INVALID, "logit_rules: the output's pitch");
  if (z->lines == 0 || z->rows == 0) return CREC_OK;
  if (!out || reinterpret_cast<uintptr_t>(out) % type_bytes(out_type)) return fail(CREC_E_INVALID, "logit_rules: the output");
  if (!output_fits(z, out, out_type, out_pitch)) return fail(CREC_E_INVALID, "logit_rules: the output overlaps the logits");
  OnDeviceOf on;
  if (const cudaError_t e = on.enter(z->logits); e != cudaSuccess) return fail.cuda(e, "logit_rules: the logits");
  LineParams p = line_params(z, rules);
  p.out = out;
  p.out_pitch = out_pitch;
  const cudaError_t e = launch_rules(p, z->type, out_type, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? CREC_OK : fail.cuda(e, "logit_rules");
}

int crec_ctc_greedy_lines(const crec_line_logits* z, const crec_rules* rules, int32_t* counts, int32_t* ids,
                          int32_t* starts, float* probs, void* stream, char* error, size_t error_size) {
  const Errors fail{error, error_size};
  if (const char* m = lines_fault(z)) return fail(CREC_E_INVALID, m);
  if (const char* m = rules_fault(rules)) return fail(CREC_E_INVALID, m);
  if (z->lines == 0) return CREC_OK;
  if (!counts || (z->rows > 0 && (!ids || !starts || !probs))) return fail(CREC_E_INVALID, "ctc_greedy_lines: no output");
  if (!aligned4({counts, ids, starts, probs})) return fail(CREC_E_INVALID, "ctc_greedy_lines: the outputs' alignment");
  OnDeviceOf on;
  if (const cudaError_t e = on.enter(counts); e != cudaSuccess) return fail.cuda(e, "ctc_greedy_lines: counts");
  LineParams p = line_params(z, rules);
  p.counts = counts;
  p.ids = ids;
  p.starts = starts;
  p.probs = probs;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = p.rows > 0 ? launch_decode<kOpGreedy>(p, z->type, s) : cudaSuccess;
  if (e == cudaSuccess) {
    // queued to start while the frames' last blocks run
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>((p.lines + 3) / 4));
    config.blockDim = dim3(128);
    config.stream = s;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = p.rows > 0;
    config.attrs = &early;
    config.numAttrs = 1;
    e = cudaLaunchKernelEx(&config, collapse_lines_kernel, p);
  }
  return e == cudaSuccess ? CREC_OK : fail.cuda(e, "ctc_greedy_lines");
}

int crec_candidates_lines(const crec_line_logits* z, const crec_rules* rules, int topk, int32_t* ids, float* logp,
                          float* blank, void* stream, char* error, size_t error_size) {
  const Errors fail{error, error_size};
  if (const char* m = lines_fault(z)) return fail(CREC_E_INVALID, m);
  if (const char* m = rules_fault(rules)) return fail(CREC_E_INVALID, m);
  if (topk < 0 || topk > std::min(kMaxTop, z->classes - 1))
    return fail(CREC_E_RANGE, "candidates_lines: topk is 0 to min(16, classes - 1)");
  if (z->lines == 0 || z->rows == 0) return CREC_OK;
  if (!blank || (topk > 0 && (!ids || !logp))) return fail(CREC_E_INVALID, "candidates_lines: no output");
  if (!aligned4({ids, logp, blank})) return fail(CREC_E_INVALID, "candidates_lines: the outputs' alignment");
  OnDeviceOf on;
  if (const cudaError_t e = on.enter(z->logits); e != cudaSuccess) return fail.cuda(e, "candidates_lines: the logits");
  LineParams p = line_params(z, rules);
  p.ids = ids;
  p.probs = logp;
  p.blank = blank;
  p.topk = topk;
  const cudaError_t e = launch_decode<kOpCandidates>(p, z->type, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? CREC_OK : fail.cuda(e, "candidates_lines");
}

int crec_blob_head(const void* model, size_t model_bytes, int* k, int* classes, char* error, size_t error_size) {
  const Errors fail{error, error_size};
  if (!k || !classes) return fail(CREC_E_INVALID, "blob_head: arguments");
  try {
    std::vector<uint16_t> w;
    std::vector<float> bias;
    const char* m = blob_head(static_cast<const uint8_t*>(model), model_bytes, classes, k, &w, &bias);
    return m ? fail(CREC_E_MODEL, m) : CREC_OK;
  } catch (const std::bad_alloc&) {
    return fail(CREC_E_NOMEM, "blob_head: host memory");
  }
}

int crec_adapters_open(int device, const void* model, size_t model_bytes, int n, const int32_t* ranks, const void* a,
                       const void* b, const float* scales, crec_adapters** out, char* error, size_t error_size) {
  const Errors fail{error, error_size};
  if (!out) return fail(CREC_E_INVALID, "adapters_open: no handle to fill");
  *out = nullptr;
  if (device < 0 || n < 0 || n > 1 << 16 || (n > 0 && (!ranks || !a || !b || !scales)))
    return fail(CREC_E_INVALID, "adapters_open: arguments");
  try {
    return open_adapters(device, model, model_bytes, n, ranks, static_cast<const uint16_t*>(a),
                         static_cast<const uint16_t*>(b), scales, out, fail);
  } catch (const std::bad_alloc&) {
    return fail(CREC_E_NOMEM, "adapters_open: host memory");
  } catch (const std::exception& e) {
    return fail(CREC_E_INVALID, e.what());
  }
}

int crec_adapters_close(crec_adapters* h) {
  if (!h) return CREC_OK;
  OnDeviceOf on;
  cudaError_t e = on.to(h->device);
  if (e == cudaSuccess) e = cudaDeviceSynchronize();
  const int rc = e != cudaSuccess ? CREC_E_CUDA : *h->err ? CREC_E_TIMEOUT : CREC_OK;
  free_adapters(h);
  return rc;
}

int crec_adapters_inject(crec_adapters* h) {
  if (!h) return CREC_E_INVALID;
  h->inject = true;
  return CREC_OK;
}

int crec_adapters_logits(crec_adapters* h, const void* x, int64_t x_pitch, int64_t rows, int lines,
                         const int32_t* line_at, const int32_t* adapter, void* logits, int type, int64_t pitch,
                         void* stream, char* error, size_t error_size) {
  const Errors fail{error, error_size};
  if (!h) return fail(CREC_E_INVALID, "adapters_logits: no handle");
  if (!is_logits_type(type)) return fail(CREC_E_INVALID, "adapters_logits: the logits' type");
  if (rows < 0 || rows > kMaxRows || lines < 0 || lines > kMaxLines) return fail(CREC_E_INVALID, "adapters_logits: rows or lines");
  if (!fits_pitch(x_pitch, h->k, rows) || x_pitch % 8 || reinterpret_cast<uintptr_t>(x) % 16)
    return fail(CREC_E_INVALID, "adapters_logits: x 16-byte aligned, its pitch a multiple of 8 and at least K");
  if (!fits_pitch(pitch, h->classes, rows) || reinterpret_cast<uintptr_t>(logits) % type_bytes(type))
    return fail(CREC_E_INVALID, "adapters_logits: the logits' pitch or alignment");
  if (lines == 0 || rows == 0) return CREC_OK;
  if (!aligned4({line_at, adapter})) return fail(CREC_E_INVALID, "adapters_logits: line_at's or adapter's alignment");
  if (!x || !line_at || !logits) return fail(CREC_E_INVALID, "adapters_logits: no x, line_at or logits");
  OnDeviceOf on;
  if (const cudaError_t e = on.to(h->device); e != cudaSuccess) return fail.cuda(e, "adapters_logits");
  if (*static_cast<volatile int*>(h->err)) return fail(CREC_E_TIMEOUT, "adapters_logits: an earlier launch's wait ran out");
  AdapterParams p{};
  p.rows = static_cast<int>(rows);
  p.lines = lines;
  p.classes = h->classes;
  p.line_at = line_at;
  p.adapter = h->adapters ? adapter : nullptr;
  p.adapters = h->adapters;
  p.bias = h->bias;
  p.scale = h->scale;
  p.own = h->own;
  p.z = logits;
  p.pitch = pitch;
  p.half = type == CREC_FP16;
  const size_t element = type_bytes(type);
  p.width = wide(logits, pitch, element, 32) ? 32 : wide(logits, pitch, element, 16) ? 16 : static_cast<int>(element);
  p.err = h->err;
  p.idle = h->inject.exchange(false);
  p.wait_ns = p.idle ? 1000000ull : kWaitNs;
  plan_adapters(h, &p);
  bool maps = encode(&p.x, x, true, h->k, p.rows, 1, x_pitch, 64, p.tile_rows) && encode(&p.w, h->w, true, h->k, h->classes, 1, h->k, 64, p.n);
  if (maps && h->adapters)
    maps = encode(&p.a, h->a, true, h->k, h->r16, h->adapters, h->k, 64, h->r16) &&
           encode(&p.b, h->b, false, h->rank, h->classes, h->adapters, h->rank, std::min(h->rank, 32), p.n);
  if (maps && p.boxes) maps = encode(&p.zmap, logits, p.half, h->classes, p.rows, 1, pitch, p.half ? 64 : 32, 32);
  if (!maps) return fail(CREC_E_CUDA, "adapters_logits: cuTensorMapEncodeTiled failed");
  const size_t smem = 1024 + p.nkb * 16384 + 2 * p.h_bytes + (p.boxes ? kBoxBytes : 0) + p.stages * p.stage_bytes + sizeof(AdapterShared);
  adapter_head_kernel<<<std::min(p.items, h->sms), kAdapterThreads, smem, static_cast<cudaStream_t>(stream)>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? CREC_OK : fail.cuda(e, "adapters_logits");
}

}  // extern "C"
