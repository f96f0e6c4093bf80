// A head with low-rank adapters beside it (carbon_rec.h, crec_adapters_logits): frame f of line i,
//   z[f][c] = sum_k x[f][k] W[c][k] + b[c] + sum_j h[f][j] B_a[c][j]
//   h[f][j] = scale_a * sum_k x[f][k] A_a[j][k],  a = adapter[i]
//
// One tcgen05 kernel: a tile of 128 frames stays in shared memory while the weights stream past it,
// N classes a chunk, into float32 accumulators in TMEM.  The adapters join in the same accumulators.
// The frames of a tile may belong to many lines with many adapters; each distinct one (a slot) is a
// few more MMAs whose output rows are masked to the slot's own (disable-output-lane), so no frame is
// moved, and the cost goes with the distinct adapters of a tile, not its lines.  First h: the A rows
// of as many slots as 64 columns of TMEM hold as one B operand, each such group's product kept for its
// slots' frames only, so that all groups share the columns; a frame reads its own slot's.
// Four warps scale it and put it back as an A operand, as two tf32 words whose sum is within 2^-23 of it (h
// rounded to float16 once would cost the logits 2^-11 of the adapter's part, and its range; B's
// float16 values are tf32 values exactly).  Then each slot's B rows over each chunk's accumulators.
// The float32 logits are 4.1e-7 of their norm from 64 bits (K = 256, rank 16), float32 products on CUDA
// cores 2.5e-7: the tensor cores cut what an add shifts out where those round.
// Ranks are padded to the handle's with rows of zeros; h past an adapter's own rank is written as 0,
// since a frame's infinity times those zeros is NaN.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "sm100.cuh"

namespace crec {

constexpr int kMaxRank = 64;
constexpr int kMaxHeadK = 512;
constexpr int kAdapterChunk = 224;  // classes: two accumulators and 64 columns of h in 512 columns of TMEM
constexpr int kAdapterStages = 8;   // at most
constexpr int kAdapterThreads = 14 * 32;
constexpr int kBoxBytes = 8 * 4096;
constexpr int kBiasPlaces = 4;  // chunks whose biases are in shared memory

struct AdapterParams {
  CUtensorMap x;  // [rows][k] float16, boxes of 64 x tile_rows
  CUtensorMap w;  // [classes][k] float16, boxes of 64 x n
  CUtensorMap a;  // [adapters][r16][k] float16, boxes of 64 x r16
  CUtensorMap b;  // [adapters][classes][rank] float32, boxes of min(rank, 32) x n
  CUtensorMap zmap;  // the logits, boxes of 128 bytes x 32 rows (where `boxes`)
  int rows, lines, classes;
  const int32_t* line_at;
  const int32_t* adapter;  // null: the head alone
  int adapters;
  const float* bias;   // [classes], then 256 zeros
  const float* scale;  // [adapters]
  const int32_t* own;  // [adapters] ranks before they are padded
  void* z;
  long long pitch;
  int half;
  int width;  // bytes that a row of z may be written at once: 32, 16, or an element's
  int boxes;  // z's rows are 16-byte aligned and shared memory has room: whole boxes go out by TMA
  int clipped;  // a row's classes are whole 16-byte pieces (a TMA store ends at a piece, not at an element): so do clipped ones
  // tiles
  int tile_rows;                      // frames a tile takes of the 128 rows of an MMA
  int n, chunks, splits, chunks_per;  // classes a chunk (a multiple of 128 bytes of z's); a tile's chunks, in `splits` parts
  int items;                          // tiles * splits
  int nkb, last_steps;                // 64-channel blocks of x; MMA steps (16 channels) of the last
  int rank, r16, rank_row;            // padded to 8, 16, 32 or 64; at least 16; bytes of a row of b's boxes
  int a_stage_blocks;                 // blocks of a group's A rows that a stage takes
  int stages;
  uint32_t stage_bytes, h_bytes;  // h_bytes: of one of h's two words
  int* err;
  unsigned long long wait_ns;  // every wait's limit (kWaitNs; shorter only for a test's injected timeout)
  int idle;                    // that test: nothing is loaded
};

// What the roles of a block know of a tile's frames.
struct TileSlots {
  int n;
  int pad[3];
  uint4 rows[128];  // each slot's frames, a bit each
  uint4 group[128];  // and each group's
  int id[128];      // and its adapter
  int16_t slot[128];  // each frame's slot, -1 none, -2 not a line's frame
  int16_t own[128];   // and its adapter's own rank
  float scale[128];
};

struct AdapterShared {
  uint64_t full[kAdapterStages], empty[kAdapterStages];
  uint64_t a_full, a_empty, t_full[2], t_empty[2], h_full, h2_full, h2_empty, s_full[2], s_empty[2];
  uint64_t bias_full[kBiasPlaces], bias_empty[kBiasPlaces];
  uint64_t pad;
  float bias[kBiasPlaces][kAdapterChunk];
  uint32_t tmem;
  int failed;
  TileSlots tile[2];
  int which[128];
  int first_slot[128];
  int places[129];
  int counts[4];
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

// The tile's slots, by the 128 threads of the h warps (thread t frame r0 + t), barrier 1 theirs.
__device__ __forceinline__ void find_slots(const AdapterParams& p, AdapterShared& s, TileSlots& tile, int r0, int t) {
  const int lane = t % 32, q = t / 32, r = r0 + t;
  int id = -2;
  if (p.lines > 0) {
    const int first = p.line_at[0], end = p.line_at[p.lines];
    // the last line that begins at or before the tile, by warps of 32 probes
    int lo = 0, hi = p.lines;
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) / 32, at = lo + (lane + 1) * step;
      const unsigned le = __ballot_sync(0xffffffffu, at < hi && p.line_at[at] <= r0);
      lo += (__ffs(~le) - 1) * step;
      hi = min(hi, lo + step);
    }
    s.places[t] = lo + t <= p.lines ? p.line_at[lo + t] : 0x7fffffff;
    if (t == 0) s.places[128] = lo + 128 <= p.lines ? p.line_at[lo + 128] : 0x7fffffff;
    named_bar(1, 128);
    if (t < p.tile_rows && r >= first && r < end && r < p.rows) {
      int line;
      if (r < s.places[128]) {
        int a = 0, b = 128;
        while (b - a > 1) {
          const int mid = (a + b) / 2;
          if (s.places[mid] <= r) a = mid;
          else b = mid;
        }
        line = lo + a;
      } else {  // more than 128 lines begin in the tile (empty ones among them)
        line = line_of_row(p.line_at, p.lines, r);
      }
      line = min(max(line, 0), p.lines - 1);  // (a line_at that does not ascend)
      const int a = p.adapter ? p.adapter[line] : -1;
      id = a >= 0 && a < p.adapters ? a : -1;
    }
  }
  s.which[t] = id;
  tile.rows[t] = tile.group[t] = make_uint4(0, 0, 0, 0);
  named_bar(1, 128);
  int leader = t;
  if (id >= 0) {
    const int4* w4 = reinterpret_cast<const int4*>(s.which);
    for (int i = 0; i < 32; ++i) {
      const int4 u = w4[i];
      const int f = u.x == id ? 0 : u.y == id ? 1 : u.z == id ? 2 : u.w == id ? 3 : 4;
      if (f < 4) {
        leader = 4 * i + f;
        break;
      }
    }
  }
  __syncwarp();
  const bool leads = id >= 0 && leader == t;
  const unsigned m = __ballot_sync(0xffffffffu, leads);
  if (lane == 0) s.counts[q] = __popc(m);
  named_bar(1, 128);
  int before = 0, all = 0;
  for (int i = 0; i < 4; ++i) {
    before += i < q ? s.counts[i] : 0;
    all += s.counts[i];
  }
  if (leads) {
    const int k = before + __popc(m & ((1u << lane) - 1));
    s.first_slot[t] = k;
    tile.id[k] = id;
  }
  named_bar(1, 128);
  int slot = id;
  if (id >= 0) {
    slot = s.first_slot[leader];
    atomicOr(reinterpret_cast<uint32_t*>(&tile.rows[slot]) + q, 1u << lane);
    atomicOr(reinterpret_cast<uint32_t*>(&tile.group[slot / (64 / p.r16)]) + q, 1u << lane);
  }
  tile.slot[t] = static_cast<int16_t>(slot);
  tile.own[t] = static_cast<int16_t>(id >= 0 ? p.own[id] : 0);
  tile.scale[t] = id >= 0 ? p.scale[id] : 0.0f;
  if (t == 0) tile.n = all;
}

// v as two tf32 words (10 bits of the fraction, the MMA drops the rest), each rounded to them: hi + lo is
// within 2^-23 of v.  Rounding adds half a unit to the bits, so three kinds are told apart: finite
// values that it would carry to infinity are cut instead (lo takes what is cut off), an infinity is hi
// alone, and a NaN is one that keeps its kind without its low bits (the carry would make it 0).
__device__ __forceinline__ void split_tf32(float v, uint32_t& hi, uint32_t& lo) {
  constexpr uint32_t kKept = 0xffffe000u, kInf = 0x7f800000u, kCarries = 0x7f7ff000u;
  const uint32_t b = __float_as_uint(v), size = b & 0x7fffffffu;
  hi = size > kInf ? 0x7fffe000u : size >= kCarries ? b & kKept : (b + 0x1000u) & kKept;
  lo = size >= kInf ? 0u : (__float_as_uint(__fsub_rn(v, __uint_as_float(hi))) + 0x1000u) & kKept;
}

// 16 logits of one frame (c the first's class) from their accumulators.
__device__ __forceinline__ void store_logits(const AdapterParams& p, int r, int c, const uint32_t* acc, const float* bias) {
  float v[16];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 b = *reinterpret_cast<const float4*>(bias + 4 * i);
    v[4 * i] = __fadd_rn(__uint_as_float(acc[4 * i]), b.x);
    v[4 * i + 1] = __fadd_rn(__uint_as_float(acc[4 * i + 1]), b.y);
    v[4 * i + 2] = __fadd_rn(__uint_as_float(acc[4 * i + 2]), b.z);
    v[4 * i + 3] = __fadd_rn(__uint_as_float(acc[4 * i + 3]), b.w);
  }
  const long long o = r * p.pitch + c;
  const bool whole = c + 16 <= p.classes;
  if (p.half) {
    __half* z = static_cast<__half*>(p.z) + o;
    if (whole && p.width >= 16) {
      uint4 u[2];
      uint32_t* w = reinterpret_cast<uint32_t*>(u);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        memcpy(&w[i], &h, 4);
      }
      if (p.width == 32) {
        st_global_v8(z, u[0], u[1]);
      } else {
        reinterpret_cast<uint4*>(z)[0] = u[0];
        reinterpret_cast<uint4*>(z)[1] = u[1];
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (c + i < p.classes) z[i] = __float2half_rn(v[i]);
  } else {
    float* z = static_cast<float*>(p.z) + o;
    if (whole && p.width >= 16) {
      uint4 u[4];
      memcpy(u, v, sizeof u);
      if (p.width == 32) {
        st_global_v8(z, u[0], u[1]);
        st_global_v8(z + 8, u[2], u[3]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) reinterpret_cast<uint4*>(z)[i] = u[i];
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (c + i < p.classes) z[i] = v[i];
  }
}

// A warp's 32 frames x 128 bytes of logits (32 of float32, 64 of float16, c the first's class) from
// their accumulators through `box` (4 KB, in the 128-byte swizzle) out by TMA: each of its 32 rows a
// full line of 128 bytes, where a lane's own stores would touch 32 lines an instruction.
template <bool kHalf>
__device__ __forceinline__ void store_box(const AdapterParams& p, uint8_t* box, uint32_t taddr, int lane, int r, int c, const float* bias) {
  constexpr int kWords = kHalf ? 2 : 1;
  uint4 out[8];
#pragma unroll
  for (int h = 0; h < kWords; ++h) {
    uint32_t v[32];
    tmem_ld32(taddr + 32 * h, v);
    tmem_wait_ld();
    tmem_pin(v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 b = *reinterpret_cast<const float4*>(bias + 32 * h + 4 * i);
      const float x0 = __fadd_rn(__uint_as_float(v[4 * i]), b.x), x1 = __fadd_rn(__uint_as_float(v[4 * i + 1]), b.y);
      const float x2 = __fadd_rn(__uint_as_float(v[4 * i + 2]), b.z), x3 = __fadd_rn(__uint_as_float(v[4 * i + 3]), b.w);
      if constexpr (kHalf) {
        const __half2 lo = __floats2half2_rn(x0, x1), hi = __floats2half2_rn(x2, x3);
        uint32_t* w = reinterpret_cast<uint32_t*>(&out[4 * h + i / 2]) + 2 * (i & 1);
        memcpy(w, &lo, 4);
        memcpy(w + 1, &hi, 4);
      } else {
        out[i] = make_uint4(__float_as_uint(x0), __float_as_uint(x1), __float_as_uint(x2), __float_as_uint(x3));
      }
    }
  }
  if (lane == 0) bulk_wait_read();  // the box's last logits are on their way
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(box + lane * 128 + ((i ^ (lane & 7)) << 4)) = out[i];
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    tma_store_3d(&p.zmap, box, c, r, 0);
    bulk_commit();
  }
}

// Persistent, an SM a block: warps 0-7 write logits (a lane a frame, the two halves of a chunk), 8-11
// find the slots and put h back, 12 loads, 13 issues the MMAs.  An item is a tile's chunks
// [c0, c1); its stages, in order: per slot its A rows, then per chunk W's blocks and per slot its B rows.
__global__ void __launch_bounds__(kAdapterThreads, 1) adapter_head_kernel(const __grid_constant__ AdapterParams p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* xs = smem;                                  // [nkb][128][128 bytes]
  uint8_t* hs = xs + p.nkb * 16384;                    // h's high words, then its low words
  uint8_t* boxes = hs + 2 * p.h_bytes;                 // [8][4096], where used
  uint8_t* ring = boxes + (p.boxes ? kBoxBytes : 0);   // [stages][stage_bytes]
  AdapterShared& s = *reinterpret_cast<AdapterShared*>(ring + p.stages * p.stage_bytes);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kAdapterStages; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], 1);
    }
    mbar_init(&s.a_full, 1);
    mbar_init(&s.a_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.t_full[i], 1);
      mbar_init(&s.t_empty[i], 8);
      mbar_init(&s.s_full[i], 128);
      mbar_init(&s.s_empty[i], 10);  // the loader, the MMA issuer, the eight writers
    }
    for (int i = 0; i < kBiasPlaces; ++i) {
      mbar_init(&s.bias_full[i], 1);
      mbar_init(&s.bias_empty[i], 8);
    }
    mbar_init(&s.h_full, 1);
    mbar_init(&s.h2_full, 128);
    mbar_init(&s.h2_empty, 1);
    fence_mbar_init();
    s.failed = 0;
  }
  if (warp == 13) tmem_alloc(&s.tmem, 512);
  if (warp == 12 && lane == 0) {
    prefetch_tmap(&p.x);
    prefetch_tmap(&p.w);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem, h_col = tmem + 2 * kAdapterChunk;
  const int b_pieces = (p.rank + 31) / 32, per_group = 64 / p.r16;

  if (warp == 12) {
    // ---------------------------------------------------------------- loads
    const bool leader = elect_one();
    uint32_t g = 0, st = 0, phase = 1, q = 0;  // stages issued, the next one and its phase, chunks
    bool ok = p.idle == 0;
    auto stage = [&](uint32_t bytes) -> int {  // the next stage, empty, expecting `bytes`
      const int i = st;
      ok = mbar_wait_warp(&s.empty[i], phase, p.err, kErrTimeoutEmpty, p.wait_ns);
      if (!ok) return -1;
      ++g;
      if (++st == static_cast<uint32_t>(p.stages)) {
        st = 0;
        phase ^= 1;
      }
      if (leader) mbar_expect_tx(&s.full[i], bytes);
      __syncwarp();
      return i;
    };
    uint32_t it = 0;
    for (int item = blockIdx.x; item < p.items && ok; item += gridDim.x, ++it) {
      const int t = item / p.splits, c0 = item % p.splits * p.chunks_per, c1 = min(p.chunks, c0 + p.chunks_per);
      ok = mbar_wait_warp(&s.a_empty, (it & 1) ^ 1, p.err, kErrTimeoutEmpty, p.wait_ns);
      if (!ok) break;
      if (leader) {
        mbar_expect_tx(&s.a_full, p.nkb * p.tile_rows * 128);
        for (int kb = 0; kb < p.nkb; ++kb) tma_load_3d(xs + kb * 16384, &p.x, kb * 64, t * p.tile_rows, 0, &s.a_full);
      }
      __syncwarp();
      ok = mbar_wait_warp(&s.s_full[it & 1], (it >> 1) & 1, p.err, kErrTimeoutFull, p.wait_ns);
      const TileSlots& tile = s.tile[it & 1];
      const int slots = ok ? tile.n : 0;
      for (int k = 0; k < slots && ok; k += per_group)
        for (int kb0 = 0, kb1; kb0 < p.nkb; kb0 = kb1) {
          kb1 = min(p.nkb, kb0 + p.a_stage_blocks);
          const int group = min(per_group, slots - k);
          const int i = stage((kb1 - kb0) * group * p.r16 * 128);
          if (i < 0) break;
          if (leader)
            for (int kb = kb0; kb < kb1; ++kb)
              for (int j = 0; j < group; ++j)
                tma_load_3d(ring + i * p.stage_bytes + (kb - kb0) * 8192 + j * p.r16 * 128, &p.a, kb * 64, 0, tile.id[k + j], &s.full[i]);
          __syncwarp();
        }
      for (int c = c0; c < c1 && ok; ++c, ++q) {
        const int place = q % kBiasPlaces;
        ok = mbar_wait_warp(&s.bias_empty[place], ((q / kBiasPlaces) & 1) ^ 1, p.err, kErrTimeoutEmpty, p.wait_ns);
        if (!ok) break;
        if (leader) {
          mbar_expect_tx(&s.bias_full[place], p.n * 4);
          bulk_load(s.bias[place], p.bias + c * p.n, p.n * 4, &s.bias_full[place]);
        }
        __syncwarp();
        for (int kb = 0; kb < p.nkb; ++kb) {
          const int i = stage(p.n * 128);
          if (i < 0) break;
          if (leader) tma_load_3d(ring + i * p.stage_bytes, &p.w, kb * 64, c * p.n, 0, &s.full[i]);
          __syncwarp();
        }
        for (int k = 0; k < slots && ok; ++k)
          for (int b = 0; b < b_pieces; ++b) {
            const int i = stage(p.n * p.rank_row);
            if (i < 0) break;
            if (leader) tma_load_3d(ring + i * p.stage_bytes, &p.b, b * 32, c * p.n, tile.id[k], &s.full[i]);
            __syncwarp();
          }
      }
      if (lane == 0) mbar_arrive(&s.s_empty[it & 1]);
    }
    // the last tile's MMAs done (after a failure: what is on its way has arrived)
    if (ok && it > 0) ok = mbar_wait_warp(&s.a_empty, (it & 1) ^ 1, p.err, kErrTimeoutEmpty, p.wait_ns);
    if (!ok) {
      for (uint32_t k = q > kBiasPlaces ? q - kBiasPlaces : 0; k <= q; ++k)
        mbar_wait(&s.bias_full[k % kBiasPlaces], (k / kBiasPlaces) & 1, nullptr, 0, p.wait_ns);
      mbar_wait(&s.a_full, it & 1, nullptr, 0, p.wait_ns);
      for (uint32_t k = g > static_cast<uint32_t>(p.stages) ? g - p.stages : 0; k < g; ++k)
        mbar_wait(&s.full[k % p.stages], (k / p.stages) & 1, nullptr, 0, p.wait_ns);
    }
  } else if (warp == 13) {
    // ---------------------------------------------------------------- MMAs
    // The whole warp runs the loop, so that descriptors and counters are warp-uniform, and one lane
    // issues.  Descriptors differ from their operand's first only in the start address (address >> 4:
    // a step of 32 bytes adds 2); made anew for each MMA, inside the issuing lane's branch, they took
    // 250 cycles an MMA against the tensor cores' 80.
    const bool leader = elect_one();
    const uint32_t base = __shfl_sync(0xffffffffu, tmem, 0), hbase = base + 2 * kAdapterChunk;
    const uint32_t ring0 = smem_u32(ring), h0 = smem_u32(hs);
    const uint64_t x_desc = umma_desc_sw128(smem_u32(xs)), w_desc = umma_desc_sw128(ring0);
    const bool full_rows = p.rank_row == 128;
    const uint64_t b_desc = full_rows ? w_desc : umma_desc_narrow(ring0, p.rank_row);
    const uint64_t h_desc = full_rows ? umma_desc_sw128(h0) : umma_desc_narrow(h0, p.rank_row);
    const uint64_t stage_step = p.stage_bytes >> 4, low = p.h_bytes >> 4, a_block = 8192 >> 4;
    const uint32_t id_w = idesc_f16(p.n), id_b = idesc_tf32(p.n);
    uint32_t st = 0, phase = 0, q = 0;  // the next stage and its phase, accumulators taken
    bool ok = true;
    auto arrive = [&]() {  // the next stage's operands
      ok = mbar_wait_warp(&s.full[st], phase, p.err, kErrTimeoutFull, p.wait_ns);
      tc_fence_after();
      return ok;
    };
    auto release = [&]() {
      if (leader) umma_commit(&s.empty[st]);
      __syncwarp();
      if (++st == static_cast<uint32_t>(p.stages)) {
        st = 0;
        phase ^= 1;
      }
    };
    uint32_t it = 0, hits = 0;  // items; those with slots
    for (int item = blockIdx.x; item < p.items && ok; item += gridDim.x, ++it) {
      const int c0 = item % p.splits * p.chunks_per, c1 = min(p.chunks, c0 + p.chunks_per);
      ok = mbar_wait_warp(&s.s_full[it & 1], (it >> 1) & 1, p.err, kErrTimeoutFull, p.wait_ns) &&
           mbar_wait_warp(&s.a_full, it & 1, p.err, kErrTimeoutFull, p.wait_ns);
      if (!ok) break;
      tc_fence_after();
      const TileSlots& tile = s.tile[it & 1];
      const int slots = tile.n;
      for (int k = 0; k < slots && ok; k += per_group) {
        const uint4 on = tile.group[k / per_group], off = make_uint4(~on.x, ~on.y, ~on.z, ~on.w);
        const uint32_t id_a = idesc_f16(min(per_group, slots - k) * p.r16);
        for (int kb = 0; kb < p.nkb;) {
          if (!arrive()) break;
          uint64_t ad = x_desc + kb * 1024, bd = w_desc + st * stage_step;
          for (const int kb1 = min(p.nkb, kb + p.a_stage_blocks); kb < kb1; ++kb, ad += 1024, bd += a_block) {
            const int steps = kb == p.nkb - 1 ? p.last_steps : 4;
#pragma unroll
            for (int u = 0; u < 4; ++u)
              if (u < steps && leader) umma_rows<false>(hbase, ad + 2 * u, bd + 2 * u, id_a, off, kb | u);
          }
          release();
        }
      }
      if (!ok) break;
      if (slots && leader) umma_commit(&s.h_full);
      __syncwarp();
      for (int c = c0; c < c1 && ok; ++c, ++q) {
        const int acc = q & 1;
        ok = mbar_wait_warp(&s.t_empty[acc], ((q >> 1) & 1) ^ 1, p.err, kErrTimeoutTmemEmpty, p.wait_ns);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = base + acc * kAdapterChunk;
        for (int kb = 0; kb < p.nkb; ++kb) {
          if (!arrive()) break;
          const int steps = kb == p.nkb - 1 ? p.last_steps : 4;
          const uint64_t ad = x_desc + kb * 1024, bd = w_desc + st * stage_step;
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (u < steps && leader) umma<false>(d, ad + 2 * u, bd + 2 * u, id_w, kb | u);
          release();
        }
        if (!ok) break;
        if (slots && c == c0) {
          ok = mbar_wait_warp(&s.h2_full, hits & 1, p.err, kErrTimeoutFull, p.wait_ns);
          tc_fence_after();
        }
        for (int k = 0; k < slots && ok; ++k) {
          const uint4 on = tile.rows[k], off = make_uint4(~on.x, ~on.y, ~on.z, ~on.w);
          for (int b = 0; b < b_pieces; ++b) {
            if (!arrive()) break;
            const int steps = p.rank / 8 - 4 * b;
            const uint64_t hd = h_desc + b * 1024, bd = b_desc + st * stage_step;
#pragma unroll
            for (int u = 0; u < 4; ++u)
              if (u < steps && leader) {
                umma_rows<true>(d, hd + 2 * u, bd + 2 * u, id_b, off, 1);
                umma_rows<true>(d, hd + low + 2 * u, bd + 2 * u, id_b, off, 1);
              }
            release();
          }
        }
        if (ok && leader) umma_commit(&s.t_full[acc]);
        __syncwarp();
      }
      if (!ok) break;
      if (leader) {
        if (slots) umma_commit(&s.h2_empty);
        umma_commit(&s.a_empty);
      }
      hits += slots != 0;
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.s_empty[it & 1]);
    }
  } else if (warp >= 8) {
    // ---------------------------------------------------------------- slots and h
    const int t = threadIdx.x - 256, quarter = warp & 3;
    const uint32_t taddr = h_col + (static_cast<uint32_t>(quarter * 32) << 16);
    uint32_t built = 0, hits = 0, it = 0;
    bool ok = true;
    // the four warps' common decision: none is left waiting at a barrier of theirs
    auto agree = [&]() {
      if (!ok) s.failed = 1;
      named_bar(1, 128);
      ok = s.failed == 0;
      named_bar(1, 128);
      return ok;
    };
    auto build = [&](int item) {
      ok = mbar_wait_warp(&s.s_empty[built & 1], ((built >> 1) & 1) ^ 1, p.err, kErrTimeoutEmpty, p.wait_ns);
      if (!agree()) return;
      find_slots(p, s, s.tile[built & 1], item / p.splits * p.tile_rows, t);
      mbar_arrive(&s.s_full[built & 1]);
      ++built;
    };
    int item = blockIdx.x;
    if (item < p.items) build(item);
    for (; item < p.items && ok; item += gridDim.x, ++it) {
      named_bar(1, 128);  // the slots are whole
      const TileSlots& tile = s.tile[it & 1];
      const bool more = item + static_cast<int>(gridDim.x) < p.items;
      if (tile.n == 0) {
        if (more) build(item + gridDim.x);
        continue;
      }
      const float scale = tile.scale[t];
      const int own = tile.own[t];
      const int place = max(tile.slot[t], 0) % per_group * p.r16;  // this frame's columns of h
      ok = mbar_wait_warp(&s.h_full, hits & 1, p.err, kErrTimeoutFull, p.wait_ns) &&
           mbar_wait_warp(&s.h2_empty, (hits & 1) ^ 1, p.err, kErrTimeoutEmpty, p.wait_ns);
      if (!agree()) break;
      ++hits;
      tc_fence_after();
      for (int j0 = 0; j0 < p.rank; j0 += 16) {
        uint32_t r[16];
        for (int g = 0; g < 64; g += p.r16) {  // every slot's place, a lane keeping its own
          if (!__any_sync(0xffffffffu, place == g)) continue;
          uint32_t u[16];
          tmem_ld16(taddr + g + j0, u);
          tmem_wait_ld();
          tmem_pin(u);
#pragma unroll
          for (int i = 0; i < 16; ++i) r[i] = place == g ? u[i] : r[i];
        }
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          if (j0 + j >= p.rank) break;
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            split_tf32(j0 + j + i < own ? __fmul_rn(__uint_as_float(r[j + i]), scale) : 0.0f, hi[i], lo[i]);
          // 16 bytes of row t: in rows of rank_row bytes, swizzled as the MMA reads them
          const int k = j0 + j, block = k / 32, piece = (k % 32) / 4;
          const int swz = piece ^ ((t * p.rank_row >> 7) & (p.rank_row / 16 - 1));
          uint8_t* at = hs + block * 16384 + t * p.rank_row + swz * 16;
          *reinterpret_cast<uint4*>(at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          *reinterpret_cast<uint4*>(at + p.h_bytes) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
      }
      tc_fence_before();
      fence_proxy_async_smem();
      mbar_arrive(&s.h2_full);
      if (more) build(item + gridDim.x);
    }
  } else {
    // ---------------------------------------------------------------- logits
    const int quarter = warp & 3, half = warp >> 2, row = quarter * 32 + lane;
    const int groups = p.n / 16, g0 = half ? (groups + 1) / 2 : 0, g1 = half ? groups : (groups + 1) / 2;
    uint8_t* box = boxes + warp * 4096;
    uint32_t q = 0, it = 0;
    bool ok = true;
    for (int item = blockIdx.x; item < p.items && ok; item += gridDim.x, ++it) {
      const int t = item / p.splits, c0 = item % p.splits * p.chunks_per, c1 = min(p.chunks, c0 + p.chunks_per);
      ok = mbar_wait_warp(&s.s_full[it & 1], (it >> 1) & 1, p.err, kErrTimeoutFull, p.wait_ns);
      if (!ok) break;
      const bool mine = s.tile[it & 1].slot[row] != -2;
      const int r = t * p.tile_rows + row;
      // every frame of the warp a line's (past the last, the boxes are clipped)
      const bool whole = p.boxes && t * p.tile_rows + quarter * 32 < p.rows && __all_sync(0xffffffffu, mine || r >= p.rows);
      for (int c = c0; c < c1; ++c, ++q) {
        const int acc = q & 1;
        const int place = q % kBiasPlaces;
        ok = mbar_wait_warp(&s.t_full[acc], (q >> 1) & 1, p.err, kErrTimeoutTmemFull, p.wait_ns) &&
             mbar_wait_warp(&s.bias_full[place], (q / kBiasPlaces) & 1, p.err, kErrTimeoutFull, p.wait_ns);
        if (!ok) break;
        const float* bias = s.bias[place];
        tc_fence_after();
        const uint32_t taddr = tmem + acc * kAdapterChunk + (static_cast<uint32_t>(quarter * 32) << 16);
        if (whole) {  // boxes, the two halves in turn
          const int step = p.half ? 64 : 32;
          for (int k = half * step; k < p.n && c * p.n + k < p.classes; k += 2 * step) {
            if (!p.clipped && c * p.n + k + step > p.classes) {  // what follows a row's classes is not ours to write
              for (int g = k; g < k + step && c * p.n + g < p.classes; g += 16) {
                uint32_t v[16];
                tmem_ld16(taddr + g, v);
                tmem_wait_ld();
                tmem_pin(v);
                if (mine) store_logits(p, r, c * p.n + g, v, bias + g);
              }
            } else if (p.half) store_box<true>(p, box, taddr + k, lane, t * p.tile_rows + quarter * 32, c * p.n + k, bias + k);
            else store_box<false>(p, box, taddr + k, lane, t * p.tile_rows + quarter * 32, c * p.n + k, bias + k);
          }
        } else {
          for (int g = g0; g < g1; g += 2) {
            uint32_t v[32];
            const bool two = g + 1 < g1;
            if (two) tmem_ld32(taddr + g * 16, v);
            else tmem_ld16(taddr + g * 16, *reinterpret_cast<uint32_t(*)[16]>(v));
            tmem_wait_ld();
            tmem_pin(v);
            const int k = c * p.n + g * 16;
            if (mine && k < p.classes) store_logits(p, r, k, v, bias + g * 16);
            if (mine && two && k + 16 < p.classes) store_logits(p, r, k + 16, v + 16, bias + g * 16 + 16);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&s.t_empty[acc]);
          mbar_arrive(&s.bias_empty[place]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.s_empty[it & 1]);
    }
    if (lane == 0) bulk_wait();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 13) tmem_dealloc(tmem, 512);
}

}  // namespace crec
