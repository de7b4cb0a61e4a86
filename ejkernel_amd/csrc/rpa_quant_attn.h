// Attention over the 8-bit paged cache with a scale per block of tokens and head: the kernel.
//
//   out[row] = sum_k p_k v_k vs_k / (sum_k p_k + sum_j e^(sink_j)),  p_k = exp(cap(scale q . k_k ks_k))
//
// Codes are widened to bf16, which holds all of them exactly, and multiplied on the matrix units; the scale of a key
// enters its logit and the scale of a value its probability, in fp32.  With bf16 queries p vs is two bf16 parts in
// decode rows and rounded to bf16 once in tiles of rows;
// with fp32 queries the operands that have 24 bits -- q and p vs -- are split into three bf16 parts each (8 + 8 + 8 bits),
// three products in place of one, and nothing is rounded below fp32.
//
// One launch of 2 workgroups per compute unit.  The batch is two streams of keys.  A sequence with at most 16 query rows
// per kv head (a decode step) is one item per kv head of the first stream: its rows fill one 16-wide matrix tile, and the
// four wavefronts of a workgroup take every fourth tile of 32 keys and meet in LDS at its end.  Other sequences are cut into
// tiles of rows, an item each of the second stream: each wavefront has rows of its own (quant_row_tiles times 16) and walks
// all of the item's keys.  In both a wavefront loads K and V straight into the registers that the matrix unit takes them
// from, so nothing waits for another wavefront on the way (with the tiles' codes widened through LDS, the workgroup in
// step, 16 chunks of 512 tokens after 4096 took 410 us, without it 315 us as it then stood).
//
// Each stream is cut into equal runs of keys, one per workgroup, wherever the cut falls: few long sequences, one long chunk
// and a ragged batch all fill the device.  Parts of an item that is cut meet through the workspace: those of the first
// stream are added up by the workgroup that hands in the last one, in stream order, those of the second in a binary tree.
// Either way the result does not depend on who comes last.  Half of the workgroups take their run of the second stream
// first, so that one workgroup of a compute unit waits for memory while the other multiplies.
//
// What bounds it, on a device that copies at 4.9 TB/s, reads at 6.2 TB/s and multiplies bf16 matrices at 1325 TFLOP/s:
//   - decode, 256 sequences of up to 8192 keys, 32/8 heads of 128: the reads, 2.3 GB in 413 us = 5.6 TB/s;
//   - decode behind a window of 4096 (64 x 4 tokens, 16/8 heads of 256): the reads, 172 us = 4.9 TB/s;
//   - chunks: instruction issue.  A 32-key step of a 48-row wavefront at head_dim 128 is 48 matrix instructions of 16
//     cycles and about 300 vector instructions -- 80 to widen the codes (e4m3; 210 for int8), 60 for each 16 rows' softmax,
//     eight of them exponentials of four times the cost -- so that vector instructions issue in 61 % of all cycles, the matrix
//     units are busy in 37 % and both wait for loads or each other in the rest: 820 TFLOP/s (e4m3) and 720 (int8) for 16
//     chunks of 512 tokens, 830 for 2 x 8192 tokens;
//   - fp32 queries: the same with three products for one and the splitting of probabilities on top: 125 TFLOP/s of plain
//     products for a mixed batch at head_dim 96, which runs as 128;
//   - few short sequences: the chain of dependent loads in front of the first product (lengths, their sums, page, codes),
//     12 us for 8 sequences of up to 512 keys.
#pragma once

#include "rpa_quant.h"
#include "rpa_tile_common.h"

namespace rpa {

struct QuantArgs {
  RpaQuantParams p;
  int page_shift, block_shift;
  int group;        // query heads per kv head
  int tile_group;   // rows of one token in a tile of the second stream: min(group, rows of a tile)
  int tile_tokens;  // tokens of a tile
  int tile_pad;     // what a tile costs beyond its keys, in keys
  int subs;         // tiles side by side for the heads of one token, where they are more than a tile's rows
  int grid;         // workgroups, a multiple of 16
  // zero between launches: one for each workgroup's cut item of the first stream, then [level of the tree][workgroup][wavefront]
  // of the second
  uint32_t* tickets;
  float* thin_o;            // [2 * grid][16 * D] states of cut items of the first stream, as they lie in registers
  float* thin_ml;           // [2 * grid][16][2]
  float* tile_o;            // [2 * grid][rows * D], the same of the second
  float* tile_ml;           // [2 * grid][rows][2]
};

// The second stream's tiles for a (padded) head_dim: 16-row tiles per wavefront, and keys per step.  The more of them, the more
// rows share the widening of a key: as many as there are registers for at two workgroups per compute unit, for which some of the
// queries lie in LDS.  16 chunks of 1024 tokens at head_dim 256: 1088 us with one, 711 with two; 16 of 512 at 64: 356 us with
// three, 342 with four; in fp32 at 128: 670 us with one, 567 with two; at 128 four spill (332 us, three 257).
template <int D, int kParts>
constexpr int quant_row_tiles() { return kParts == 3 ? (D == 256 ? 1 : 2) : D == 256 ? 2 : D == 128 ? 3 : 4; }
// The queries that stay in registers: of a row's pieces of 32 elements the first so many, and of their bf16 parts.  The others
// are read from LDS for every step.  At head_dim 128 all in registers spill outside of the loops (decode of 256 sequences 424 us, 16
// chunks of 512 tokens 258 us), half of the pieces do not (411 and 257 us), none cost the loop more reads (411 and 266 us).
template <int D, int kParts>
constexpr int quant_reg_pieces() { return D == 128 && kParts == 1 ? 2 : D / 32; }
template <int D, int kParts>
constexpr int quant_reg_parts() { return D == 256 && kParts == 1 ? 0 : D == 128 && kParts == 3 ? 1 : kParts; }
// Whether the second stream is a function of its own: it then has the whole register file at the price of a few us at its
// start.  At head_dim 256 its spills would cost the first stream more (64 x 4 tokens behind a window: 195 us against 175).
template <int D, int kParts>
constexpr bool quant_apart() { return D == 256 && kParts == 1; }
constexpr int kTileStep = 32;

constexpr uint64_t kQuantTicketBytes = 1u << 18;  // of the workspace's head
constexpr int kThinStep = 128;     // keys a workgroup takes at once in the first stream
// What an item costs beyond its keys, in keys: its queries, its rows' way out, a join.  First stream: 256 sequences of up to 512
// keys take 49 us at 128, 45 at 256, 44 at 384.  Second, three row tiles: 16 chunks of 512 tokens 295 us at 64, 278 at 128,
// 266 at 192, 264 at 256, so 224 for three and four; with one a step takes less time but so does the rest (16 chunks of 1024 tokens at
// head_dim 256: 1152 us at 64, 1112 at 128, 1128 at 256): 112, and 160 for two (QuantArgs::tile_pad).
constexpr int kThinPad = 384;
constexpr int kThinLeast = 256;    // least run of keys per workgroup
constexpr int kThinUneven = 1024;  // what cuts at any place cost over cuts into equal parts, in keys of a run
constexpr int kThinMeet = 384;     // what a cut costs at all
constexpr int kTileLeast = 256;
constexpr float kNoKey = -3.0e38f; // row maximum before any key
constexpr float kLazy = 2048.f;    // the running maximum follows when eight probabilities under it are more than that
constexpr int kAgentScope = 16;    // auxiliary bit of a buffer access: coherent across the device's L2s

namespace quant {

// The launch's arguments where the hardware keeps them: constant memory, read through the scalar cache.
typedef const __attribute__((address_space(4))) QuantArgs Args;

struct Seq {
  int q0, q_len, kv_len;
};

__device__ __forceinline__ int64_t ramp(int n, int c, int d) {  // sum over i < n of max(0, c + i d)
  const int i0 = c >= 0 ? 0 : static_cast<int>(static_cast<uint32_t>(d - 1 - c) / static_cast<uint32_t>(d));
  const int m = max(n - i0, 0);
  return static_cast<int64_t>(m) * (c + static_cast<int64_t>(i0) * d) + d * (static_cast<int64_t>(m) * (m - 1) >> 1);
}

// Keys of the rows of tokens [t0, t1) of a sequence: [first, end).
struct Range {
  int first, end;
};
__device__ __forceinline__ Range key_range(Args& a, const Seq& q, int t0, int t1) {
  const int base = q.kv_len - q.q_len;
  Range r;
  r.end = max(base + t1, 0);
  const int64_t f = static_cast<int64_t>(base) + t0 - a.p.sliding_window + 1;
  r.first = a.p.sliding_window > 0 && f > 0 ? static_cast<int>(f) : 0;
  return r;
}

// The second stream: tiles of one (sequence, head).
__device__ __forceinline__ int tiles_of(Args& a, const Seq& q) { return (q.q_len + a.tile_tokens - 1) / a.tile_tokens; }
// Stream positions in front of tile n (n below the number of tiles), or of all tiles.
__device__ __forceinline__ int64_t tiles_before(Args& a, const Seq& q, int n, bool all) {
  const int base = q.kv_len - q.q_len, d = a.tile_tokens;
  int64_t sum = ramp(n, base + d, d) + static_cast<int64_t>(n) * a.tile_pad;
  if (a.p.sliding_window > 0) sum -= ramp(n, max(base - a.p.sliding_window + 1, -0x40000000), d);  // (a window beyond every key)
  if (all) sum -= max(base + n * d, 0) - max(base + q.q_len, 0);
  return sum;
}

__device__ __forceinline__ bool is_thin(Args& a, const Seq& q) { return static_cast<int64_t>(q.q_len) * a.group <= 16; }

__device__ __forceinline__ int thin_keys(Args& a, const Seq& q) {
  const Range r = key_range(a, q, 0, q.q_len);
  return r.end - r.first;
}

// Lengths of sequence s, clipped to what the buffers hold; empty from sequence n on.  The loads do not wait for n.
__device__ __forceinline__ Seq load_seq(Args& a, int n, int s) {
  const int at = min(s, a.p.max_num_seqs - 1);
  const int q0 = a.p.query_start_loc[at], q1 = a.p.query_start_loc[at + 1], len = a.p.context_lens[at];
  Seq q;
  q.q0 = min(max(q0, 0), a.p.total_tokens);
  q.q_len = s < n ? max(min(max(q1, 0), a.p.total_tokens) - q.q0, 0) : 0;
  q.kv_len = min(max(len, 0), a.p.pages_per_seq << a.page_shift);  // at most 2^30
  return q;
}

// A cut of a stream of `total` positions over `n` workgroups: run w is [bound(w), bound(w + 1)).  Where the whole grid takes
// part, two workgroups share a compute unit, and the one that was there first gets the larger part of its issue slots and
// of its memory requests: with equal runs it ends at three quarters of the other's time.  So it gets the longer run: kFirst of
// kPairUnits, the other the rest (2 x 8192 tokens: 746 us at 64, 724 at 72, 707 at 80; 16 chunks of 512 after 4096: 260, 255
// and 256; decode steps of 64 x 4 tokens behind a window 173, 173 and 169, of 256 up to 8192 keys alike).  The workgroups of
// an XCD hold `block` neighbouring runs; those of its first workgroups lie in front in the first stream and behind in the second,
// which is dealt out from the grid's back.
constexpr int kPairUnits = 128, kFirst = 78;
// x / y of numbers that are not negative: 32 bits nearly always; the rest bit by bit, since the code on the way to the
// first load is fetched anew by every launch and a 64-bit division is long.
__device__ __forceinline__ int64_t divide(int64_t x, int64_t y) {
  if (static_cast<uint64_t>(x | y) >> 32 == 0) return static_cast<uint32_t>(x) / static_cast<uint32_t>(y);
  int64_t quotient = 0;
#pragma unroll 1
  for (int b = 62; b >= 0; --b) {
    if ((x >> b) < y) continue;
    x -= y << b;
    quotient |= int64_t{1} << b;
  }
  return quotient;
}
struct Cut {
  int64_t per_unit, rest;  // positions of a unit; the first `rest` units have one more
  int n, block, pair, lead;  // workgroups; a block of them; units of two runs, one of each half of a block; of the one in front
  __device__ __forceinline__ void set(int64_t total) {
    const int64_t units = static_cast<int64_t>(n) * pair / 2;
    per_unit = divide(total, units);
    rest = total - per_unit * units;
  }
  __device__ __forceinline__ int64_t bound(int w) const {
    const int b = w / block, r = w - b * block, half = block / 2;
    const int64_t u = static_cast<int64_t>(b) * half * pair + (r <= half ? r * lead : half * lead + (r - half) * (pair - lead));
    return u * per_unit + min(u, rest);
  }
  __device__ __forceinline__ int owner(int64_t x) const {  // the run that holds position x
    const int64_t big = rest * (per_unit + 1);
    const int64_t u = x < big ? divide(x, per_unit + 1) : rest + divide(x - big, per_unit);
    const int half = block / 2, b = static_cast<int>(divide(u, half * pair)), r = static_cast<int>(u - static_cast<int64_t>(b) * half * pair);
    return b * block + (r < half * lead ? r / lead : half + (r - half * lead) / (pair - lead));
  }
};

// Lengths of 64 sequences at a time, a lane each.
struct Window {
  Seq mine;
  int base = -1;
  __device__ __forceinline__ void at(Args& a, int n, int s) {
    if (base >= 0 && s >= base && s < base + 64) return;
    base = s;
    mine = load_seq(a, n, s + (threadIdx.x & 63));
  }
  __device__ __forceinline__ Seq get(int s) const {
    const int l = s - base;
    return {__builtin_amdgcn_readlane(mine.q0, l), __builtin_amdgcn_readlane(mine.q_len, l), __builtin_amdgcn_readlane(mine.kv_len, l)};
  }
  // The first sequence from s on that is in the stream, or n.
  __device__ __forceinline__ int next(Args& a, int n, int s, bool thin) {
    while (s < n) {
      at(a, n, s);
      const uint64_t m = __ballot(mine.q_len > 0 && is_thin(a, mine) == thin) >> (s - base);
      if (m != 0) return s + __ffsll(static_cast<unsigned long long>(m)) - 1;
      s = base + 64;
    }
    return n;
  }
};

// bf16 parts of eight fp32 values: part 0 is the value rounded, part 1 the rest of it rounded, part 2 the rest of that.
template <int kParts>
__device__ __forceinline__ void split(const float (&x)[8], bf16x8_t (&part)[kParts]) {
  float r[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = x[e];
#pragma unroll
  for (int s = 0; s < kParts; ++s) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      part[s][e] = static_cast<__bf16>(r[e]);
      if (s + 1 < kParts) r[e] -= static_cast<float>(part[s][e]);
    }
  }
}

// Eight query elements from element d of a row (zeros where the row or the element does not exist), with the sign of the
// softmax scale.
template <typename T, int kParts>
__device__ __forceinline__ void load_q(Args& a, const T* row, bool real, int d, bf16x8_t (&part)[kParts]) {
  const int head_dim = a.p.head_dim;
  const uint32_t sign = __float_as_uint(a.p.softmax_scale) & 0x80000000u;
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if constexpr (sizeof(T) == 2) {
    u32x4_t w = {0u, 0u, 0u, 0u};
    if (real && d < head_dim) w = *reinterpret_cast<const u32x4_t*>(row + d);
    w ^= sign | sign >> 16;
    part[0] = __builtin_bit_cast(bf16x8_t, w);
  } else {
    if (real && d < head_dim) {
      const f32x4_t lo = *reinterpret_cast<const f32x4_t*>(row + d), hi = *reinterpret_cast<const f32x4_t*>(row + d + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = __uint_as_float(__float_as_uint(lo[e]) ^ sign);
        x[4 + e] = __uint_as_float(__float_as_uint(hi[e]) ^ sign);
      }
    }
    split<kParts>(x, part);
  }
}

// 16 codes -> two operands of eight bf16.
template <int kCode>
__device__ __forceinline__ void widen16(u32x4_t w, bf16x8_t (&op)[2]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    u32x4_t o;
    o[0] = codes_to_bf16<kCode, false>(w[2 * h]);
    o[1] = codes_to_bf16<kCode, true>(w[2 * h]);
    o[2] = codes_to_bf16<kCode, false>(w[2 * h + 1]);
    o[3] = codes_to_bf16<kCode, true>(w[2 * h + 1]);
    op[h] = __builtin_bit_cast(bf16x8_t, o);
  }
}

// Byte b of two words (two keys) as a pair of bf16, for all four bytes.
template <int kCode>
__device__ __forceinline__ void widen_pairs(uint32_t x, uint32_t y, uint32_t (&pair)[4]) {
  if constexpr (kCode == kCodeI8) {
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const float f = static_cast<float>(static_cast<int8_t>(x >> (8 * b))), g = static_cast<float>(static_cast<int8_t>(y >> (8 * b)));
      pair[b] = __builtin_amdgcn_perm(__float_as_uint(g), __float_as_uint(f), 0x07060302u);
    }
  } else {
    const uint32_t lo = __builtin_amdgcn_perm(y, x, 0x05010400u), hi = __builtin_amdgcn_perm(y, x, 0x07030602u);
    pair[0] = codes_to_bf16<kCode, false>(lo);
    pair[1] = codes_to_bf16<kCode, true>(lo);
    pair[2] = codes_to_bf16<kCode, false>(hi);
    pair[3] = codes_to_bf16<kCode, true>(hi);
  }
}

// A lane offset as it stands beside its load, where the load takes it with a scalar base (hoisted, it becomes a pair of
// registers that is added to the base for every load).
__device__ __forceinline__ uint32_t here(uint32_t off) {
  asm volatile("" : "+v"(off));
  return off;
}
// Loads on either side stay there: they are counted as they come in, so a wait for one that the compiler had moved behind
// the others would be a wait for all of them.
__device__ __forceinline__ void in_order() { asm volatile("" ::: "memory"); }

__device__ __forceinline__ f32x4_t mfma(bf16x8_t a, bf16x8_t b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// A product under its scale: capped in units of log2, or just scaled.  The quick tanh is off by 1e-7 of the cap, nothing beside
// probabilities that are rounded to bf16; with fp32 queries the library's is taken, to a unit of its own size.
template <bool kCap, bool kExact>
__device__ __forceinline__ float scaled(float s, float c, float cap, float inv_cap) {
  if constexpr (kCap) return cap * (kExact ? tanhf(s * c * inv_cap) : tanh_fast(s * c * inv_cap));
  return s * c;
}

// Adds the row's sinks to its sum: (m, l) -> weight of the output and sum under the larger of the two maxima.
__device__ __forceinline__ void add_sinks(Args& a, int head, float m, float& l, float& weight) {
  weight = 1.f;
  if (a.p.num_sinks == 0 || !(l > 0.f)) return;
  const float* sink = a.p.sinks + static_cast<size_t>(head) * a.p.num_sinks;
  float top = m;
  for (int j = 0; j < a.p.num_sinks; ++j) top = fmaxf(top, sink[j] * kLog2e);
  weight = __builtin_amdgcn_exp2f(m - top);
  l *= weight;
  for (int j = 0; j < a.p.num_sinks; ++j) l += __builtin_amdgcn_exp2f(sink[j] * kLog2e - top);
}

// Register r of lane group g <-> register g of lane group r.
template <int W>
__device__ __forceinline__ void transpose_groups(uint32_t (&w)[4][W]) {
#pragma unroll
  for (int k = 0; k < W; ++k) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const auto x = __builtin_amdgcn_permlane32_swap(w[r][k], w[r + 2][k], false, false);
      w[r][k] = x[0], w[r + 2][k] = x[1];
    }
#pragma unroll
    for (int r = 0; r < 4; r += 2) {
      const auto x = __builtin_amdgcn_permlane16_swap(w[r][k], w[r + 1][k], false, false);
      w[r][k] = x[0], w[r + 1][k] = x[1];
    }
  }
}

// N fp32 results to the output, N a multiple of 4.
template <typename T, int N>
__device__ __forceinline__ void store_row(T* dst, const float (&o)[N]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int k = 0; k < N / 4; ++k) *reinterpret_cast<f32x4_t*>(dst + 4 * k) = f32x4_t{o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]};
  } else {
    uint32_t w[N / 2];
#pragma unroll
    for (int k = 0; k < N / 2; ++k) w[k] = pack_bf16x2(o[2 * k], o[2 * k + 1]);
    if constexpr (N % 8 == 0) {
#pragma unroll
      for (int k = 0; k < N / 8; ++k) *reinterpret_cast<u32x4_t*>(dst + 8 * k) = u32x4_t{w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]};
    } else {
      *reinterpret_cast<u32x2_t*>(dst) = u32x2_t{w[0], w[1]};
    }
  }
}

// Who else holds parts of an item that starts at stream position x0 and has `keys` keys (`step` of them at once).
struct Parts {
  int first, count;  // workgroup of the first part, number of parts
  bool head;         // the first part begins the item (else the workgroup where the item starts has none of its keys)
};
__device__ __forceinline__ Parts parts_of(const Cut& cut, int64_t x0, int keys, int step) {
  Parts r;
  const int w0 = cut.owner(x0), w1 = cut.owner(x0 + keys - 1);
  r.head = w1 == w0 || cut.bound(w0 + 1) - x0 >= step;
  r.first = r.head ? w0 : w0 + 1;
  r.count = w1 - r.first + 1;
  return r;
}
// A part's place in the workspace: the run's first item (begun by an earlier workgroup) or its last.
__device__ __forceinline__ int slot_of(const Parts& parts, int k) { return 2 * (parts.first + k) + (parts.head && k == 0 ? 1 : 0); }

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc_of(void* base, uint64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(base, 0, static_cast<int>(min(bytes, static_cast<uint64_t>(0x7fffffff))), 0x00027000);
}

// Hands in a part: the workgroup's stores have left for memory-side storage before the ticket is drawn.  True for the
// workgroup that draws the last one; the ticket is then zero again.
__device__ __forceinline__ bool last_part(uint32_t* ticket, int parts, int* lds_flag) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t t = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *lds_flag = t + 1 == static_cast<uint32_t>(parts);
    if (t + 1 == static_cast<uint32_t>(parts)) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  return *lds_flag != 0;
}

// One wavefront's pass over keys k_begin, k_begin + stride, ... < k_end, 32 at a time (all multiples of 32): MT tiles of 16
// rows against one kv head of sequence s.  Lane (i, g) = (lane % 16, lane / 16) holds column i, a query row, of every
// product.  K: rows i of two 16-key subtiles, pieces g, g + 4, ... of 16 elements, straight from the cache in the order in
// which the matrix unit takes them (q is loaded in the same order).  The logits come out as keys 4 g + r and 16 + 4 g + r,
// which is how the second product wants them, so probabilities stay in their lanes; V: those eight keys, D / 16
// neighbouring elements of each, which byte permutes turn into operands along the keys.  K of the next tile is asked for
// when this tile's has been multiplied, V likewise: one set of registers each, filled for half of the time.
template <int MT, int kD>
struct RowState {
  f32x4_t acc[MT][kD / 16];  // output element (kD / 16) (4 g + r) + n of row i, unnormalised
  float m[MT], l[MT];        // running maximum (log2) of the row, this lane's share of its sum
};
template <int kCode, int D, int kParts, bool kCap, bool kWide, int MT, typename Q>
__device__ __forceinline__ void walk(Args& a, const Seq& q, int s, int h, const Q& query,
                                     const int (&hi)[MT], const Range& range, int full_lo, int full_hi, int k_begin, int k_end, int stride,
                                     RowState<MT, D>& st) {
  constexpr int NP = D / 64, NV = D / 64, NO = D / 16;
  // Bf16 parts of the probabilities.  The first stream waits for memory, so that with bf16 queries a second part costs it nothing and
  // leaves the result's own rounding alone.
  constexpr int kWeightParts = kParts == 1 && MT == 1 ? 2 : kParts;
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4, dim = a.p.head_dim;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    st.m[mt] = kNoKey, st.l[mt] = 0.f;
#pragma unroll
    for (int n = 0; n < NO; ++n) st.acc[mt][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  if (k_begin >= k_end) return;
  const int32_t* __restrict__ table = a.p.block_tables + static_cast<size_t>(s) * a.p.pages_per_seq;
  const int last_page = max(q.kv_len - 1, 0) >> a.page_shift;
  // Lane offsets inside 16 keys of a head.  Pieces beyond head_dim read the row's first again (the queries are zero there,
  // the outputs not stored).
  uint32_t k_off[NP], v_off[4];
#pragma unroll
  for (int n = 0; n < NP; ++n) k_off[n] = (kWide ? i * dim : 0) + (16 * (g + 4 * n) < dim ? 16 * (g + 4 * n) : 0);
#pragma unroll
  for (int r = 0; r < 4; ++r) v_off[r] = ((kWide ? 4 * g : 0) + r) * dim + (NO * i < dim ? NO * i : 0);
  const uint32_t sc_off = 4 * g >> a.block_shift;

  // Pages of 16 tokens and more (kWide): 16 keys have one page, whose address is scalar.  Shorter ones: a page for each
  // lane's key of K and for each lane's four keys of V.  A page is fewer than 2^32 bytes.
  struct Pages {
    int k[2] = {0, 0}, v[2] = {0, 0};
  };
  const int page_mask = (1 << a.page_shift) - 1;
  const uint32_t head_bytes = static_cast<uint32_t>(dim) << a.page_shift, page_bytes = 2 * a.p.num_kv_heads * head_bytes;
  const uint32_t head_scales = 1u << (a.page_shift - a.block_shift), page_scales = 2 * a.p.num_kv_heads * head_scales;
  const char* k_codes = static_cast<const char*>(a.p.kv_cache) + static_cast<uint64_t>(2 * h) * head_bytes;
  const float* k_scales = a.p.kv_scales + static_cast<uint64_t>(2 * h) * head_scales;
  auto codes_at = [&](int page, int k) { return k_codes + (static_cast<uint64_t>(static_cast<uint32_t>(page)) * page_bytes + static_cast<uint32_t>((k & page_mask) * dim)); };
  auto scales_at = [&](int page, int k) { return k_scales + (static_cast<uint64_t>(static_cast<uint32_t>(page)) * page_scales + static_cast<uint32_t>((k & page_mask) >> a.block_shift)); };
  auto load_pages = [&](int k0) {
    Pages pg;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if constexpr (kWide) {
        pg.k[u] = ((const_i32_ptr)table)[min((k0 + 16 * u) >> a.page_shift, last_page)];
      } else {
        pg.k[u] = table[min((k0 + 16 * u + i) >> a.page_shift, last_page)];
        pg.v[u] = table[min((k0 + 16 * u + 4 * g) >> a.page_shift, last_page)];
      }
    }
    return pg;
  };
  u32x4_t kr[2][NP];
  uint32_t vr[2][4][NV];
  float ks[2], vs[2];
  const char* v_rows[2];    // where V of the tile in flight begins, and its scales: known when its K was asked for
  const float* v_scale[2];
  auto load_k = [&](int k0, const Pages& pg) {
    const char* rows[2];
    const float* sc[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      // the pages are clamped here, where they are used, so that nothing waits for them where they are loaded
      const int page = clamp_page(pg.k[u], a.p.num_pages), v_page = kWide ? page : clamp_page(pg.v[u], a.p.num_pages);
      rows[u] = codes_at(page, k0 + 16 * u + (kWide ? 0 : i));
      sc[u] = scales_at(v_page, k0 + 16 * u + (kWide ? 0 : 4 * g));
      v_rows[u] = (kWide ? rows[u] : codes_at(v_page, k0 + 16 * u + 4 * g)) + head_bytes;
      v_scale[u] = sc[u] + head_scales;
    }
#pragma unroll
    for (int n = 0; n < NP; ++n)  // in the order of their use
#pragma unroll
      for (int u = 0; u < 2; ++u) kr[u][n] = *reinterpret_cast<const u32x4_t*>(rows[u] + here(k_off[n]));
#pragma unroll
    for (int u = 0; u < 2; ++u) ks[u] = kWide ? sc[u][here(sc_off)] : *sc[u];
  };
  auto load_v = [&] {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      vs[u] = kWide ? v_scale[u][here(sc_off)] : *v_scale[u];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint32_t* src = reinterpret_cast<const uint32_t*>(v_rows[u] + here(v_off[r]));
        if constexpr (NV == 1) {
          vr[u][r][0] = src[0];
        } else if constexpr (NV == 2) {
          const u32x2_t w = *reinterpret_cast<const u32x2_t*>(src);
          vr[u][r][0] = w[0], vr[u][r][1] = w[1];
        } else {
          const u32x4_t w = *reinterpret_cast<const u32x4_t*>(src);
#pragma unroll
          for (int j = 0; j < 4; ++j) vr[u][r][j] = w[j];
        }
      }
    }
  };

  const float cap = a.p.logits_soft_cap, inv_cap = kCap ? 1.f / cap : 0.f;
  const float magnitude = fabsf(a.p.softmax_scale);  // its sign is in the queries: logits grow with the products
  const float c_scale = kCap ? magnitude : magnitude * kLog2e, cap2 = cap * kLog2e;
  // Loads run ahead without a branch, so that every path to a wait has the same loads behind it: the last tile reads itself
  // again (from the caches).
  Pages pg = load_pages(k_begin), pg_next = load_pages(k_begin + stride);
  load_k(k_begin, pg);
  in_order();
  load_v();
  in_order();
  for (int k0 = k_begin; k0 < k_end; k0 += stride) {
    f32x4_t sa[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) sa[mt][0] = sa[mt][1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      bf16x8_t op[2][2];
#pragma unroll
      for (int u = 0; u < 2; ++u) widen16<kCode>(kr[u][n], op[u]);
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int sp = 0; sp < kParts; ++sp) {
            const bf16x8_t x = query(mt, 2 * n + hf, sp);
#pragma unroll
            for (int u = 0; u < 2; ++u) sa[mt][u] = mfma(op[u][hf], x, sa[mt][u]);
          }
    }
    float c[2] = {ks[0] * c_scale, ks[1] * c_scale}, w[2] = {vs[0], vs[1]};
    const bool more = k0 + stride < k_end;
    const int ahead = more ? k0 + stride : k0;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      pg.k[u] = more ? pg_next.k[u] : pg.k[u];
      pg.v[u] = more ? pg_next.v[u] : pg.v[u];
    }
    pg_next = load_pages(k0 + 2 * stride);
    in_order();
    load_k(ahead, pg);
    in_order();
    const bool edge = k0 < full_lo || k0 + 32 > full_hi;
    const int window = a.p.sliding_window > 0 ? a.p.sliding_window : 0x40000000;  // hi - window: the row's first key, or below 0
    if (kCap || edge) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int k = k0 + 16 * u + 4 * g;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float x = scaled<kCap, kParts == 3>(sa[mt][u][r], c[u], cap2, inv_cap);
            sa[mt][u][r] = !edge || (k + r < hi[mt] && k + r >= hi[mt] - window) ? x : -INFINITY;
          }
        c[u] = 1.f;
        if (edge) {  // what no row sees may be anything
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (k + r < range.first || k + r >= range.end) {
#pragma unroll
              for (int j = 0; j < NV; ++j) vr[u][r][j] = 0u;
            }
          if (k + 3 < range.first || k >= range.end) w[u] = 0.f;
        }
      }
    }
    // Probabilities under the running maximum as it stands.  Where some of them are so large that a logit must have passed it
    // by far (or there was none yet), it follows, which happens a few times in a row's walk: no maximum is taken in the others.
    bf16x8_t pf[MT][kWeightParts];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float pv[8], sum;
      const auto weigh = [&] {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          pv[e] = __builtin_amdgcn_exp2f(fmaf(sa[mt][e >> 2][e & 3], c[e >> 2], -st.m[mt]));
          sum = e == 0 ? pv[0] : sum + pv[e];
        }
      };
      weigh();
      if (__any(sum > kLazy)) {
        const float x0 = fmaxf(fmaxf(fmaxf(sa[mt][0][0], sa[mt][0][1]), sa[mt][0][2]), sa[mt][0][3]) * c[0];  // (scales are not negative)
        const float x1 = fmaxf(fmaxf(fmaxf(sa[mt][1][0], sa[mt][1][1]), sa[mt][1][2]), sa[mt][1][3]) * c[1];
        const float m_new = fmaxf(st.m[mt], row_groups_max(fmaxf(x0, x1)));
        const float alpha = __builtin_amdgcn_exp2f(st.m[mt] - m_new);
#pragma unroll
        for (int n = 0; n < NO; ++n) st.acc[mt][n] *= alpha;
        st.l[mt] *= alpha;
        st.m[mt] = m_new;
        weigh();
      }
      st.l[mt] += sum;
#pragma unroll
      for (int e = 0; e < 8; ++e) pv[e] *= w[e >> 2];
      split<kWeightParts>(pv, pf[mt]);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      uint32_t pair[4][4];  // keys (0 1) (2 3) (16 17) (18 19) of the group, bytes 0..3
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        widen_pairs<kCode>(vr[u][0][j], vr[u][1][j], pair[2 * u]);
        widen_pairs<kCode>(vr[u][2][j], vr[u][3][j], pair[2 * u + 1]);
      }
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const bf16x8_t v = __builtin_bit_cast(bf16x8_t, u32x4_t{pair[0][b], pair[1][b], pair[2][b], pair[3][b]});
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int sp = 0; sp < kWeightParts; ++sp) st.acc[mt][4 * j + b] = mfma(v, pf[mt][sp], st.acc[mt][4 * j + b]);
      }
    }
    in_order();
    load_v();
    in_order();
  }
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) st.l[mt] = row_groups_sum(st.l[mt]);
}

template <int D>
struct ThinLds {
  float o[4][4][D / 64][64][4];  // wavefront, r, piece, lane
  float ml[4][16][2];
};

// A run of keys [ka, kb) (from the range's first key rounded down to 32) of one (sequence, kv head) with R <= 16 rows.
// `self`: this workgroup's place in the cut; x0: the item's first position in the stream.
template <int kCode, int D, typename T, int kParts, bool kCap, bool kWide>
__device__ __forceinline__ void thin_item(Args& a, const Seq& q, int s, int h, int ka, int kb, const Cut& cut, int self, int64_t x0,
                                          ThinLds<D>& lds, int* lds_flag) {
  constexpr int NO = D / 16;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
  const int G = a.group, R = q.q_len * G, dim = a.p.head_dim;
  const Range range = key_range(a, q, 0, q.q_len);
  const int base = range.first & ~31, keys = range.end - base;
  const int token = i / G, head = h * G + i - token * G;
  const bool real = i < R;
  // keys of row i
  const int pos = q.kv_len - q.q_len + token;
  const int hi = real ? pos + 1 : 0;
  const int full_lo = a.p.sliding_window > 0 ? max(q.kv_len - a.p.sliding_window, 0) : 0;  // keys every row sees
  const int full_hi = q.kv_len - q.q_len + 1;

  bf16x8_t qf[1][D / 32][kParts];
  {
    const T* row = static_cast<const T*>(a.p.queries) + (q.q0 + (real ? token : 0)) * a.p.query_token_stride + (real ? head : 0) * a.p.query_head_stride;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) load_q<T, kParts>(a, row, real, 16 * (g + 4 * (k >> 1)) + 8 * (k & 1), qf[0][k]);
  }
  RowState<1, D> st;
  walk<kCode, D, kParts, kCap, kWide, 1>(a, q, s, h, [&](int, int k, int sp) { return qf[0][k][sp]; }, {hi}, range, full_lo, full_hi, base + ka + 32 * wave, base + ((min(kb, keys) + 31) & ~31), 128, st);
  const auto& acc = st.acc[0];
  const float m = st.m[0], l = st.l[0];

  // The four wavefronts meet: wavefront w adds up outputs NO (4 g + w) .. + NO of every row.
  __syncthreads();  // LDS may hold what came before
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int n = 0; n < NO / 4; ++n)
      *reinterpret_cast<f32x4_t*>(lds.o[wave][r][n][lane]) = f32x4_t{acc[4 * n][r], acc[4 * n + 1][r], acc[4 * n + 2][r], acc[4 * n + 3][r]};
  if (g == 0) lds.ml[wave][i][0] = m, lds.ml[wave][i][1] = l;
  __syncthreads();
  float top = kNoKey, sum = 0.f, o[NO];
#pragma unroll
  for (int v = 0; v < 4; ++v) top = fmaxf(top, lds.ml[v][i][0]);
#pragma unroll
  for (int n = 0; n < NO; ++n) o[n] = 0.f;
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    const float f = __builtin_amdgcn_exp2f(lds.ml[v][i][0] - top);
    sum = fmaf(f, lds.ml[v][i][1], sum);
#pragma unroll
    for (int n = 0; n < NO / 4; ++n) {
      const f32x4_t y = *reinterpret_cast<const f32x4_t*>(lds.o[v][wave][n][lane]);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[4 * n + e] = fmaf(f, y[e], o[4 * n + e]);
    }
  }

  if (ka > 0 || kb < keys) {  // a part: hand it in, and add all of them up if it is the last
    const Parts parts = parts_of(cut, x0, range.end - range.first, kThinStep);
    const int slots = 2 * a.grid;
    const auto o_rsrc = rsrc_of(a.thin_o, static_cast<uint64_t>(slots) * 16 * D * 4);
    const int part = self - parts.first;
    const auto place = [&](int k, int n) { return ((slot_of(parts, k) * 4 + wave) * (NO / 4) + n) * 1024 + lane * 16; };
#pragma unroll
    for (int n = 0; n < NO / 4; ++n)
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, f32x4_t{o[4 * n], o[4 * n + 1], o[4 * n + 2], o[4 * n + 3]}), o_rsrc, place(part, n), 0, kAgentScope);
    if (wave == 0 && g == 0) {
      const uint64_t both = (static_cast<uint64_t>(__float_as_uint(sum)) << 32) | __float_as_uint(top);
      __hip_atomic_store(reinterpret_cast<uint64_t*>(a.thin_ml) + slot_of(parts, part) * 16 + i, both, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (!last_part(a.tickets + parts.first, parts.count, lds_flag)) return;
    top = kNoKey, sum = 0.f;
#pragma unroll
    for (int n = 0; n < NO; ++n) o[n] = 0.f;
    constexpr int kAtOnce = 4;  // parts whose loads are in flight together
    for (int k0 = 0; k0 < parts.count; k0 += kAtOnce) {
      uint64_t both[kAtOnce];
      u32x4_t y[kAtOnce][NO / 4];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        const int k = min(k0 + j, parts.count - 1);
        both[j] = __hip_atomic_load(reinterpret_cast<uint64_t*>(a.thin_ml) + slot_of(parts, k) * 16 + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
        for (int n = 0; n < NO / 4; ++n) y[j][n] = __builtin_amdgcn_raw_buffer_load_b128(o_rsrc, place(k, n), 0, kAgentScope);
      }
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        if (k0 + j >= parts.count) break;
        const float mk = __uint_as_float(static_cast<uint32_t>(both[j])), lk = __uint_as_float(static_cast<uint32_t>(both[j] >> 32));
        const float t_new = fmaxf(top, mk), f = __builtin_amdgcn_exp2f(top - t_new), fk = __builtin_amdgcn_exp2f(mk - t_new);
        top = t_new;
        sum = sum * f + lk * fk;
#pragma unroll
        for (int n = 0; n < NO / 4; ++n) {
          const f32x4_t z = __builtin_bit_cast(f32x4_t, y[j][n]);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[4 * n + e] = o[4 * n + e] * f + z[e] * fk;
        }
      }
    }
  }
  if (!real) return;
  float weight;
  add_sinks(a, head, top, sum, weight);
  const float f = sum > 0.f ? weight / sum : 0.f;
  T* dst = static_cast<T*>(a.p.out) + (static_cast<size_t>(q.q0 + token) * a.p.num_q_heads + head) * dim;
#pragma unroll
  for (int n = 0; n < NO; ++n) o[n] *= f;
  if (NO * (4 * g + wave) < dim) store_row<T, NO>(dst + NO * (4 * g + wave), o);
}

// Queries of a tile that are not in registers: every wavefront's own, as the matrix unit takes them.
template <int D, int kParts>
struct TileLds {
  static constexpr bool kAllParts = quant_reg_pieces<D, kParts>() < D / 32;  // of the pieces behind the first, else the last parts of all
  static constexpr int kPieces = kAllParts ? D / 32 - quant_reg_pieces<D, kParts>() : D / 32;
  static constexpr int kLds = kAllParts ? kParts : kParts - quant_reg_parts<D, kParts>();
  bf16x8_t q[4][quant_row_tiles<D, kParts>()][kPieces][kLds > 0 ? kLds : 1][kLds > 0 ? 64 : 1];
  __device__ __forceinline__ bf16x8_t& at(int wave, int mt, int k, int sp) {
    return q[wave][mt][k - (D / 32 - kPieces)][kAllParts ? sp : sp - (kParts - kLds)][threadIdx.x & 63];
  }
};

// A run of keys [ka, kb) of one tile of rows.
template <int kCode, int D, typename T, int kParts, bool kCap, bool kWide>
__device__ __forceinline__ void tile_item(Args& a, const Seq& q, int s, int hs, int tile, int ka, int kb, const Cut& cut, int self, int64_t x0,
                                          TileLds<D, kParts>& lds) {
  constexpr int kRowTiles = quant_row_tiles<D, kParts>(), NO = D / 16;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
  const int dim = a.p.head_dim;
  const int h = hs / a.subs, sub = hs - h * a.subs;
  const int t0 = tile * a.tile_tokens, t1 = min(t0 + a.tile_tokens, q.q_len);
  const Range range = key_range(a, q, t0, t1);
  const int base = range.first & ~31, keys = range.end - base;
  const int q_base = q.kv_len - q.q_len;

  // row i of row tile m of this wavefront: its token in the sequence (negative: none) and its head
  struct Row {
    int token, head;
  };
  auto row_of_tile = [&](int mt) {
    const int rr = (wave * kRowTiles + mt) * 16 + i;
    const int dt = rr / a.tile_group, gg = sub * a.tile_group + rr - dt * a.tile_group;
    return Row{dt < t1 - t0 && gg < a.group ? t0 + dt : -1, h * a.group + gg};
  };
  int hi[kRowTiles];
  constexpr int kReg = quant_reg_parts<D, kParts>(), kPieces = quant_reg_pieces<D, kParts>();
  bf16x8_t qf[kRowTiles][D / 32][kReg > 0 ? kReg : 1];
#pragma unroll
  for (int mt = 0; mt < kRowTiles; ++mt) {
    const Row row = row_of_tile(mt);
    const bool real = row.token >= 0;
    hi[mt] = real ? q_base + row.token + 1 : 0;
    const T* src = static_cast<const T*>(a.p.queries) + (q.q0 + (real ? row.token : 0)) * a.p.query_token_stride + (real ? row.head : 0) * a.p.query_head_stride;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) {
      bf16x8_t part[kParts];
      load_q<T, kParts>(a, src, real, 16 * (g + 4 * (k >> 1)) + 8 * (k & 1), part);
#pragma unroll
      for (int sp = 0; sp < kParts; ++sp) {
        if (sp < kReg && k < kPieces) qf[mt][k][sp] = part[sp];
        else lds.at(wave, mt, k, sp) = part[sp];
      }
    }
  }
  const auto query = [&](int mt, int k, int sp) { return sp < kReg && k < kPieces ? qf[mt][k][sp] : lds.at(wave, mt, k, sp); };
  const int full_lo = a.p.sliding_window > 0 ? max(q_base + t1 - a.p.sliding_window, 0) : 0;  // keys every row sees
  const int full_hi = q_base + t0 + 1;
  RowState<kRowTiles, D> st;
  walk<kCode, D, kParts, kCap, kWide, kRowTiles>(a, q, s, h, query, hi, range, full_lo, full_hi, base + ka, base + ((min(kb, keys) + 31) & ~31), 32, st);
  auto& acc = st.acc;
  auto& m = st.m;
  auto& l = st.l;

  if (ka > 0 || kb < keys) {
    const Parts parts = parts_of(cut, x0, range.end - range.first, kTileStep);
    const int slots = 2 * a.grid;
    const auto o_rsrc = rsrc_of(a.tile_o, static_cast<uint64_t>(slots) * 64 * kRowTiles * D * 4);
    const int part = self - parts.first;
    // The parts meet in a tree, pairs of neighbours first: whoever comes to a node second adds the other's state to its own,
    // which it still has in registers, and goes on to the next; whoever comes first leaves its state behind.  A wavefront's
    // rows are its own, so each goes its own way.  A ticket holds the part that waits at its node, plus one.
    const int wait_part = part + 1;
    const auto slot_at = [&](int k) { return slot_of(parts, k) * 4 + wave; };
    const auto place = [&](int k, int mt, int n) { return ((slot_at(k) * kRowTiles + mt) * NO + n) * 1024 + lane * 16; };
    const auto ml_at = [&](int k, int mt) { return reinterpret_cast<uint64_t*>(a.tile_ml) + (slot_at(k) * kRowTiles + mt) * 16 + i; };
    int level = 0;
    for (int span = 1; span < parts.count; span *= 2, ++level) {
#pragma clang fp contract(off)  // one of the two weights is 1: with both products rounded the sum is the same whoever adds
      const int node = part & -(2 * span), sibling = (part & span) != 0 ? node : node + span;
      if (sibling >= parts.count) continue;  // nobody to meet on this level
      uint32_t* ticket = a.tickets + a.grid + ((level * a.grid + parts.first + node) * 4 + wave);
      int other = __hip_atomic_load(ticket, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      other = __builtin_amdgcn_readfirstlane(other);
      if (other == 0) {
#pragma unroll
        for (int mt = 0; mt < kRowTiles; ++mt) {
#pragma unroll
          for (int n = 0; n < NO; ++n) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, acc[mt][n]), o_rsrc, place(part, mt, n), 0, kAgentScope);
          if (g == 0) {
            const uint64_t both = (static_cast<uint64_t>(__float_as_uint(l[mt])) << 32) | __float_as_uint(m[mt]);
            __hip_atomic_store(ml_at(part, mt), both, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the state is in memory before anybody is told
        if (lane == 0) other = __hip_atomic_exchange(ticket, static_cast<uint32_t>(wait_part), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        other = __builtin_amdgcn_readfirstlane(other);
        if (other == 0) return;
      }
      asm volatile("" ::: "memory");
      if (lane == 0) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      const int from = other - 1;
      uint64_t both[kRowTiles];
      u32x4_t y[kRowTiles][NO];  // all of a state is in flight at once
#pragma unroll
      for (int mt = 0; mt < kRowTiles; ++mt) {
        both[mt] = __hip_atomic_load(ml_at(from, mt), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
        for (int n = 0; n < NO; ++n) y[mt][n] = __builtin_amdgcn_raw_buffer_load_b128(o_rsrc, place(from, mt, n), 0, kAgentScope);
      }
#pragma unroll
      for (int mt = 0; mt < kRowTiles; ++mt) {
        const float mk = __uint_as_float(static_cast<uint32_t>(both[mt])), lk = __uint_as_float(static_cast<uint32_t>(both[mt] >> 32));
        const float t_new = fmaxf(m[mt], mk), f = __builtin_amdgcn_exp2f(m[mt] - t_new), fk = __builtin_amdgcn_exp2f(mk - t_new);
        m[mt] = t_new;
        l[mt] = l[mt] * f + lk * fk;
#pragma unroll
        for (int n = 0; n < NO; ++n) {
          const f32x4_t z = __builtin_bit_cast(f32x4_t, y[mt][n]);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[mt][n][e] = acc[mt][n][e] * f + z[e] * fk;
        }
      }
    }
  }
#pragma unroll
  for (int mt = 0; mt < kRowTiles; ++mt) {
    const Row row = row_of_tile(mt);
    float weight;
    add_sinks(a, row.token < 0 ? 0 : row.head, m[mt], l[mt], weight);
    const float f = l[mt] > 0.f ? weight / l[mt] : 0.f;
    // A lane has four pieces of a row that follow each other; the four lanes of a row exchange them, so that a store writes
    // whole cache lines.
    constexpr int W = NO * static_cast<int>(sizeof(T)) / 4;
    uint32_t w[4][W];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int k = 0; k < W; ++k) {
        if constexpr (sizeof(T) == 4) w[r][k] = __float_as_uint(acc[mt][k][r] * f);
        else w[r][k] = pack_bf16x2(acc[mt][2 * k][r] * f, acc[mt][2 * k + 1][r] * f);
      }
    transpose_groups<W>(w);
    if (row.token < 0) continue;
    T* dst = static_cast<T*>(a.p.out) + (static_cast<size_t>(q.q0 + row.token) * a.p.num_q_heads + row.head) * dim;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = NO * (4 * r + g);
      if (d >= dim) continue;
      if constexpr (W == 2) {
        *reinterpret_cast<u32x2_t*>(dst + d) = u32x2_t{w[r][0], w[r][1]};
      } else {
#pragma unroll
        for (int k = 0; k < W / 4; ++k) reinterpret_cast<u32x4_t*>(dst + d)[k] = u32x4_t{w[r][4 * k], w[r][4 * k + 1], w[r][4 * k + 2], w[r][4 * k + 3]};
      }
    }
  }
}

// Place of workgroup b in a stream's cut over n workgroups (-1: none): the workgroups of one XCD hold neighbouring runs.
__device__ __forceinline__ int place_in_cut(int b, int n) {
  const int xcd = b & 7, j = b >> 3, per = n >> 3, rem = n & 7;
  return j < per + (xcd < rem ? 1 : 0) ? xcd * per + min(xcd, rem) + j : -1;
}

// A workgroup's run of a stream: [x, x_end) of `cut`, beginning `off` positions into sequence `seq` of n.
struct Run {
  Cut cut;
  int self, seq, n;
  int fixed;  // first stream: positions of every item (a multiple of the run), 0 where they are its keys and kThinPad
  Seq first;  // lengths of sequence `seq`
  int64_t x, x_end, off;
};

struct SchedLds {
  int64_t sums[4][2];
  int seqs[4], longest[4];
  Run run[2];
  int flag;
};

template <int D, int kParts>
struct Lds {
  union {
    ThinLds<D> thin;
    TileLds<D, kParts> tile;
  };
  SchedLds sched;
};
template <int D, int kParts>
__device__ __forceinline__ Lds<D, kParts>& lds_of() {
  __shared__ __align__(16) char bytes[sizeof(Lds<D, kParts>)];
  return *reinterpret_cast<Lds<D, kParts>*>(bytes);
}

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<int>(x)), hi = __builtin_amdgcn_readfirstlane(static_cast<int>(x >> 32));
  return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ Run uniform(const Run& r) {
  return {{uniform(r.cut.per_unit), uniform(r.cut.rest), uniform(r.cut.n), uniform(r.cut.block), uniform(r.cut.pair), uniform(r.cut.lead)}, uniform(r.self), uniform(r.seq), uniform(r.n), uniform(r.fixed),
          {uniform(r.first.q0), uniform(r.first.q_len), uniform(r.first.kv_len)}, uniform(r.x), uniform(r.x_end), uniform(r.off)};
}


template <int kCode, int D, typename T, int kParts, bool kCap, bool kWide>
__device__ __forceinline__ void thin_phase(uint64_t args) {
  Args& a = *reinterpret_cast<Args*>(uniform(static_cast<int64_t>(args)));
  Lds<D, kParts>& lds = lds_of<D, kParts>();
  const Run run = uniform(lds.sched.run[0]);
  Window window;
  int s = run.seq;
  int64_t off = run.off, x = run.x;
  Seq q = run.first;
  while (x < run.x_end && s < run.n) {
    const int keys = thin_keys(a, q), len = run.fixed > 0 ? run.fixed : keys + kThinPad;
    const Range range = key_range(a, q, 0, q.q_len);
    const int all = range.end - (range.first & ~31);  // keys as they are walked
    int h = static_cast<int>(divide(off, len));
    int begin = static_cast<int>(off - static_cast<int64_t>(h) * len);
    for (; h < a.p.num_kv_heads && x < run.x_end; ++h, begin = 0) {
      const int end = static_cast<int>(min(static_cast<int64_t>(len), begin + (run.x_end - x)));
      const int ka = begin >= keys ? all : begin / kThinStep * kThinStep, kb = end >= keys ? all : end / kThinStep * kThinStep;
      if (ka < kb || (keys == 0 && begin == 0))
        thin_item<kCode, D, T, kParts, kCap, kWide>(a, q, s, h, keys == 0 ? 0 : ka, kb, run.cut, run.self, x - begin, lds.thin, &lds.sched.flag);
      x += end - begin;
    }
    off = 0;
    if (x < run.x_end) s = window.next(a, run.n, s + 1, true);
    if (x < run.x_end && s < run.n) q = window.get(s);
  }
}

template <int kCode, int D, typename T, int kParts, bool kCap, bool kWide>
__device__ __forceinline__ void tile_phase(uint64_t args) {
  constexpr int kStep = kTileStep;
  Args& a = *reinterpret_cast<Args*>(uniform(static_cast<int64_t>(args)));
  Lds<D, kParts>& lds = lds_of<D, kParts>();
  const Run run = uniform(lds.sched.run[1]);
  __syncthreads();  // the other stream's items may still be read from LDS
  Window window;
  int s = run.seq;
  int64_t off = run.off, x = run.x;
  const int heads = a.p.num_kv_heads * a.subs;
  Seq q = run.first;
  while (x < run.x_end && s < run.n) {
    const int tiles = tiles_of(a, q);
    const int64_t len = tiles_before(a, q, tiles, true);
    int h = static_cast<int>(divide(off, len));
    int64_t rest = off - static_cast<int64_t>(h) * len;
    int tile = 0;  // the last tile that starts at or before the position: 64 of them tried at once
    for (int span = tiles; span > 1;) {
      const int step = (span + 63) >> 6, k = static_cast<int>(threadIdx.x & 63) * step;
      const int before = __popcll(__ballot(k < span && tiles_before(a, q, tile + min(k, span - 1), false) <= rest)) - 1;
      tile += before * step;
      span = min(step, span - before * step);
    }
    int begin = static_cast<int>(rest - tiles_before(a, q, tile, false));
    for (; h < heads && x < run.x_end; ++h, tile = 0) {
      for (; tile < tiles && x < run.x_end; ++tile, begin = 0) {
        const Range range = key_range(a, q, tile * a.tile_tokens, min((tile + 1) * a.tile_tokens, q.q_len));
        const int keys = range.end - range.first, all = range.end - (range.first & ~31), item = keys + a.tile_pad;
        const int end = static_cast<int>(min(static_cast<int64_t>(item), begin + (run.x_end - x)));
        const int ka = begin >= keys ? all : begin / kStep * kStep, kb = end >= keys ? all : end / kStep * kStep;
        if (ka < kb || (keys == 0 && begin == 0))
          tile_item<kCode, D, T, kParts, kCap, kWide>(a, q, s, h, tile, keys == 0 ? 0 : ka, kb, run.cut, run.self, x - begin, lds.tile);
        x += end - begin;
      }
    }
    off = 0;
    if (x < run.x_end) s = window.next(a, run.n, s + 1, false);
    if (x < run.x_end && s < run.n) q = window.get(s);
  }
}

template <int kCode, int D, typename T, int kParts, bool kCap, bool kWide>
__device__ __attribute__((noinline)) void tile_phase_apart(uint64_t args) {
  tile_phase<kCode, D, T, kParts, kCap, kWide>(args);
}

template <int kCode, int D, typename T, int kParts, bool kCap, bool kWide>
__global__ __launch_bounds__(256, 2) void quant_attention_kernel(QuantArgs) {
  Args& a = *(Args*)__builtin_amdgcn_kernarg_segment_ptr();
  SchedLds& sched = lds_of<D, kParts>().sched;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = min(max(a.p.num_seqs[0], 0), a.p.max_num_seqs);

  // Lengths of the two streams; of the first also the longest item and how many sequences there are.
  const int per = (a.p.max_num_seqs + 255) >> 8;
  const int s0 = min(static_cast<int>(threadIdx.x) * per, a.p.max_num_seqs), s1 = min(s0 + per, a.p.max_num_seqs);
  auto length = [&](const Seq& q, bool thin) {
    return thin ? static_cast<int64_t>(thin_keys(a, q) + kThinPad) * a.p.num_kv_heads : tiles_before(a, q, tiles_of(a, q), true) * a.p.num_kv_heads * a.subs;
  };
  int64_t sum[2] = {0, 0};
  int seqs = 0, longest = 0;
  Seq only = {0, 0, 0};
  for (int s = s0; s < s1; ++s) {
    const Seq q = load_seq(a, n, s);
    only = q;
    if (q.q_len == 0) continue;
    const bool thin = is_thin(a, q);
    sum[thin ? 0 : 1] += length(q, thin);
    if (thin) ++seqs, longest = max(longest, thin_keys(a, q));
  }
  int64_t inc[2] = {sum[0], sum[1]};
  int seqs_inc = seqs;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t x = __shfl_up(inc[0], o), y = __shfl_up(inc[1], o);
    const int z = __shfl_up(seqs_inc, o);
    if (lane >= o) inc[0] += x, inc[1] += y, seqs_inc += z;
    longest = max(longest, __shfl_xor(longest, o));
  }
  if (lane == 63) {
    sched.sums[wave][0] = inc[0], sched.sums[wave][1] = inc[1];
    sched.seqs[wave] = seqs_inc, sched.longest[wave] = longest;
  }
  __syncthreads();
  int64_t before[2] = {inc[0] - sum[0], inc[1] - sum[1]}, total[2] = {0, 0};
  int seqs_before = seqs_inc - seqs, seqs_all = 0;
  longest = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < wave) before[0] += sched.sums[w][0], before[1] += sched.sums[w][1], seqs_before += sched.seqs[w];
    total[0] += sched.sums[w][0], total[1] += sched.sums[w][1];
    seqs_all += sched.seqs[w];
    longest = max(longest, sched.longest[w]);
  }
  // Few items: as many equal parts for each as there are workgroups, one for a compute unit, and places for the longest.  A
  // run that holds the end of an item and the start of the next takes 6 us longer, in which a workgroup walks kThinUneven
  // keys, so items of different lengths get places of their own unless the longest is that much longer than an even run
  // (8 x 8192 keys of 8 heads: 39 us cut anywhere, 34 us in equal parts; 24 x 1024: 27 and 20 us); and parts that meet
  // take 2 us, kThinMeet keys, so short items are not cut (8 x 512 keys: 15.2 us in two parts, 14.7 us in one; 8 x 1024:
  // 15.8 us in four, 18.8 us in one).
  const int64_t items = static_cast<int64_t>(seqs_all) * a.p.num_kv_heads;
  int parts = 0, piece = 0;
  // Nearly as many items as workgroups are whole as well (64 x 4 tokens of 8 heads behind a window: 176 us cut evenly, 171 us so).
  const int places = items <= a.grid / 2 ? a.grid / 2 : a.grid;
  if (items > 0 && items <= places && (places < a.grid || items * 10 >= a.grid * 9)) {
    parts = max(min(places / static_cast<int>(items), longest / kThinLeast), 1);
    if (longest - longest / parts < kThinMeet) parts = 1;
    piece = max(((longest - 1) / parts + kThinStep) & -kThinStep, kThinStep);  // parts * piece >= longest
    if (piece > total[0] / places + kThinUneven) parts = 0;
  }
  const int fixed = parts * piece;
  if (fixed > 0) {
    sum[0] = static_cast<int64_t>(seqs) * a.p.num_kv_heads * fixed;
    before[0] = static_cast<int64_t>(seqs_before) * a.p.num_kv_heads * fixed;
    total[0] = items * fixed;
  }
  bool has[2];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    Run r;
    r.n = n;
    r.fixed = c == 0 ? fixed : 0;
    const int64_t most = max(total[c] / (c == 0 ? kThinLeast : kTileLeast), static_cast<int64_t>(1));  // workgroups worth their while
    const bool whole = most >= a.grid && r.fixed == 0;
    r.cut.n = whole ? a.grid : static_cast<int>(r.fixed > 0 ? items * parts : min(most, static_cast<int64_t>(a.grid / 2)));
    r.cut.block = whole ? a.grid / 8 : 2 * r.cut.n;
    r.cut.pair = whole ? kPairUnits : 2;
    r.cut.lead = !whole ? 1 : c == 0 ? kFirst : kPairUnits - kFirst;
    r.cut.set(total[c]);
    // the first stream from the grid's front, the second from its back: where both are short they meet different workgroups
    r.self = total[c] > 0 ? place_in_cut(c == 0 ? blockIdx.x : a.grid - 1 - blockIdx.x, r.cut.n) : -1;
    r.x = r.self >= 0 ? r.cut.bound(r.self) : 0;
    r.x_end = r.self >= 0 ? r.cut.bound(r.self + 1) : 0;
    has[c] = r.x < r.x_end;
    // the thread whose sequences hold the run's first position finds it
    if (r.self >= 0 && r.x >= before[c] && r.x < before[c] + sum[c]) {
      int64_t off = r.x - before[c];
      for (int s = s0; s < s1; ++s) {
        const Seq q = per == 1 ? only : load_seq(a, n, s);
        if (q.q_len == 0 || is_thin(a, q) != (c == 0)) continue;
        const int64_t len = r.fixed > 0 ? static_cast<int64_t>(r.fixed) * a.p.num_kv_heads : length(q, c == 0);
        if (off < len) {
          r.seq = s;
          r.first = q;
          r.off = off;
          sched.run[c] = r;
          break;
        }
        off -= len;
      }
    }
  }
  __syncthreads();
  const bool thin_first = static_cast<int>(blockIdx.x) * 2 < a.grid;
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {
    const int c = (k == 0) == thin_first ? 0 : 1;
    const uint64_t args = reinterpret_cast<uint64_t>(&a);
    if (c == 0 && has[0]) thin_phase<kCode, D, T, kParts, kCap, kWide>(args);
    if (c == 1 && has[1]) {
      if constexpr (quant_apart<D, kParts>()) tile_phase_apart<kCode, D, T, kParts, kCap, kWide>(args);
      else tile_phase<kCode, D, T, kParts, kCap, kWide>(args);
    }
  }

  // Rows in front of the first sequence and behind the last are zeros.
  const int row_first = n > 0 ? min(max(a.p.query_start_loc[0], 0), a.p.total_tokens) : 0;
  const int row_last = n > 0 ? max(row_first, min(max(a.p.query_start_loc[n], 0), a.p.total_tokens)) : 0;
  const int64_t row_words = static_cast<int64_t>(a.p.num_q_heads) * a.p.head_dim * sizeof(T) / 16;
  u32x4_t* out = static_cast<u32x4_t*>(a.p.out);
  const int64_t at = blockIdx.x * 256 + threadIdx.x, stride = static_cast<int64_t>(a.grid) * 256;
  for (int64_t k = at; k < row_first * row_words; k += stride) out[k] = u32x4_t{0u, 0u, 0u, 0u};
  for (int64_t k = row_last * row_words + at; k < a.p.total_tokens * row_words; k += stride) out[k] = u32x4_t{0u, 0u, 0u, 0u};
}

}  // namespace quant

// Launches the kernel for one type of codes; head_dim is padded to 64, 128 or 256.
template <int kCode>
int launch_quant_codes(const QuantArgs& a, hipStream_t stream) {
  const bool f32 = a.p.dtype == RPA_DTYPE_F32, cap = a.p.logits_soft_cap != 0.f;
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(a.grid), dim3(256), 0, stream, a);
    return hipGetLastError() == hipSuccess ? RPA_OK : RPA_ERR_LAUNCH;
  };
  auto width = [&](auto d) {
    constexpr int D = decltype(d)::value;
    auto pages = [&](auto wide) {
      constexpr bool W = decltype(wide)::value;
      if (f32) return cap ? go(quant::quant_attention_kernel<kCode, D, float, 3, true, W>) : go(quant::quant_attention_kernel<kCode, D, float, 3, false, W>);
      return cap ? go(quant::quant_attention_kernel<kCode, D, bf16_t, 1, true, W>) : go(quant::quant_attention_kernel<kCode, D, bf16_t, 1, false, W>);
    };
    return a.page_shift >= 4 ? pages(std::true_type{}) : pages(std::false_type{});
  };
  if (a.p.head_dim <= 64) return width(std::integral_constant<int, 64>{});
  if (a.p.head_dim <= 128) return width(std::integral_constant<int, 128>{});
  return width(std::integral_constant<int, 256>{});
}

int launch_quant_i8(const QuantArgs& a, hipStream_t stream);
int launch_quant_e4m3(const QuantArgs& a, hipStream_t stream);
int launch_quant_e5m2(const QuantArgs& a, hipStream_t stream);

}  // namespace rpa
