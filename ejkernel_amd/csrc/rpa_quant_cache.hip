// Writing to and reading from the 8-bit paged cache with a scale per block of tokens and head.
//
// Update.  For every run of new tokens inside one block and every combined head (K or V of a kv head):
//   a = max |x| over the run's finite elements,  s = a / 127  or  2^ceil(log2(a / qmax)),  at least the block's old scale
//   if the run begins inside the block;  code = round(x / s);  if s grew, the codes in front of the run are re-expressed.
// One wavefront takes one (run, combined head).  It keeps the rows in registers between the maximum and the codes (runs of
// more than 64 elements a lane are read twice, the second time from the caches) and writes one byte per element, so what
// bounds it is the traffic of the rows, and for single tokens the chain slot -> row and old scale -> code.  Runs are found
// from the slots alone: a wavefront looks at 64 tokens at once.
#include <algorithm>
#include <type_traits>

#include "rpa_quant.h"
#include "rpa_tile_common.h"

namespace rpa {

namespace {

constexpr int kPiece = 8;         // elements a lane handles at once
constexpr int kTokensPerChunk = 64;
constexpr int kBatch = 8;         // pieces a lane has in flight

typedef __attribute__((ext_vector_type(2))) uint16_t u16x2_t;

// Eight elements as they lie in memory, and as floats.
template <typename T>
struct Piece {
  uint4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* __restrict__ src) {
#pragma unroll
    for (unsigned k = 0; k < sizeof(T) / 2; ++k) w[k] = reinterpret_cast<const uint4*>(src)[k];
  }
  // Largest magnitude so far as an integer, which orders magnitudes as the numbers do, infinity and then NaN on top; bf16 in
  // both halves of a word at once.
  __device__ __forceinline__ uint32_t top(uint32_t most) const {
#pragma unroll
    for (unsigned k = 0; k < sizeof(T) / 2; ++k) {
      const uint32_t u[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if constexpr (sizeof(T) == 4) most = max(most, u[c] & 0x7fffffffu);
        else most = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, most), __builtin_bit_cast(u16x2_t, u[c] & 0x7fff7fffu)));
      }
    }
    return most;
  }
  __device__ __forceinline__ void get(float (&x)[kPiece]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        x[4 * k] = __uint_as_float(w[k].x), x[4 * k + 1] = __uint_as_float(w[k].y);
        x[4 * k + 2] = __uint_as_float(w[k].z), x[4 * k + 3] = __uint_as_float(w[k].w);
      }
    } else {
      const uint32_t u[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[2 * k] = __uint_as_float(u[k] << 16);
        x[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u);
      }
    }
  }
};

// round(x / s) with ties to even, decided on the exact quotient.  `inv` is 1 / s rounded, so x * inv is off by three
// roundings at most and its nearest integer q by one; r = x - q s is exact in fp32: x and q s are multiples of one unit
// in the last place of s (or of x, where |x| < s and q is 0 or 1), and |r| < 2 s.
__device__ __forceinline__ float round_quotient(float x, float s, float inv) {
  float q = rintf(x * inv);
  const float r = fmaf(-q, s, x), h = 0.5f * s;
  const bool odd = (static_cast<int>(q) & 1) != 0;
  if (r > h || (r == h && odd)) q += 1.f;
  else if (r < -h || (r == -h && odd)) q -= 1.f;
  return q;
}

// A quotient in fp64 as an fp32 number that an 8-bit floating type rounds alike: cut off towards zero, with the last bit set
// where that is not exact.  Such a number lies on the quotient's side of every middle between two codes, whose last bit is
// clear.  (Quotients of 32-bit products lie on a middle or further from it than fp64 rounds.)
__device__ __forceinline__ float off_the_middle(double v) {
  const float f = static_cast<float>(v);
  const double d = static_cast<double>(f);
  if (d == v) return f;
  return __uint_as_float((__float_as_uint(f) - (fabs(d) > fabs(v) ? 1u : 0u)) | 1u);
}

// Code of x under scale s (0 where the block is all zeros).  Infinities saturate, NaN is 0.  Where the scale of a floating
// type is a power of two, as an update makes it, x * inv is exact (or below the type's least step, too small for its
// rounding to matter); an old scale that somebody else wrote need not be one.
template <int kCode>
__device__ __forceinline__ uint32_t pack4(const float* x, float s, float inv) {
  float y[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float v = x[k];
    v = v != v ? 0.f : v;
    if constexpr (kCode == kCodeI8) {
      v = s > 0.f ? (isinf(v) ? copysignf(127.f, v) : round_quotient(v, s, inv)) : 0.f;
    } else {
      v = !(s > 0.f) ? 0.f : (__float_as_uint(s) & 0x7fffffu) == 0 ? v * inv : off_the_middle(static_cast<double>(v) / static_cast<double>(s));
      v = fminf(fmaxf(v, -code_max<kCode>()), code_max<kCode>());
    }
    y[k] = v;
  }
  if constexpr (kCode == kCodeI8) {
    uint32_t w = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) w |= (static_cast<uint32_t>(static_cast<int>(y[k])) & 0xffu) << (8 * k);
    return w;
  } else if constexpr (kCode == kCodeE4m3) {
    return __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false), true);
  } else {
    return __builtin_amdgcn_cvt_pk_bf8_f32(y[2], y[3], __builtin_amdgcn_cvt_pk_bf8_f32(y[0], y[1], 0, false), true);
  }
}

// The same for finite x of at most code_max * s, without the cases that pack4 looks for.  For int8, adding 1.5 * 2^23 leaves
// round(x * inv) in the low bits of the sum; `odd` is set where the remainder reaches half a step, which pack4 then decides.
template <int kCode>
__device__ __forceinline__ uint32_t pack4_finite(const float* x, float s, float inv, bool& odd) {
  if constexpr (kCode == kCodeI8) {
    constexpr float kRound = 12582912.f;
    uint32_t u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float y = fmaf(x[k], inv, kRound);
      odd |= fabsf(fmaf(-(y - kRound), s, x[k])) >= 0.5f * s;
      u[k] = __float_as_uint(y);
    }
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(u[3], u[2], 0x0c0c0400u), __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400u), 0x05040100u);
  } else if constexpr (kCode == kCodeE4m3) {
    return __builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inv, x[3] * inv, __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inv, x[1] * inv, 0, false), true);
  } else {
    return __builtin_amdgcn_cvt_pk_bf8_f32(x[2] * inv, x[3] * inv, __builtin_amdgcn_cvt_pk_bf8_f32(x[0] * inv, x[1] * inv, 0, false), true);
  }
}

// round(code * old / s): the codes of a word under a larger scale, in fp64, where code * old and q * s are exact products
// of 32 bits and the quotient is too fine to be mistaken for a middle.  A code that is no number (a cache that somebody
// else wrote) becomes 0.
template <int kCode>
__device__ __forceinline__ uint32_t requantize4(uint32_t w, float old, float s) {
  if constexpr (kCode == kCodeI8) {
    uint32_t out = 0;
    const double ratio = static_cast<double>(old) / static_cast<double>(s), h = 0.5 * s;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const double v = static_cast<double>(code_to_f32<kCode>(w, k));
      double q = rint(v * ratio);
      const double r = v * old - q * s;
      const bool odd = (static_cast<int>(q) & 1) != 0;
      if (r > h || (r == h && odd)) q += 1.0;
      else if (r < -h || (r == -h && odd)) q -= 1.0;
      out |= (static_cast<uint32_t>(static_cast<int>(q)) & 0xffu) << (8 * k);
    }
    return out;
  } else {
    float y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) y[k] = off_the_middle(static_cast<double>(code_to_f32<kCode>(w, k)) * old / s);
    return pack4<kCode>(y, 1.f, 1.f);
  }
}

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), o)));
  return v;
}

// The scale a run of largest magnitude `a` asks for.
template <int kCode>
__device__ __forceinline__ float fresh_scale(float a) {
  if (!(a > 0.f)) return 0.f;
  if constexpr (kCode == kCodeI8) {
    return fmaxf(__fdiv_rn(a, 127.f), 0x1p-126f);
  } else {
    // qmax = 1.75 * 2^e_max: a = m * 2^e with m in [1, 2) asks for 2^(e - e_max), doubled if m > 1.75
    constexpr int e_max = kCode == kCodeE4m3 ? 8 : 15;
    const uint32_t u = __float_as_uint(a);
    const int e = static_cast<int>(u >> 23) - e_max + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return __uint_as_float(static_cast<uint32_t>(max(e, 1)) << 23);  // at least 2^-126
  }
}

// The scale of rows that were given: at least the block's old one (one that is no number counts as none).
template <int kCode>
__device__ __forceinline__ float next_scale(float a, float old) {
  const float want = fresh_scale<kCode>(a);
  return want > old ? want : old > 0.f ? old : want;
}

// Codes of a piece; `plain`: all of its elements are finite, under a scale that an update made.
template <int kCode, typename T>
__device__ __forceinline__ uint2 codes_of(const Piece<T>& x, float s, float inv, bool plain) {
  float y[kPiece];
  x.get(y);
  uint2 w = {0u, 0u};
  bool odd = !plain;
  if (plain) {
    w.x = pack4_finite<kCode>(y, s, inv, odd);
    w.y = pack4_finite<kCode>(y + 4, s, inv, odd);
  }
  if (odd) {
    w.x = pack4<kCode>(y, s, inv);
    w.y = pack4<kCode>(y + 4, s, inv);
  }
  return w;
}
template <int kCode>
__device__ __forceinline__ bool is_plain(bool finite, float s) {
  return finite && s > 0.f && (kCode == kCodeI8 || (__float_as_uint(s) & 0x7fffffu) == 0);
}

// Re-expresses the pieces lane, lane + lanes, ... < n in front of `rows` under a scale that has grown.
template <int kCode>
__device__ __forceinline__ void requantize(char* rows, int n, int lane, int lanes, float old, float s) {
  const float was = old > 0.f ? old : 0.f;
  for (int e = lane; e < n; e += lanes) {
    uint2* at = reinterpret_cast<uint2*>(rows + static_cast<size_t>(e) * kPiece);
    uint2 w = *at;
    w.x = requantize4<kCode>(w.x, was, s);
    w.y = requantize4<kCode>(w.y, was, s);
    *at = w;
  }
}

// 64 tokens of which no two are neighbours in a block (a decode step): a row of head_dim elements fills only a part of a
// wavefront, so that 64 / lanes rows are taken at once, `lanes` being the power of two that holds one.
template <int kCode, typename T>
__device__ __forceinline__ void update_single_rows(const RpaQuantUpdateParams& p, int page_shift, int block_shift, int slot, int worker, int workers) {
  const int lane = threadIdx.x & 63, heads = 2 * p.num_kv_heads, pieces = p.head_dim / kPiece, lane_bits = 32 - __clz(pieces - 1), lanes = 1 << lane_bits;
  const int piece = lane & (lanes - 1), units = min(kTokensPerChunk, p.total_tokens - static_cast<int>(blockIdx.x) * kTokensPerChunk) * heads;
  for (int unit0 = worker << (6 - lane_bits); unit0 < units; unit0 += workers << (6 - lane_bits)) {
    const int unit = min(unit0 + (lane >> lane_bits), units - 1), token = unit / heads, head = unit - token * heads, j = head >> 1;
    const int s0 = __shfl(slot, token);
    const bool real = s0 >= 0 && unit0 + (lane >> lane_bits) < units;
    const int page = real ? s0 >> page_shift : 0, off = s0 & ((1 << page_shift) - 1), inside = s0 & ((1 << block_shift) - 1);
    const int64_t t = static_cast<int64_t>(blockIdx.x) * kTokensPerChunk + token;
    const T* src = (head & 1) ? static_cast<const T*>(p.values) + t * p.value_token_stride + j * p.value_head_stride
                              : static_cast<const T*>(p.keys) + t * p.key_token_stride + j * p.key_head_stride;
    const size_t line = static_cast<size_t>(page) * heads + head;
    float* scale = p.kv_scales + (line << (page_shift - block_shift)) + (off >> block_shift);
    const float old = real && inside > 0 ? *scale : 0.f;
    Piece<T> x;
    x.load(src + (piece < pieces ? piece * kPiece : 0));  // lanes behind the row hold its first piece: no change to the maximum
    uint32_t most = x.top(0u);
    if constexpr (sizeof(T) == 2) most = max(most & 0xffff0000u, most << 16);
    uint32_t row_most = most;
    for (int o = lanes >> 1; o > 0; o >>= 1) row_most = max(row_most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(row_most), o)));
    const bool finite = row_most < 0x7f800000u;
    float a = __uint_as_float(row_most);
    if (__any(!finite)) {  // seldom: only the finite elements count
      float y[kPiece], b = 0.f;
      x.get(y);
#pragma unroll
      for (int c = 0; c < kPiece; ++c) b = fabsf(y[c]) < INFINITY ? fmaxf(b, fabsf(y[c])) : b;
      for (int o = lanes >> 1; o > 0; o >>= 1) b = fmaxf(b, __shfl_xor(b, o));
      a = b;
    }
    const float s = next_scale<kCode>(a, old), inv = s > 0.f ? 1.f / s : 0.f;
    if (!real) continue;
    char* dst = static_cast<char*>(p.kv_cache) + ((line << page_shift) + off) * p.head_dim;
    if (piece < pieces) *reinterpret_cast<uint2*>(dst + piece * kPiece) = codes_of<kCode>(x, s, inv, is_plain<kCode>(finite, s));
    if (inside > 0 && s != old) requantize<kCode>(dst - static_cast<size_t>(inside) * p.head_dim, inside * pieces, piece, lanes, old, s);
    if (piece == 0 && (inside == 0 || s != old)) *scale = s;
  }
}

template <int kCode, typename T>
__global__ __launch_bounds__(256) void quant_update_kernel(RpaQuantUpdateParams p, int page_shift, int block_shift) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t pool = static_cast<int64_t>(p.num_pages) << page_shift;
  const int t = blockIdx.x * kTokensPerChunk + lane;
  const int block_mask = (1 << block_shift) - 1;
  // run starts among this chunk's 64 tokens
  int slot = -1, before = -1;
  if (t < p.total_tokens) {
    slot = p.slot_mapping[t];
    if (slot >= pool) slot = -1;
    if (t > 0) before = p.slot_mapping[t - 1];
  }
  const bool follows = slot >= 0 && before >= 0 && before == slot - 1 && (slot & block_mask) != 0;
  uint64_t mask = __ballot(slot >= 0 && !follows);
  const uint64_t follow = __ballot(follows);
  const int runs = __popcll(mask), heads = 2 * p.num_kv_heads;
  const int pieces = p.head_dim / kPiece, step_rows = 64 / pieces, step_pieces = 64 - step_rows * pieces;
  const int row0 = lane / pieces, piece0 = lane - row0 * pieces;  // this lane's first piece; the next one lies 64 pieces on
  const int worker = blockIdx.y * (blockDim.x >> 6) + wave, workers = gridDim.y * (blockDim.x >> 6);
  const int behind_chunk = (blockIdx.x + 1) * kTokensPerChunk;
  if (follow == 0) {
    const int last = __builtin_amdgcn_readlane(slot, 63);
    if (last < 0 || behind_chunk >= p.total_tokens || p.slot_mapping[behind_chunk] != last + 1 || ((last + 1) & block_mask) == 0) {
      update_single_rows<kCode, T>(p, page_shift, block_shift, slot, worker, workers);
      return;
    }
  }
  int at_run = 0;
  for (int64_t unit = worker; unit < static_cast<int64_t>(runs) * heads; unit += workers) {
    const int run = static_cast<int>(unit) / heads, head = static_cast<int>(unit) - run * heads;
    for (; at_run < run; ++at_run) mask &= mask - 1;  // the runs come in order
    const int src_lane = __ffsll(static_cast<unsigned long long>(mask)) - 1;
    const int t0 = blockIdx.x * kTokensPerChunk + src_lane;
    const int s0 = __builtin_amdgcn_readlane(slot, src_lane);
    const int inside = s0 & block_mask;
    // Length of the run: the tokens that follow in this chunk, and if it reaches the chunk's end, those behind it.
    const uint64_t behind = src_lane == 63 ? 0 : follow >> (src_lane + 1);
    int n = __ffsll(static_cast<unsigned long long>(~behind));
    if (src_lane + n == 64) {
      const int most = min((1 << block_shift) - inside, p.total_tokens - t0);
      while (n < most) {
        const int k = n + lane;
        const uint64_t b = __ballot(k < most && p.slot_mapping[t0 + min(k, most - 1)] == s0 + k);
        const int more = b == ~0ull ? 64 : __ffsll(static_cast<unsigned long long>(~b)) - 1;
        n += more;
        if (more < 64) break;
      }
    }
    const int j = head >> 1;
    const T* __restrict__ src = (head & 1) ? static_cast<const T*>(p.values) + t0 * p.value_token_stride + j * p.value_head_stride
                                           : static_cast<const T*>(p.keys) + t0 * p.key_token_stride + j * p.key_head_stride;
    const int64_t stride = (head & 1) ? p.value_token_stride : p.key_token_stride;
    const int page = s0 >> page_shift, off = s0 & ((1 << page_shift) - 1);
    const size_t first_row = ((static_cast<size_t>(page) * heads + head) << page_shift) + off;
    float* scale = p.kv_scales + ((static_cast<size_t>(page) * heads + head) << (page_shift - block_shift)) + (off >> block_shift);
    const float old = inside > 0 ? *scale : 0.f;

    // Batches of kBatch pieces a lane, all in flight at once; most runs are one batch.
    const int total = n * pieces;
    Piece<T> x[kBatch];
    uint32_t most = 0;
    int row = row0, piece = piece0;
    for (int e0 = 0; e0 < total; e0 += 64 * kBatch) {
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        if (e0 + 64 * k >= total) break;
        const bool real = e0 + 64 * k + lane < total;
        x[k].load(src + (real ? row * stride + piece * kPiece : 0));
        row += step_rows, piece += step_pieces;
        if (piece >= pieces) piece -= pieces, ++row;
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        if (e0 + 64 * k >= total) break;
        most = x[k].top(most);  // a lane behind the last piece holds the first one: it does not change the maximum
      }
    }
    if constexpr (sizeof(T) == 2) most = max(most & 0xffff0000u, most << 16);
    most = wave_max_u32(most);
    const bool finite = most < 0x7f800000u;
    float a = __uint_as_float(most);
    if (!finite) {  // seldom: only the finite elements count
      a = 0.f;
      row = row0, piece = piece0;
#pragma unroll 1
      for (int e = lane; e < total; e += 64) {
        Piece<T> one;
        one.load(src + row * stride + piece * kPiece);
        float y[kPiece];
        one.get(y);
#pragma unroll
        for (int c = 0; c < kPiece; ++c) a = fabsf(y[c]) < INFINITY ? fmaxf(a, fabsf(y[c])) : a;
        row += step_rows, piece += step_pieces;
        if (piece >= pieces) piece -= pieces, ++row;
      }
      a = wave_max(a);
    }
    const float s = next_scale<kCode>(a, old), inv = s > 0.f ? 1.f / s : 0.f;
    const bool plain = is_plain<kCode>(finite, s);
    char* dst = static_cast<char*>(p.kv_cache) + first_row * p.head_dim;
    row = row0, piece = piece0;
    for (int e0 = 0; e0 < total; e0 += 64 * kBatch) {
      if (total > 64 * kBatch) {
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          if (e0 + 64 * k >= total) break;
          const bool real = e0 + 64 * k + lane < total;
          x[k].load(src + (real ? row * stride + piece * kPiece : 0));
          row += step_rows, piece += step_pieces;
          if (piece >= pieces) piece -= pieces, ++row;
        }
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int e = e0 + 64 * k + lane;
        if (e0 + 64 * k >= total) break;
        const uint2 w = codes_of<kCode>(x[k], s, inv, plain);
        if (e < total) *reinterpret_cast<uint2*>(dst + static_cast<size_t>(e) * kPiece) = w;  // the rows of a block lie together
      }
    }
    if (inside > 0 && s != old) requantize<kCode>(dst - static_cast<size_t>(inside) * p.head_dim, inside * pieces, lane, 64, old, s);
    if (lane == 0 && (inside == 0 || s != old)) *scale = s;
  }
}

// Read-back: a lane takes eight elements of kGatherRows rows, whose loads are in flight together.  What bounds it is the
// traffic, two thirds of it stores that nobody reads out of the L2 in time, so they are not kept there: 32768 tokens of 8
// heads of 128 (202 MB) take 30 us; 41 us with stores that stay, 48 us with one row and either.
constexpr int kGatherRows = 2;
template <int kCode, typename T>
__global__ __launch_bounds__(256) void quant_gather_kernel(RpaQuantGatherParams p, int page_shift, int block_shift) {
  const int64_t pool = static_cast<int64_t>(p.num_pages) << page_shift;
  const int heads = 2 * p.num_kv_heads, pieces = p.head_dim / kPiece;
  const int t0 = blockIdx.x * kGatherRows;
  int slot[kGatherRows];
#pragma unroll
  for (int r = 0; r < kGatherRows; ++r) slot[r] = p.slot_mapping[min(t0 + r, p.total_tokens - 1)];
  for (int e = threadIdx.x; e < heads * pieces; e += blockDim.x) {
    const int head = e / pieces, piece = e - head * pieces;
    uint2 w[kGatherRows];
    float s[kGatherRows];
#pragma unroll
    for (int r = 0; r < kGatherRows; ++r) {
      const bool real = slot[r] >= 0 && slot[r] < pool;
      const int at = real ? slot[r] : 0, off = at & ((1 << page_shift) - 1);
      const size_t line = static_cast<size_t>(at >> page_shift) * heads + head;
      w[r] = *reinterpret_cast<const uint2*>(static_cast<const char*>(p.kv_cache) + ((line << page_shift) + off) * p.head_dim + piece * kPiece);
      s[r] = p.kv_scales[(line << (page_shift - block_shift)) + (off >> block_shift)];
    }
#pragma unroll
    for (int r = 0; r < kGatherRows; ++r) {
      if (t0 + r >= p.total_tokens) break;
      const bool real = slot[r] >= 0 && slot[r] < pool;
      float y[kPiece];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        y[k] = real ? code_to_f32<kCode>(w[r].x, k) * s[r] : 0.f;
        y[4 + k] = real ? code_to_f32<kCode>(w[r].y, k) * s[r] : 0.f;
      }
      T* dst = static_cast<T*>((head & 1) ? p.values : p.keys) + (static_cast<size_t>(t0 + r) * p.num_kv_heads + (head >> 1)) * p.head_dim + piece * kPiece;
      u32x4_t* out = reinterpret_cast<u32x4_t*>(dst);
      if constexpr (sizeof(T) == 4) {
        __builtin_nontemporal_store(u32x4_t{__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]), __float_as_uint(y[3])}, out);
        __builtin_nontemporal_store(u32x4_t{__float_as_uint(y[4]), __float_as_uint(y[5]), __float_as_uint(y[6]), __float_as_uint(y[7])}, out + 1);
      } else {
        u32x4_t u;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          bf16x2_t b;
          b[0] = static_cast<__bf16>(y[2 * k]);
          b[1] = static_cast<__bf16>(y[2 * k + 1]);
          u[k] = __builtin_bit_cast(uint32_t, b);
        }
        __builtin_nontemporal_store(u, out);
      }
    }
  }
}

template <typename F>
void by_types(int cache_dtype, int dtype, F&& f) {
  auto with = [&](auto code) {
    if (dtype == RPA_DTYPE_F32) f(code, float{});
    else f(code, bf16_t{});
  };
  switch (code_of_dtype(cache_dtype)) {
    case kCodeI8: with(std::integral_constant<int, kCodeI8>{}); break;
    case kCodeE4m3: with(std::integral_constant<int, kCodeE4m3>{}); break;
    default: with(std::integral_constant<int, kCodeE5m2>{}); break;
  }
}

}  // namespace

int launch_quant_update(const RpaQuantUpdateParams& p, hipStream_t stream) {
  if (p.total_tokens == 0) return RPA_OK;
  const int chunks = (p.total_tokens + kTokensPerChunk - 1) / kTokensPerChunk;
  // Enough lanes for all rows of a chunk at once where every token is a run of its own (a decode step), and 4096 workgroups
  // at most where the runs are longer and fewer than the tokens.
  int lanes = 1;
  while (lanes * kPiece < p.head_dim) lanes *= 2;
  const int most = (2 * p.num_kv_heads * kTokensPerChunk * lanes + 255) / 256;
  const int per_chunk = std::max(1, std::min(most, 4096 / chunks));
  by_types(p.cache_dtype, p.dtype, [&](auto code, auto t) {
    hipLaunchKernelGGL((quant_update_kernel<decltype(code)::value, decltype(t)>), dim3(chunks, per_chunk), dim3(256), 0, stream, p,
                       __builtin_ctz(p.page_size), __builtin_ctz(p.scale_block));
  });
  return hipGetLastError() == hipSuccess ? RPA_OK : RPA_ERR_LAUNCH;
}

int launch_quant_gather(const RpaQuantGatherParams& p, hipStream_t stream) {
  if (p.total_tokens == 0) return RPA_OK;
  by_types(p.cache_dtype, p.dtype, [&](auto code, auto t) {
    hipLaunchKernelGGL((quant_gather_kernel<decltype(code)::value, decltype(t)>), dim3((p.total_tokens + kGatherRows - 1) / kGatherRows), dim3(256), 0, stream, p,
                       __builtin_ctz(p.page_size), __builtin_ctz(p.scale_block));
  });
  return hipGetLastError() == hipSuccess ? RPA_OK : RPA_ERR_LAUNCH;
}

}  // namespace rpa
