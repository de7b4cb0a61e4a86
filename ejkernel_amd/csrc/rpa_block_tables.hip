// Block tables and slot maps from request lengths: one step of a paged cache's bookkeeping.
//
// Three prefix sums over the requests -- query tokens, pages needed, pages given back -- decide who is admitted and
// which places of the ring of free pages each request takes from and gives to; after them every table entry and every
// token's slot stands alone.  The sums are taken by one workgroup (a few thousand lengths: what bounds it is the latency
// of its loads and barriers); the entries are written by the same workgroup where they are few, by a second launch over
// the device where they are many.
#include "rpa_device.h"
#include "rpa_host.h"

namespace rpa {

namespace {

constexpr int kThreads = 1024, kFewThreads = 256;

struct Request {
  int q;       // new tokens, negative: ended
  int cached;  // tokens in the cache, within what the table can hold
  int have;    // pages it holds
};

__device__ __forceinline__ int pages_of(int tokens, int page_size) { return tokens / page_size + (tokens % page_size != 0 ? 1 : 0); }

__device__ __forceinline__ Request request(const RpaBlockTablesParams& p, int n, int s) {
  Request r;
  const int64_t room = static_cast<int64_t>(p.pages_per_seq) * p.page_size;
  const int cap = room > 0x7fffffff ? 0x7fffffff : static_cast<int>(room);
  r.q = s < n ? p.query_lens[s] : 0;
  r.cached = s < n ? min(max(p.cached_lens[s], 0), cap) : 0;
  r.have = pages_of(r.cached, p.page_size);
  return r;
}

// Pages request r takes if its new tokens run: `end` = its last token's place in the flat batch.
__device__ __forceinline__ bool fits(const RpaBlockTablesParams& p, const Request& r, int64_t end) {
  return r.q >= 0 && static_cast<int64_t>(r.cached) + r.q <= static_cast<int64_t>(p.pages_per_seq) * p.page_size && end <= p.total_tokens;
}
__device__ __forceinline__ int need_of(const RpaBlockTablesParams& p, const Request& r) {
  return r.q > 0 ? pages_of(r.cached + r.q, p.page_size) - r.have : 0;
}

// Exclusive prefix sums of two values over the workgroup; `total` gets the sums.
struct Pair {
  int64_t a, b;
};
template <int kWaves>
__device__ __forceinline__ Pair block_prefix(Pair v, Pair* lds, Pair* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Pair inc = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t a = __shfl_up(inc.a, o), b = __shfl_up(inc.b, o);
    if (lane >= o) inc.a += a, inc.b += b;
  }
  if (lane == 63) lds[wave] = inc;
  __syncthreads();
  Pair base = {0, 0}, all = {0, 0};
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const Pair x = lds[w];
    if (w < wave) base.a += x.a, base.b += x.b;
    all.a += x.a, all.b += x.b;
  }
  *total = all;
  return {base.a + inc.a - v.a, base.b + inc.b - v.b};
}

// What the entries' writers need of a request besides its lengths, four words of scratch: pages taken and their place
// in the ring, pages given back and theirs.
struct Move {
  int taken, from, given, to;
};

// Ring state {head, count} as the kernels use it.
__device__ __forceinline__ int2 ring_state(const RpaBlockTablesParams& p) {
  const int cap = p.num_free_slots;
  int head = p.free_state[0] % cap;
  head += head < 0 ? cap : 0;
  return make_int2(head, min(max(p.free_state[1], 0), cap));
}

// Place i of the ring, i below twice its size.
__device__ __forceinline__ int ring_place(int64_t i, int cap) { return static_cast<int>(i >= cap ? i - cap : i); }

// Table entries of request s: taken pages behind those it holds, given pages into the ring.  The places written lie
// behind the ring's free pages, those read among them.
__device__ __forceinline__ void move_pages(const RpaBlockTablesParams& p, const Move& m, int have, int s, int first, int step) {
  int32_t* row = p.block_tables + static_cast<size_t>(s) * p.pages_per_seq;
  for (int k = first; k < m.taken; k += step) row[have + k] = p.free_pages[ring_place(static_cast<int64_t>(m.from) + k, p.num_free_slots)];
  for (int k = first; k < m.given; k += step) p.free_pages[ring_place(static_cast<int64_t>(m.to) + k, p.num_free_slots)] = row[k];
}

// Last s with start[s] <= t of n_all + 1 starts: it holds t where t lies in front of the last of them.
__device__ __forceinline__ int sequence_of(const int32_t* start, int n_all, int t) {
  int lo = 0, hi = n_all;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Slot of position pos of request s, which held `have` pages before this step and takes others from place `from` of the
// ring on.  The page is read where it lay before the step, so it does not matter who has moved already.
__device__ __forceinline__ int slot_of(const RpaBlockTablesParams& p, int s, int pos, int have, int from) {
  const int j = pos / p.page_size;
  const int page = j < have ? p.block_tables[static_cast<size_t>(s) * p.pages_per_seq + j]
                            : p.free_pages[ring_place(static_cast<int64_t>(from) + (j - have), p.num_free_slots)];
  return static_cast<int>(static_cast<int64_t>(page) * p.page_size + (pos - j * p.page_size));
}

__device__ __forceinline__ int clipped_count(const RpaBlockTablesParams& p) { return min(max(p.num_seqs[0], 0), p.max_num_seqs); }

// What the slots need of the requests, where a thread has one at most.
template <int kN>
struct FewLds {
  int start[kN + 1], cached[kN], from[kN];  // cached: -1 where the request's tokens do not run
};

// kPer: requests that a thread keeps in registers, all loaded at once; 0: as many as there are, loaded for every pass.
template <int kN, int kPer>
__global__ __launch_bounds__(kN) void block_tables_plan_kernel(RpaBlockTablesParams p, int write_entries) {
  constexpr int kWaves = kN / 64;
  __shared__ Pair lds[3][kWaves];
  __shared__ FewLds<kN> few;
  const int n_all = p.max_num_seqs, cap = p.num_free_slots, lane = threadIdx.x & 63;
  const int per = (n_all + kN - 1) / kN;
  const int s0 = static_cast<int>(min(static_cast<int64_t>(threadIdx.x) * per, static_cast<int64_t>(n_all))), s1 = min(s0 + per, n_all);
  const int n = clipped_count(p);
  const int2 ring = ring_state(p);
  Move* moves = reinterpret_cast<Move*>(p.scratch);
  Request kept[kPer > 0 ? kPer : 1];
#pragma unroll
  for (int k = 0; k < kPer; ++k) kept[k] = request(p, n, min(s0 + k, n_all - 1));
  const auto each = [&](auto&& f) {
    if constexpr (kPer > 0) {
#pragma unroll
      for (int k = 0; k < kPer; ++k)
        if (s0 + k < s1) f(s0 + k, kept[k]);
    } else {
      for (int s = s0; s < s1; ++s) f(s, request(p, n, s));
    }
  };

  Pair sum = {0, 0}, total;
  each([&](int, const Request& r) {
    sum.a += max(r.q, 0);
    sum.b += r.q < 0 ? r.have : 0;
  });
  const Pair at = block_prefix<kWaves>(sum, lds[0], &total);  // first token and first page given back of this thread's requests
  sum = {0, 0};
  int64_t end = at.a;
  each([&](int, const Request& r) {
    end += max(r.q, 0);
    sum.a += fits(p, r, end) ? need_of(p, r) : 0;
  });
  const Pair taken = block_prefix<kWaves>(sum, lds[1], &total);
  Pair last = {0, 0};  // behind the last page taken and given back: whoever does not fit, nobody behind it does
  int64_t start = at.a, back = at.b, need = taken.a;
  Move m = {0, 0, 0, 0};
  int first_token = 0, cached = -1;
  each([&](int s, const Request& r) {
    end = start + max(r.q, 0);
    const bool ok = fits(p, r, end);
    const int want = ok ? need_of(p, r) : 0, gives = r.q < 0 ? r.have : 0;
    const bool in = r.q == 0 || (ok && (want == 0 || need + want <= ring.y));
    const bool out = r.q < 0 && ring.y + back + gives <= cap;  // a ring that cannot hold them: the request stays
    first_token = static_cast<int>(min(start, static_cast<int64_t>(p.total_tokens)));
    cached = in && r.q > 0 ? r.cached : -1;
    p.query_start_loc[s] = first_token;
    p.context_lens[s] = in ? r.cached + r.q : 0;
    p.admitted[s] = in ? 1 : 0;
    p.cached_lens_out[s] = s >= n ? p.cached_lens[s] : in ? r.cached + r.q : out ? 0 : r.cached;
    m.taken = in ? want : 0;
    m.from = ring_place(ring.x + min(need, static_cast<int64_t>(cap)), cap);
    m.given = out ? gives : 0;
    m.to = ring_place(ring.x + ring.y + min(back, static_cast<int64_t>(cap)), cap);
    if (!write_entries) moves[s] = m;
    start = end;
    need += want;
    back += gives;
    if (m.taken > 0) last.a = need;
    if (m.given > 0) last.b = back;
  });
  const int behind_last = static_cast<int>(min(start, static_cast<int64_t>(p.total_tokens)));
  if (s0 < n_all && s1 == n_all) p.query_start_loc[n_all] = behind_last;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    last.a = max(last.a, __shfl_xor(last.a, o));
    last.b = max(last.b, __shfl_xor(last.b, o));
  }
  if (lane == 0) lds[2][threadIdx.x >> 6] = last;
  const int s = threadIdx.x;
  if (write_entries && s < n_all) {
    few.start[s] = first_token;
    few.cached[s] = cached;
    few.from[s] = m.from;
    if (s == n_all - 1) few.start[n_all] = behind_last;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 0; w < kWaves; ++w) last.a = max(last.a, lds[2][w].a), last.b = max(last.b, lds[2][w].b);
    p.free_state_out[0] = ring_place(ring.x + last.a, cap);
    p.free_state_out[1] = static_cast<int>(ring.y - last.a + last.b);
  }
  if (!write_entries) return;  // else: a thread has one request at most
  const int have = kept[0].have;
  // Pages: one for most requests of a decode step, which its thread moves; longer moves by the wavefront, one after another.
  if (m.taken == 1) p.block_tables[static_cast<size_t>(s) * p.pages_per_seq + have] = p.free_pages[m.from];
  for (uint64_t long_moves = __ballot(m.taken > 1 || m.given > 0); long_moves != 0; long_moves &= long_moves - 1) {
    const int l = __ffsll(static_cast<unsigned long long>(long_moves)) - 1;
    const Move w = {__builtin_amdgcn_readlane(m.taken, l), __builtin_amdgcn_readlane(m.from, l), __builtin_amdgcn_readlane(m.given, l),
                    __builtin_amdgcn_readlane(m.to, l)};
    move_pages(p, w, __builtin_amdgcn_readlane(have, l), __builtin_amdgcn_readlane(s, l), lane, 64);
  }
  for (int t = threadIdx.x; t < p.total_tokens; t += kN) {
    int slot = -1, pos = -1;
    if (t < few.start[n_all]) {
      const int s = sequence_of(few.start, n_all, t), cached = few.cached[s];
      if (cached >= 0) {
        pos = cached + (t - few.start[s]);
        slot = slot_of(p, s, pos, pages_of(cached, p.page_size), few.from[s]);
      }
    }
    p.slot_mapping[t] = slot;
    p.positions[t] = pos;
  }
}

// 256 tokens or the pages of four requests a workgroup.  The tokens' request is looked for among the 256 behind the first
// token's, which is found 64 at a time, and beyond them (256 idle requests in a row) in memory: 11 dependent loads for 2048
// requests become three.
__global__ __launch_bounds__(256) void block_tables_entries_kernel(RpaBlockTablesParams p, int token_groups) {
  constexpr int kNear = 256;
  __shared__ int near_start[kNear + 1];
  const int n = clipped_count(p), n_all = p.max_num_seqs, lane = threadIdx.x & 63;
  const Move* moves = reinterpret_cast<const Move*>(p.scratch);
  const int32_t* start = p.query_start_loc;
  if (static_cast<int>(blockIdx.x) >= token_groups) {
    const int s = (blockIdx.x - token_groups) * 4 + (threadIdx.x >> 6);
    if (s < n) move_pages(p, moves[s], request(p, n, s).have, s, lane, 64);
    return;
  }
  const int t0 = blockIdx.x * 256, t = t0 + threadIdx.x;
  int first = 0;  // the last s with start[s] <= t0; starts do not decrease
  for (int span = n_all; span > 1;) {
    const int step = (span + 63) >> 6, k = lane * step;
    const int before = __popcll(__ballot(k < span && start[first + min(k, span - 1)] <= t0)) - 1;
    first += before * step;
    span = min(step, span - before * step);
  }
  for (int k = threadIdx.x; k <= kNear; k += 256) near_start[k] = start[min(first + k, n_all)];
  __syncthreads();
  if (t >= p.total_tokens) return;
  int slot = -1, pos = -1;
  if (t < start[n_all]) {
    const int most = min(kNear, n_all - first);
    const int s = first + (near_start[most] <= t && first + most < n_all ? most + sequence_of(start + first + most, n_all - first - most, t)
                                                                        : sequence_of(near_start, most, t));
    if (p.admitted[s]) {
      const Request r = request(p, n, s);
      pos = r.cached + (t - start[s]);
      slot = slot_of(p, s, pos, r.have, moves[s].from);
    }
  }
  p.slot_mapping[t] = slot;
  p.positions[t] = pos;
}

}  // namespace

int launch_block_tables(const RpaBlockTablesParams& p, hipStream_t stream) {
  // The sums take one workgroup: a small one is through its barriers sooner.  It also writes the entries where a thread has
  // one request and a few tokens.
  const bool few = p.max_num_seqs <= kThreads && p.total_tokens <= 4 * kThreads;
  const bool fewer = p.max_num_seqs <= kFewThreads && p.total_tokens <= 4 * kFewThreads;
  if (fewer) hipLaunchKernelGGL((block_tables_plan_kernel<kFewThreads, 1>), dim3(1), dim3(kFewThreads), 0, stream, p, 1);
  else if (p.max_num_seqs <= kThreads) hipLaunchKernelGGL((block_tables_plan_kernel<kThreads, 1>), dim3(1), dim3(kThreads), 0, stream, p, few ? 1 : 0);
  else if (p.max_num_seqs <= 4 * kThreads) hipLaunchKernelGGL((block_tables_plan_kernel<kThreads, 4>), dim3(1), dim3(kThreads), 0, stream, p, 0);
  else hipLaunchKernelGGL((block_tables_plan_kernel<kThreads, 0>), dim3(1), dim3(kThreads), 0, stream, p, 0);
  if (hipGetLastError() != hipSuccess) return RPA_ERR_LAUNCH;
  if (few) return RPA_OK;
  const int token_groups = (p.total_tokens + 255) / 256, seq_groups = (p.max_num_seqs + 3) / 4;
  hipLaunchKernelGGL(block_tables_entries_kernel, dim3(token_groups + seq_groups), dim3(256), 0, stream, p, token_groups);
  return hipGetLastError() == hipSuccess ? RPA_OK : RPA_ERR_LAUNCH;
}

}  // namespace rpa
