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

constexpr int kThreads = 1024;

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
__device__ __forceinline__ Pair block_prefix(Pair v, Pair* lds, Pair* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Pair inc = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t a = __shfl_up(inc.a, o), b = __shfl_up(inc.b, o);
    if (lane >= o) inc.a += a, inc.b += b;
  }
  __syncthreads();  // lds may still be read from the call before
  if (lane == 63) lds[wave] = inc;
  __syncthreads();
  Pair base = {0, 0}, all = {0, 0};
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
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

__device__ __forceinline__ int ring_place(int64_t i, int cap) { return static_cast<int>(i % cap); }

// Table entries of request s: taken pages behind those it holds, given pages into the ring.  The places written lie
// behind the ring's free pages, those read among them.
__device__ __forceinline__ void move_pages(const RpaBlockTablesParams& p, const Move& m, int have, int s, int first, int step) {
  int32_t* row = p.block_tables + static_cast<size_t>(s) * p.pages_per_seq;
  for (int k = first; k < m.taken; k += step) row[have + k] = p.free_pages[ring_place(static_cast<int64_t>(m.from) + k, p.num_free_slots)];
  for (int k = first; k < m.given; k += step) p.free_pages[ring_place(static_cast<int64_t>(m.to) + k, p.num_free_slots)] = row[k];
}

// Slot and position of flat token t.  `start` are the query starts (n_all + 1 of them).
__device__ __forceinline__ void map_token(const RpaBlockTablesParams& p, const int32_t* start, const Move* moves, int n, int t) {
  int slot = -1, pos = -1;
  const int n_all = p.max_num_seqs;
  if (t < start[n_all]) {
    int lo = 0, hi = n_all;  // last s with start[s] <= t: it holds t, since start[s + 1] > t
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (start[mid] <= t) lo = mid;
      else hi = mid;
    }
    const int s = lo;
    if (p.admitted[s]) {
      const Request r = request(p, n, s);
      pos = r.cached + (t - start[s]);
      const int j = pos / p.page_size;
      const int page = j < r.have ? p.block_tables[static_cast<size_t>(s) * p.pages_per_seq + j]
                                  : p.free_pages[ring_place(static_cast<int64_t>(moves[s].from) + (j - r.have), p.num_free_slots)];
      slot = static_cast<int>(static_cast<int64_t>(page) * p.page_size + (pos - j * p.page_size));
    }
  }
  p.slot_mapping[t] = slot;
  p.positions[t] = pos;
}

__device__ __forceinline__ int clipped_count(const RpaBlockTablesParams& p) { return min(max(p.num_seqs[0], 0), p.max_num_seqs); }

__global__ __launch_bounds__(kThreads) void block_tables_plan_kernel(RpaBlockTablesParams p, int write_entries) {
  __shared__ Pair lds[kThreads / 64];
  const int n_all = p.max_num_seqs, n = clipped_count(p), cap = p.num_free_slots;
  const int per = (n_all + kThreads - 1) / kThreads;
  const int s0 = min(static_cast<int64_t>(threadIdx.x) * per, static_cast<int64_t>(n_all)), s1 = min(s0 + per, n_all);
  const int2 ring = ring_state(p);
  Move* moves = reinterpret_cast<Move*>(p.scratch);

  Pair sum = {0, 0}, total;
  for (int s = s0; s < s1; ++s) {
    const Request r = request(p, n, s);
    sum.a += max(r.q, 0);
    sum.b += r.q < 0 ? r.have : 0;
  }
  const Pair at = block_prefix(sum, lds, &total);  // first token and first page given back of this thread's requests
  sum = {0, 0};
  int64_t end = at.a;
  for (int s = s0; s < s1; ++s) {
    const Request r = request(p, n, s);
    end += max(r.q, 0);
    sum.a += fits(p, r, end) ? need_of(p, r) : 0;
  }
  const Pair taken = block_prefix(sum, lds, &total);
  Pair moved = {0, 0};  // pages taken and given back
  int64_t start = at.a, back = at.b, need = taken.a;
  for (int s = s0; s < s1; ++s) {
    const Request r = request(p, n, s);
    end = start + max(r.q, 0);
    const bool ok = fits(p, r, end);
    const int want = ok ? need_of(p, r) : 0, gives = r.q < 0 ? r.have : 0;
    const bool in = r.q == 0 || (ok && (want == 0 || need + want <= ring.y));
    const bool out = r.q < 0 && ring.y + back + gives <= cap;  // a ring that cannot hold them: the request stays
    p.query_start_loc[s] = static_cast<int>(min(start, static_cast<int64_t>(p.total_tokens)));
    p.context_lens[s] = in ? r.cached + r.q : 0;
    p.admitted[s] = in ? 1 : 0;
    p.cached_lens_out[s] = s >= n ? p.cached_lens[s] : in ? r.cached + r.q : out ? 0 : r.cached;
    Move m;
    m.taken = in ? want : 0;
    m.from = ring_place(ring.x + min(need, static_cast<int64_t>(cap)), cap);
    m.given = out ? gives : 0;
    m.to = ring_place(ring.x + ring.y + min(back, static_cast<int64_t>(cap)), cap);
    moves[s] = m;
    moved.a += m.taken;
    moved.b += m.given;
    start = end;
    need += want;
    back += gives;
  }
  block_prefix(moved, lds, &total);
  if (s0 < n_all && s1 == n_all) p.query_start_loc[n_all] = static_cast<int>(min(start, static_cast<int64_t>(p.total_tokens)));
  if (threadIdx.x == 0) {
    p.free_state_out[0] = ring_place(ring.x + total.a, cap);
    p.free_state_out[1] = static_cast<int>(ring.y - total.a + total.b);
  }
  if (!write_entries) return;
  __syncthreads();
  const int lane = threadIdx.x & 63;
  for (int s = threadIdx.x >> 6; s < n; s += kThreads / 64) move_pages(p, moves[s], request(p, n, s).have, s, lane, 64);
  for (int t = threadIdx.x; t < p.total_tokens; t += kThreads) map_token(p, p.query_start_loc, moves, n, t);
}

__global__ __launch_bounds__(256) void block_tables_entries_kernel(RpaBlockTablesParams p, int token_groups) {
  const int n = clipped_count(p);
  const Move* moves = reinterpret_cast<const Move*>(p.scratch);
  if (static_cast<int>(blockIdx.x) < token_groups) {
    const int t = blockIdx.x * 256 + threadIdx.x;
    if (t < p.total_tokens) map_token(p, p.query_start_loc, moves, n, t);
  } else {
    const int s = (blockIdx.x - token_groups) * 4 + (threadIdx.x >> 6);
    if (s < n) move_pages(p, moves[s], request(p, n, s).have, s, threadIdx.x & 63, 64);
  }
}

}  // namespace

int launch_block_tables(const RpaBlockTablesParams& p, hipStream_t stream) {
  const bool few = p.max_num_seqs <= kThreads && p.total_tokens <= 4 * kThreads;
  hipLaunchKernelGGL(block_tables_plan_kernel, dim3(1), dim3(kThreads), 0, stream, p, few ? 1 : 0);
  if (hipGetLastError() != hipSuccess) return RPA_ERR_LAUNCH;
  if (few) return RPA_OK;
  const int token_groups = (p.total_tokens + 255) / 256, seq_groups = (p.max_num_seqs + 3) / 4;
  hipLaunchKernelGGL(block_tables_entries_kernel, dim3(token_groups + seq_groups), dim3(256), 0, stream, p, token_groups);
  return hipGetLastError() == hipSuccess ? RPA_OK : RPA_ERR_LAUNCH;
}

}  // namespace rpa
