// Block tables and slot maps of a paged token pool, built on the GPU from the requests'
// lengths: the device form of what a serving engine does per forward with
// TokenToKVPoolAllocator.alloc and ReqToTokenPool (reference src/qwenquest/memory.py:28-76).
//
// A block is 64 consecutive pool rows; block 0 is padding.  Request r holds held[r] blocks,
// table[r, 0 .. held[r]).  The free blocks are a stack, free[0 .. count).  A call gives request
// i, which is to hold tokens 0 .. prefix_i + n_i,
//   need_i = max(0, ceil((prefix_i + n_i) / 64) - held_i)
// blocks from the stack's top, in request order, and writes for its token t (position
// p = prefix_i + t)
//   row = table[r, p / 64] * 64 + p % 64,   position = p,   req_to_token[r, p] = row.
// Asked again with the same lengths it takes nothing and answers the same.
//
// assign_plan_kernel: one block; a thread per request (a loop over more), two block-wide
// prefix sums (tokens, blocks).  All requests are judged before anything is written, so a
// refused call leaves the pool as it was and answers the padding row.  Up to a request per
// thread, what the judging read stays in registers.  assign_fill_kernel:
// a thread per token and per new block, each finding its request by bisection of the
// prefix sums; a thread per token writes 20 bytes, coalesced.
// Bound: launches and the latency of dependent loads at decode sizes, the 20 bytes a token
// of the slot map at prompts.  Measured: a decode batch of 64 requests is one launch of 4.2 us
// (12 us a call with the host's part); 16 prompts of 362945 tokens in all 3.0 + 6.0 us to assign
// and 3.2 + 5.4 to release.
#include "qq_fp8.h"

namespace qq {
namespace {

constexpr int kPlan = 1024;      // threads of the planning block, at most
constexpr int kErrExhausted = 1, kErrRequest = 2, kErrTwice = 4, kErrTotal = 8, kErrKinds = 4;
constexpr int kMaxPoolReqs = 1 << 18;  // the planning block's bitmap of requests: 32 KiB

// What the planning block hands to the fill: a header, then a record per request.
struct PlanHead {
  int32_t ok, count, tokens, blocks;  // count: the stack's height before the call
  int32_t pad[4];
};
struct PlanRow {
  int32_t tok, blk;   // tokens and blocks of the requests before this one
  int32_t req, prefix, held;
  int32_t pad[3];
};

struct BlockArgs {
  const int64_t* rpi;
  const int64_t* prefix;  // decode: the context's length, the new token included
  const int64_t* fresh;   // new tokens, or nullptr: decode, one at the context's end
  int bs;
  int64_t total;
  int32_t* table;
  int64_t table_stride;
  int32_t* r2t;
  int64_t r2t_stride, width;
  int reqs;
  int32_t* held;
  int32_t* stack;
  int32_t* count;
  int64_t cap;  // entries of the stack
  int64_t* loc;
  int64_t* pos;
  int32_t* err;         // [kErrKinds] refused calls
  int32_t* err_mirror;  // the same in host memory, or nullptr
  PlanHead* head;
  PlanRow* rows;
  int here;  // the planning block writes the slots itself
};

struct PlanSmem {
  int64_t a[kPlan / 64], b[kPlan / 64];
  int32_t err;
};

// Exclusive prefix sums of (a, b) over the block's threads; the totals come back in ta, tb.
template <int NT>
__device__ inline void block_sums(PlanSmem& sm, int64_t& a, int64_t& b, int64_t& ta, int64_t& tb) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int64_t x = a, y = b;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t u = __shfl_up((long long)x, d, 64), v = __shfl_up((long long)y, d, 64);
    if (lane >= d) {
      x += u;
      y += v;
    }
  }
  __syncthreads();
  if (lane == 63) {
    sm.a[wave] = x;
    sm.b[wave] = y;
  }
  __syncthreads();
  int64_t ba = 0, bb = 0;
  ta = tb = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    const int64_t u = sm.a[w], v = sm.b[w];
    if (w < wave) {
      ba += u;
      bb += v;
    }
    ta += u;
    tb += v;
  }
  a = ba + x - a;
  b = bb + y - b;
}

struct Asked {
  int64_t req, prefix, n;
};

__device__ inline Asked asked(const BlockArgs& a, int i) {
  Asked q{0, 0, 0};
  if (i >= a.bs) return q;
  q.req = a.rpi[i];
  q.prefix = a.prefix[i];
  if (a.fresh) {
    q.n = a.fresh[i];
  } else {  // decode; a padded entry has no context
    q.n = q.prefix >= 1 ? 1 : 0;
    q.prefix -= 1;
  }
  return q;
}

__device__ inline bool sound(const BlockArgs& a, const Asked& q) {
  return q.req >= 0 && q.req < a.reqs && q.prefix >= 0 && q.n >= 0 && q.prefix <= a.width && q.n <= a.width - q.prefix;
}

__device__ inline int blocks_of(int64_t tokens) { return (int)((tokens + 63) >> 6); }

// Marks request `req`; whether it was marked before.
__device__ inline bool mark(uint32_t* seen, int64_t req) {
  const uint32_t bit = 1u << (req & 31);
  return atomicOr(&seen[req >> 5], bit) & bit;
}

// Counts a refused call under each of its reasons.  The counts only grow, so that a host that reads
// them at any time misses no call.
__device__ inline void report(const BlockArgs& a, int err) {
  for (int kind = 0; kind < kErrKinds; ++kind)
    if (err >> kind & 1) {
      const int32_t n = a.err[kind] + 1;
      a.err[kind] = n;
      if (a.err_mirror) a.err_mirror[kind] = n;
    }
}

// The last request whose first token (BLK: block) is at or before `at`, among those with any.
template <bool BLK>
__device__ inline int find_row(const PlanRow* rows, int bs, int at) {
  int lo = 0, hi = bs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if ((BLK ? rows[mid].blk : rows[mid].tok) <= at) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Table entries and slots of a planned call, item by item from `first`.
__device__ inline void fill_slots(const BlockArgs& a, const PlanHead& h, int64_t first, int64_t step) {
  for (int64_t k = first; k < h.blocks; k += step) {
    const PlanRow r = a.rows[find_row<true>(a.rows, a.bs, (int)k)];
    a.table[r.req * a.table_stride + r.held + (k - r.blk)] = a.stack[h.count - 1 - k];
  }
  for (int64_t t = first; t < a.total; t += step) {
    int64_t row = 0, p = 0;
    if (t < h.tokens) {
      const PlanRow r = a.rows[find_row<false>(a.rows, a.bs, (int)t)];
      p = r.prefix + (t - r.tok);
      const int64_t j = p >> 6;  // a block held before, or one of this call's (other threads write those)
      const int32_t block = j < r.held ? a.table[r.req * a.table_stride + j] : a.stack[h.count - 1 - (r.blk + j - r.held)];
      row = (int64_t)block * 64 + (p & 63);
      a.r2t[r.req * a.r2t_stride + p] = (int32_t)row;
    }
    a.loc[t] = row;
    a.pos[t] = p;
  }
}

__global__ __launch_bounds__(256) void assign_fill_kernel(BlockArgs a) {
  fill_slots(a, *a.head, (int64_t)blockIdx.x * 256 + threadIdx.x, (int64_t)gridDim.x * 256);
}

// What request i takes: its tokens and the blocks it lacks (after a call: none).
struct Taken {
  Asked q;
  int held, need;
};

template <int NT>
__global__ __launch_bounds__(NT) void assign_plan_kernel(BlockArgs a) {
  extern __shared__ uint32_t seen[];
  __shared__ PlanSmem sm;
  const int tid = threadIdx.x;
  auto look = [&](int i, int& err) {
    Taken t{asked(a, i), 0, 0};
    if (t.q.n == 0) return t;
    if (sound(a, t.q)) {
      t.held = a.held[t.q.req];
      t.need = max(0, blocks_of(t.q.prefix + t.q.n) - t.held);
    } else {
      err |= kErrRequest;
      t.q.n = 0;
    }
    return t;
  };
  int err = 0;
  const Taken mine = look(tid, err);  // in flight while the bitmap is cleared
  const int count = *a.count;
  for (int i = tid; i < (a.reqs + 31) / 32; i += NT) seen[i] = 0;
  if (tid == 0) sm.err = 0;
  __syncthreads();
  int64_t tokens = 0, blocks = 0;
  int64_t t0 = 0, b0 = 0;  // before this thread's request, in the only round
  for (int i0 = 0; i0 < a.bs; i0 += NT) {
    const Taken x = i0 == 0 ? mine : look(i0 + tid, err);
    if (x.q.n > 0 && mark(seen, x.q.req)) err |= kErrTwice;
    int64_t t = x.q.n, b = x.need, tt, tb;
    block_sums<NT>(sm, t, b, tt, tb);
    tokens += tt;
    blocks += tb;
    t0 = t;
    b0 = b;
  }
  if (err) atomicOr(&sm.err, err);
  if (tid == 0) {
    if (blocks > count) atomicOr(&sm.err, kErrExhausted);
    if (a.fresh && tokens > a.total) atomicOr(&sm.err, kErrTotal);
  }
  __syncthreads();
  err = sm.err;
  if (tid == 0) {
    if (err) report(a, err);
    else *a.count = count - (int)blocks;
    if (a.fresh) *a.head = {err == 0, count, err ? 0 : (int)tokens, err ? 0 : (int)blocks, {0, 0, 0, 0}};
  }
  if (err) {
    if (a.here)
      for (int64_t i = tid; i < a.total; i += NT) a.loc[i] = a.pos[i] = 0;
    return;
  }
  const PlanHead planned{1, count, (int)tokens, (int)blocks, {0, 0, 0, 0}};
  tokens = blocks = 0;
  for (int i0 = 0; i0 < a.bs; i0 += NT) {
    const int i = i0 + tid;
    const Taken x = i0 == 0 ? mine : look(i, err);
    int64_t t = t0, b = b0;
    if (a.bs > NT) {  // block-uniform
      int64_t tt, tb;
      t = x.q.n;
      b = x.need;
      block_sums<NT>(sm, t, b, tt, tb);
      t += tokens;
      b += blocks;
      tokens += tt;
      blocks += tb;
    }
    if (i >= a.bs) continue;
    const Asked& q = x.q;
    if (x.need > 0) a.held[q.req] = x.held + x.need;
    if (a.fresh) {
      a.rows[i] = {(int)t, (int)b, (int)q.req, (int)q.prefix, x.held, {0, 0, 0}};
      continue;
    }
    // decode: the request's one token here and now
    int64_t row = 0;
    if (q.n) {
      int32_t* tr = a.table + q.req * a.table_stride;
      int32_t block = x.need ? 0 : tr[q.prefix >> 6];
      for (int j = 0; j < x.need; ++j) tr[x.held + j] = block = a.stack[count - 1 - (b + j)];
      row = (int64_t)block * 64 + (q.prefix & 63);
      a.r2t[q.req * a.r2t_stride + q.prefix] = (int32_t)row;
    }
    a.loc[i] = row;
    a.pos[i] = q.n ? q.prefix : 0;
  }
  if (a.fresh && a.here) {
    __syncthreads();  // the records are written
    fill_slots(a, planned, tid, NT);
  }
}

// The blocks of the listed requests back on the stack, such that the k-th of them (request
// order, then block order) lies where assigning them took the k-th from.
__global__ __launch_bounds__(kPlan) void release_plan_kernel(BlockArgs a) {
  extern __shared__ uint32_t seen[];
  __shared__ PlanSmem sm;
  const int tid = threadIdx.x;
  for (int i = tid; i < (a.reqs + 31) / 32; i += kPlan) seen[i] = 0;
  if (tid == 0) sm.err = 0;
  const int count = *a.count;
  __syncthreads();
  int64_t blocks = 0;
  int err = 0;
  for (int i0 = 0; i0 < a.bs; i0 += kPlan) {
    const int i = i0 + tid;
    int64_t held = 0;
    const int64_t req = i < a.bs ? a.rpi[i] : 0;
    if (i < a.bs) {
      if (req < 0 || req >= a.reqs) err |= kErrRequest;
      else if (mark(seen, req)) err |= kErrTwice;
      else held = a.held[req];
    }
    int64_t t = 0, b = held, tt, tb;
    block_sums<kPlan>(sm, t, b, tt, tb);
    if (i < a.bs) a.rows[i] = {0, (int)(blocks + b), (int)req, 0, (int)held, {0, 0, 0}};
    blocks += tb;
  }
  if (err) atomicOr(&sm.err, err);
  __syncthreads();
  err = sm.err;
  if (count + blocks > a.cap) err |= kErrTotal;  // not blocks that this stack gave out
  if (!err)
    for (int i = tid; i < a.bs; i += kPlan) a.held[a.rpi[i]] = 0;
  if (tid == 0) {
    if (err) report(a, err);
    else *a.count = count + (int)blocks;
    *a.head = {err == 0, count, 0, err ? 0 : (int)blocks, {0, 0, 0, 0}};
  }
}

__global__ __launch_bounds__(256) void release_fill_kernel(BlockArgs a) {
  const PlanHead h = *a.head;
  const int64_t step = (int64_t)gridDim.x * 256;
  // 64 threads a block of the pool: one returns it, each clears a position
  for (int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x; k < (int64_t)h.blocks * 64; k += step) {
    const int at = (int)(k >> 6), slot = (int)(k & 63);
    const PlanRow r = a.rows[find_row<true>(a.rows, a.bs, at)];
    const int64_t j = at - r.blk, p = j * 64 + slot;
    if (slot == 0) {
      int32_t* e = a.table + r.req * a.table_stride + j;
      a.stack[h.count + h.blocks - 1 - at] = *e;
      *e = 0;
    }
    if (p < a.width) a.r2t[r.req * a.r2t_stride + p] = 0;
  }
}

int check_pool(const BlockArgs& a, const char* what) {
  QQ_REQUIRE(a.bs >= 0 && a.total >= 0 && a.total < (int64_t)1 << 31, "%s: bad sizes", what);
  QQ_REQUIRE(a.reqs > 0 && a.reqs <= kMaxPoolReqs, "%s: %d requests, at most %d", what, a.reqs, kMaxPoolReqs);
  QQ_REQUIRE(a.width > 0 && a.width < (int64_t)1 << 30 && a.r2t_stride >= a.width && a.table_stride >= (a.width + 63) / 64,
             "%s: bad table sizes", what);
  QQ_REQUIRE(a.cap >= 0 && a.cap < kMaxPoolBlocks, "%s: at most %d blocks", what, kMaxPoolBlocks);
  QQ_REQUIRE(a.bs == 0 || (a.rpi && a.table && a.r2t && a.held && a.stack && a.count && a.err), "%s: null pointer", what);
  return QQ_OK;
}

int set_workspace(BlockArgs& a, void* workspace, int64_t bytes, const char* what) {
  const int64_t need = qq_block_workspace_bytes(a.bs);
  QQ_REQUIRE(workspace && bytes >= need, "%s: workspace %lld bytes < %lld needed", what, (long long)bytes, (long long)need);
  a.head = static_cast<PlanHead*>(workspace);
  a.rows = reinterpret_cast<PlanRow*>(a.head + 1);
  return QQ_OK;
}

size_t seen_bytes(const BlockArgs& a) { return (size_t)((a.reqs + 31) / 32) * 4; }

// Blocks of 256 threads for n items, four items a thread at most where the chip is full.
int fill_blocks(int64_t n) { return (int)max((int64_t)1, min((n + 255) / 256, (int64_t)4096)); }

}  // namespace
}  // namespace qq

using namespace qq;

extern "C" int64_t qq_block_workspace_bytes(int bs) {
  return bs <= 0 ? 0 : (int64_t)sizeof(PlanHead) + (int64_t)bs * sizeof(PlanRow);
}

extern "C" int qq_block_assign(const int64_t* req_pool_indices, const int64_t* lens, const int64_t* new_lens, int bs,
                               int64_t total, int32_t* block_table, int64_t block_table_stride, int32_t* req_to_token,
                               int64_t req_to_token_stride, int64_t max_context_len, int max_reqs, int32_t* held,
                               int32_t* free_blocks, int32_t* free_count, int64_t free_cap, int64_t* loc, int64_t* pos,
                               int32_t* error_counts, int32_t* error_mirror, void* workspace, int64_t workspace_bytes,
                               void* stream) {
  const char* what = "qq_block_assign";
  BlockArgs a{req_pool_indices, lens, new_lens, bs, total, block_table, block_table_stride, req_to_token,
              req_to_token_stride, max_context_len, max_reqs, held, free_blocks, free_count, free_cap, loc, pos,
              error_counts, error_mirror, nullptr, nullptr, 0};
  int st = check_pool(a, what);
  if (st != QQ_OK) return st;
  QQ_REQUIRE(bs == 0 || lens, "%s: null pointer", what);
  QQ_REQUIRE(new_lens || total == bs, "%s: a decode batch has one row per request", what);
  QQ_REQUIRE(total == 0 || (loc && pos), "%s: null pointer", what);
  if (total == 0 && bs == 0) return QQ_OK;
  QQ_REQUIRE(bs > 0, "%s: %lld tokens of no request", what, (long long)total);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (new_lens && (st = set_workspace(a, workspace, workspace_bytes, what)) != QQ_OK) return st;
  // a launch less is worth up to four tokens a thread of the planning block
  a.here = !new_lens || total <= 4 * (bs <= 256 ? 256 : kPlan);
  // one round of threads where that is enough; few waves meet at a barrier sooner
  if (bs <= 256) assign_plan_kernel<256><<<1, 256, seen_bytes(a), s>>>(a);
  else assign_plan_kernel<kPlan><<<1, kPlan, seen_bytes(a), s>>>(a);
  if (!a.here) assign_fill_kernel<<<fill_blocks(total), 256, 0, s>>>(a);
  return check_launch(what);
}

extern "C" int qq_block_release(const int64_t* req_pool_indices, int bs, int32_t* block_table,
                                int64_t block_table_stride, int32_t* req_to_token, int64_t req_to_token_stride,
                                int64_t max_context_len, int max_reqs, int32_t* held, int32_t* free_blocks,
                                int32_t* free_count, int64_t free_cap, int32_t* error_counts, int32_t* error_mirror,
                                void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "qq_block_release";
  BlockArgs a{req_pool_indices, nullptr, nullptr, bs, 0, block_table, block_table_stride, req_to_token,
              req_to_token_stride, max_context_len, max_reqs, held, free_blocks, free_count, free_cap, nullptr, nullptr,
              error_counts, error_mirror, nullptr, nullptr, 0};
  int st = check_pool(a, what);
  if (st != QQ_OK) return st;
  if (bs == 0) return QQ_OK;
  if ((st = set_workspace(a, workspace, workspace_bytes, what)) != QQ_OK) return st;
  hipStream_t s = static_cast<hipStream_t>(stream);
  release_plan_kernel<<<1, kPlan, seen_bytes(a), s>>>(a);
  release_fill_kernel<<<1024, 256, 0, s>>>(a);
  return check_launch(what);
}
