// The bookkeeping of one serving step, from request lengths that live on the GPU: blocks
// taken from and given back to a ring of free blocks, block tables, and the position and
// cache slot of every token of the step.
//
// With ctx tokens held and n new ones, request s needs
//   need = ceil((ctx + n) / bs) - ceil(ctx / bs)
// blocks. Requests are served in order until one does not fit (its tokens in max_tokens,
// its blocks in the ring, its length in the table); that one and those after it get no
// tokens. Block j >= have = ceil(ctx / bs) of request s is ring entry
// head + pop[s] + (j - have), pop the exclusive prefix sum of need; a finished request's
// blocks go to the ring's tail first-row-first and its row starts again at length 0.
//
// One launch, no waiting between CTAs: every CTA forms the three prefix sums (tokens,
// blocks taken, blocks given back) of all requests in its own shared memory (12 bytes a
// request) and then writes its share of the tokens, one a thread. A token takes its block
// from the ring directly and not from the table, so no CTA reads what another one writes:
// the ring's popped and pushed ranges are disjoint, and the only table entry a token reads
// is the request's last, partly filled block. Rows of finished requests are read and
// rewritten by a warp. What bounds it is latency: the lengths' loads, the
// sums (all loads first, then a contiguous range of requests a thread and one block-wide
// scan of the ranges' sums), a binary search a token and the load of its block. 256 requests
// of one token: 4.2 to 4.8 us a call; 4096 requests with 58 thousand tokens and 203 finished
// rows: 8.5 us (24.6 us with the lengths loaded tile by tile and four tokens a thread; 2.3
// more with one entry of a finished row in flight a lane, 0.6 more with 64-bit divisions).
#include <limits.h>

#include <algorithm>

#include "internal.h"
#include "paged_step.h"
#include "ptx.cuh"

namespace fe {
namespace step {

constexpr int kPlanThreads = 512;

// Sums saturate at kMaxPlanCount, above every capacity: min(a + b, cap) is associative, so
// lengths that would overflow 32 bits still fail the capacity tests.
__device__ __forceinline__ unsigned sat_add(unsigned a, unsigned b) {
  return min(a + b, static_cast<unsigned>(kMaxPlanCount));
}

__device__ __forceinline__ unsigned warp_scan_sat(unsigned v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned n = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v = sat_add(v, n);
  }
  return v;
}

// Where entry s of a prefix sum lies: one word in 33 is left out, so that threads that walk
// ranges of 2^k entries side by side hit different banks.
__device__ __forceinline__ int at(int s) { return s + (s >> 5); }
__host__ __device__ constexpr int padded(int n) { return n + (n >> 5) + 1; }

// ceil(n / d) without an overflow
__device__ __forceinline__ unsigned ceil_div(unsigned n, unsigned d) {
  return n == 0 ? 0 : (n - 1) / d + 1;
}

// Largest s in [0, S) with cu[s] <= t, for t < cu[S].
__device__ __forceinline__ int request_of(const unsigned* cu, int S, unsigned t) {
  int lo = 0, hi = S;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[at(mid)] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PlanParams p) {
  extern __shared__ unsigned smem[];
  constexpr int NW = kPlanThreads / 32;
  __shared__ unsigned wsum[3][NW];
  __shared__ int first_fail;
  const int S = p.num_seqs, bs = p.block_size, nb = p.num_blocks;
  // [S + 1] each: tokens, blocks taken and blocks given back before request s
  unsigned* cu = smem;
  unsigned* pop = cu + padded(S + 1);
  unsigned* push = pop + padded(S + 1);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int head = max(0, __ldg(p.state)) % nb;
  const int count = min(max(0, __ldg(p.state + 1)), nb);
  // tokens a row can hold: its blocks', and a length has 31 bits
  const unsigned room = static_cast<unsigned>(
      min(static_cast<long long>(p.width) * bs, static_cast<long long>(INT_MAX)));
  auto finished = [&](int s) { return p.finished && p.finished[s]; };
  // ring entry head + k, k < 2^30
  auto ring = [&](unsigned k) -> int& {
    unsigned i = head + k % nb;
    if (i >= static_cast<unsigned>(nb)) i -= nb;
    return p.free_blocks[i];
  };
  if (tid == 0) {
    first_fail = S;
    cu[0] = pop[0] = push[0] = 0;
  }
  // what each request asks for, as entry s + 1
#pragma unroll 4
  for (int s = tid; s < S; s += kPlanThreads) {
    const int held = max(0, __ldg(p.context_lens + s)), add = max(0, __ldg(p.new_lens + s));
    const bool fin = finished(s);
    const int ctx = fin ? 0 : held;
    const unsigned end = static_cast<unsigned>(ctx) + static_cast<unsigned>(add);  // < 2^32
    const unsigned have = ceil_div(held, bs);
    const unsigned need = ceil_div(end, bs) - (fin ? 0 : have);
    // a request that its row cannot hold asks for more than there is
    cu[at(s + 1)] = end <= room ? min(add, kMaxPlanCount) : kMaxPlanCount;
    pop[at(s + 1)] = min(need, static_cast<unsigned>(kMaxPlanCount));
    push[at(s + 1)] = fin ? min(have, static_cast<unsigned>(p.width)) : 0;
  }
  __syncthreads();
  // prefix sums: this thread's range, then the ranges before it
  const int per = (S + kPlanThreads - 1) / kPlanThreads;
  const int s0 = min(S, tid * per), s1 = min(S, s0 + per);
  unsigned own[3] = {0, 0, 0};
  for (int s = s0; s < s1; ++s) {
    own[0] = sat_add(own[0], cu[at(s + 1)]);
    own[1] = sat_add(own[1], pop[at(s + 1)]);
    own[2] = sat_add(own[2], push[at(s + 1)]);
  }
  unsigned run[3];
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const unsigned inc = warp_scan_sat(own[k], lane);
    if (lane == 31) wsum[k][warp] = inc;
    const unsigned before = __shfl_up_sync(0xffffffffu, inc, 1);
    run[k] = lane == 0 ? 0 : before;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    if (w < warp) {
#pragma unroll
      for (int k = 0; k < 3; ++k) run[k] = sat_add(run[k], wsum[k][w]);
    }
  }
  int fail = S;
  for (int s = s0; s < s1; ++s) {
    const int i = at(s + 1);
    cu[i] = run[0] = sat_add(run[0], cu[i]);
    pop[i] = run[1] = sat_add(run[1], pop[i]);
    push[i] = run[2] = sat_add(run[2], push[i]);
    if (run[0] > static_cast<unsigned>(p.max_tokens) || run[1] > static_cast<unsigned>(count))
      fail = min(fail, s);
  }
  if (fail < S) atomicMin(&first_fail, fail);
  __syncthreads();
  const int served = first_fail;
  const unsigned total = cu[at(served)], taken = pop[at(served)];
  if (served < S) {
    __syncthreads();
    for (int s = served + 1 + tid; s <= S; s += kPlanThreads) cu[at(s)] = total;
    __syncthreads();
  }

  const int gtid = blockIdx.x * kPlanThreads + tid, nth = gridDim.x * kPlanThreads;
  // tokens
  for (int t = gtid; t < p.max_tokens; t += nth) {
    int pos = -1;
    long long slot = -1;
    if (static_cast<unsigned>(t) < total) {
      const int s = request_of(cu, S, t);
      const bool fresh = finished(s);
      const int ctx = fresh ? 0 : max(0, __ldg(p.context_lens + s));
      const int have = static_cast<int>((static_cast<unsigned>(ctx) + bs - 1u) / bs);  // < 2^32
      pos = ctx + t - static_cast<int>(cu[at(s)]);
      const int j = pos / bs, off = pos - j * bs;
      int* entry = p.block_tables + static_cast<long long>(s) * p.width + j;
      int block;
      if (j < have) {
        block = *entry;
      } else {
        block = ring(pop[at(s)] + (j - have));
        if (off == 0 && !fresh) *entry = block;
      }
      slot = static_cast<long long>(block) * bs + off;
    }
    p.positions[t] = pos;
    p.slots[t] = slot;
  }
  // lengths and offsets
  if (gtid == 0) {
    const long long left = static_cast<long long>(count) - taken + push[at(S)];
    p.state_out[0] = static_cast<int>((static_cast<unsigned>(head) + taken) % nb);
    p.state_out[1] = static_cast<int>(min(left, static_cast<long long>(nb)));
    p.state_out[2] = served;
    p.state_out[3] = total;
    p.cu_seqlens[0] = 0;
    if (static_cast<long long>(count) + push[at(S)] > nb) atomicOr(p.err, kErrBadBlock);
  }
  for (int s = gtid; s < S; s += nth) {
    const unsigned end = cu[at(s + 1)];
    p.cu_seqlens[s + 1] = end;
    p.context_lens_out[s] =
        (finished(s) ? 0 : max(0, __ldg(p.context_lens + s))) + static_cast<int>(end - cu[at(s)]);
  }
  // finished rows, a warp each: entry j goes back to the ring and then takes the row's new
  // block j
  if (p.finished) {
    for (int s = gtid >> 5; s < S; s += nth >> 5) {
      if (!p.finished[s]) continue;
      const int held = static_cast<int>(push[at(s + 1)] - push[at(s)]);
      const int now = static_cast<int>((cu[at(s + 1)] - cu[at(s)] + bs - 1u) / bs);  // < 2^32
      int* row = p.block_tables + static_cast<long long>(s) * p.width;
      // 8 entries a lane in flight: a long row's entries are one round trip, not one each
      for (int j0 = lane; j0 < max(held, now); j0 += 256) {
        int old[8], fresh[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int j = j0 + 32 * k;
          if (j < held) old[k] = row[j];
          if (j < now) fresh[k] = ring(pop[at(s)] + j);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int j = j0 + 32 * k;
          const unsigned to = static_cast<unsigned>(count) + push[at(s)] + j;
          if (j < held && to < static_cast<unsigned>(nb)) ring(to) = old[k];
          if (j < now) row[j] = fresh[k];
        }
      }
    }
  }
}

cudaError_t launch_plan(const PlanParams& p, cudaStream_t stream) {
  const int smem = 3 * padded(p.num_seqs + 1) * static_cast<int>(sizeof(int));
  const cudaError_t e = ensure_smem_optin(reinterpret_cast<const void*>(plan_kernel), smem);
  if (e != cudaSuccess) return e;
  // a token a thread; 8 threads a request for the finished rows
  const long long threads = std::max<long long>(p.max_tokens, 8LL * p.num_seqs);
  const long long blocks = (threads + kPlanThreads - 1) / kPlanThreads;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(std::min<long long>(std::max<long long>(blocks, 1), sm_count())));
  cfg.blockDim = dim3(kPlanThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  // placed while the kernel before finishes (it waits for it); a decode that comes next reads
  // lengths and tables before its own wait, and is told to start after this kernel
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  tables_written(stream);
  return cudaLaunchKernelEx(&cfg, plan_kernel, p);
}

}  // namespace step
}  // namespace fe
