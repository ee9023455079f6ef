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
// request) and then writes its share of the tokens, 4 consecutive ones a thread. A token
// takes its block from the ring directly and not from the table, so no CTA reads what
// another one writes: the ring's popped and pushed ranges are disjoint, and the only table
// entry a token reads is the request's last, partly filled block. Rows of finished
// requests are read and rewritten by one thread an entry.
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

// Largest s in [0, S) with cu[s] <= t, for t < cu[S].
__device__ __forceinline__ int request_of(const int* cu, int S, int t) {
  int lo = 0, hi = S;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PlanParams p) {
  extern __shared__ int smem[];
  constexpr int NW = kPlanThreads / 32;
  __shared__ unsigned wsum[3][NW];
  __shared__ int first_fail;
  const int S = p.num_seqs, bs = p.block_size, nb = p.num_blocks;
  int* cu = smem;            // [S + 1] tokens before request s
  int* pop = cu + S + 1;     // [S + 1] blocks taken before request s
  int* push = pop + S + 1;   // [S + 1] blocks given back before request s
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int head = max(0, __ldg(p.state)) % nb;
  const int count = min(max(0, __ldg(p.state + 1)), nb);
  const long long room = static_cast<long long>(p.width) * bs;
  if (tid == 0) {
    first_fail = S;
    cu[0] = pop[0] = push[0] = 0;
  }
  __syncthreads();
  unsigned run0 = 0, run1 = 0, run2 = 0;  // sums of the tiles so far
  for (int base = 0; base < S; base += kPlanThreads) {
    const int s = base + tid;
    unsigned n = 0, need = 0, give = 0;
    bool fits = true;
    if (s < S) {
      int ctx = max(0, __ldg(p.context_lens + s));
      const int add = max(0, __ldg(p.new_lens + s));
      if (p.finished && p.finished[s]) {
        give = static_cast<unsigned>(min((static_cast<long long>(ctx) + bs - 1) / bs,
                                         static_cast<long long>(p.width)));
        ctx = 0;
      }
      const long long end = static_cast<long long>(ctx) + add;
      fits = end <= room;
      n = min(static_cast<unsigned>(add), static_cast<unsigned>(kMaxPlanCount));
      need = static_cast<unsigned>(
          min((end + bs - 1) / bs - (static_cast<long long>(ctx) + bs - 1) / bs,
              static_cast<long long>(kMaxPlanCount)));
    }
    unsigned i0 = warp_scan_sat(n, lane), i1 = warp_scan_sat(need, lane),
             i2 = warp_scan_sat(give, lane);
    if (lane == 31) {
      wsum[0][warp] = i0;
      wsum[1][warp] = i1;
      wsum[2][warp] = i2;
    }
    __syncthreads();
    unsigned b0 = run0, b1 = run1, b2 = run2;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const unsigned w0 = wsum[0][w], w1 = wsum[1][w], w2 = wsum[2][w];
      if (w < warp) {
        b0 = sat_add(b0, w0);
        b1 = sat_add(b1, w1);
        b2 = sat_add(b2, w2);
      }
      run0 = sat_add(run0, w0);
      run1 = sat_add(run1, w1);
      run2 = sat_add(run2, w2);
    }
    i0 = sat_add(i0, b0);
    i1 = sat_add(i1, b1);
    i2 = sat_add(i2, b2);
    if (s < S) {
      cu[s + 1] = static_cast<int>(i0);
      pop[s + 1] = static_cast<int>(i1);
      push[s + 1] = static_cast<int>(i2);
      if (!fits || i0 > static_cast<unsigned>(p.max_tokens) || i1 > static_cast<unsigned>(count))
        atomicMin(&first_fail, s);
    }
    __syncthreads();
  }
  const int served = first_fail;
  const int total = cu[served];
  __syncthreads();
  for (int s = served + 1 + tid; s <= S; s += kPlanThreads) cu[s] = total;
  __syncthreads();
  const int taken = pop[served];

  const int gtid = blockIdx.x * kPlanThreads + tid, nth = gridDim.x * kPlanThreads;
  if (gtid == 0) {
    const long long left = static_cast<long long>(count) - taken + run2;
    p.state_out[0] = static_cast<int>((static_cast<long long>(head) + taken) % nb);
    p.state_out[1] = static_cast<int>(min(left, static_cast<long long>(nb)));
    p.state_out[2] = served;
    p.state_out[3] = total;
    p.cu_seqlens[0] = 0;
    if (static_cast<long long>(count) + run2 > nb) atomicOr(p.err, kErrBadBlock);
  }
  for (int s = gtid; s < S; s += nth) {
    const int ctx = p.finished && p.finished[s] ? 0 : max(0, __ldg(p.context_lens + s));
    p.cu_seqlens[s + 1] = cu[s + 1];
    p.context_lens_out[s] = ctx + cu[s + 1] - cu[s];
  }
  // finished rows, a warp each: entry j goes back to the ring and then takes the row's new
  // block j
  if (p.finished) {
    for (int s = gtid >> 5; s < S; s += nth >> 5) {
      if (!p.finished[s]) continue;
      const int held = static_cast<int>(
          min((max(0LL, static_cast<long long>(__ldg(p.context_lens + s))) + bs - 1) / bs,
              static_cast<long long>(p.width)));
      const int now = (cu[s + 1] - cu[s] + bs - 1) / bs;
      int* row = p.block_tables + static_cast<long long>(s) * p.width;
      for (int j = lane; j < max(held, now); j += 32) {
        const long long to = static_cast<long long>(count) + push[s] + j;
        if (j < held && to < nb) p.free_blocks[(head + to) % nb] = row[j];
        if (j < now) row[j] = p.free_blocks[(static_cast<long long>(head) + pop[s] + j) % nb];
      }
    }
  }
  // tokens, 4 a thread
  for (long long t0 = 4LL * gtid; t0 < p.max_tokens; t0 += 4LL * nth) {
    int pos[4];
    long long slot[4];
    int s = -1, ctx = 0, have = 0, beg = 0, end = 0;
    bool fresh = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = static_cast<int>(t0) + i;
      pos[i] = -1;
      slot[i] = -1;
      if (t0 + i >= total) continue;
      if (s < 0 || t >= end) {
        s = request_of(cu, S, t);
        beg = cu[s];
        end = cu[s + 1];
        fresh = p.finished && p.finished[s];
        ctx = fresh ? 0 : max(0, __ldg(p.context_lens + s));
        have = (ctx + bs - 1) / bs;
      }
      const int at = ctx + t - beg;
      const int j = at / bs, off = at - j * bs;
      int* row = p.block_tables + static_cast<long long>(s) * p.width;
      int block;
      if (j < have) {
        block = row[j];
      } else {
        block = p.free_blocks[(static_cast<long long>(head) + pop[s] + (j - have)) % nb];
        if (off == 0 && !fresh) row[j] = block;
      }
      pos[i] = at;
      slot[i] = static_cast<long long>(block) * bs + off;
    }
    if (t0 + 4 <= p.max_tokens && (reinterpret_cast<uintptr_t>(p.positions) & 15) == 0 &&
        (reinterpret_cast<uintptr_t>(p.slots) & 15) == 0) {
      *reinterpret_cast<int4*>(p.positions + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
      *reinterpret_cast<longlong2*>(p.slots + t0) = make_longlong2(slot[0], slot[1]);
      *reinterpret_cast<longlong2*>(p.slots + t0 + 2) = make_longlong2(slot[2], slot[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (t0 + i < p.max_tokens) {
          p.positions[t0 + i] = pos[i];
          p.slots[t0 + i] = slot[i];
        }
      }
    }
  }
}

cudaError_t launch_plan(const PlanParams& p, cudaStream_t stream) {
  const int smem = 3 * (p.num_seqs + 1) * static_cast<int>(sizeof(int));
  const cudaError_t e = ensure_smem_optin(reinterpret_cast<const void*>(plan_kernel), smem);
  if (e != cudaSuccess) return e;
  // 4 tokens a thread; 8 threads a request for the finished rows
  const long long threads = std::max<long long>((p.max_tokens + 3LL) / 4, 8LL * p.num_seqs);
  const long long blocks = (threads + kPlanThreads - 1) / kPlanThreads;
  const int grid = static_cast<int>(std::min<long long>(std::max<long long>(blocks, 1), sm_count()));
  plan_kernel<<<grid, kPlanThreads, smem, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace step
}  // namespace fe
