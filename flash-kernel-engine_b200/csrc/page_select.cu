// Page selection of the sparse paged decode: every page of a sequence is scored against
// the query through the int8 box of its keys (page_bounds.cu), and the num_pages best of
// each KV head are listed in ascending order.
//
// The query is rounded to whole numbers like a box: qi = round(q / 2^eq), eq the smallest
// exponent with amax(q) <= 127 * 2^eq. With box [lo, hi] 2^ek,
//   score(page) = max over the group's heads of  sum_c max(qi_c hi_c, qi_c lo_c) 2^eq 2^ek,
// an upper bound of the rounded query's product with every key of the page. Since
// max(q hi, q lo) = q+ hi + q- lo, the sum is a product of the int8 row [q+ | q-] with the
// stored row [hi | lo] and runs on the integer tensor path, 16 pages x 8 heads a warp
// instruction. It is a whole number below 2^24 (256 channels at most of 127 * 127), so
// fp32 holds it exactly, the powers of two scale it exactly, and the choice of pages does
// not depend on the order of any sum. Ties go to the lower page. The first keep_first and
// the last keep_last pages are always chosen; the last one may be partly filled.
//
// A cluster of CTAs serves one (sequence, KV head): each scores a contiguous range of the
// pages and keeps their scores as ordered 32-bit keys in its shared memory. The threshold
// comes from histograms of the keys between the smallest and the largest one, refined
// until the wanted count ends at a bin's edge or a bin is a single key; with several CTAs
// each adds up all histograms over distributed shared memory. Then the warps count and
// write their chosen pages in order. One launch, nothing but the lists goes to memory; the
// boxes are read once (d / 32 bytes a token at 16-token pages: 1/32 of bf16 keys and values).
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <limits.h>
#include <stdint.h>

#include <algorithm>

#include "internal.h"
#include "page_box.cuh"
#include "paged_decode.h"
#include "paged_step.h"
#include "ptx.cuh"

namespace cg = cooperative_groups;

namespace fe {
namespace step {

constexpr int kBinBits = 10;
constexpr int kBins = 1 << kBinBits;
constexpr unsigned kForced = 0xffffffffu;  // key of an always-chosen page, above every score

// Order-preserving map of a float (no NaN, no -0) to 32 bits.
__device__ __forceinline__ unsigned key_of(float x) {
  const unsigned u = __float_as_uint(x);
  return u ^ (static_cast<unsigned>(static_cast<int>(u) >> 31) | 0x80000000u);
}

// D = A(16x32, row) * B(32x8, col) + D, int8 inputs, int32 accumulate.
__device__ __forceinline__ void mma_s8_16832(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                             uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, "
      "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int NTHR>
struct SelectShared {
  unsigned hist[kBins];
  unsigned suffix[NTHR / 32];
  unsigned warp_above[NTHR / 32], warp_equal[NTHR / 32];
  unsigned kmin, kmax;             // of this CTA's unforced keys
  unsigned cta_above, cta_equal;   // chosen above / equal to the threshold in this CTA
  unsigned bin, above, in_bin;     // result of one histogram round
};

template <typename T, int D, int NTHR>
__global__ void __launch_bounds__(NTHR) page_select_kernel(const SelectParams p, int ctas,
                                                           int cap) {
  constexpr int NW = NTHR / 32;
  constexpr int QB = 2 * D;   // bytes of a box, and of a head's [q+ | q-] row
  constexpr int CH = QB / 64; // 64-byte pieces a quad of lanes reads
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ SelectShared<NTHR> sh;
  unsigned* keys = reinterpret_cast<unsigned*>(dyn);          // [cap]
  const int G = p.heads / p.kv_heads, GP = (G + 7) / 8 * 8;
  signed char* qrow = reinterpret_cast<signed char*>(keys + cap);   // [GP][QB]
  float* qscale = reinterpret_cast<float*>(qrow + GP * QB);   // [GP]: 2^eq, +inf, or 0 (no head)
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / ctas, rank = blockIdx.x % ctas;
  const int seq = row / p.kv_heads, kvh = row % p.kv_heads;
  cg::cluster_group cluster = cg::this_cluster();
  auto sync = [&] {
    if (ctas > 1) cluster.sync(); else __syncthreads();
  };

  int ctx = max(0, __ldg(p.context_lens + seq));
  const long long room = static_cast<long long>(p.width) * p.block_size;
  if (ctx > room) {
    if (tid == 0) atomicOr(p.err, kErrBadBlock);
    ctx = static_cast<int>(room);
  }
  const int P = (ctx + p.block_size - 1) / p.block_size, K = p.num_pages;
  const int* table = p.block_tables + static_cast<long long>(seq) * p.width;
  int* sel = p.selected + static_cast<long long>(row) * K;
  int* blocks = p.sel_blocks + static_cast<long long>(row) * K;
  // virtual block of a page: the cache seen as [num_blocks * Hkv, 1, ...]
  auto vblock = [&](int page) {
    const int b = __ldg(table + page);
    if (b < 0 || b >= p.num_blocks) {
      atomicOr(p.err, kErrBadBlock);
      return -1;
    }
    return b * p.kv_heads + kvh;
  };
  if (P <= K) {  // every page (uniform over the cluster: no CTA waits for another)
    for (int i = rank * NTHR + tid; i < K; i += ctas * NTHR) {
      sel[i] = i < P ? i : -1;
      if (i < P) blocks[i] = vblock(i);
    }
    if (rank == 0 && tid == 0) p.sel_lens[row] = ctx;
    return;
  }

  // ---- the query as whole numbers, a warp a head
  for (int g = warp; g < GP; g += NW) {
    constexpr int E = D / 32;
    float x[E], amax = 0.f;
    bool fin = true;
    const T* q = static_cast<const T*>(p.q) +
                 (static_cast<long long>(seq) * p.heads + kvh * G + g) * D;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      x[i] = g < G ? static_cast<float>(q[i * 32 + lane]) : 0.f;
      fin = fin && is_finite(x[i]);
      amax = fmaxf(amax, fabsf(x[i]));
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    fin = __all_sync(0xffffffffu, fin);
    const int e = box_exponent(fin ? amax : 0.f);
    const float inv = exp2_int(-e);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int v = fin ? __float2int_rn(x[i] * inv) : 0;
      qrow[g * QB + i * 32 + lane] = static_cast<signed char>(max(v, 0));
      qrow[g * QB + D + i * 32 + lane] = static_cast<signed char>(min(v, 0));
    }
    if (lane == 0)
      qscale[g] = g >= G ? 0.f : fin ? exp2_int(e) : __int_as_float(0x7f800000);
  }
  if (tid == 0) {
    sh.kmin = kForced;
    sh.kmax = 0;
  }
  __syncthreads();

  // ---- scores of this CTA's pages [beg, end), 16 a warp at a time
  const int per = ((P + ctas - 1) / ctas + 15) / 16 * 16;
  const int beg = min(P, rank * per), n = min(P, beg + per) - beg;
  const int gq = lane >> 2, cq = lane & 3;
  unsigned kmin = kForced, kmax = 0;
  for (int tile = warp; tile * 16 < n; tile += NW) {
    const int mine = tile * 16 + (lane & 15);  // the page whose block this lane looks up
    int b = 0;
    if (mine < n) {
      b = __ldg(table + beg + mine);
      if (b < 0 || b >= p.num_blocks) b = 0;  // flagged where the page is listed
    }
    const long long page = static_cast<long long>(b) * p.kv_heads + kvh;
    const float ks = __ldg(p.scales + page);
    const long long p0 = __shfl_sync(0xffffffffu, page, gq),
                    p1 = __shfl_sync(0xffffffffu, page, gq + 8);
    const uint4* r0 = reinterpret_cast<const uint4*>(p.values + p0 * QB) + cq;
    const uint4* r1 = reinterpret_cast<const uint4*>(p.values + p1 * QB) + cq;
    uint4 a0[CH], a1[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      a0[i] = __ldg(r0 + 4 * i);
      a1[i] = __ldg(r1 + 4 * i);
    }
    float best0 = -__int_as_float(0x7f800000), best1 = best0;
    for (int h0 = 0; h0 < GP; h0 += 8) {
      int acc[4] = {0, 0, 0, 0};
      const uint4* qv = reinterpret_cast<const uint4*>(qrow + (h0 + gq) * QB) + cq;
      // the k index of both operands is the byte's place in this lane's 16-byte pieces
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const uint4 v = qv[4 * i];
        mma_s8_16832(acc, a0[i].x, a1[i].x, a0[i].y, a1[i].y, v.x, v.y);
        mma_s8_16832(acc, a0[i].z, a1[i].z, a0[i].w, a1[i].w, v.z, v.w);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float qs = qscale[h0 + 2 * cq + j];
        if (qs == 0.f) continue;  // past the group's heads
        const bool open = qs == __int_as_float(0x7f800000);
        best0 = fmaxf(best0, open ? qs : static_cast<float>(acc[j]) * qs);
        best1 = fmaxf(best1, open ? qs : static_cast<float>(acc[2 + j]) * qs);
      }
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      best0 = fmaxf(best0, __shfl_xor_sync(0xffffffffu, best0, o));
      best1 = fmaxf(best1, __shfl_xor_sync(0xffffffffu, best1, o));
    }
    const float ks0 = __shfl_sync(0xffffffffu, ks, gq), ks1 = __shfl_sync(0xffffffffu, ks, gq + 8);
    if (cq < 2) {
      const int at = tile * 16 + gq + 8 * cq;
      const float sc = cq ? ks1 : ks0, best = cq ? best1 : best0;
      if (at < n) {
        const int j = beg + at;
        unsigned key;
        if (j < p.keep_first || j >= P - p.keep_last) {
          key = kForced;
        } else {
          const bool open = sc == __int_as_float(0x7f800000);
          key = key_of((open ? sc : best * sc) + 0.f);  // + 0: no -0
          kmin = min(kmin, key);
          kmax = max(kmax, key);
        }
        keys[at] = key;
      }
    }
  }
  kmin = __reduce_min_sync(0xffffffffu, kmin);
  kmax = __reduce_max_sync(0xffffffffu, kmax);
  if (lane == 0) {
    atomicMin(&sh.kmin, kmin);
    atomicMax(&sh.kmax, kmax);
  }
  sync();

  // ---- the threshold: chosen are the keys above thr and the first `need` equal to it
  unsigned rem = K - p.keep_first - p.keep_last;  // still to choose (P > K: all forced are in)
  unsigned lo = kForced, hi = 0;
  for (int r = 0; r < ctas; ++r) {
    SelectShared<NTHR>* o = ctas > 1 ? cluster.map_shared_rank(&sh, r) : &sh;
    lo = min(lo, o->kmin);
    hi = max(hi, o->kmax);
  }
  unsigned thr = kForced - 1, need = 0;
  if (rem > 0) {
    for (;;) {
      if (lo == hi) {
        thr = lo;
        need = rem;
        break;
      }
      const int bits = 32 - __clz(hi - lo);
      const int shift = max(0, bits - kBinBits);
      for (int i = tid; i < kBins; i += NTHR) sh.hist[i] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += NTHR) {
        const unsigned k = keys[i];
        if (k >= lo && k <= hi) atomicAdd(&sh.hist[(k - lo) >> shift], 1u);
      }
      sync();
      // this thread's bins, the highest ones first over the threads
      constexpr int BPT = kBins / NTHR;
      unsigned c[BPT], sum = 0;
#pragma unroll
      for (int i = 0; i < BPT; ++i) c[i] = 0;
      const int b0 = kBins - (tid + 1) * BPT;
      for (int r = 0; r < ctas; ++r) {
        const unsigned* hr = ctas > 1 ? cluster.map_shared_rank(sh.hist, r) : sh.hist;
#pragma unroll
        for (int i = 0; i < BPT; ++i) c[i] += hr[b0 + i];
      }
#pragma unroll
      for (int i = 0; i < BPT; ++i) sum += c[i];
      unsigned inc = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      if (lane == 31) sh.suffix[warp] = inc;
      __syncthreads();
      unsigned above = inc - sum;
      for (int w = 0; w < warp; ++w) above += sh.suffix[w];
      if (above < rem && rem <= above + sum) {
#pragma unroll
        for (int i = BPT - 1; i >= 0; --i) {
          if (rem > above && rem <= above + c[i]) {
            sh.bin = b0 + i;
            sh.above = above;
            sh.in_bin = c[i];
            break;
          }
          above += c[i];
        }
      }
      sync();  // the result, and every CTA done with the histograms
      const unsigned from = lo + (sh.bin << shift);
      const unsigned width = (1u << shift) - 1;
      rem -= sh.above;
      if (sh.in_bin == rem) {  // the whole bin is chosen
        thr = from - 1;
        need = 0;
        break;
      }
      hi = min(hi, from + width);
      lo = from;
    }
  }

  // ---- the lists: each warp takes a contiguous range of the CTA's pages
  const int span = ((n + NW - 1) / NW + 31) / 32 * 32;
  const int wb = min(n, warp * span), we = min(n, wb + span);
  unsigned na = 0, ne = 0;
  for (int i = wb + lane; i < we; i += 32) {
    const unsigned k = keys[i];
    na += k > thr;
    ne += k == thr;
  }
  na = __reduce_add_sync(0xffffffffu, na);
  ne = __reduce_add_sync(0xffffffffu, ne);
  if (lane == 0) {
    sh.warp_above[warp] = na;
    sh.warp_equal[warp] = ne;
  }
  __syncthreads();
  if (tid == 0) {
    unsigned a = 0, e = 0;
    for (int w = 0; w < NW; ++w) {
      a += sh.warp_above[w];
      e += sh.warp_equal[w];
    }
    sh.cta_above = a;
    sh.cta_equal = e;
  }
  sync();
  unsigned a = 0, e = 0;
  for (int r = 0; r < rank; ++r) {
    SelectShared<NTHR>* o = cluster.map_shared_rank(&sh, r);
    a += o->cta_above;
    e += o->cta_equal;
  }
  for (int w = 0; w < warp; ++w) {
    a += sh.warp_above[w];
    e += sh.warp_equal[w];
  }
  const unsigned below = (1u << lane) - 1;
  for (int i0 = wb; i0 < we; i0 += 32) {
    const int i = i0 + lane;
    const unsigned k = i < we ? keys[i] : 0;
    const unsigned ma = __ballot_sync(0xffffffffu, i < we && k > thr);
    const unsigned me = __ballot_sync(0xffffffffu, i < we && k == thr);
    const unsigned ea = e + __popc(me & below);  // equal ones before this page
    const bool chosen = (ma >> lane & 1) || ((me >> lane & 1) && ea < need);
    if (chosen) {
      const unsigned at = a + __popc(ma & below) + min(ea, need);
      sel[at] = beg + i;
      blocks[at] = vblock(beg + i);
    }
    a += __popc(ma);
    e += __popc(me);
  }
  if (rank == 0 && tid == 0)
    p.sel_lens[row] = (K - 1) * p.block_size + ctx - (P - 1) * p.block_size;
  if (ctas > 1) cluster.sync();  // no CTA leaves while another reads its shared memory
}

static int select_smem(int cap, int group, int d) {
  const int gp = (group + 7) / 8 * 8;
  return cap * 4 + gp * 2 * d + gp * 4;
}
// Keys a CTA holds: the pages of the widest table over `ctas`, in 16-page tiles.
static long long select_cap(long long width, int ctas) {
  return ((width + ctas - 1) / ctas + 15) / 16 * 16;
}
constexpr int kSelectSmem = 200 * 1024;

bool select_width_ok(long long width, int group, int d) {
  const long long cap = select_cap(width, kMaxSelectCtas);
  return group <= 128 && cap * 4 + (group + 7) / 8 * 8 * (2LL * d + 4) <= kSelectSmem;
}

template <typename T, int D, int NTHR>
static cudaError_t launch_cfg(const SelectParams& p, int ctas, cudaStream_t st) {
  auto kern = page_select_kernel<T, D, NTHR>;
  const int cap = static_cast<int>(select_cap(p.width, ctas));
  const int smem = select_smem(cap, p.heads / p.kv_heads, D);
  cudaError_t e = ensure_smem_optin(reinterpret_cast<const void*>(kern), smem);
  if (e != cudaSuccess) return e;
  if (ctas > 8) {  // more than the portable cluster size
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(static_cast<long long>(p.num_seqs) * p.kv_heads * ctas));
  cfg.blockDim = dim3(NTHR);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p, ctas, cap);
}

template <typename T, int D>
static cudaError_t launch_d(const SelectParams& p, cudaStream_t st) {
  // CTAs a row: enough to fill the GPU, at least 128 pages each, and as many as the
  // shared memory needs for the widest table
  const long long rows = static_cast<long long>(p.num_seqs) * p.kv_heads;
  int ctas = 1;
  while (ctas < kMaxSelectCtas &&
         ((rows * ctas * 2 <= sm_count() && p.width / (2 * ctas) >= 128) ||
          select_smem(static_cast<int>(select_cap(p.width, ctas)), p.heads / p.kv_heads, D) >
              kSelectSmem))
    ctas *= 2;
  if (rows * ctas <= sm_count()) return launch_cfg<T, D, 512>(p, ctas, st);
  return launch_cfg<T, D, 256>(p, ctas, st);
}

template <typename T>
static cudaError_t launch_t(const SelectParams& p, int d, cudaStream_t st) {
  if (d == 64) return launch_d<T, 64>(p, st);
  if (d == 128) return launch_d<T, 128>(p, st);
  return cudaErrorInvalidValue;
}

cudaError_t launch_page_select(const SelectParams& p, int d, int dtype, cudaStream_t st) {
  if (dtype == paged::kBf16) return launch_t<__nv_bfloat16>(p, d, st);
  if (dtype == paged::kF16) return launch_t<half>(p, d, st);
  if (dtype == paged::kF32) return launch_t<float>(p, d, st);
  return cudaErrorInvalidValue;
}

}  // namespace step
}  // namespace fe
