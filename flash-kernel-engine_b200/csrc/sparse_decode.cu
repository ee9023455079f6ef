// Sparse paged decode: every page of a sequence is scored against the query through the
// int8 box of its keys (page_bounds.cu), the num_pages best of each KV head are chosen, and
// the query's heads attend to those.
//
// Score. The query is rounded to whole numbers like a box: qi = round(q / 2^eq), eq the
// smallest exponent with amax(q) <= 127 * 2^eq. With box [lo, hi] 2^ek,
//   score(page) = max over the group's heads of  sum_c max(qi_c hi_c, qi_c lo_c) 2^eq 2^ek,
// an upper bound of the rounded query's product with every key of the page (the query is
// rounded to nearest, so its own product can be larger). Since
// max(q hi, q lo) = q+ hi + q- lo, the sum is a product of the int8 row [q+ | q-] with the
// stored row [hi | lo] and runs on the integer tensor path, 16 pages x 8 heads an
// instruction. It is a whole number below 2^24 (256 terms at most of 127 * 127), so fp32
// holds it exactly, the powers of two scale it exactly (while the score is inside fp32's
// range; beyond it pages tie at 0 or infinity), and the choice of pages does not depend on
// the order of any sum. Ties go to the lower page. The first keep_first and the
// last keep_last pages are always chosen; the last one may be partly filled.
//
// Attention. Softmax over the chosen pages' tokens with a running maximum and sum a warp,
// in fp32; the weights are rounded to the element type for the product with V, as in
// paged_decode.cu, since the 16-bit matrix instructions take no wider ones. The relative
// error of the outputs is 0.0019 in bf16 (0.0017 with fp32 weights, nearly all of it the
// output's own rounding) and 0.00023 in fp16 (0.00021). Weights in two 16-bit parts cost
// nearly no time (4 x 131072 tokens: 41.1 and 41.0 us), but their second part is 0 or
// negative for many of them, and times an infinite value that makes a NaN where the value
// itself is right.
//
// Choice. A score is kept as an ordered 32-bit key, with the largest key of every 8 pages.
// Up to 8 pages a thread are held in registers, and a threshold is found bit by bit from the
// first bit in which the keys differ, one barrier a bit, until no more keys reach it than
// there are threads; the K-th largest of those is then found with one key a thread, which
// the barrier itself counts. Longer rows first look at the groups' maxima: the m-th largest
// of them is a lower bound of the m-th largest key, so that only keys that reach it matter:
// a few hundred of thousands. Where those are too many (equal scores, say), all keys are
// read again for every bit.
//
// Two launches. page_score_kernel reads the boxes: one CTA an SM takes an equal share of all
// sequences' 16-page tiles, whatever their lengths, and all KV heads of a tile at once, whose
// boxes are neighbours in memory. sparse_decode_kernel gives each (sequence, KV head) a
// cluster of CTAs: each finds the threshold by itself, lists the chosen pages, attends to
// its share of them, and the partial (m, l, O) are joined over distributed shared memory.
//
// fp32 caches, the x-packed layout and groups of more than 16 heads take the same scores and
// choice, which then writes a block table for each (sequence, KV head) that paged_decode.cu
// runs over.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <limits.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "internal.h"
#include "page_box.cuh"
#include "page_key.h"
#include "paged_decode.h"
#include "paged_step.h"
#include "ptx.cuh"

namespace cg = cooperative_groups;

namespace fe {
namespace step {

constexpr int kMaxCtas = 8;            // of one (sequence, KV head): the portable cluster; of
                                       // clusters of 16 only four were resident at a time
constexpr int kScoreWarps = 16;        // of a CTA of the score launch
constexpr int kScoreRing = 150 * 1024; // bytes of boxes of a CTA in flight, at most
constexpr int kScoreStages = 32;       // and tiles
constexpr int kScoreSeqs = 4096;       // most sequences of one launch of it
constexpr int kMaxFusedPages = 8192;   // most chosen pages whose list fits shared memory
constexpr int kGroup = 8;              // pages whose largest key is kept

// D = A(16x32, row) * B(32x8, col) + D, int8 inputs, int32 accumulate.
__device__ __forceinline__ void mma_s8_16832(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                             uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, "
      "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <typename T>
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1) {
  const uint32_t a[4] = {a0, a1, a2, a3};
  if constexpr (std::is_same<T, half>::value) mma_f16_16816(d, a, b0, b1);
  else mma_bf16_16816(d, a, b0, b1);
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, half>::value) return pack_f16x2(lo, hi);
  else return pack_bf16x2(lo, hi);
}
// 16 bytes that are read once.
__device__ __forceinline__ uint4 ld_once(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ void named_bar(int id, int nthreads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(nthreads) : "memory");
}
__device__ __forceinline__ void griddep_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void griddep_launch() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// One sequence: its length within the table's room, pages, and block table.
struct Seq {
  int ctx, pages;
  const int* table;
};
__device__ __forceinline__ int pages_of(int ctx, int block_size) {  // 16 or 32
  return static_cast<int>((static_cast<unsigned>(ctx) + block_size - 1) >> (4 + (block_size >> 5)));
}
// Pages of a sequence of `ctx` tokens within the table's width.
__device__ __forceinline__ int pages_within(const SelectParams& p, int ctx) {
  return min(pages_of(max(0, ctx), p.block_size), p.width);
}
__device__ __forceinline__ Seq seq_of(const SelectParams& p, int seq) {
  Seq r;
  r.ctx = max(0, __ldg(p.context_lens + seq));
  const long long room = static_cast<long long>(p.width) * p.block_size;
  if (r.ctx > room) {
    if (threadIdx.x == 0) atomicOr(p.err, kErrBadBlock);
    r.ctx = static_cast<int>(room);
  }
  r.pages = pages_of(r.ctx, p.block_size);
  r.table = p.block_tables + static_cast<long long>(seq) * p.width;
  return r;
}

// A query head as whole numbers, one warp: [q+ | q-] of 2 D bytes, and (mul, add) that make
// a score of a sum: (2^eq, 0); with a NaN or an infinity (0, +inf); (0, -inf) without a
// query, the padding to 8 heads.
template <typename T, int D>
struct QueryHead {
  static constexpr int PW = 4 / sizeof(T);  // channels a word
  static constexpr int W = D / 32 / PW;     // words of a lane, 32 lanes side by side
  uint32_t raw[W];
  bool real;
  __device__ __forceinline__ void load(const T* q) {  // nullptr: no query
    real = q != nullptr;
    const uint32_t* w = reinterpret_cast<const uint32_t*>(q);
#pragma unroll
    for (int i = 0; i < W; ++i) raw[i] = real ? __ldg(w + i * 32 + (threadIdx.x & 31)) : 0;
  }
  __device__ __forceinline__ void store(signed char* out, float2* scale) const {
    const int lane = threadIdx.x & 31;
    if (!real) {
#pragma unroll
      for (int i = 0; i < D / 64; ++i)
        *reinterpret_cast<uint32_t*>(out + (i * 32 + lane) * 4) = 0;
      if (lane == 0) *scale = make_float2(0.f, -kInf);
      return;
    }
    float x[W][PW], amax = 0.f;
    bool fin = true;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if constexpr (PW == 1) {
        x[i][0] = __uint_as_float(raw[i]);
      } else {
        x[i][0] = static_cast<float>(reinterpret_cast<const T*>(&raw[i])[0]);
        x[i][1] = static_cast<float>(reinterpret_cast<const T*>(&raw[i])[1]);
      }
#pragma unroll
      for (int j = 0; j < PW; ++j) {
        fin = fin && is_finite(x[i][j]);
        amax = fmaxf(amax, fabsf(x[i][j]));
      }
    }
    // non-negative floats are ordered as their bits
    amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)));
    fin = __all_sync(0xffffffffu, fin);
    const int e = box_exponent(fin ? amax : 0.f);
    const float inv = exp2_int(-e);
#pragma unroll
    for (int i = 0; i < W; ++i) {
#pragma unroll
      for (int j = 0; j < PW; ++j) {
        const int at = (i * 32 + lane) * PW + j;
        const int v = fin ? __float2int_rn(x[i][j] * inv) : 0;
        out[at] = static_cast<signed char>(max(v, 0));
        out[D + at] = static_cast<signed char>(min(v, 0));
      }
    }
    if (lane == 0) *scale = fin ? make_float2(exp2_int(e), 0.f) : make_float2(0.f, kInf);
  }
};

// Keys of the 16 pages from `first` on into keys[0..15], 0 past the row's end, and of their
// two groups of 8 the largest key that is not always chosen into maxima[0..1], one warp.
// tile: the boxes of one head in shared memory, rows `pitch` bytes apart; an odd number of
// 64 bytes, so that a quarter warp's 16-byte reads (2 rows x 4 pieces) hit different banks.
// sc: the scale of page gq + 8 (cq & 1).
template <int D>
__device__ __forceinline__ void score_tile(const SelectParams& p, int pages,
                                           const unsigned char* tile, int pitch, float sc,
                                           const signed char* qrow, const float2* qscale, int GP,
                                           int first, unsigned* keys, unsigned* maxima) {
  constexpr int CH = 2 * D / 64;
  const int lane = threadIdx.x & 31, gq = lane >> 2, cq = lane & 3;
  uint4 a[2][CH];
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int i = 0; i < CH; ++i)
      a[k][i] = *reinterpret_cast<const uint4*>(tile + (gq + 8 * k) * pitch + (cq + 4 * i) * 16);
  float best[2] = {-kInf, -kInf};
  for (int h0 = 0; h0 < GP; h0 += 8) {
    int acc[2][4] = {};
    const uint4* qv = reinterpret_cast<const uint4*>(qrow + (h0 + gq) * 2 * D) + cq;
    // the k index of both operands is the byte's place in this lane's 16-byte pieces
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const uint4 v = qv[4 * i];
      mma_s8_16832(acc[0], a[0][i].x, a[1][i].x, a[0][i].y, a[1][i].y, v.x, v.y);
      mma_s8_16832(acc[1], a[0][i].z, a[1][i].z, a[0][i].w, a[1][i].w, v.z, v.w);
    }
    const float4 ms = *reinterpret_cast<const float4*>(qscale + h0 + 2 * cq);
#pragma unroll
    for (int k = 0; k < 2; ++k) {  // exact: a sum below 2^24 times a power of two, plus 0
      best[k] = fmaxf(best[k], fmaf(static_cast<float>(acc[0][2 * k] + acc[1][2 * k]), ms.x, ms.y));
      best[k] = fmaxf(best[k],
                      fmaf(static_cast<float>(acc[0][2 * k + 1] + acc[1][2 * k + 1]), ms.z, ms.w));
    }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    best[k] = fmaxf(best[k], __shfl_xor_sync(0xffffffffu, best[k], 1));
    best[k] = fmaxf(best[k], __shfl_xor_sync(0xffffffffu, best[k], 2));
  }
  // lanes with an even cq have page gq, those with an odd one page gq + 8
  const int at = gq + 8 * (cq & 1), j = first + at;
  const float mine = cq & 1 ? best[1] : best[0];
  unsigned key = page_key(mine, sc);
  const bool in = j < pages, kept = j < p.keep_first || j >= pages - p.keep_last;
  unsigned open = in && !kept ? key : 0;
  key = !in ? 0 : kept ? kForced : key;
  if (cq < 2) keys[at] = key;
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) open = max(open, __shfl_xor_sync(0xffffffffu, open, o));
  if (lane < 2) maxima[lane] = open;
}

template <int NTHR>
struct SelectShared {
  unsigned count[32];
  unsigned above[NTHR / 32], equal[NTHR / 32];
  int groups[NTHR];    // groups that matter
  unsigned key[NTHR];  // candidates, and the pages they are of
  int page[NTHR];
};

// The sum of a count over the block in turn `row`, each of which is used once after
// block_range.
template <int NW, typename Shared>
__device__ __forceinline__ unsigned block_count(Shared& sh, unsigned c, int row) {
  c = __reduce_add_sync(0xffffffffu, c);
  if constexpr (NW > 1) {
    if ((threadIdx.x & 31) == 0) atomicAdd(&sh.count[row], c);
    __syncthreads();
    c = sh.count[row];
  }
  return c;
}

// The smallest and the largest of a value of each thread over the block. Clears the counts.
template <int NW, typename Shared>
__device__ __forceinline__ void block_range(Shared& sh, unsigned& lo, unsigned& hi) {
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  if constexpr (NW > 1) {
    __syncthreads();  // sh.above, sh.equal and sh.count are read
    if ((threadIdx.x & 31) == 0) {
      sh.above[threadIdx.x >> 5] = lo;
      sh.equal[threadIdx.x >> 5] = hi;
    }
    if (threadIdx.x < 32) sh.count[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      lo = min(lo, sh.above[w]);
      hi = max(hi, sh.equal[w]);
    }
  }
}

// A threshold with at least K and at most `most` keys at or above it where there is one, else
// the K-th largest key. More than the always-chosen ones are wanted, so that it is one of
// the others, which lie between lo and hi. count(at): this thread's keys at or above `at`.
template <int NW, typename Shared, typename Count>
__device__ __forceinline__ unsigned find_threshold(Shared& sh, unsigned lo, unsigned hi,
                                                   unsigned K, unsigned most, Count count) {
  const int bits = 32 - __clz(lo ^ hi);  // those below the first one in which the keys differ
  unsigned thr = bits == 32 ? 0 : (hi >> bits) << bits;
  for (int bit = bits - 1; bit >= 0; --bit) {
    const unsigned at = thr | (1u << bit);
    const unsigned c = block_count<NW>(sh, count(at), bit);
    if (c >= K) {
      thr = at;
      if (c <= most) break;
    }
  }
  return thr;
}

// How many keys are above / equal to the threshold: in the warps before, and in all.
struct Before {
  unsigned above, equal, all_above, all_equal;
};
template <int NW, typename Shared>
__device__ __forceinline__ Before block_before(Shared& sh, unsigned above, unsigned equal) {
  above = __reduce_add_sync(0xffffffffu, above);
  equal = __reduce_add_sync(0xffffffffu, equal);
  Before b{0, 0, above, equal};
  if constexpr (NW > 1) {
    const int warp = threadIdx.x >> 5;
    __syncthreads();  // sh.above and sh.equal are read
    if ((threadIdx.x & 31) == 0) {
      sh.above[warp] = above;
      sh.equal[warp] = equal;
    }
    __syncthreads();
    b.all_above = b.all_equal = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      b.above += w < warp ? sh.above[w] : 0;
      b.equal += w < warp ? sh.equal[w] : 0;
      b.all_above += sh.above[w];
      b.all_equal += sh.equal[w];
    }
  }
  return b;
}

// 32 consecutive places of a warp: put(place in the list, i, k) where `k` is above thr, or
// equal to it and among the first `need` equal ones. b moves on past them.
template <typename Put>
__device__ __forceinline__ void list_32(Before& b, unsigned k, unsigned thr, unsigned need, int i,
                                        Put put) {
  const unsigned below = (1u << (threadIdx.x & 31)) - 1;
  const unsigned ma = __ballot_sync(0xffffffffu, k > thr);
  const unsigned me = __ballot_sync(0xffffffffu, k == thr);
  const unsigned e = b.equal + __popc(me & below);  // equal ones before this place
  if (k > thr || (k == thr && e < need))
    put(static_cast<int>(b.above + __popc(ma & below) + min(e, need)), i, k);
  b.above += __popc(ma);
  b.equal += __popc(me);
}

// Keys of up to NTHR * J places in registers: warp w holds places [32 J w, 32 J (w + 1)),
// lane l those with place % 32 == l.
template <int NTHR, int J>
struct KeyRegisters {
  static constexpr int NW = NTHR / 32;
  unsigned k[J];
  int first;
  template <typename Key>
  __device__ __forceinline__ void load(int n, Key key) {  // key(i): the key of place i < n
    first = (threadIdx.x >> 5) * 32 * J + (threadIdx.x & 31);
#pragma unroll
    for (int j = 0; j < J; ++j) k[j] = first + j * 32 < n ? key(first + j * 32) : 0;
  }
  template <typename Shared>
  __device__ __forceinline__ unsigned threshold(Shared& sh, unsigned K, unsigned most) const {
    unsigned lo = kForced, hi = 0;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (k[j] != 0) lo = min(lo, k[j]);
      if (k[j] != kForced) hi = max(hi, k[j]);
    }
    block_range<NW>(sh, lo, hi);
    return find_threshold<NW>(sh, lo, hi, K, most, [&](unsigned at) {
      unsigned c = 0;
#pragma unroll
      for (int j = 0; j < J; ++j) c += k[j] >= at;
      return c;
    });
  }
  template <typename Shared>
  __device__ __forceinline__ Before before(Shared& sh, unsigned thr) const {
    unsigned above = 0, equal = 0;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      above += k[j] > thr;
      equal += k[j] == thr;
    }
    return block_before<NW>(sh, above, equal);
  }
  template <typename Put>
  __device__ __forceinline__ void list(Before b, unsigned thr, unsigned need, Put put) const {
#pragma unroll
    for (int j = 0; j < J; ++j) list_32(b, k[j], thr, need, first + j * 32, put);
  }
};

// put(place, page) for the K best of n <= NTHR candidates in sh.key, one a thread, `rem` of
// them not kForced: the barrier itself counts.
template <int NTHR, typename Put>
__device__ __forceinline__ void choose_candidates(SelectShared<NTHR>& sh, int n, unsigned K,
                                                  unsigned rem, Put put) {
  constexpr int NW = NTHR / 32;
  const int tid = threadIdx.x;
  const unsigned k = tid < n ? sh.key[tid] : 0;
  unsigned thr = kForced - 1;
  if (rem > 0) {
    unsigned lo = k != 0 ? k : kForced, hi = k != kForced ? k : 0;
    block_range<NW>(sh, lo, hi);
    const int bits = 32 - __clz(lo ^ hi);
    thr = bits == 32 ? 0 : (hi >> bits) << bits;
    for (int bit = bits - 1; bit >= 0; --bit) {
      const unsigned at = thr | (1u << bit);
      const unsigned c = __syncthreads_count(k >= at);
      if (c >= K) {
        thr = at;
        if (c == K) break;
      }
    }
  }
  Before b = block_before<NW>(sh, k > thr, k == thr);
  list_32(b, k, thr, K - b.all_above, tid,
          [&](int at, int i, unsigned) { put(at, sh.page[i]); });
}

// put(place, i) for the K best of n places i in ascending order, `rem` of them not kForced.
template <int NTHR, int J, typename Shared, typename Key, typename Put>
__device__ __forceinline__ void choose_in_registers(Shared& sh, int n, unsigned K, unsigned rem,
                                                    Key key, Put put) {
  KeyRegisters<NTHR, J> r;
  r.load(n, key);
  unsigned thr = kForced - 1;
  if constexpr (NTHR > 32) {
    if (rem > 0 && K <= NTHR - NTHR / 8) {  // down to one candidate a thread first
      thr = r.threshold(sh, K, NTHR) - 1;
      const Before b = r.before(sh, thr);
      if (b.all_above <= NTHR) {
        r.list(b, thr, 0, [&](int at, int i, unsigned k) {
          sh.key[at] = k;
          sh.page[at] = i;
        });
        __syncthreads();
        return choose_candidates<NTHR>(sh, static_cast<int>(b.all_above), K, rem, put);
      }
    }
  }
  if (rem > 0) thr = r.threshold(sh, K, K);
  const Before b = r.before(sh, thr);
  r.list(b, thr, K - b.all_above, [&](int at, int i, unsigned) { put(at, i); });
}

// The groups of 8 pages that matter into sh.groups: those whose largest open key reaches a
// lower bound of the rem-th largest open key (thr), and those of always-chosen pages
// (outside [first_end, last_beg)). Returns their number, above NTHR where they do not fit.
template <int NTHR, int J>
__device__ __forceinline__ int find_groups(SelectShared<NTHR>& sh, const unsigned* gmaxima, int ng,
                                           unsigned rem, int first_end, int last_beg,
                                           unsigned& thr) {
  KeyRegisters<NTHR, J> m;
  m.load(ng, [&](int i) { return __ldcg(gmaxima + i); });
  thr = m.threshold(sh, rem, rem + rem / 4 + 8);
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int i = m.first + j * 32;
    if (i < ng && (i < first_end || i >= last_beg)) m.k[j] = kForced;
  }
  const Before b = m.before(sh, thr);
  const int listed = static_cast<int>(b.all_above + b.all_equal);
  if (listed <= NTHR) m.list(b, thr, b.all_equal, [&](int at, int i, unsigned) { sh.groups[at] = i; });
  __syncthreads();
  return listed;
}

// put(place, page) for the K chosen pages of a row (of more than K pages), in ascending order.
template <int NTHR, typename Put>
__device__ __forceinline__ void choose_pages(SelectShared<NTHR>& sh, const SelectParams& p,
                                             const Seq& r, const unsigned* gkeys,
                                             const unsigned* gmaxima, Put put) {
  constexpr int NW = NTHR / 32;
  const unsigned K = p.num_pages, rem = K - p.keep_first - p.keep_last;
  const int n = r.pages, ng = (n + kGroup - 1) / kGroup;
  auto key = [&](int i) { return __ldcg(gkeys + i); };
  if (n <= 256) {  // one warp: the barriers would cost more than the longer turns
    if (threadIdx.x >= 32) return;
    if (n <= 128) choose_in_registers<32, 4>(sh, n, K, rem, key, put);
    else choose_in_registers<32, 8>(sh, n, K, rem, key, put);
    return;
  }
  if (n <= NTHR * 3) return choose_in_registers<NTHR, 3>(sh, n, K, rem, key, put);
  if (n <= NTHR * 8) return choose_in_registers<NTHR, 8>(sh, n, K, rem, key, put);
  const int first_end = (p.keep_first + kGroup - 1) / kGroup;
  const int last_beg = (n - p.keep_last) / kGroup;
  if (rem > 0 && ng <= NTHR * 16 && static_cast<int>(rem) <= (last_beg - first_end) / 2) {
    unsigned bound;
    const int listed =
        ng <= NTHR * 3 ? find_groups<NTHR, 3>(sh, gmaxima, ng, rem, first_end, last_beg, bound)
        : ng <= NTHR * 8
            ? find_groups<NTHR, 8>(sh, gmaxima, ng, rem, first_end, last_beg, bound)
            : find_groups<NTHR, 16>(sh, gmaxima, ng, rem, first_end, last_beg, bound);
    if (listed <= NTHR) {
      // their keys that reach the bound, one a thread where they are few enough
      auto page = [&](int i) { return sh.groups[i / kGroup] * kGroup + i % kGroup; };
      KeyRegisters<NTHR, kGroup> k;
      k.load(listed * kGroup, [&](int i) { return key(page(i)); });
      const Before b = k.before(sh, bound - 1);
      if (b.all_above <= NTHR) {
        k.list(b, bound - 1, 0, [&](int at, int i, unsigned x) {
          sh.key[at] = x;
          sh.page[at] = page(i);
        });
        __syncthreads();
        return choose_candidates<NTHR>(sh, static_cast<int>(b.all_above), K, rem, put);
      }
    }
  }
  // all keys, read again for every bit
  unsigned thr = kForced - 1;
  if (rem > 0) {
    unsigned lo = kForced, hi = 0;
#pragma unroll 8
    for (int i = threadIdx.x; i < n; i += NTHR) {
      const unsigned k = key(i);
      lo = min(lo, k);
      if (k != kForced) hi = max(hi, k);
    }
    block_range<NW>(sh, lo, hi);
    thr = find_threshold<NW>(sh, lo, hi, K, K, [&](unsigned at) {
      unsigned c = 0;
#pragma unroll 8
      for (int i = threadIdx.x; i < n; i += NTHR) c += key(i) >= at;
      return c;
    });
  }
  // each warp lists a range of them
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int span = ((n + NW - 1) / NW + 31) / 32 * 32;
  const int beg = min(n, warp * span), end = min(n, beg + span);
  unsigned above = 0, equal = 0;
#pragma unroll 8
  for (int i = beg + lane; i < end; i += 32) {
    const unsigned k = key(i);
    above += k > thr;
    equal += k == thr;
  }
  Before b = block_before<NW>(sh, above, equal);
  const unsigned need = K - b.all_above;
  for (int i = beg; i < end; i += 32)
    list_32(b, i + lane < end ? key(i + lane) : 0, thr, need, i + lane,
            [&](int at, int j, unsigned) { put(at, j); });
}

// ---------------------------------------------------------------------------
// Scores of all pages into p.keys [rows, key_stride] and p.maxima [rows, key_stride / 8].
// CTA x takes an equal share of the 16-page tiles of all sequences with more than num_pages
// pages, blockIdx.y a group of KV heads (a power of two). A producer warp copies each
// block's boxes of all these heads, which are neighbours in memory, with one bulk copy into
// a ring of tiles; consumer warp w scores head w % head_group of every (16 / head_group)th
// tile. A tile's place in the ring always belongs to the same consumer warps (`stages` is a
// multiple of 16 / head_group), so a parity wait cannot be satisfied by an older phase.
// HBM bound once it streams: four contexts of 131072 tokens (67 MB of boxes) take 14 us, of
// which 1.2 go to the prefix sum and 3 to the block table, the query and the first tiles;
// then a CTA takes 46 GB/s, 6.8 TB/s in all. A change of the sequence inside a CTA's share
// costs it 2 us, its query's (3.5 with its length, table and scales loaded only then). With
// the boxes read into registers, one row a CTA, the launch took 20 us: 256-byte reads of one
// head at a time, and two tiles a warp in flight.
template <typename T, int D>
__global__ void __launch_bounds__(32 * (kScoreWarps + 1), 1)
    page_score_kernel(const SelectParams p, int head_group, int stages) {
  constexpr int NW = kScoreWarps, NTH = 32 * (NW + 1);
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ int warp_tot[NW + 1];
  __shared__ uint64_t full[kScoreStages], empty[kScoreStages];
  __shared__ int dead;  // a wait ran out
  const int G = p.heads / p.kv_heads, GP = (G + 7) / 8 * 8;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int pitch = head_group * 2 * D + 64;  // bytes of a page's boxes in the ring
  unsigned char* ring = dyn;
  signed char* qrow = reinterpret_cast<signed char*>(dyn + stages * 16 * pitch);
  // two sequences' query rows
  float2* qscale = reinterpret_cast<float2*>(qrow + 2 * head_group * GP * 2 * D);
  int* pre = reinterpret_cast<int*>(qscale + 2 * head_group * GP);  // [S + 1] tiles before
  const int head0 = blockIdx.y * head_group, nh = min(head_group, p.kv_heads - head0);
  if (tid == 0) {
    dead = 0;
    for (int i = 0; i < stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], nh);
    }
    fence_mbar_init();
  }
  griddep_launch();  // the next kernel's CTAs take the SMs as this one's leave them
  griddep_wait();
  // prefix sum of the tiles: a contiguous range of sequences a thread
  {
    auto count = [&](int i) {
      const int pages = pages_within(p, __ldg(p.context_lens + i));
      return pages > p.num_pages ? (pages + 15) / 16 : 0;
    };
    const int per = (p.num_seqs + NTH - 1) / NTH;
    const int b0 = min(p.num_seqs, tid * per), b1 = min(p.num_seqs, b0 + per);
    int local = 0;
    for (int i = b0; i < b1; ++i) local += count(i);
    int inc = local;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) warp_tot[warp] = inc;
    __syncthreads();
    int run = inc - local, all = 0;
#pragma unroll
    for (int w = 0; w <= NW; ++w) {
      run += w < warp ? warp_tot[w] : 0;
      all += warp_tot[w];
    }
    for (int i = b0; i < b1; ++i) {
      pre[i] = run;
      run += count(i);
    }
    if (tid == 0) pre[p.num_seqs] = all;
    __syncthreads();
  }
  const int total = pre[p.num_seqs];
  const unsigned each = static_cast<unsigned>(total) / gridDim.x, more = total - each * gridDim.x;
  // total * x / grid: where the sequences are equal and their number divides the grid, none
  // of them changes inside a CTA's share
  int at = each * blockIdx.x + more * blockIdx.x / gridDim.x;
  const int stop = each * (blockIdx.x + 1) + more * (blockIdx.x + 1) / gridDim.x;
  if (at >= stop) return;
  // the sequence of tile `at`: the last one that starts at or before it
  int seq = 0, hi = p.num_seqs;
  while (hi - seq > 1) {
    const int mid = (seq + hi) >> 1;
    if (pre[mid] <= at) seq = mid; else hi = mid;
  }
  int slot = 0, phase = 0;  // of tile `at`
  while (pre[seq + 1] <= at) ++seq;

  // The table's entry for page j, looked at when it is used: nothing waits for a load that is
  // for later. Past the sequence's pages it may be anything; an entry out of range counts as
  // block 0 here (it is flagged where the page is listed).
  auto entry = [&](int sq, int j) {
    return j < p.width ? __ldg(p.block_tables + static_cast<long long>(sq) * p.width + j) : 0;
  };
  // the first of this CTA's boxes and scales of a block
  auto box_of = [&](int b) {
    return static_cast<long long>(b < 0 || b >= p.num_blocks ? 0 : b) * p.kv_heads + head0;
  };

  if (warp == NW) {
    // ---- producer: two tiles a step, lanes 0..15 the first one's pages, the others the next
    const uint64_t policy = l2_policy_evict_first();
    const uint32_t bytes = nh * 2 * D;
    // for this lane's page of tiles t and t + 1
    auto mine = [&](int sq, int t) { return entry(sq, t * 16 + lane); };
    int t0 = at - pre[seq];
    int b0 = mine(seq, t0), b1 = mine(seq, t0 + 2), b2 = mine(seq, t0 + 4);
    while (true) {
      const int t1 = min(stop, pre[seq + 1]) - pre[seq];
      at += t1 - t0;
      // the next sequence's first entries are on their way while this one's tiles are copied
      int next = seq, n0 = 0, n1 = 0, n2 = 0;
      if (at < stop) {
        while (pre[next + 1] <= at) ++next;
        n0 = mine(next, 0);
        n1 = mine(next, 2);
        n2 = mine(next, 4);
      }
      for (int t = t0; t < t1; t += 2) {
        const signed char* src = p.values + box_of(b0) * (2 * D);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if (t + k >= t1) break;
          const bool free_ =
              __all_sync(0xffffffffu, mbar_wait(&empty[slot], (phase & 1) ^ 1));
          if (!free_) {
            if (lane == 0) atomicOr(p.err, kErrWaitTimeout);
            return;  // the consumers' waits run out too, after the copies in flight
          }
          if (lane == 0) mbar_arrive_expect_tx(&full[slot], 16 * bytes);
          __syncwarp();
          if (lane >> 4 == k)
            bulk_load(ring + (slot * 16 + (lane & 15)) * pitch, src, bytes, &full[slot], policy);
          if (++slot == stages) {
            slot = 0;
            ++phase;
          }
        }
        b0 = b1;
        b1 = b2;
        b2 = t + 6 < t1 ? mine(seq, t + 6) : 0;
      }
      if (at >= stop) return;
      seq = next;
      t0 = 0;
      b0 = n0;
      b1 = n1;
      b2 = n2;
    }
  }

  // ---- consumers
  const int head = warp % head_group, group = warp / head_group, step = NW / head_group;
  const int gq = lane >> 2, cq = lane & 3, page_at = gq + 8 * (cq & 1);
  // the query rows of a sequence into buffer `buf`
  auto query = [&](int sq, int buf) {
    const T* q = static_cast<const T*>(p.q) + (static_cast<long long>(sq) * p.heads + head0 * G) * D;
    auto head_of = [&](int i) {
      const int h = i / GP, g = i - h * GP;
      return i < nh * GP && g < G ? q + (h * G + g) * D : nullptr;
    };
    signed char* rows = qrow + buf * head_group * GP * 2 * D;
    float2* scales = qscale + buf * head_group * GP;
    for (int i = warp; i < nh * GP; i += 4 * NW) {
      QueryHead<T, D> qh[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) qh[k].load(head_of(i + k * NW));
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + k * NW < nh * GP) qh[k].store(rows + (i + k * NW) * 2 * D, scales + i + k * NW);
    }
  };
  auto scale_of = [&](int b) { return __ldg(p.scales + box_of(b) + min(head, nh - 1)); };
  // this warp's first tile: its ring places are those with slot % step == group
  auto skip_at = [&](int slot) { return (group - slot % step + step) % step; };
  int t0 = at - pre[seq], skip = skip_at(slot), ctx = __ldg(p.context_lens + seq);
  int b1 = entry(seq, (t0 + skip) * 16 + page_at);
  int b2 = entry(seq, (t0 + skip + step) * 16 + page_at);
  for (int buf = 0;; buf ^= 1) {
    const int t1 = min(stop, pre[seq + 1]) - pre[seq], n = slot + t1 - t0;
    float sc = scale_of(b1);
    query(seq, buf);  // the other buffer was read before the last barrier but one
    at += t1 - t0;
    // the next sequence's length and first entries are on their way while this one is scored
    int next = seq, next_ctx = 0, n1 = 0, n2 = 0;
    const int next_skip = skip_at(n % stages);
    if (at < stop) {
      while (pre[next + 1] <= at) ++next;
      next_ctx = __ldg(p.context_lens + next);
      n1 = entry(next, next_skip * 16 + page_at);
      n2 = entry(next, (next_skip + step) * 16 + page_at);
    }
    const int end = head < nh ? t1 : 0, pages = pages_within(p, ctx);
    const signed char* qr = qrow + (buf * head_group + head) * GP * 2 * D;
    const float2* qs = qscale + (buf * head_group + head) * GP;
    const long long row = static_cast<long long>(seq) * p.kv_heads + head0 + head;
    unsigned* keys = p.keys + row * p.key_stride;
    unsigned* maxima = p.maxima + row * (p.key_stride / kGroup);
    int s = slot + skip, ph = phase;
    if (s >= stages) {
      s -= stages;
      ++ph;
    }
    named_bar(1, NW * 32);  // this sequence's query rows are there
    for (int t = t0 + skip; t < end; t += step) {
      const float sc_next = scale_of(b2);
      b2 = t + 2 * step < end ? entry(seq, (t + 2 * step) * 16 + page_at) : 0;
      const bool ok = __all_sync(
          0xffffffffu, *static_cast<volatile int*>(&dead) == 0 && mbar_wait(&full[s], ph & 1));
      if (!ok && lane == 0) {
        dead = 1;
        atomicOr(p.err, kErrWaitTimeout);
      }
      if (ok) {
        score_tile<D>(p, pages, ring + s * 16 * pitch + head * 2 * D, pitch, sc,
                      qr, qs, GP, t * 16, keys + t * 16, maxima + t * 2);
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[s]);
      }
      sc = sc_next;
      s += step;
      if (s >= stages) {
        s -= stages;
        ++ph;
      }
    }
    if (at >= stop) return;
    slot = n % stages;
    phase += n / stages;
    seq = next;
    ctx = next_ctx;
    skip = next_skip;
    t0 = 0;
    b1 = n1;
    b2 = n2;
  }
}

// ---------------------------------------------------------------------------
// Attention of one warp over 16-token pieces of the chosen pages, heads in groups of 8.
template <typename T, int D, int NT>
struct WarpAttention {
  static constexpr int KC = D / 32;  // 16-byte pieces of a key row a lane holds
  static constexpr int VH = D / 64;  // 64-channel halves of a value row
  uint4 q[NT][KC];
  uint4 k[2][KC];       // tokens g and g + 8
  uint4 v[VH][4];       // tokens 2c, 2c + 1, 2c + 8, 2c + 9, channels 8g..8g+7
  float o[VH * 4][NT][4];
  float m[NT][2], l[NT][2];

  __device__ __forceinline__ void init(const T* query, int G) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        q[nt][i] = make_uint4(0, 0, 0, 0);
        if (nt * 8 + g < G) {  // rows are 4-byte aligned at least
          const uint32_t* w =
              reinterpret_cast<const uint32_t*>(query + (nt * 8 + g) * D + (c + 4 * i) * 8);
          q[nt][i] = make_uint4(__ldg(w), __ldg(w + 1), __ldg(w + 2), __ldg(w + 3));
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        m[nt][j] = -kInf;
        l[nt][j] = 0.f;
      }
#pragma unroll
      for (int t = 0; t < VH * 4; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[t][nt][j] = 0.f;
    }
  }
  __device__ __forceinline__ void load_k(const T* rows) {  // [16, D]
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      k[0][i] = ld_once(rows + g * D + (c + 4 * i) * 8);
      k[1][i] = ld_once(rows + (g + 8) * D + (c + 4 * i) * 8);
    }
  }
  // Rows past the sequence's end are zeros: their weights are 0, and 0 * NaN is not.
  __device__ __forceinline__ void load_v(const T* rows, int limit) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int h = 0; h < VH; ++h)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int tok = 2 * c + (t & 1) + (t >> 1) * 8;
        v[h][t] = tok < limit ? ld_once(rows + tok * D + h * 64 + g * 8) : make_uint4(0, 0, 0, 0);
      }
  }
  // s[nt] = scores of tokens g (0, 1) and g + 8 (2, 3) with heads 2c and 2c + 1.
  __device__ __forceinline__ void scores(float (&s)[NT][4]) const {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < 4; ++j) s[nt][j] = 0.f;
      // the k index of both operands is the channel's place in this lane's 16-byte pieces
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        mma_16816<T>(s[nt], k[0][i].x, k[1][i].x, k[0][i].y, k[1][i].y, q[nt][i].x, q[nt][i].y);
        mma_16816<T>(s[nt], k[0][i].z, k[1][i].z, k[0][i].w, k[1][i].w, q[nt][i].z, q[nt][i].w);
      }
    }
  }
  // Folds 16 tokens (those below limit) into (m, l, O).
  __device__ __forceinline__ void weights(float (&s)[NT][4], int limit, float scale_log2,
                                          uint32_t (&b)[NT][2]) {
    const int lane = threadIdx.x & 31, g = lane >> 2;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      bool grew = false;
      float alpha[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        s[nt][j] = g < limit ? s[nt][j] * scale_log2 : -kInf;
        s[nt][2 + j] = g + 8 < limit ? s[nt][2 + j] * scale_log2 : -kInf;
        float mx = fmaxf(s[nt][j], s[nt][2 + j]);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float mn = fmaxf(m[nt][j], mx);
        const float base = mn == -kInf ? 0.f : mn;
        alpha[j] = ex2(m[nt][j] - base);
        grew = grew || mn > m[nt][j];
        m[nt][j] = mn;
        s[nt][j] = ex2(s[nt][j] - base);
        s[nt][2 + j] = ex2(s[nt][2 + j] - base);
        l[nt][j] = l[nt][j] * alpha[j] + s[nt][j] + s[nt][2 + j];
      }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int t = 0; t < VH * 4; ++t) {
          o[t][nt][0] *= alpha[0];
          o[t][nt][1] *= alpha[1];
          o[t][nt][2] *= alpha[0];
          o[t][nt][3] *= alpha[1];
        }
      }
      // tokens x heads -> heads x tokens
      b[nt][0] = movmatrix_t(pack2<T>(s[nt][0], s[nt][1]));
      b[nt][1] = movmatrix_t(pack2<T>(s[nt][2], s[nt][3]));
    }
  }
  // O^T += V^T P^T. Row g of product 4h + w is channel 64h + 8g + 2w, row g + 8 the next one:
  // a lane's own 16 bytes, two tokens of a channel put together by byte permutes.
  __device__ __forceinline__ void accumulate(const uint32_t (&b)[NT][2]) {
#pragma unroll
    for (int h = 0; h < VH; ++h) {
      const uint32_t w[4][4] = {{v[h][0].x, v[h][0].y, v[h][0].z, v[h][0].w},
                                {v[h][1].x, v[h][1].y, v[h][1].z, v[h][1].w},
                                {v[h][2].x, v[h][2].y, v[h][2].z, v[h][2].w},
                                {v[h][3].x, v[h][3].y, v[h][3].z, v[h][3].w}};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a0 = __byte_perm(w[0][i], w[1][i], 0x5410);
        const uint32_t a1 = __byte_perm(w[0][i], w[1][i], 0x7632);
        const uint32_t a2 = __byte_perm(w[2][i], w[3][i], 0x5410);
        const uint32_t a3 = __byte_perm(w[2][i], w[3][i], 0x7632);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          mma_16816<T>(o[h * 4 + i][nt], a0, a1, a2, a3, b[nt][0], b[nt][1]);
      }
    }
  }
  // This warp's (m, l) and O rows [8 NT][D + 4] into shared memory.
  __device__ __forceinline__ void store(float* om, float* ol, float* oo) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float x = l[nt][j];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        const int head = nt * 8 + 2 * c + j;
        if (g == 0) {
          om[head] = m[nt][j];
          ol[head] = x;
        }
#pragma unroll
        for (int h = 0; h < VH; ++h) {
          float4* dst = reinterpret_cast<float4*>(oo + head * (D + 4) + h * 64 + g * 8);
          dst[0] = make_float4(o[h * 4][nt][j], o[h * 4][nt][2 + j], o[h * 4 + 1][nt][j],
                               o[h * 4 + 1][nt][2 + j]);
          dst[1] = make_float4(o[h * 4 + 2][nt][j], o[h * 4 + 2][nt][2 + j], o[h * 4 + 3][nt][j],
                               o[h * 4 + 3][nt][2 + j]);
        }
      }
  }
};

// The factor of a part (m, l, O) in a join with maximum M. A part without tokens has m = -inf
// and l = 0; one whose scores are all -inf or NaN keeps its own NaN.
__device__ __forceinline__ float join_weight(float m, float l, float M) {
  return m == -kInf ? (l != 0.f ? 1.f : 0.f) : ex2(m - M);
}
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}

// Bytes of the warps' partial results.
template <int D, int NT, int NTHR>
constexpr int merge_bytes() {
  return NTHR / 32 * 8 * NT * (D + 4 + 2) * 4;
}

// Byte offsets of the fused kernel's shared memory after the warps' partial results.
struct SparseSmem {
  int chosen, got, total;
};

// Selection and attention of one (sequence, KV head) by a cluster of `ctas` CTAs. Of 24 us for
// four contexts of 131072 tokens and 256 pages (67 MB of keys and values), the choice takes
// 6.4, the attention 13 (5 TB/s on 128 SMs) and the joins 2.7; 512 rows of 64 pages (268 MB)
// take 47 us in the attention, 5.7 TB/s.
template <typename T, int D, int NT, int NTHR>
__global__ void __launch_bounds__(NTHR, NT == 2 ? 1 : 512 / NTHR) sparse_decode_kernel(const SelectParams p, int ctas, const SparseSmem lay) {
  constexpr int NW = NTHR / 32, HP = 8 * NT;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ SelectShared<NTHR> sh;
  int* chosen = reinterpret_cast<int*>(dyn + lay.chosen);  // [num_pages]
  float* got_m = reinterpret_cast<float*>(dyn + lay.got);  // [ctas][HP] of every CTA
  float* got_l = got_m + ctas * HP;
  float* got_o = got_l + ctas * HP;  // [ctas][share] of this CTA's share of the output
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, warp = tid >> 5;
  const int row = blockIdx.x / ctas, rank = blockIdx.x % ctas;
  const int seq = row / p.kv_heads, kvh = row - seq * p.kv_heads;
  const int G = p.heads / p.kv_heads, K = p.num_pages;
  if (ctas > 1) cluster_arrive();  // waited for before the first store to another CTA
  griddep_wait();
  const Seq r = seq_of(p, seq);
  const int P = r.pages, n = min(P, K);
  int* sel = p.selected + static_cast<long long>(row) * K;

  WarpAttention<T, D, NT> w;
  w.init(static_cast<const T*>(p.q) + (static_cast<long long>(seq) * p.heads + kvh * G) * D, G);

  // ---- the chosen pages, in every CTA's shared memory
  if (P > K) {
    auto put = [&](int at, int page) {
      chosen[at] = page;
      if (rank == 0) sel[at] = page;
    };
    choose_pages<NTHR>(sh, p, r, p.keys + row * p.key_stride,
                       p.maxima + row * (p.key_stride / kGroup), put);
  } else {
    for (int i = tid; i < K; i += NTHR) {
      if (i < P) chosen[i] = i;
      if (rank == 0) sel[i] = i < P ? i : -1;
    }
  }
  __syncthreads();

  // ---- this CTA's share of them
  const int lg = 31 - __clz(ctas);  // ctas is a power of two, n at most kMaxFusedPages
  const int beg = n * rank >> lg, end = n * (rank + 1) >> lg;
  const int spp = p.block_size / 16, pieces = (end - beg) * spp;
  const T* kc = static_cast<const T*>(p.k_cache);
  const T* vc = static_cast<const T*>(p.v_cache);
  // rows of piece u and the tokens in it
  auto locate = [&](int u, long long& at, int& limit) {
    const int i = u >> (spp >> 1), half_ = u - i * spp;  // spp is 1 or 2
    const int page = chosen[beg + i];
    const int b = __ldg(r.table + page);
    limit = r.ctx - page * p.block_size - half_ * 16;
    if (b < 0 || b >= p.num_blocks) {
      if ((tid & 31) == 0) atomicOr(p.err, kErrBadBlock);
      limit = 0;
      at = 0;
      return;
    }
    at = ((static_cast<long long>(b) * p.kv_heads + kvh) * p.block_size + half_ * 16) * D;
  };
  {
    long long at = 0, at_next = 0;
    int limit = 0, limit_next = 0;
    int u = warp;
    if (u < pieces) {
      locate(u, at, limit);
      w.load_k(kc + at);
      w.load_v(vc + at, limit);
    }
    if (u + NW < pieces) locate(u + NW, at_next, limit_next);
    for (; u < pieces; u += NW) {
      float s[NT][4];
      uint32_t b[NT][2];
      w.scores(s);
      const bool more = u + NW < pieces;
      if (more) w.load_k(kc + at_next);
      if (limit > 0) {
        w.weights(s, limit, p.scale_log2, b);
        w.accumulate(b);
      }
      if (more) w.load_v(vc + at_next, limit_next);
      at = at_next;
      limit = limit_next;
      if (u + 2 * NW < pieces) locate(u + 2 * NW, at_next, limit_next);
    }
  }

  // ---- joined over the warps, then over the cluster
  float* om = reinterpret_cast<float*>(dyn);  // [NW][HP]
  float* ol = om + NW * HP;                   // [NW][HP]
  float* oo = ol + NW * HP;                   // [NW][HP][D + 4]
  w.store(om + warp * HP, ol + warp * HP, oo + warp * HP * (D + 4));
  __syncthreads();
  T* out = static_cast<T*>(p.out) +
           (static_cast<long long>(seq) * p.heads + kvh * G) * D;
  const int share = (G * D + ctas - 1) / ctas;
  if (ctas > 1) cluster_wait();  // every CTA runs: its shared memory takes stores
  for (int i = tid; i < G * D; i += NTHR) {
    const int h = i / D, d = i - h * D;
    float M = -kInf, L = 0.f, O = 0.f;
#pragma unroll
    for (int x = 0; x < NW; ++x) M = fmaxf(M, om[x * HP + h]);
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      const float f = join_weight(om[x * HP + h], ol[x * HP + h], M);
      L += ol[x * HP + h] * f;
      O += oo[(x * HP + h) * (D + 4) + d] * f;
    }
    if (ctas == 1) {
      out[i] = static_cast<T>(n > 0 ? O / L : 0.f);
    } else {
      const int to = i / share;
      cluster.map_shared_rank(got_o, to)[rank * share + i - to * share] = O;
      if (d < ctas) {
        cluster.map_shared_rank(got_m, d)[rank * HP + h] = M;
        cluster.map_shared_rank(got_l, d)[rank * HP + h] = L;
      }
    }
  }
  if (ctas == 1) return;
  cluster.sync();  // all stores to this CTA have arrived, and nothing else will
  for (int k = tid; k < share && rank * share + k < G * D; k += NTHR) {
    const int i = rank * share + k, h = i / D;
    float M = -kInf, L = 0.f, O = 0.f;
    for (int c = 0; c < ctas; ++c) M = fmaxf(M, got_m[c * HP + h]);
    for (int c = 0; c < ctas; ++c) {
      const float f = join_weight(got_m[c * HP + h], got_l[c * HP + h], M);
      L += got_l[c * HP + h] * f;
      O += got_o[c * share + k] * f;
    }
    out[i] = static_cast<T>(n > 0 ? O / L : 0.f);
  }
}

// ---------------------------------------------------------------------------
// Selection alone, a CTA a row: the block table (block * Hkv + head) and the length that
// paged_decode.cu runs over.
template <int NTHR>
__global__ void __launch_bounds__(NTHR) page_select_kernel(const SelectParams p) {
  __shared__ SelectShared<NTHR> sh;
  const int tid = threadIdx.x, row = blockIdx.x, K = p.num_pages;
  const int seq = row / p.kv_heads, kvh = row - seq * p.kv_heads;
  griddep_wait();
  const Seq r = seq_of(p, seq);
  int* sel = p.selected + static_cast<long long>(row) * K;
  int* blocks = p.sel_blocks + static_cast<long long>(row) * K;
  auto block = [&](int page) {
    const int b = __ldg(r.table + page);
    const bool ok = b >= 0 && b < p.num_blocks;
    if (!ok) atomicOr(p.err, kErrBadBlock);
    return ok ? b * p.kv_heads + kvh : -1;
  };
  const int P = r.pages;
  if (tid == 0)
    p.sel_lens[row] = P <= K ? r.ctx : (K - 1) * p.block_size + r.ctx - (P - 1) * p.block_size;
  if (P <= K) {
    for (int i = tid; i < K; i += NTHR) {
      sel[i] = i < P ? i : -1;
      if (i < P) blocks[i] = block(i);
    }
    return;
  }
  auto put = [&](int at, int page) { sel[at] = page; };
  choose_pages<NTHR>(sh, p, r, p.keys + row * p.key_stride,
                     p.maxima + row * (p.key_stride / kGroup), put);
  __syncthreads();  // the list is written, and read back by its CTA
#pragma unroll 4
  for (int i = tid; i < K; i += NTHR) blocks[i] = block(sel[i]);
}

// ---------------------------------------------------------------------------
// host launch

// Ints of a row's keys (whole 16-page tiles), and of all keys and maxima.
static long long key_stride(int width) { return (width + 15LL) / 16 * 16; }
long long sparse_key_ints(long long rows, int width) {
  return rows * (key_stride(width) + key_stride(width) / kGroup);
}

bool sparse_fused(const SelectParams& p, int dtype, int kv_layout) {
  return dtype != paged::kF32 && kv_layout == paged::kKvFlat && p.heads / p.kv_heads <= 16 &&
         p.num_pages <= kMaxFusedPages;
}

// Every kernel waits for its predecessor before it reads anything, so they may all be
// placed while it finishes. Only the score kernel lets its successor be placed early, which
// is one of this file.
static void launch_config(cudaLaunchConfig_t& cfg, cudaLaunchAttribute* attr, long long grid,
                          int threads, int smem, int ctas, cudaStream_t st) {
  cfg = cudaLaunchConfig_t{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (ctas > 1) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
}

template <typename T, int D>
static cudaError_t launch_scores(const SelectParams& all, cudaStream_t st) {
  auto kern = page_score_kernel<T, D>;
  const int G = all.heads / all.kv_heads, GP = (G + 7) / 8 * 8;
  // KV heads of a CTA, a power of two: 8 (whose boxes fill 2 KB of memory), fewer where
  // there are fewer or where their query rows would take more than 16 KB
  int hg = 8;
  while (hg > 1 && (hg / 2 >= all.kv_heads || hg * GP * 2 * D > 16384)) hg /= 2;
  const int groups = (all.kv_heads + hg - 1) / hg;
  const int pitch = hg * 2 * D + 64, step = kScoreWarps / hg;
  const int stages = std::min(kScoreStages, kScoreRing / (16 * pitch)) / step * step;
  for (int s0 = 0; s0 < all.num_seqs; s0 += kScoreSeqs) {
    SelectParams p = all;
    p.num_seqs = std::min(kScoreSeqs, all.num_seqs - s0);
    p.q = static_cast<const T*>(all.q) + static_cast<long long>(s0) * all.heads * D;
    p.context_lens += s0;
    p.block_tables += static_cast<long long>(s0) * all.width;
    p.keys += static_cast<long long>(s0) * all.kv_heads * all.key_stride;
    p.maxima += static_cast<long long>(s0) * all.kv_heads * (all.key_stride / kGroup);
    const int smem = stages * 16 * pitch + 2 * hg * GP * (2 * D + 8) + (p.num_seqs + 1) * 4;
    const cudaError_t e = ensure_smem_optin(reinterpret_cast<const void*>(kern), smem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr[2];
    launch_config(cfg, attr, std::max(1, sm_count() / groups), 32 * (kScoreWarps + 1), smem, 1,
                  st);
    cfg.gridDim.y = groups;
    const cudaError_t l = cudaLaunchKernelEx(&cfg, kern, p, hg, stages);
    if (l != cudaSuccess) return l;
  }
  return cudaSuccess;
}

template <typename T, int D, int NT, int NTHR>
static cudaError_t launch_fused(const SelectParams& p, int ctas, cudaStream_t st) {
  auto kern = sparse_decode_kernel<T, D, NT, NTHR>;
  const int share = (p.heads / p.kv_heads * D + ctas - 1) / ctas;
  SparseSmem lay;
  lay.chosen = (merge_bytes<D, NT, NTHR>() + 15) / 16 * 16;
  lay.got = lay.chosen + (p.num_pages + 3) / 4 * 16;
  lay.total = lay.got + (ctas > 1 ? ctas * (share + 16 * NT) * 4 : 0);
  const cudaError_t e = ensure_smem_optin(reinterpret_cast<const void*>(kern), lay.total);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[2];
  launch_config(cfg, attr, static_cast<long long>(p.num_seqs) * p.kv_heads * ctas, NTHR, lay.total,
                ctas, st);
  return cudaLaunchKernelEx(&cfg, kern, p, ctas, lay);
}

static cudaError_t launch_select(const SelectParams& p, cudaStream_t st) {
  constexpr int NTHR = 512;
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[2];
  launch_config(cfg, attr, static_cast<long long>(p.num_seqs) * p.kv_heads, NTHR, 0, 1, st);
  return cudaLaunchKernelEx(&cfg, page_select_kernel<NTHR>, p);
}

template <typename T, int D>
static cudaError_t launch_d(SelectParams& p, bool fused, cudaStream_t st) {
  p.key_stride = key_stride(p.width);
  p.maxima = p.keys + p.key_stride * p.num_seqs * p.kv_heads;
  const cudaError_t e = launch_scores<T, D>(p, st);
  if (e != cudaSuccess) return e;
  if constexpr (!std::is_same<T, float>::value) {
    if (fused) {
      // CTAs a row: enough to fill the GPU, with 4 pieces of 16 tokens each at least
      const long long rows = static_cast<long long>(p.num_seqs) * p.kv_heads;
      int ctas = 1;
      while (ctas < kMaxCtas && rows * ctas * 2 <= sm_count() &&
             p.num_pages * (p.block_size / 16) >= 4 * ctas)
        ctas *= 2;
      if (p.heads / p.kv_heads > 8) return launch_fused<T, D, 2, 256>(p, ctas, st);
      // more rows than SMs: four CTAs of 4 warps an SM, so that one's choice runs beside
      // the others' copies (batch of 64 mixed contexts: 76 us; 90 us with two of 8 warps)
      if (rows * ctas > sm_count()) return launch_fused<T, D, 1, 128>(p, ctas, st);
      return launch_fused<T, D, 1, 512>(p, ctas, st);
    }
  }
  return launch_select(p, st);
}

template <typename T>
static cudaError_t launch_t(SelectParams& p, int d, bool fused, cudaStream_t st) {
  if (d == 64) return launch_d<T, 64>(p, fused, st);
  if (d == 128) return launch_d<T, 128>(p, fused, st);
  return cudaErrorInvalidValue;
}

cudaError_t launch_sparse(SelectParams p, int d, int dtype, bool fused, cudaStream_t st) {
  if (dtype == paged::kBf16) return launch_t<__nv_bfloat16>(p, d, fused, st);
  if (dtype == paged::kF16) return launch_t<half>(p, d, fused, st);
  if (dtype == paged::kF32) return launch_t<float>(p, d, fused, st);
  return cudaErrorInvalidValue;
}

}  // namespace step
}  // namespace fe
