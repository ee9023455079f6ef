// Sparse paged decode: every page of a sequence is scored against the query through the
// int8 box of its keys (page_bounds.cu), the num_pages best of each KV head are chosen, and
// the query's heads attend to those.
//
// Score. The query is rounded to whole numbers like a box: qi = round(q / 2^eq), eq the
// smallest exponent with amax(q) <= 127 * 2^eq. With box [lo, hi] 2^ek,
//   score(page) = max over the group's heads of  sum_c max(qi_c hi_c, qi_c lo_c) 2^eq 2^ek,
// an upper bound of the rounded query's product with every key of the page. Since
// max(q hi, q lo) = q+ hi + q- lo, the sum is a product of the int8 row [q+ | q-] with the
// stored row [hi | lo] and runs on the integer tensor path, 16 pages x 8 heads an
// instruction. It is a whole number below 2^24 (256 terms at most of 127 * 127), so fp32
// holds it exactly, the powers of two scale it exactly, and the choice of pages does not
// depend on the order of any sum. Ties go to the lower page. The first keep_first and the
// last keep_last pages are always chosen; the last one may be partly filled.
//
// Attention. Softmax over the chosen pages' tokens with a running maximum and sum a warp,
// in fp32; the weights are rounded to the element type for the product with V, as in
// paged_decode.cu.
//
// One launch where the block tables are at most kOnePassPages wide: a cluster of CTAs
// serves one (sequence, KV head). Each scores a share of the pages and stores the keys
// (scores as ordered 32-bit words) into the shared memory of all; each then finds the
// threshold by itself from histograms of its copy, lists the chosen pages, attends to its
// share of them, and the partial (m, l, O) are joined over distributed shared memory.
// Wider tables take a launch of their own for the scores, cut into 256-page pieces whatever
// the lengths of the sequences, with the keys in global memory.
//
// fp32 caches, the x-packed layout and groups of more than 16 heads take the same
// selection, which then writes a block table for each (sequence, KV head) that
// paged_decode.cu runs over.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <limits.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "internal.h"
#include "page_box.cuh"
#include "paged_decode.h"
#include "paged_step.h"
#include "ptx.cuh"

namespace cg = cooperative_groups;

namespace fe {
namespace step {

constexpr int kBinBits = 11;
constexpr int kBins = 1 << kBinBits;
constexpr unsigned kForced = 0xffffffffu;  // key of an always-chosen page, above every score
constexpr float kInf = __builtin_huge_valf();
constexpr int kMaxCtas = 8;            // of one (sequence, KV head)
constexpr int kOnePassPages = 1024;    // widest table scored in the attention's launch
constexpr int kScorePages = 256;       // pages a CTA of the score launch takes
constexpr int kMaxFusedPages = 8192;   // most chosen pages whose list fits shared memory
constexpr int kKeysInSmem = 40960;     // more keys of a row stay in global memory

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
__device__ __forceinline__ void griddep_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// The row of one (sequence, KV head).
struct Row {
  int seq, kvh, ctx, pages;
  const int* table;
};
__device__ __forceinline__ Row row_of(const SelectParams& p, int row) {
  Row r;
  r.seq = row / p.kv_heads;
  r.kvh = row - r.seq * p.kv_heads;
  r.ctx = max(0, __ldg(p.context_lens + r.seq));
  const long long room = static_cast<long long>(p.width) * p.block_size;
  if (r.ctx > room) {
    if (threadIdx.x == 0) atomicOr(p.err, kErrBadBlock);
    r.ctx = static_cast<int>(room);
  }
  r.pages = (r.ctx + p.block_size - 1) / p.block_size;
  r.table = p.block_tables + static_cast<long long>(r.seq) * p.width;
  return r;
}

// The group's query heads as whole numbers, a warp a head: rows [q+ | q-] of 2 D bytes and
// scales 2^eq (+inf for a head with a NaN or an infinity, 0 for the padding to 8 heads).
template <typename T, int D, int NW>
__device__ __forceinline__ void quantise_query(const SelectParams& p, const Row& r,
                                               signed char* qrow, float* qscale) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int G = p.heads / p.kv_heads, GP = (G + 7) / 8 * 8;
  for (int g = warp; g < GP; g += NW) {
    constexpr int E = D / 32;
    float x[E], amax = 0.f;
    bool fin = true;
    const T* q = static_cast<const T*>(p.q) +
                 (static_cast<long long>(r.seq) * p.heads + r.kvh * G + g) * D;
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
      qrow[g * 2 * D + i * 32 + lane] = static_cast<signed char>(max(v, 0));
      qrow[g * 2 * D + D + i * 32 + lane] = static_cast<signed char>(min(v, 0));
    }
    if (lane == 0) qscale[g] = g >= G ? 0.f : fin ? exp2_int(e) : kInf;
  }
}

// Keys of pages [first, first + 32) of a row by one warp, those below `end`: store(page,
// key). All of the 32 boxes' bytes are in flight at once.
template <int D, typename Store>
__device__ __forceinline__ void score_32(const SelectParams& p, const Row& r,
                                         const signed char* qrow, const float* qscale, int first,
                                         int end, Store store) {
  constexpr int QB = 2 * D;    // bytes of a box, and of a head's row
  constexpr int CH = QB / 64;  // 64-byte pieces that a quad of lanes reads
  const int lane = threadIdx.x & 31, gq = lane >> 2, cq = lane & 3;
  const int GP = (p.heads / p.kv_heads + 7) / 8 * 8;
  int b = 0;
  if (first + lane < end) {
    b = __ldg(r.table + first + lane);
    if (b < 0 || b >= p.num_blocks) b = 0;  // flagged where the page is listed
  }
  const long long page = static_cast<long long>(b) * p.kv_heads + r.kvh;
  const float ks = __ldg(p.scales + page);
  uint4 a[4][CH];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const long long pk = __shfl_sync(0xffffffffu, page, gq + 8 * k);
    const uint4* v = reinterpret_cast<const uint4*>(p.values + pk * QB) + cq;
#pragma unroll
    for (int i = 0; i < CH; ++i) a[k][i] = ld_once(v + 4 * i);
  }
  float best[4] = {-kInf, -kInf, -kInf, -kInf};
  for (int h0 = 0; h0 < GP; h0 += 8) {
    int acc[2][4] = {};
    const uint4* qv = reinterpret_cast<const uint4*>(qrow + (h0 + gq) * QB) + cq;
    // the k index of both operands is the byte's place in this lane's 16-byte pieces
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const uint4 v = qv[4 * i];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        mma_s8_16832(acc[t], a[2 * t][i].x, a[2 * t + 1][i].x, a[2 * t][i].y, a[2 * t + 1][i].y,
                     v.x, v.y);
        mma_s8_16832(acc[t], a[2 * t][i].z, a[2 * t + 1][i].z, a[2 * t][i].w, a[2 * t + 1][i].w,
                     v.z, v.w);
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float qs = qscale[h0 + 2 * cq + j];
      if (qs == 0.f) continue;  // past the group's heads
#pragma unroll
      for (int k = 0; k < 4; ++k)
        best[k] = fmaxf(best[k],
                        qs == kInf ? qs : static_cast<float>(acc[k >> 1][(k & 1) * 2 + j]) * qs);
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    best[k] = fmaxf(best[k], __shfl_xor_sync(0xffffffffu, best[k], 1));
    best[k] = fmaxf(best[k], __shfl_xor_sync(0xffffffffu, best[k], 2));
  }
  // lane (gq, cq) keeps page gq + 8 cq
  const float mine = cq == 0 ? best[0] : cq == 1 ? best[1] : cq == 2 ? best[2] : best[3];
  const float sc = __shfl_sync(0xffffffffu, ks, gq + 8 * cq);
  const int j = first + gq + 8 * cq;
  if (j < end) {
    const bool kept = j < p.keep_first || j >= r.pages - p.keep_last;
    store(j, kept ? kForced : key_of((sc == kInf ? sc : mine * sc) + 0.f));  // + 0: no -0
  }
}

template <int NTHR>
struct SelectShared {
  unsigned hist[kBins];
  unsigned sums[NTHR / 32], above[NTHR / 32], equal[NTHR / 32];
  unsigned kmin, kmax;
  unsigned bin, over, in_bin;  // result of one histogram round
};

// The threshold of the K best of `n` > K keys, `kept` of them kForced: chosen are the keys
// above thr and the first `need` equal to it. Histograms of the keys between the smallest
// and the largest one, refined until the count ends at a bin's edge or a bin is one key.
template <int NTHR>
__device__ __forceinline__ void find_threshold(SelectShared<NTHR>& sh, const unsigned* keys, int n,
                                               unsigned rem, unsigned& thr, unsigned& need) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int NW = NTHR / 32, BPT = kBins / NTHR;
  thr = kForced - 1;
  need = 0;
  if (rem == 0) return;
  if (tid == 0) {
    sh.kmin = kForced;
    sh.kmax = 0;
  }
  for (int i = tid; i < kBins; i += NTHR) sh.hist[i] = 0;
  __syncthreads();
  unsigned lo = kForced, hi = 0;
  for (int i = tid; i < n; i += NTHR) {
    const unsigned k = keys[i];
    lo = min(lo, k);
    if (k != kForced) hi = max(hi, k);
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  if (lane == 0) {
    atomicMin(&sh.kmin, lo);
    atomicMax(&sh.kmax, hi);
  }
  __syncthreads();
  lo = sh.kmin;
  hi = sh.kmax;
  for (;;) {
    if (lo == hi) {
      thr = lo;
      need = rem;
      return;
    }
    const int shift = max(0, 32 - __clz(hi - lo) - kBinBits);
    for (int i = tid; i < n; i += NTHR) {
      const unsigned k = keys[i];
      if (k >= lo && k <= hi) atomicAdd(&sh.hist[(k - lo) >> shift], 1u);
    }
    __syncthreads();
    // this thread's bins, the highest ones first over the threads
    unsigned c[BPT], sum = 0;
    const int b0 = kBins - (tid + 1) * BPT;
#pragma unroll
    for (int i = 0; i < BPT; ++i) {
      c[i] = sh.hist[b0 + i];
      sum += c[i];
      sh.hist[b0 + i] = 0;
    }
    unsigned inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) sh.sums[warp] = inc;
    __syncthreads();
    unsigned over = inc - sum;
#pragma unroll
    for (int w = 0; w < NW; ++w) over += w < warp ? sh.sums[w] : 0;
    if (over < rem && rem <= over + sum) {
      bool done = false;
#pragma unroll
      for (int i = BPT - 1; i >= 0; --i) {
        if (!done && rem <= over + c[i]) {
          sh.bin = b0 + i;
          sh.over = over;
          sh.in_bin = c[i];
          done = true;
        }
        over += c[i];
      }
    }
    __syncthreads();
    const unsigned from = lo + (sh.bin << shift);
    rem -= sh.over;
    if (sh.in_bin == rem) {  // the whole bin is chosen
      thr = from - 1;
      return;
    }
    hi = min(hi, from + ((1u << shift) - 1));
    lo = from;
  }
}

// put(place, page) for the chosen pages in ascending order; each warp takes a range.
template <int NTHR, typename Put>
__device__ __forceinline__ void list_chosen(SelectShared<NTHR>& sh, const unsigned* keys, int n,
                                            unsigned thr, unsigned need, Put put) {
  constexpr int NW = NTHR / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
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
    sh.above[warp] = na;
    sh.equal[warp] = ne;
  }
  __syncthreads();
  unsigned a = 0, e = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    a += w < warp ? sh.above[w] : 0;
    e += w < warp ? sh.equal[w] : 0;
  }
  if (na == 0 && (ne == 0 || e >= need)) return;  // uniform in the warp
  const unsigned below = (1u << lane) - 1;
  for (int i0 = wb; i0 < we; i0 += 32) {
    const int i = i0 + lane;
    const unsigned k = i < we ? keys[i] : 0;
    const unsigned ma = __ballot_sync(0xffffffffu, i < we && k > thr);
    const unsigned me = __ballot_sync(0xffffffffu, i < we && k == thr);
    const unsigned ea = e + __popc(me & below);  // equal ones before this page
    if ((ma >> lane & 1) || ((me >> lane & 1) && ea < need))
      put(static_cast<int>(a + __popc(ma & below) + min(ea, need)), i);
    a += __popc(ma);
    e += __popc(me);
  }
}

// ---------------------------------------------------------------------------
// Scores of wide tables: CTA x takes kScorePages pages of row y into p.keys [rows, width].
template <typename T, int D>
__global__ void __launch_bounds__(256) page_score_kernel(const SelectParams p) {
  extern __shared__ __align__(16) signed char qrow[];
  const int GP = (p.heads / p.kv_heads + 7) / 8 * 8;
  float* qscale = reinterpret_cast<float*>(qrow + GP * 2 * D);
  griddep_wait();
  const Row r = row_of(p, blockIdx.x / p.pieces);
  const int beg = static_cast<int>(blockIdx.x % p.pieces) * kScorePages;
  if (r.pages <= p.num_pages || beg >= r.pages) return;
  quantise_query<T, D, 8>(p, r, qrow, qscale);
  __syncthreads();
  const int first = beg + (threadIdx.x >> 5) * 32;
  if (first >= r.pages) return;
  unsigned* keys = p.keys + static_cast<long long>(blockIdx.x / p.pieces) * p.width;
  score_32<D>(p, r, qrow, qscale, first, r.pages, [&](int j, unsigned key) { keys[j] = key; });
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

// Bytes of the region that holds first the keys, then the warps' partial results.
template <int D, int NT, int NTHR>
constexpr int merge_bytes() {
  return NTHR / 32 * 8 * NT * (D + 4 + 2) * 4;
}

// Selection and attention of one (sequence, KV head) by a cluster of `ctas` CTAs.
// key_cap: keys that fit shared memory (0: none are needed there).
template <typename T, int D, int NT, int NTHR>
__global__ void __launch_bounds__(NTHR, NTHR == 256 && NT == 1 ? 2 : 1)
    sparse_decode_kernel(const SelectParams p, int ctas,
                         int key_cap, int region) {
  constexpr int NW = NTHR / 32, HP = 8 * NT;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ SelectShared<NTHR> sh;
  __shared__ float part_m[HP], part_l[HP];  // this CTA's joined (m, l)
  unsigned* keys_s = reinterpret_cast<unsigned*>(dyn);
  int* chosen = reinterpret_cast<int*>(dyn + region);             // [num_pages]
  signed char* qrow = reinterpret_cast<signed char*>(chosen + (p.num_pages + 3) / 4 * 4);
  float* qscale = reinterpret_cast<float*>(qrow + HP * 2 * D);
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, warp = tid >> 5;
  const int row = blockIdx.x / ctas, rank = blockIdx.x % ctas;
  const int G = p.heads / p.kv_heads, K = p.num_pages;
  griddep_wait();
  const Row r = row_of(p, row);
  const int P = r.pages, n = min(P, K);
  int* sel = p.selected + static_cast<long long>(row) * K;

  // ---- the chosen pages, in every CTA's shared memory
  if (P > K) {
    const unsigned* keys = keys_s;
    if (p.keys) {  // scored by page_score_kernel
      const unsigned* g = p.keys + static_cast<long long>(row) * p.width;
      if (P <= key_cap) {
        for (int i = tid; i < P; i += NTHR) keys_s[i] = __ldcg(g + i);
        __syncthreads();
      } else {
        keys = g;
      }
    } else {
      quantise_query<T, D, NW>(p, r, qrow, qscale);
      if (ctas > 1) cluster.sync(); else __syncthreads();  // all CTAs run: they are stored to
      for (int first = (rank * NW + warp) * 32; first < P; first += ctas * NW * 32) {
        score_32<D>(p, r, qrow, qscale, first, P, [&](int j, unsigned key) {
          if (ctas == 1) {
            keys_s[j] = key;
          } else {
            for (int c = 0; c < ctas; ++c) cluster.map_shared_rank(keys_s, c)[j] = key;
          }
        });
      }
      if (ctas > 1) cluster.sync(); else __syncthreads();
    }
    unsigned thr, need;
    find_threshold<NTHR>(sh, keys, P, K - p.keep_first - p.keep_last, thr, need);
    list_chosen<NTHR>(sh, keys, P, thr, need, [&](int at, int page) {
      chosen[at] = page;
      if (rank == 0) sel[at] = page;
    });
  } else {
    for (int i = tid; i < K; i += NTHR) {
      if (i < P) chosen[i] = i;
      if (rank == 0) sel[i] = i < P ? i : -1;
    }
  }
  __syncthreads();

  // ---- this CTA's share of them: block << 32 is not needed, the list becomes (page, block)
  const int beg = static_cast<int>(static_cast<long long>(n) * rank / ctas);
  const int end = static_cast<int>(static_cast<long long>(n) * (rank + 1) / ctas);
  const int spp = p.block_size / 16, pieces = (end - beg) * spp;
  const T* kc = static_cast<const T*>(p.k_cache);
  const T* vc = static_cast<const T*>(p.v_cache);
  // rows of piece u and the tokens in it
  auto locate = [&](int u, long long& at, int& limit) {
    const int i = u / spp, half_ = u - i * spp;
    const int page = chosen[beg + i];
    const int b = __ldg(r.table + page);
    limit = r.ctx - page * p.block_size - half_ * 16;
    if (b < 0 || b >= p.num_blocks) {
      if ((tid & 31) == 0) atomicOr(p.err, kErrBadBlock);
      limit = 0;
      at = 0;
      return;
    }
    at = ((static_cast<long long>(b) * p.kv_heads + r.kvh) * p.block_size + half_ * 16) * D;
  };
  WarpAttention<T, D, NT> w;
  w.init(static_cast<const T*>(p.q) + (static_cast<long long>(r.seq) * p.heads + r.kvh * G) * D, G);
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
  __syncthreads();  // the keys are read: their region takes the partial results
  float* om = reinterpret_cast<float*>(dyn);  // [NW][HP]
  float* ol = om + NW * HP;                   // [NW][HP]
  float* oo = ol + NW * HP;                   // [NW][HP][D + 4]
  w.store(om + warp * HP, ol + warp * HP, oo + warp * HP * (D + 4));
  __syncthreads();
  T* out = static_cast<T*>(p.out) +
           (static_cast<long long>(r.seq) * p.heads + r.kvh * G) * D;
  for (int i = tid; i < G * D; i += NTHR) {
    const int h = i / D, d = i - h * D;
    float M = -kInf, L = 0.f, O = 0.f;
#pragma unroll
    for (int x = 0; x < NW; ++x) M = fmaxf(M, om[x * HP + h]);
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      const float mx = om[x * HP + h];
      const float f = mx == -kInf ? (ol[x * HP + h] != 0.f ? 1.f : 0.f) : ex2(mx - M);
      L += ol[x * HP + h] * f;
      O += oo[(x * HP + h) * (D + 4) + d] * f;
    }
    if (ctas == 1) {
      out[i] = static_cast<T>(n > 0 ? O / L : 0.f);
    } else {
      oo[h * (D + 4) + d] = O;  // only this thread reads column d of any warp's row h
      if (d == 0) {
        part_m[h] = M;
        part_l[h] = L;
      }
    }
  }
  if (ctas == 1) return;
  cluster.sync();
  for (int i = rank * NTHR + tid; i < G * D; i += ctas * NTHR) {
    const int h = i / D, d = i - h * D;
    float M = -kInf, mm[kMaxCtas], ll[kMaxCtas], o[kMaxCtas];
#pragma unroll
    for (int c = 0; c < kMaxCtas; ++c) {
      mm[c] = -kInf;
      ll[c] = o[c] = 0.f;
      if (c < ctas) {
        mm[c] = *cluster.map_shared_rank(&part_m[h], c);
        ll[c] = *cluster.map_shared_rank(&part_l[h], c);
        o[c] = *cluster.map_shared_rank(&oo[h * (D + 4) + d], c);
      }
      M = fmaxf(M, mm[c]);
    }
    float L = 0.f, O = 0.f;
#pragma unroll
    for (int c = 0; c < kMaxCtas; ++c) {
      const float f = mm[c] == -kInf ? (ll[c] != 0.f ? 1.f : 0.f) : ex2(mm[c] - M);
      L += ll[c] * f;
      O += o[c] * f;
    }
    out[i] = static_cast<T>(n > 0 ? O / L : 0.f);
  }
  cluster.sync();  // no CTA leaves while another reads its shared memory
}

// ---------------------------------------------------------------------------
// Selection alone, a CTA a row: the block table (block * Hkv + head) and the length that
// paged_decode.cu runs over.
template <typename T, int D, int NTHR>
__global__ void __launch_bounds__(NTHR) page_select_kernel(const SelectParams p, int key_cap) {
  constexpr int NW = NTHR / 32;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ SelectShared<NTHR> sh;
  unsigned* keys_s = reinterpret_cast<unsigned*>(dyn);
  signed char* qrow = reinterpret_cast<signed char*>(keys_s + key_cap);
  const int GP = (p.heads / p.kv_heads + 7) / 8 * 8;
  float* qscale = reinterpret_cast<float*>(qrow + GP * 2 * D);
  const int tid = threadIdx.x, warp = tid >> 5, row = blockIdx.x, K = p.num_pages;
  griddep_wait();
  const Row r = row_of(p, row);
  int* sel = p.selected + static_cast<long long>(row) * K;
  int* blocks = p.sel_blocks + static_cast<long long>(row) * K;
  auto put = [&](int at, int page) {
    sel[at] = page;
    const int b = __ldg(r.table + page);
    const bool ok = b >= 0 && b < p.num_blocks;
    if (!ok) atomicOr(p.err, kErrBadBlock);
    blocks[at] = ok ? b * p.kv_heads + r.kvh : -1;
  };
  const int P = r.pages;
  if (tid == 0)
    p.sel_lens[row] = P <= K ? r.ctx : (K - 1) * p.block_size + r.ctx - (P - 1) * p.block_size;
  if (P <= K) {
    for (int i = tid; i < K; i += NTHR) {
      if (i < P) put(i, i); else sel[i] = -1;
    }
    return;
  }
  const unsigned* keys = keys_s;
  if (p.keys) {
    keys = p.keys + static_cast<long long>(row) * p.width;
  } else {
    quantise_query<T, D, NW>(p, r, qrow, qscale);
    __syncthreads();
    for (int first = warp * 32; first < P; first += NW * 32)
      score_32<D>(p, r, qrow, qscale, first, P, [&](int j, unsigned key) { keys_s[j] = key; });
    __syncthreads();
  }
  unsigned thr, need;
  find_threshold<NTHR>(sh, keys, P, K - p.keep_first - p.keep_last, thr, need);
  list_chosen<NTHR>(sh, keys, P, thr, need, put);
}

// ---------------------------------------------------------------------------
// host launch

bool sparse_two_pass(int width) { return width > kOnePassPages; }

bool sparse_fused(const SelectParams& p, int dtype, int kv_layout) {
  return dtype != paged::kF32 && kv_layout == paged::kKvFlat && p.heads / p.kv_heads <= 16 &&
         p.num_pages <= kMaxFusedPages;
}

// Every kernel waits for its predecessor before it reads anything, so they may all be
// placed while it finishes; none lets its successor start early.
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
static cudaError_t launch_scores(SelectParams& p, cudaStream_t st) {
  const int GP = (p.heads / p.kv_heads + 7) / 8 * 8;
  const int smem = GP * (2 * D + 4);
  const cudaError_t e =
      ensure_smem_optin(reinterpret_cast<const void*>(page_score_kernel<T, D>), smem);
  if (e != cudaSuccess) return e;
  p.pieces = (p.width + kScorePages - 1) / kScorePages;
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[2];
  launch_config(cfg, attr, static_cast<long long>(p.num_seqs) * p.kv_heads * p.pieces, 256, smem, 1,
                st);
  return cudaLaunchKernelEx(&cfg, page_score_kernel<T, D>, p);
}

template <typename T, int D, int NT, int NTHR>
static cudaError_t launch_fused(const SelectParams& p, int ctas, cudaStream_t st) {
  auto kern = sparse_decode_kernel<T, D, NT, NTHR>;
  const int key_cap = std::min(p.width, kKeysInSmem);
  const int region = (std::max(key_cap * 4, merge_bytes<D, NT, NTHR>()) + 15) / 16 * 16;
  const int smem = region + (p.num_pages + 3) / 4 * 16 + 8 * NT * (2 * D + 4);
  const cudaError_t e = ensure_smem_optin(reinterpret_cast<const void*>(kern), smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[2];
  launch_config(cfg, attr, static_cast<long long>(p.num_seqs) * p.kv_heads * ctas, NTHR, smem, ctas,
                st);
  return cudaLaunchKernelEx(&cfg, kern, p, ctas, key_cap, region);
}

template <typename T, int D>
static cudaError_t launch_select(const SelectParams& p, cudaStream_t st) {
  constexpr int NTHR = 512;
  auto kern = page_select_kernel<T, D, NTHR>;
  const int key_cap = p.keys ? 0 : (p.width + 3) / 4 * 4;
  const int smem = key_cap * 4 + (p.heads / p.kv_heads + 7) / 8 * 8 * (2 * D + 4);
  const cudaError_t e = ensure_smem_optin(reinterpret_cast<const void*>(kern), smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[2];
  launch_config(cfg, attr, static_cast<long long>(p.num_seqs) * p.kv_heads, NTHR, smem, 1, st);
  return cudaLaunchKernelEx(&cfg, kern, p, key_cap);
}

template <typename T, int D>
static cudaError_t launch_d(SelectParams& p, bool fused, cudaStream_t st) {
  if (p.keys) {
    const cudaError_t e = launch_scores<T, D>(p, st);
    if (e != cudaSuccess) return e;
  }
  if constexpr (!std::is_same<T, float>::value) {
    if (fused) {
      // CTAs a row: enough to fill the GPU, at least two 16-token pieces a warp's turn each
      const long long rows = static_cast<long long>(p.num_seqs) * p.kv_heads;
      int ctas = 1;
      while (ctas < kMaxCtas && rows * ctas * 2 <= sm_count() &&
             p.num_pages * (p.block_size / 16) >= 4 * ctas)
        ctas *= 2;
      if (p.heads / p.kv_heads > 8) return launch_fused<T, D, 2, 256>(p, ctas, st);
      if (rows * ctas <= sm_count()) return launch_fused<T, D, 1, 512>(p, ctas, st);
      return launch_fused<T, D, 1, 256>(p, ctas, st);
    }
  }
  return launch_select<T, D>(p, st);
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
