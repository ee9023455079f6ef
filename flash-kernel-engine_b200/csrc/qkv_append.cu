// One pass over a step's QKV projection: per-head RMS norm of the queries and keys, the
// rotary embedding of both, queries out, keys and values into their cache slots.
//
//   y = x / sqrt(mean(x^2) + eps) * w          (per head of a token; w shared by the heads)
//   pair (a, b) of y at position p -> (a c - b s, a s + b c),  c, s = cos/sin[p][i]
// with pair i the elements (2i, 2i + 1) or (i, i + r / 2) of the first r = rotary_dim
// ones. fp32 arithmetic, one rounding to the element type at the end.
//
// Vector paths (r = d or no rotation, d = 64, 128 or 256, 16-byte aligned rows): a warp
// takes 32 / (d / 16) heads of a token at a time, 16 elements a lane: 8 in each half of the
// head, so that either pairing stays inside a lane. The token's cos / sin entries sit in 16
// registers for all of its heads (reading them per head would double the traffic), and the
// sum of squares takes log2(d / 16) shuffles.
//   - Few tokens: their heads are cut into parts, a warp each, loads first.
//   - Many: persistent CTAs of 4 such warps and a producer that copies whole token rows and
//     their cos / sin entries into a ring with bulk copies, so that the loads neither wait
//     for positions nor take registers. HBM bound: the projection is read and written once.
//     8192 tokens of 48 heads of 128 in bf16 (206 MB): 36 us, 5.7 TB/s, 87% of a plain copy
//     (51 us with rows read into registers). The arithmetic is close behind: 228 instructions
//     for 512 elements took 49 us, with two fp32 operations an instruction it hides.
// Other shapes take a warp per head, two reads.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>
#include <type_traits>

#include "internal.h"
#include "paged_decode.h"
#include "paged_step.h"
#include "ptx.cuh"

namespace fe {
namespace step {

template <typename T>
__device__ __forceinline__ T round_to(float x) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return __float2bfloat16_rn(x);
  else if constexpr (std::is_same<T, half>::value) return __float2half_rn(x);
  else return x;
}

__device__ __forceinline__ float weight_at(const void* w, int f32, int i, const float*) {
  return static_cast<const float*>(w)[i];
}
template <typename T>
__device__ __forceinline__ float weight_at(const void* w, int f32, int i, const T*) {
  return f32 ? static_cast<const float*>(w)[i] : static_cast<float>(static_cast<const T*>(w)[i]);
}

// 8 consecutive elements: 16 bytes of bf16 / fp16, 32 of fp32.
template <typename T>
struct Oct {
  uint4 v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = v; }
  __device__ __forceinline__ void get(float2* x) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        x[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
      } else {
        half2 h;
        memcpy(&h, &w[i], 4);
        x[i] = __half22float2(h);
      }
    }
  }
  __device__ __forceinline__ void set(const float2* x) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) w[i] = pack_bf16x2(x[i].x, x[i].y);
      else w[i] = pack_f16x2(x[i].x, x[i].y);
    }
    v = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct Oct<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = *reinterpret_cast<const float4*>(p);
    b = *reinterpret_cast<const float4*>(p + 4);
  }
  __device__ __forceinline__ void store(float* p) const {
    *reinterpret_cast<float4*>(p) = a;
    *reinterpret_cast<float4*>(p + 4) = b;
  }
  __device__ __forceinline__ void get(float2* x) const {
    x[0] = make_float2(a.x, a.y);
    x[1] = make_float2(a.z, a.w);
    x[2] = make_float2(b.x, b.y);
    x[3] = make_float2(b.z, b.w);
  }
  __device__ __forceinline__ void set(const float2* x) {
    a = make_float4(x[0].x, x[0].y, x[1].x, x[1].y);
    b = make_float4(x[2].x, x[2].y, x[3].x, x[3].y);
  }
};

// Two fp32 operations an instruction.
__device__ __forceinline__ uint64_t bits2(float2 a) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.x), "f"(a.y));
  return r;
}
__device__ __forceinline__ float2 from_bits2(uint64_t a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)));
  return from_bits2(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)), "l"(bits2(c)));
  return from_bits2(r);
}

__device__ __forceinline__ void griddep_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// What a token's position and slot allow.
struct Token {
  int pos;
  bool live;         // position >= 0 and inside the rotary tables
  bool cached;       // its K and V are written
  long long block;
  int off;
};
__device__ __forceinline__ Token token_of(const QkvParams& p, int t) {
  Token k;
  k.pos = __ldg(p.positions + t);
  const long long slot = __ldg(p.slots + t);
  k.live = k.pos >= 0;
  bool bad = false;
  if (k.live && p.rope_cos && k.pos >= p.rope_max_pos) {
    k.live = false;
    bad = true;
  }
  k.cached = k.live && slot >= 0;
  k.block = slot / p.block_size;
  k.off = static_cast<int>(slot - k.block * p.block_size);
  if (k.cached && k.block >= p.num_blocks) {
    k.cached = false;
    bad = true;
  }
  if (bad) atomicOr(p.err, kErrBadBlock);
  return k;
}

// A lane's cos / sin entries of a token: adjacent pairs: octet a holds pairs 4 l .., octet b
// D / 4 + 4 l ..; half pairs: (a[i], b[i]) is pair 8 l + i.
struct Turns {
  float2 c[4], s[4];
  template <int D>
  __device__ __forceinline__ void load(const float* cos, const float* sin, int l, int interleaved) {
    const int c0 = interleaved ? l * 4 : l * 8, c1 = interleaved ? D / 4 + l * 4 : l * 8 + 4;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 x = *reinterpret_cast<const float4*>(cos + (i ? c1 : c0));
      const float4 y = *reinterpret_cast<const float4*>(sin + (i ? c1 : c0));
      c[2 * i] = make_float2(x.x, x.y);
      c[2 * i + 1] = make_float2(x.z, x.w);
      s[2 * i] = make_float2(y.x, y.y);
      s[2 * i + 1] = make_float2(y.z, y.w);
    }
  }
};

// One head in the octets (a, b) of D / 16 lanes: norm, rotation and the write to its place.
// Every lane of the warp calls it (shuffles); `in`: its head exists. values: every lane's
// head is a value head, or none.
template <typename T, int D>
__device__ __forceinline__ void finish_head(const QkvParams& p, const Token& tok, int t, int h,
                                            bool in, bool values, int l, Oct<T>& a, Oct<T>& b,
                                            const Turns& turn, const float* wq, const float* wk) {
  constexpr int L = D / 16;
  const int ea = l * 8, eb = D / 2 + l * 8;
  const bool is_q = h < p.heads, is_v = h >= p.heads + p.kv_heads;
  float2 x[8];
  if (!values) {
    if (in) {
      a.get(x);
      b.get(x + 4);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = make_float2(0.f, 0.f);
    }
    float2 sq = mul2(x[0], x[0]), sr = mul2(x[4], x[4]);
#pragma unroll
    for (int i = 1; i < 4; ++i) {
      sq = fma2(x[i], x[i], sq);
      sr = fma2(x[4 + i], x[4 + i], sr);
    }
    float ss = (sq.x + sq.y) + (sr.x + sr.y);
#pragma unroll
    for (int o = 1; o < L; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (in && !is_v) {
      if (is_q ? p.q_weight != nullptr : p.k_weight != nullptr) {
        const float r = rsqrtf(ss * (1.f / D) + p.eps);
        const float2 rr = make_float2(r, r);
        const float* w = is_q ? wq : wk;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float4 u = *reinterpret_cast<const float4*>(w + ea + 4 * i);
          const float4 v = *reinterpret_cast<const float4*>(w + eb + 4 * i);
          x[2 * i] = mul2(mul2(x[2 * i], rr), make_float2(u.x, u.y));
          x[2 * i + 1] = mul2(mul2(x[2 * i + 1], rr), make_float2(u.z, u.w));
          x[4 + 2 * i] = mul2(mul2(x[4 + 2 * i], rr), make_float2(v.x, v.y));
          x[5 + 2 * i] = mul2(mul2(x[5 + 2 * i], rr), make_float2(v.z, v.w));
        }
      }
      if (p.rope_cos) {
        if (p.interleaved) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 u = x[i];
            const float c = i & 1 ? turn.c[i / 2].y : turn.c[i / 2].x;
            const float s = i & 1 ? turn.s[i / 2].y : turn.s[i / 2].x;
            x[i] = make_float2(u.x * c - u.y * s, u.x * s + u.y * c);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 u = x[i], v = x[4 + i], c = turn.c[i], s = turn.s[i];
            x[i] = fma2(v, make_float2(-s.x, -s.y), mul2(u, c));
            x[4 + i] = fma2(v, c, mul2(u, s));
          }
        }
      }
    }
  }
  if (!in) return;
  if (is_q) {
    if (!tok.live) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = make_float2(0.f, 0.f);
    }
    T* q = static_cast<T*>(p.q_out) + (static_cast<long long>(t) * p.heads + h) * D;
    a.set(x);
    b.set(x + 4);
    a.store(q + ea);
    b.store(q + eb);
  } else if (tok.cached) {
    if (!is_v) {
      a.set(x);
      b.set(x + 4);
    }
    const int hk = h - p.heads - (is_v ? p.kv_heads : 0);
    const long long page = (tok.block * p.kv_heads + hk) * p.block_size * D;
    T* dst = static_cast<T*>(is_v ? p.v_cache : p.k_cache) + page;
    if (p.kv_layout == paged::kKvFlat) {
      a.store(dst + tok.off * D + ea);
      b.store(dst + tok.off * D + eb);
    } else if (!is_v) {  // [D / 8, BS, 8]
      a.store(dst + (ea / 8 * p.block_size + tok.off) * 8);
      b.store(dst + (eb / 8 * p.block_size + tok.off) * 8);
    } else {  // [D, BS]
      a.get(x);
      b.get(x + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        dst[(ea + 2 * i) * p.block_size + tok.off] = round_to<T>(x[i].x);
        dst[(ea + 2 * i + 1) * p.block_size + tok.off] = round_to<T>(x[i].y);
        dst[(eb + 2 * i) * p.block_size + tok.off] = round_to<T>(x[4 + i].x);
        dst[(eb + 2 * i + 1) * p.block_size + tok.off] = round_to<T>(x[4 + i].y);
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ void load_weights(const QkvParams& p, float* wq, float* wk, int d) {
  for (int i = threadIdx.x; i < d; i += blockDim.x) {
    if (p.q_weight) wq[i] = weight_at(p.q_weight, p.weight_f32, i, static_cast<const T*>(nullptr));
    if (p.k_weight) wk[i] = weight_at(p.k_weight, p.weight_f32, i, static_cast<const T*>(nullptr));
  }
}

constexpr int kAppendWarps = 8;

// Few tokens. U: reads of 32 / L heads in flight a warp.
template <typename T, int D, int U>
__global__ void __launch_bounds__(32 * kAppendWarps, 3) qkv_vec_kernel(const QkvParams p, int parts,
                                                                   int per_part) {
  constexpr int L = D / 16;    // lanes a head takes
  constexpr int HPI = 32 / L;  // heads a warp reads at once
  __shared__ __align__(16) float wq[D], wk[D];
  const int lane = threadIdx.x & 31;
  const int l = lane % L, sub = lane / L;
  const long long unit = blockIdx.x * static_cast<long long>(kAppendWarps) + (threadIdx.x >> 5);
  const int t = static_cast<int>(unit / parts), part = static_cast<int>(unit % parts);
  const bool on = t < p.tokens;
  const int heads = p.heads + 2 * p.kv_heads;
  const int h_end = min(heads, (part + 1) * per_part);
  int h0 = part * per_part + sub;
  const T* row = static_cast<const T*>(p.qkv) + (on ? t : 0) * p.row_stride;
  Oct<T> a[U], b[U];
  auto fetch = [&](int h) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (on && h + u * HPI < h_end) {
        const T* x = row + static_cast<long long>(h + u * HPI) * D + l * 8;
        a[u].load(x);
        b[u].load(x + D / 2);
      }
    }
  };
  griddep_wait();
  fetch(h0);
  load_weights<T>(p, wq, wk, D);
  Token tok{};
  Turns turn;
  if (on) {
    tok = token_of(p, t);
    if (p.rope_cos && tok.live) {
      const long long at = static_cast<long long>(tok.pos) * (D / 2);
      turn.load<D>(p.rope_cos + at, p.rope_sin + at, l, p.interleaved);
    }
  }
  __syncthreads();
  if (!on) return;
  // every lane of the warp runs the same number of rounds: the shuffles need all of them
  for (int base = part * per_part; base < h_end; base += U * HPI, h0 += U * HPI) {
    if (base != part * per_part) fetch(h0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (base + u * HPI >= h_end) break;
      const int h = h0 + u * HPI;
      finish_head<T, D>(p, tok, t, h, h < h_end, base + u * HPI >= p.heads + p.kv_heads, l, a[u],
                        b[u], turn, wq, wk);
    }
  }
}

constexpr int kRowWarps = 4;    // consumer warps of a CTA of the row kernel
constexpr int kRowStages = 3;   // token rows of a CTA in flight, at most
constexpr int kRowCtas = 4;     // CTAs an SM

// Many tokens: CTA x takes tokens x, x + grid, ..; `stages` rows of `stage_bytes` in flight.
template <typename T, int D>
__global__ void __launch_bounds__(32 * (kRowWarps + 1), kRowCtas) qkv_row_kernel(const QkvParams p,
                                                                       int stages,
                                                                       int stage_bytes) {
  constexpr int L = D / 16, HPI = 32 / L;
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ __align__(16) float wq[D], wk[D];
  __shared__ Token token[kRowStages];
  __shared__ uint64_t full[kRowStages], empty[kRowStages];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int heads = p.heads + 2 * p.kv_heads;
  const uint32_t row_bytes = heads * D * sizeof(T);
  if (tid == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kRowWarps);
    }
    fence_mbar_init();
  }
  griddep_wait();
  load_weights<T>(p, wq, wk, D);
  __syncthreads();
  int slot = 0, phase = 0;
  auto advance = [&] {
    if (++slot == stages) {
      slot = 0;
      ++phase;
    }
  };
  if (warp == kRowWarps) {
    // ---- producer, one lane
    if (lane != 0) return;
    const uint64_t policy = l2_policy_evict_first(), keep = l2_policy_evict_last();
    Token next = token_of(p, min(static_cast<int>(blockIdx.x), p.tokens - 1));
    for (long long t = blockIdx.x; t < p.tokens; t += gridDim.x) {
      if (!mbar_wait(&empty[slot], (phase & 1) ^ 1)) {
        atomicOr(p.err, kErrWaitTimeout);
        return;  // the consumers' waits run out too, after the copies in flight
      }
      const bool turn = p.rope_cos && next.live;
      unsigned char* dst = ring + slot * stage_bytes;
      token[slot] = next;
      mbar_arrive_expect_tx(&full[slot], row_bytes + (turn ? 4 * D : 0));
      bulk_load(dst, static_cast<const T*>(p.qkv) + t * p.row_stride, row_bytes, &full[slot], policy);
      if (turn) {
        const long long at = static_cast<long long>(next.pos) * (D / 2);
        bulk_load(dst + row_bytes, p.rope_cos + at, 2 * D, &full[slot], keep);
        bulk_load(dst + row_bytes + 2 * D, p.rope_sin + at, 2 * D, &full[slot], keep);
      }
      if (t + gridDim.x < p.tokens) next = token_of(p, static_cast<int>(t + gridDim.x));
      advance();
    }
    return;
  }
  // ---- consumers: heads sub, sub + HPI, .. of every kRowWarps-th read
  const int l = lane % L, sub = lane / L;
  for (long long t = blockIdx.x; t < p.tokens; t += gridDim.x) {
    if (!__all_sync(0xffffffffu, mbar_wait(&full[slot], phase & 1))) {
      if (lane == 0) atomicOr(p.err, kErrWaitTimeout);
      return;  // the producer's wait for this place runs out too
    }
    const unsigned char* src = ring + slot * stage_bytes;
    const Token tok = token[slot];
    Turns turn;
    if (p.rope_cos && tok.live) {
      const float* turns = reinterpret_cast<const float*>(src + row_bytes);
      turn.load<D>(turns, turns + D / 2, l, p.interleaved);
    }
    const T* row = reinterpret_cast<const T*>(src) + l * 8;
    for (int h0 = warp * HPI; h0 < heads; h0 += kRowWarps * HPI) {
      const int h = h0 + sub;
      Oct<T> a, b;
      if (h < heads) {
        a.load(row + h * D);
        b.load(row + h * D + D / 2);
      }
      finish_head<T, D>(p, tok, static_cast<int>(t), h, h < heads, h0 >= p.heads + p.kv_heads, l,
                        a, b, turn, wq, wk);
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[slot]);
    advance();
  }
}

// Any even or odd head_dim, partial rotation, any alignment: a warp per head of a token.
template <typename T>
__global__ void __launch_bounds__(256) qkv_head_kernel(const QkvParams p) {
  const int lane = threadIdx.x & 31;
  griddep_wait();
  const int heads = p.heads + 2 * p.kv_heads, D = p.head_dim;
  const long long total = static_cast<long long>(p.tokens) * heads;
  for (long long w = blockIdx.x * 8LL + (threadIdx.x >> 5); w < total; w += gridDim.x * 8LL) {
    const int t = static_cast<int>(w / heads), h = static_cast<int>(w % heads);
    const bool is_q = h < p.heads, is_v = h >= p.heads + p.kv_heads;
    const Token tok = token_of(p, t);
    if (!is_q && !tok.cached) continue;
    const T* x = static_cast<const T*>(p.qkv) + t * p.row_stride + static_cast<long long>(h) * D;
    const int hk = h - p.heads - (is_v ? p.kv_heads : 0);
    T* dst = is_q ? static_cast<T*>(p.q_out) + (static_cast<long long>(t) * p.heads + h) * D
                  : static_cast<T*>(is_v ? p.v_cache : p.k_cache) +
                        (tok.block * p.kv_heads + hk) * p.block_size * D;
    auto put = [&](int e, T v) {
      if (is_q) dst[e] = v;
      else if (p.kv_layout == paged::kKvFlat) dst[static_cast<long long>(tok.off) * D + e] = v;
      else if (is_v) dst[static_cast<long long>(e) * p.block_size + tok.off] = v;
      else dst[(static_cast<long long>(e / 8) * p.block_size + tok.off) * 8 + e % 8] = v;
    };
    if (is_v) {
      for (int e = lane; e < D; e += 32) put(e, x[e]);
      continue;
    }
    const void* wt = is_q ? p.q_weight : p.k_weight;
    float r = 1.f;
    if (wt) {
      float ss = 0.f;
      for (int e = lane; e < D; e += 32) {
        const float y = static_cast<float>(x[e]);
        ss = fmaf(y, y, ss);
      }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      r = rsqrtf(ss / D + p.eps);
    }
    auto norm = [&](int e) {
      const float y = static_cast<float>(x[e]);
      return wt ? y * r * weight_at(wt, p.weight_f32, e, static_cast<const T*>(nullptr)) : y;
    };
    const int rd = p.rope_cos ? p.rotary_dim : 0, half_r = rd / 2;
    for (int i = lane; i < half_r; i += 32) {
      const int e0 = p.interleaved ? 2 * i : i, e1 = p.interleaved ? 2 * i + 1 : i + half_r;
      float y0 = 0.f, y1 = 0.f;
      if (tok.live) {
        const long long at = static_cast<long long>(tok.pos) * half_r + i;
        const float c = __ldg(p.rope_cos + at), s = __ldg(p.rope_sin + at);
        const float u0 = norm(e0), u1 = norm(e1);
        y0 = u0 * c - u1 * s;
        y1 = u0 * s + u1 * c;
      }
      put(e0, round_to<T>(y0));
      put(e1, round_to<T>(y1));
    }
    for (int e = rd + lane; e < D; e += 32) put(e, round_to<T>(tok.live ? norm(e) : 0.f));
  }
}

// Placed while the kernel before finishes, which it waits for before it reads anything.
template <typename... Args>
static cudaError_t launch_dependent(void (*kern)(Args...), long long blocks, int threads, int smem,
                                    cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

// Rows of many tokens. 3 rows in flight in each of 4 CTAs an SM, fewer where they would
// take more than 200 KB (8192 tokens of 48 heads: 36 us; 40 with 4 rows in 3 CTAs, 37 with 2
// in 5, whose 80 registers a thread spill).
template <typename T, int D>
static cudaError_t launch_rows(const QkvParams& p, int stage_bytes, cudaStream_t st) {
  const int stages = std::max(2, std::min(kRowStages, 50 * 1024 / stage_bytes));
  const int smem = stages * stage_bytes;
  const cudaError_t e =
      ensure_smem_optin(reinterpret_cast<const void*>(qkv_row_kernel<T, D>), smem);
  if (e != cudaSuccess) return e;
  const int per_sm = std::max(1, std::min(kRowCtas, 200 * 1024 / smem));
  const long long blocks = std::min<long long>(p.tokens, static_cast<long long>(per_sm) * sm_count());
  return launch_dependent(qkv_row_kernel<T, D>, blocks, 32 * (kRowWarps + 1), smem, st, p, stages,
                          stage_bytes);
}

template <typename T, int D>
static cudaError_t launch_vec(const QkvParams& p, cudaStream_t st) {
  constexpr int HPI = 32 / (D / 16);
  const int heads = p.heads + 2 * p.kv_heads;
  // From 4 tokens an SM on the ring pays: 1237 fp32 tokens take 6.4 us with it and 7.0
  // without, 256 tokens of 80 heads 5.8 us with it and 3.8 without.
  const long long stage_bytes = static_cast<long long>(heads) * D * sizeof(T) + 4 * D;
  if (p.tokens >= 4LL * sm_count() && 2 * stage_bytes <= 200 * 1024)
    return launch_rows<T, D>(p, static_cast<int>(stage_bytes), st);
  // Fewer tokens are cut into parts of whole reads, for 16 warps an SM where they give them
  // (one read in flight a warp: 3.8 us for those 256 tokens, 4.7 with two or four and fewer
  // warps an SM).
  constexpr int U = 1;
  const int reads = (heads + HPI - 1) / HPI;
  const long long want = 16LL * sm_count();  // warps
  const long long parts_wanted = std::max<long long>(1, want / std::max(1, p.tokens));
  const int per = static_cast<int>(std::max<long long>(1, reads / std::min<long long>(parts_wanted, reads)));
  const int parts = (reads + per - 1) / per;
  const long long units = static_cast<long long>(p.tokens) * parts;
  const long long blocks = (units + kAppendWarps - 1) / kAppendWarps;
  return launch_dependent(qkv_vec_kernel<T, D, U>, blocks, 32 * kAppendWarps, 0, st, p, parts,
                          per * HPI);
}

template <typename T>
static cudaError_t launch_t(const QkvParams& p, cudaStream_t st) {
  const uintptr_t ptrs = reinterpret_cast<uintptr_t>(p.qkv) | reinterpret_cast<uintptr_t>(p.q_out) |
                         reinterpret_cast<uintptr_t>(p.k_cache) |
                         reinterpret_cast<uintptr_t>(p.v_cache) |
                         reinterpret_cast<uintptr_t>(p.rope_cos) |
                         reinterpret_cast<uintptr_t>(p.rope_sin);
  const bool vec = (ptrs & 15) == 0 && (p.row_stride * static_cast<long long>(sizeof(T))) % 16 == 0 &&
                   (!p.rope_cos || p.rotary_dim == p.head_dim);
  if (vec && p.head_dim == 64) return launch_vec<T, 64>(p, st);
  if (vec && p.head_dim == 128) return launch_vec<T, 128>(p, st);
  if (vec && p.head_dim == 256) return launch_vec<T, 256>(p, st);
  const long long total = static_cast<long long>(p.tokens) * (p.heads + 2 * p.kv_heads);
  const long long blocks = std::min<long long>((total + 7) / 8, 32LL * sm_count());
  return launch_dependent(qkv_head_kernel<T>, blocks, 256, 0, st, p);
}

cudaError_t launch_qkv_append(const QkvParams& p, int dtype, cudaStream_t st) {
  if (dtype == paged::kBf16) return launch_t<__nv_bfloat16>(p, st);
  if (dtype == paged::kF16) return launch_t<half>(p, st);
  if (dtype == paged::kF32) return launch_t<float>(p, st);
  return cudaErrorInvalidValue;
}

}  // namespace step
}  // namespace fe
