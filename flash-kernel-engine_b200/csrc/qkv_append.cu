// One pass over a step's QKV projection: per-head RMS norm of the queries and keys, the
// rotary embedding of both, queries out, keys and values into their cache slots.
//
//   y = x / sqrt(mean(x^2) + eps) * w          (per head of a token; w shared by the heads)
//   pair (a, b) of y at position p -> (a c - b s, a s + b c),  c, s = cos/sin[p][i]
// with pair i the elements (2i, 2i + 1) or (i, i + r / 2) of the first r = rotary_dim
// ones. fp32 arithmetic, one rounding to the element type at the end.
//
// Vector path (r = d or no rotation, d = 64, 128 or 256, 16-byte aligned rows): a warp
// takes one token and reads 32 / (d / 16) of its heads at a time, 16 elements a lane: 8 in
// each half of the head, so that either pairing stays inside a lane. The token's cos / sin
// entries then sit in 16 registers for all of its heads (reading them per head would
// double the traffic), and the sum of squares takes log2(d / 16) shuffles. HBM bound: the
// projection is read once and written once. Other shapes take a warp per head, two reads.
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
  __device__ __forceinline__ void get(float* x) const {
    T e[8];
    memcpy(e, &v, 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(e[i]);
  }
  __device__ __forceinline__ void set(const float* x) {
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = round_to<T>(x[i]);
    memcpy(&v, e, 16);
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
  __device__ __forceinline__ void get(float* x) const {
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  }
  __device__ __forceinline__ void set(const float* x) {
    a = make_float4(x[0], x[1], x[2], x[3]);
    b = make_float4(x[4], x[5], x[6], x[7]);
  }
};

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

constexpr int kAppendWarps = 8;

// U: reads of 32 / L heads in flight a warp.
template <typename T, int D, int U>
__global__ void __launch_bounds__(32 * kAppendWarps) qkv_vec_kernel(const QkvParams p, int parts,
                                                                   int per_part) {
  constexpr int L = D / 16;    // lanes a head takes
  constexpr int HPI = 32 / L;  // heads a warp reads at once
  __shared__ float wq[D], wk[D];
  const int lane = threadIdx.x & 31;
  const int l = lane % L, sub = lane / L;
  const long long unit = blockIdx.x * static_cast<long long>(kAppendWarps) + (threadIdx.x >> 5);
  const int t = static_cast<int>(unit / parts), part = static_cast<int>(unit % parts);
  const bool on = t < p.tokens;
  const int heads = p.heads + 2 * p.kv_heads;
  const int h_end = min(heads, (part + 1) * per_part);
  int h0 = part * per_part + sub;
  const T* row = static_cast<const T*>(p.qkv) + (on ? t : 0) * p.row_stride;
  const int ea = l * 8, eb = D / 2 + l * 8;  // first elements of the lane's two octets
  Oct<T> a[U], b[U];
  auto fetch = [&](int h) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (on && h + u * HPI < h_end) {
        a[u].load(row + static_cast<long long>(h + u * HPI) * D + ea);
        b[u].load(row + static_cast<long long>(h + u * HPI) * D + eb);
      }
    }
  };
  fetch(h0);
  const bool nq = p.q_weight != nullptr, nk = p.k_weight != nullptr;
  for (int i = threadIdx.x; i < D; i += 32 * kAppendWarps) {
    if (nq) wq[i] = weight_at(p.q_weight, p.weight_f32, i, static_cast<const T*>(nullptr));
    if (nk) wk[i] = weight_at(p.k_weight, p.weight_f32, i, static_cast<const T*>(nullptr));
  }
  Token tok{};
  float c[8], s[8];
  const bool rot = p.rope_cos != nullptr;
  if (on) {
    tok = token_of(p, t);
    if (rot && tok.live) {
      const long long at = static_cast<long long>(tok.pos) * (D / 2);
      // adjacent pairs: octet a holds pairs l * 4 .., octet b D / 4 + l * 4 ..;
      // half pairs: (a[i], b[i]) is pair l * 8 + i
      const int c0 = p.interleaved ? l * 4 : l * 8, c1 = p.interleaved ? D / 4 + l * 4 : l * 8 + 4;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 x = __ldg(reinterpret_cast<const float4*>(p.rope_cos + at + (i ? c1 : c0)));
        const float4 y = __ldg(reinterpret_cast<const float4*>(p.rope_sin + at + (i ? c1 : c0)));
        c[4 * i] = x.x; c[4 * i + 1] = x.y; c[4 * i + 2] = x.z; c[4 * i + 3] = x.w;
        s[4 * i] = y.x; s[4 * i + 1] = y.y; s[4 * i + 2] = y.z; s[4 * i + 3] = y.w;
      }
    }
  }
  __syncthreads();
  if (!on) return;
  // every lane of the warp runs the same number of rounds: the shuffles need all of them
  for (int base = part * per_part; base < h_end; base += U * HPI, h0 += U * HPI) {
    if (base != part * per_part) fetch(h0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * HPI;
      if (base + u * HPI >= h_end) break;
      const bool in = h < h_end;
      const bool is_q = h < p.heads, is_v = h >= p.heads + p.kv_heads;
      float x[16], ss = 0.f;
      if (in) {
        a[u].get(x);
        b[u].get(x + 8);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
      for (int o = 1; o < L; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (!in) continue;
      if (!is_v) {
        if (is_q ? nq : nk) {
          const float r = 1.f / sqrtf(ss * (1.f / D) + p.eps);
          const float* w = is_q ? wq : wk;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            x[i] = x[i] * r * w[ea + i];
            x[8 + i] = x[8 + i] * r * w[eb + i];
          }
        }
        if (rot) {
          if (p.interleaved) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float u0 = x[2 * i], u1 = x[2 * i + 1];
              x[2 * i] = u0 * c[i] - u1 * s[i];
              x[2 * i + 1] = u0 * s[i] + u1 * c[i];
            }
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float u0 = x[i], u1 = x[8 + i];
              x[i] = u0 * c[i] - u1 * s[i];
              x[8 + i] = u0 * s[i] + u1 * c[i];
            }
          }
        }
      }
      if (is_q) {
        if (!tok.live) {
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] = 0.f;
        }
        T* q = static_cast<T*>(p.q_out) + (static_cast<long long>(t) * p.heads + h) * D;
        a[u].set(x);
        b[u].set(x + 8);
        a[u].store(q + ea);
        b[u].store(q + eb);
      } else if (tok.cached) {
        if (!is_v) {
          a[u].set(x);
          b[u].set(x + 8);
        }
        const int hk = h - p.heads - (is_v ? p.kv_heads : 0);
        const long long page = (tok.block * p.kv_heads + hk) * p.block_size * D;
        T* dst = static_cast<T*>(is_v ? p.v_cache : p.k_cache) + page;
        if (p.kv_layout == paged::kKvFlat) {
          a[u].store(dst + tok.off * D + ea);
          b[u].store(dst + tok.off * D + eb);
        } else if (!is_v) {  // [D / 8, BS, 8]
          a[u].store(dst + (ea / 8 * p.block_size + tok.off) * 8);
          b[u].store(dst + (eb / 8 * p.block_size + tok.off) * 8);
        } else {  // [D, BS]
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            dst[(ea + i) * p.block_size + tok.off] = round_to<T>(x[i]);
            dst[(eb + i) * p.block_size + tok.off] = round_to<T>(x[8 + i]);
          }
        }
      }
    }
  }
}

// Any even or odd head_dim, partial rotation, any alignment: a warp per head of a token.
template <typename T>
__global__ void __launch_bounds__(256) qkv_head_kernel(const QkvParams p) {
  const int lane = threadIdx.x & 31;
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
      r = 1.f / sqrtf(ss / D + p.eps);
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

template <typename T, int D>
static cudaError_t launch_vec(const QkvParams& p, cudaStream_t st) {
  constexpr int U = sizeof(T) == 4 ? 2 : 4;
  constexpr int HPI = 32 / (D / 16);
  const int heads = p.heads + 2 * p.kv_heads;
  // A warp walks all of a token's heads where there are tokens enough to fill the GPU (the
  // cos / sin entries are read once); fewer tokens are cut into parts of whole reads.
  const int reads = (heads + HPI - 1) / HPI;
  const long long want = 16LL * sm_count();  // warps
  const long long parts_wanted = std::max<long long>(1, want / std::max(1, p.tokens));
  const int per = static_cast<int>(std::max<long long>(1, reads / std::min<long long>(parts_wanted, reads)));
  const int parts = (reads + per - 1) / per;
  const long long units = static_cast<long long>(p.tokens) * parts;
  const long long blocks = (units + kAppendWarps - 1) / kAppendWarps;
  qkv_vec_kernel<T, D, U><<<static_cast<unsigned>(blocks), 32 * kAppendWarps, 0, st>>>(p, parts,
                                                                                    per * HPI);
  return cudaGetLastError();
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
  qkv_head_kernel<T><<<static_cast<unsigned>(blocks), 256, 0, st>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_qkv_append(const QkvParams& p, int dtype, cudaStream_t st) {
  if (dtype == paged::kBf16) return launch_t<__nv_bfloat16>(p, st);
  if (dtype == paged::kF16) return launch_t<half>(p, st);
  if (dtype == paged::kF32) return launch_t<float>(p, st);
  return cudaErrorInvalidValue;
}

}  // namespace step
}  // namespace fe
