// int8 boxes of the keys of full cache pages, the summary that sparse_decode.cu scores.
//
// For page b, KV head h and channel c let hi = max_t k[t, c], lo = min_t k[t, c] over the
// page's block_size tokens, amax = max |k|, and e the smallest exponent with
// amax <= 127 * 2^e (at least -120, so that 2^-e stays finite). The page stores
// ceil(hi / 2^e) and floor(lo / 2^e) as int8 and 2^e as fp32. Rounding outwards keeps
// every key inside its box, and powers of two keep every step exact: a box does not depend
// on the order of the reductions. A page with a NaN or an infinity stores an empty box and
// the scale +inf (it is always chosen, so the attention shows the value as the dense one
// does).
//
// Pages are named by the step's slot list: the token whose slot ends a page closes it. One
// warp takes 32 slots and one KV head; the heads of a block are neighbours in the cache
// and in the launch order. Each lane owns 16 bytes of channels and keeps the packed max
// and min in the element type. HBM bound: each closed page's keys are read once, a page's 4 KB
// in one go of 16-byte loads. Four contexts of 131072 tokens, 8 heads of 128 (1.15 GB): 174 to
// 181 us, 6.3 to 6.6 TB/s, the rate of a plain copy.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

#include "internal.h"
#include "page_box.cuh"
#include "paged_decode.h"
#include "paged_step.h"
#include "ptx.cuh"

namespace fe {
namespace step {

// Max / min of 16 bytes of elements that keep a NaN once they met one.
template <typename T>
struct Ext;
template <>
struct Ext<__nv_bfloat16> {
  static constexpr int N = 8;
  __nv_bfloat162 hi[4], lo[4];
  __device__ __forceinline__ void init(uint4 v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) hi[i] = lo[i] = *reinterpret_cast<const __nv_bfloat162*>(&w[i]);
  }
  __device__ __forceinline__ void add(uint4 v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 x = *reinterpret_cast<const __nv_bfloat162*>(&w[i]);
      hi[i] = __hmax2_nan(hi[i], x);
      lo[i] = __hmin2_nan(lo[i], x);
    }
  }
  __device__ __forceinline__ void get(float (&h)[N], float (&l)[N]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = __bfloat1622float2(hi[i]), b = __bfloat1622float2(lo[i]);
      h[2 * i] = a.x; h[2 * i + 1] = a.y;
      l[2 * i] = b.x; l[2 * i + 1] = b.y;
    }
  }
};
template <>
struct Ext<half> {
  static constexpr int N = 8;
  half2 hi[4], lo[4];
  __device__ __forceinline__ void init(uint4 v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) hi[i] = lo[i] = *reinterpret_cast<const half2*>(&w[i]);
  }
  __device__ __forceinline__ void add(uint4 v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const half2 x = *reinterpret_cast<const half2*>(&w[i]);
      hi[i] = __hmax2_nan(hi[i], x);
      lo[i] = __hmin2_nan(lo[i], x);
    }
  }
  __device__ __forceinline__ void get(float (&h)[N], float (&l)[N]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = __half22float2(hi[i]), b = __half22float2(lo[i]);
      h[2 * i] = a.x; h[2 * i + 1] = a.y;
      l[2 * i] = b.x; l[2 * i + 1] = b.y;
    }
  }
};
template <>
struct Ext<float> {
  static constexpr int N = 4;
  float hi[4], lo[4];
  __device__ __forceinline__ void init(uint4 v) {
    hi[0] = lo[0] = __uint_as_float(v.x);
    hi[1] = lo[1] = __uint_as_float(v.y);
    hi[2] = lo[2] = __uint_as_float(v.z);
    hi[3] = lo[3] = __uint_as_float(v.w);
  }
  __device__ __forceinline__ void add(uint4 v) {
    const float x[4] = {__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z),
                        __uint_as_float(v.w)};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      hi[i] = x[i] != x[i] || hi[i] < x[i] ? x[i] : hi[i];
      lo[i] = x[i] != x[i] || lo[i] > x[i] ? x[i] : lo[i];
    }
  }
  __device__ __forceinline__ void get(float (&h)[N], float (&l)[N]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      h[i] = hi[i];
      l[i] = lo[i];
    }
  }
};

template <typename T, int D, int BS, int KVL>
__global__ void __launch_bounds__(256) page_bounds_kernel(const BoundsParams p) {
  constexpr int N = Ext<T>::N;            // channels a lane owns
  constexpr int CPR = D / N;              // lanes (16-byte chunks) a row takes: 8, 16 or 32
  constexpr int RPI = 32 / CPR;           // rows a warp reads at once
  constexpr int IT = BS / RPI;            // reads a page takes
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const long long item = blockIdx.x * 8LL + (threadIdx.x >> 5);
  const int h = static_cast<int>(item % p.kv_heads);
  const long long t = item / p.kv_heads * 32 + lane;
  const long long slot = t < p.tokens ? p.slots[t] : -1;
  const bool ends = slot >= 0 && slot % BS == BS - 1;
  const bool bad = slot >= static_cast<long long>(p.num_blocks) * BS;
  if (bad) atomicOr(p.err, kErrBadBlock);
  unsigned todo = __ballot_sync(0xffffffffu, ends && !bad);
  const int ch = lane % CPR, r0 = lane / CPR;
  while (todo) {
    const int who = __ffs(todo) - 1;
    todo &= todo - 1;
    const long long block = __shfl_sync(0xffffffffu, slot, who) / BS;
    const long long page = block * p.kv_heads + h;
    const T* k = static_cast<const T*>(p.k_cache) + page * (BS * D);
    uint4 v[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int r = i * RPI + r0;
      // flat [BS, D], or x-packed [D / 8, BS, 8]
      v[i] = __ldg(reinterpret_cast<const uint4*>(
          KVL == paged::kKvFlat ? k + r * D + ch * N : k + (ch * BS + r) * N));
    }
    Ext<T> x;
    x.init(v[0]);
#pragma unroll
    for (int i = 1; i < IT; ++i) x.add(v[i]);
    float hi[N], lo[N];
    x.get(hi, lo);
    float amax = 0.f;
    bool fin = true;
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int o = CPR; o < 32; o <<= 1) {
        const float a = __shfl_xor_sync(0xffffffffu, hi[i], o);
        const float b = __shfl_xor_sync(0xffffffffu, lo[i], o);
        hi[i] = a != a || hi[i] < a ? a : hi[i];
        lo[i] = b != b || lo[i] > b ? b : lo[i];
      }
      fin = fin && is_finite(hi[i]) && is_finite(lo[i]);
      amax = fmaxf(amax, fmaxf(fabsf(hi[i]), fabsf(lo[i])));
    }
#pragma unroll
    for (int o = 1; o < CPR; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    fin = __all_sync(0xffffffffu, fin);
    const int e = box_exponent(fin ? amax : 0.f);
    const float inv = exp2_int(-e);
    if (lane < CPR) {
      uint32_t a[N / 4], b[N / 4];
#pragma unroll
      for (int w = 0; w < N / 4; ++w) {
        a[w] = b[w] = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int u = fin ? __float2int_ru(hi[4 * w + i] * inv) : 0;
          const int l = fin ? __float2int_rd(lo[4 * w + i] * inv) : 0;
          a[w] |= (static_cast<uint32_t>(u) & 0xffu) << (8 * i);
          b[w] |= (static_cast<uint32_t>(l) & 0xffu) << (8 * i);
        }
      }
      uint32_t* out = reinterpret_cast<uint32_t*>(p.values + page * (2 * D)) + ch * (N / 4);
#pragma unroll
      for (int w = 0; w < N / 4; ++w) {
        out[w] = a[w];
        out[D / 4 + w] = b[w];
      }
      if (lane == 0) p.scales[page] = fin ? exp2_int(e) : __int_as_float(0x7f800000);
    }
  }
}

template <typename T>
static cudaError_t launch_bounds_t(const BoundsParams& p, int d, int bs, cudaStream_t st) {
  const long long items = (p.tokens + 31LL) / 32 * p.kv_heads;
  // placed while the kernel before finishes, which it waits for before it reads anything
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((items + 7) / 8));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
#define FE_CASE(D_, BS_, L_)                     \
  if (d == D_ && bs == BS_ && p.kv_layout == L_) \
    return cudaLaunchKernelEx(&cfg, page_bounds_kernel<T, D_, BS_, L_>, p);
  FE_CASE(64, 16, paged::kKvFlat)
  FE_CASE(64, 32, paged::kKvFlat)
  FE_CASE(128, 16, paged::kKvFlat)
  FE_CASE(128, 32, paged::kKvFlat)
  if constexpr (!std::is_same<T, float>::value) {
    FE_CASE(64, 16, paged::kKvVllm)
    FE_CASE(128, 16, paged::kKvVllm)
  }
#undef FE_CASE
  return cudaErrorInvalidValue;
}

cudaError_t launch_page_bounds(const BoundsParams& p, int d, int bs, int dtype, cudaStream_t st) {
  if (dtype == paged::kBf16) return launch_bounds_t<__nv_bfloat16>(p, d, bs, st);
  if (dtype == paged::kF16) return launch_bounds_t<half>(p, d, bs, st);
  if (dtype == paged::kF32) return launch_bounds_t<float>(p, d, bs, st);
  return cudaErrorInvalidValue;
}

}  // namespace step
}  // namespace fe
