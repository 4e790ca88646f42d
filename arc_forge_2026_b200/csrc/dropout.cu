// Dropout from a counter-based generator: y = x * scale where kept, else 0 (+ residual). The mask is a function of
// (seed, offset + i / 8) alone -- Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as
// 1, 2, 3", 2011), 128 bits for eight elements, 16 bits each -- so the backward pass makes it again and nothing is
// stored. An element stays when its 16 bits are below threshold = round((1 - p) 65536); scale = 65536 / threshold, so
// the expectation is exact for the rounded p. A dropped element is 0 whatever it held (NaN and infinity included).
// Memory bounds it: at 16 bits an element the ten rounds cost about 10 integer operations an element.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "ffn.h"

namespace afb {
namespace drop {

AFB_DEV uint4 philox(uint64_t ctr, uint64_t key) {
  uint32_t x0 = (uint32_t)ctr, x1 = (uint32_t)(ctr >> 32), x2 = 0, x3 = 0;
  uint32_t k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)x0 * 0xD2511F53u, b = (uint64_t)x2 * 0xCD9E8D57u;
    x0 = (uint32_t)(b >> 32) ^ x1 ^ k0;
    x1 = (uint32_t)b;
    x2 = (uint32_t)(a >> 32) ^ x3 ^ k1;
    x3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(x0, x1, x2, x3);
}

template <typename T>
AFB_DEV float to_f(T v) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return __bfloat162float(v);
  else if constexpr (std::is_same<T, __half>::value) return __half2float(v);
  else return v;
}
template <typename T>
AFB_DEV T from_f(float v) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return __float2bfloat16(v);
  else if constexpr (std::is_same<T, __half>::value) return __float2half(v);
  else return v;
}
template <typename T>
struct alignas(16) Vec8 {
  T v[8];
};

// a thread takes groups of eight elements; VEC: every base is 16-byte aligned
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) dropout_kernel(const T* __restrict__ x, const T* __restrict__ res,
                                                      T* __restrict__ y, int64_t n, uint32_t threshold, float scale,
                                                      uint64_t seed, uint64_t offset, const int64_t* __restrict__ rng) {
  grid_dep_wait();
  grid_dep_trigger();
  if (rng) {
    seed += (uint64_t)rng[0];
    offset += (uint64_t)rng[1];
  }
  const int64_t groups = (n + 7) / 8;
  for (int64_t q = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; q < groups; q += (int64_t)gridDim.x * blockDim.x) {
    const int64_t i0 = q * 8;
    const bool whole = VEC && i0 + 8 <= n;
    Vec8<T> a, r;
    if (whole) {
      a = *reinterpret_cast<const Vec8<T>*>(x + i0);
      if (res) r = *reinterpret_cast<const Vec8<T>*>(res + i0);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (i0 + j < n) {
          a.v[j] = x[i0 + j];
          if (res) r.v[j] = res[i0 + j];
        }
      }
    }
    const uint4 w = philox(offset + (uint64_t)q, seed);
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t bits = (words[j >> 1] >> (16 * (j & 1))) & 0xFFFFu;
      float f = bits < threshold ? __fmul_rn(to_f(a.v[j]), scale) : 0.f;
      if (res) f = __fadd_rn(f, to_f(r.v[j]));
      a.v[j] = from_f<T>(f);
    }
    if (whole) {
      *reinterpret_cast<Vec8<T>*>(y + i0) = a;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i0 + j < n) y[i0 + j] = a.v[j];
    }
  }
}

template <typename T>
static int run(const void* x, const void* res, void* y, int64_t n, uint32_t threshold, uint64_t seed, uint64_t offset,
               const int64_t* rng, int num_sms, cudaStream_t st) {
  const int64_t groups = (n + 7) / 8;
  const int grid = (int)std::min<int64_t>((groups + 255) / 256, (int64_t)num_sms * 8);
  const float scale = threshold ? (float)(65536.0 / threshold) : 0.f;
  const bool vec = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(res) | reinterpret_cast<uintptr_t>(y)) & 15) == 0;
  return launch_pdl(vec ? dropout_kernel<T, true> : dropout_kernel<T, false>, dim3(grid), dim3(256), 0, st,
                    (const T*)x, (const T*)res, (T*)y, n, threshold, scale, seed, offset, rng);
}

}  // namespace drop

int dropout(const void* x, const void* residual, void* y, int64_t n, int dtype, uint32_t threshold, uint64_t seed,
            uint64_t offset, const int64_t* rng, int num_sms, cudaStream_t st) {
  if (n < 0 || threshold > 65536 || dtype < 0 || dtype > 2) return 3;
  if (n == 0) return 0;
  if (dtype == ELEM_BF16)
    return drop::run<__nv_bfloat16>(x, residual, y, n, threshold, seed, offset, rng, num_sms, st);
  if (dtype == ELEM_FP16) return drop::run<__half>(x, residual, y, n, threshold, seed, offset, rng, num_sms, st);
  return drop::run<float>(x, residual, y, n, threshold, seed, offset, rng, num_sms, st);
}

}  // namespace afb
