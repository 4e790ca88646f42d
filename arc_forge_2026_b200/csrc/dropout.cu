// Dropout from a counter-based generator: y = x * scale where kept, else 0 (+ residual). The mask is a function of
// (seed, offset + i / 8) alone -- Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as
// 1, 2, 3", 2011), 128 bits for eight elements, 16 bits each -- so the backward pass makes it again and nothing is
// stored. An element stays when its 16 bits are below threshold = round((1 - p) 65536); scale = 65536 / threshold, so
// the expectation is exact for the rounded p. A dropped element is 0 whatever it held (NaN and infinity included).
// At 16 bits an element the ten rounds cost about 9 integer operations an element, and the choice, the scale and the
// conversions 6. 16,384 x 2,560 takes 36 us in bf16 (4.7 TB/s), 54 with a residual, 8,192 x 2,560 36 and 43 in fp32 (4.6
// and 5.8 TB/s). No unit is full: the integer pipe is 59 % busy and the multiplier 57 %, the issue slots 57 %. A thread's
// loads and its arithmetic take turns, and a warp waits about as long for memory as for the two pipes; of the grid's six CTAs
// an SM five are resident at a time, by registers.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "ffn.h"

namespace afb {
namespace drop {

// the ten round keys, made once a thread
struct Keys {
  uint32_t a[10], b[10];
  AFB_DEV explicit Keys(uint64_t seed) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
      a[r] = (uint32_t)seed + r * 0x9E3779B9u;
      b[r] = (uint32_t)(seed >> 32) + r * 0xBB67AE85u;
    }
  }
};
AFB_DEV uint4 philox(uint64_t ctr, const Keys& key) {
  uint32_t x0 = (uint32_t)ctr, x1 = (uint32_t)(ctr >> 32), x2 = 0, x3 = 0;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p = (uint64_t)x0 * 0xD2511F53u, q = (uint64_t)x2 * 0xCD9E8D57u;
    x0 = (uint32_t)(q >> 32) ^ x1 ^ key.a[r];
    x1 = (uint32_t)q;
    x2 = (uint32_t)(p >> 32) ^ x3 ^ key.b[r];
    x3 = (uint32_t)p;
  }
  return make_uint4(x0, x1, x2, x3);
}

template <typename T>
struct alignas(16) Vec8 {
  T v[8];
};

template <typename T>
AFB_DEV void unpack(const Vec8<T>& r, float* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 p;
    if constexpr (std::is_same<T, __half>::value) p = __half22float2(reinterpret_cast<const __half2*>(&r)[i]);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value)
      p = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162*>(&r)[i]);
    else p = make_float2(r.v[2 * i], r.v[2 * i + 1]);
    f[2 * i] = p.x;
    f[2 * i + 1] = p.y;
  }
}
template <typename T>
AFB_DEV Vec8<T> pack(const float* f) {
  Vec8<T> r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, __half>::value) reinterpret_cast<uint32_t*>(&r)[i] = pack_f16x2(f[2 * i], f[2 * i + 1]);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value)
      reinterpret_cast<uint32_t*>(&r)[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
    else r.v[2 * i] = f[2 * i], r.v[2 * i + 1] = f[2 * i + 1];
  }
  return r;
}
template <typename T>
AFB_DEV Vec8<T> load8(const T* p) {
  Vec8<T> r;
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(&r)[0] = reinterpret_cast<const float4*>(p)[0];
    reinterpret_cast<float4*>(&r)[1] = reinterpret_cast<const float4*>(p)[1];
  } else {
    *reinterpret_cast<uint4*>(&r) = *reinterpret_cast<const uint4*>(p);
  }
  return r;
}
template <typename T>
AFB_DEV void store8(T* p, const Vec8<T>& r) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = reinterpret_cast<const float4*>(&r)[0];
    reinterpret_cast<float4*>(p)[1] = reinterpret_cast<const float4*>(&r)[1];
  } else {
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&r);
  }
}

// The eight elements of group q: 16 bits of a word are below t when the word, with them in front, is at most
// (t - 1) 2^16 + 65535 -- one comparison, and a shift for the low half; `some` is t > 0
template <typename T, bool RES>
AFB_DEV Vec8<T> apply(const Vec8<T>& x, const Vec8<T>& res, const uint4& w, uint32_t top, bool some, float scale) {
  const uint32_t words[4] = {w.x, w.y, w.z, w.w};
  float f[8], r[8];
  unpack(x, f);
  if (RES) unpack(res, r);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t bits = j & 1 ? words[j >> 1] : words[j >> 1] << 16;
    f[j] = some && bits <= top ? __fmul_rn(f[j], scale) : 0.f;
    if (RES) f[j] = __fadd_rn(f[j], r[j]);
  }
  return pack<T>(f);
}

// a thread takes PER groups of eight elements at a time, a grid apart; VEC: every base is 16-byte aligned
template <typename T, bool VEC, bool RES>
__global__ void __launch_bounds__(256) dropout_kernel(const T* __restrict__ x, const T* __restrict__ res,
                                                      T* __restrict__ y, int64_t n, uint32_t threshold, float scale,
                                                      uint64_t seed, uint64_t offset, const int64_t* __restrict__ rng) {
  constexpr int PER = sizeof(T) == 4 ? 2 : 4;
  grid_dep_wait();
  grid_dep_trigger();
  if (rng) {
    seed += (uint64_t)rng[0];
    offset += (uint64_t)rng[1];
  }
  const Keys key(seed);
  const bool some = threshold > 0;
  const uint32_t top = ((threshold - 1) << 16) | 0xFFFFu;
  const int64_t whole = VEC ? n / 8 : 0, groups = (n + 7) / 8, step = (int64_t)gridDim.x * blockDim.x;
  int64_t q = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  for (; q + (PER - 1) * step < whole; q += PER * step) {
    Vec8<T> a[PER], r[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      a[k] = load8(x + (q + k * step) * 8);
      if (RES) r[k] = load8(res + (q + k * step) * 8);
    }
#pragma unroll
    for (int k = 0; k < PER; ++k)
      store8(y + (q + k * step) * 8,
             apply<T, RES>(a[k], r[k], philox(offset + (uint64_t)(q + k * step), key), top, some, scale));
  }
  for (; q < groups; q += step) {  // the rest, by elements where a group is cut short or unaligned
    const int64_t i0 = q * 8;
    Vec8<T> a, r;
    const uint4 w = philox(offset + (uint64_t)q, key);
    if (q < whole) {
      a = load8(x + i0);
      if (RES) r = load8(res + i0);
      store8(y + i0, apply<T, RES>(a, r, w, top, some, scale));
      continue;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i0 + j < n) {
        a.v[j] = x[i0 + j];
        if (RES) r.v[j] = res[i0 + j];
      }
    a = apply<T, RES>(a, r, w, top, some, scale);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i0 + j < n) y[i0 + j] = a.v[j];
  }
}

template <typename T>
static int run(const void* x, const void* res, void* y, int64_t n, uint32_t threshold, uint64_t seed, uint64_t offset,
               const int64_t* rng, int num_sms, cudaStream_t st) {
  const int64_t groups = (n + 7) / 8;
  const int grid = (int)std::min<int64_t>((groups + 255) / 256, (int64_t)num_sms * 6);
  const float scale = threshold ? (float)(65536.0 / threshold) : 0.f;
  const bool vec = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(res) | reinterpret_cast<uintptr_t>(y)) & 15) == 0;
  auto kern = vec ? (res ? dropout_kernel<T, true, true> : dropout_kernel<T, true, false>)
                  : (res ? dropout_kernel<T, false, true> : dropout_kernel<T, false, false>);
  return launch_pdl(kern, dim3(grid), dim3(256), 0, st, (const T*)x, (const T*)res, (T*)y, n, threshold, scale, seed,
                    offset, rng);
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
