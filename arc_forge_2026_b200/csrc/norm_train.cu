// LayerNorm and zero-centred RMSNorm with trainable weights, forward and backward (dx, dw, db):
//
//   layer  y = xh w + b, xh = (x - mean) rstd      rms  y = xh (1 + w), xh = x rstd
//   v = dy w (or dy (1 + w)); dx = rstd (v - mean(v) - xh mean(v xh))   (rms: without mean(v))
//   dw = sum_rows dy xh, db = sum_rows dy
//
// Memory bounds both directions (forward 2, backward 3 row transfers). A row lives in the registers of WPR warps
// (NV chunks of 8 elements a lane), so it is read once: the variance is the mean square about the mean already known,
// not a difference of two sums. In the backward pass a thread owns the same columns in every row its CTA takes, so dw
// and db add up in its registers over the rows; each CTA writes one row of partial sums and a second kernel adds
// those in a fixed order (no atomics: results are bitwise reproducible).
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "ffn.h"

namespace afb {
namespace norm {

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
// 8 elements from a 16-byte aligned address
template <typename T>
AFB_DEV void load8(const T* p, float* f) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  } else {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    const T* h = reinterpret_cast<const T*>(&q);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = to_f(h[i]);
  }
}
template <typename T>
AFB_DEV void store8(T* p, const float* f) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    uint4 q;
    T* h = reinterpret_cast<T*>(&q);
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = from_f<T>(f[i]);
    *reinterpret_cast<uint4*>(p) = q;
  }
}
// chunk at column c of a row of `width`: elements past the row's end read 0. VEC: width and every row start are
// multiples of 16 bytes, so a chunk is whole or absent.
template <bool VEC, typename T>
AFB_DEV void load_chunk(const T* row, int c, int width, float* f) {
  if constexpr (VEC) {
    if (c < width) {
      load8(row + c, f);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = c + i < width ? to_f(row[c + i]) : 0.f;
  }
}
template <bool VEC, typename T>
AFB_DEV void store_chunk(T* row, int c, int width, const float* f) {
  if constexpr (VEC) {
    if (c < width) store8(row + c, f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < width) row[c + i] = from_f<T>(f[i]);
  }
}
// weights: fp32 or the rows' type
template <bool VEC, typename T>
AFB_DEV void load_weight(const void* w, int w32, int c, int width, float* f) {
  if (w32) load_chunk<VEC>(reinterpret_cast<const float*>(w), c, width, f);
  else load_chunk<VEC>(reinterpret_cast<const T*>(w), c, width, f);
}

// sums over the WPR warps of a row; `red` holds WPR slots per row group, `bar` is the group's named barrier
template <int WPR>
AFB_DEV float2 row_sum2(float2 v, float2* red, int wr, int bar) {
  v.x = warp_sum(v.x);
  v.y = warp_sum(v.y);
  if constexpr (WPR > 1) {
    if ((threadIdx.x & 31) == 0) red[wr] = v;
    named_bar_sync(bar, WPR * 32);
    v = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < WPR; ++i) {
      const float2 r = red[i];
      v.x += r.x;
      v.y += r.y;
    }
    named_bar_sync(bar, WPR * 32);  // the slots may be written again
  }
  return v;
}

template <int WPR>
struct Block {
  static constexpr int THREADS = WPR > 8 ? WPR * 32 : 256, GROUPS = THREADS / (WPR * 32);
};

template <typename T, int WPR, int NV, bool VEC>
__global__ void __launch_bounds__(Block<WPR>::THREADS) norm_fwd_kernel(NormArgs a) {
  grid_dep_wait();
  grid_dep_trigger();
  constexpr int G = Block<WPR>::GROUPS;
  __shared__ float2 red[G][WPR];
  const int grp = threadIdx.x / (WPR * 32), t = threadIdx.x % (WPR * 32), wr = t >> 5;
  const int w32 = a.wtype == ELEM_FP32;
  const float inv = 1.f / a.width;
  for (int64_t row = (int64_t)blockIdx.x * G + grp; row < a.rows; row += (int64_t)gridDim.x * G) {
    const T* x = reinterpret_cast<const T*>(a.x) + row * a.ldx;
    float v[NV][8];
#pragma unroll
    for (int p = 0; p < NV; ++p) load_chunk<VEC>(x, (p * WPR * 32 + t) * 8, a.width, v[p]);
    float mean = 0.f;
    if (!a.rms) {
      float s = 0.f;
#pragma unroll
      for (int p = 0; p < NV; ++p)
#pragma unroll
        for (int i = 0; i < 8; ++i) s += v[p][i];
      mean = row_sum2<WPR>(make_float2(s, 0.f), red[grp], wr, 1 + grp).x * inv;
    }
    float q = 0.f;
#pragma unroll
    for (int p = 0; p < NV; ++p)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = v[p][i] - mean;
        if ((p * WPR * 32 + t) * 8 + i < a.width) q += d * d;
      }
    const float rstd = rsqrtf(row_sum2<WPR>(make_float2(q, 0.f), red[grp], wr, 1 + grp).x * inv + a.eps);
    if (t == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
    T* y = reinterpret_cast<T*>(a.y) + row * a.width;
#pragma unroll
    for (int p = 0; p < NV; ++p) {
      const int c = (p * WPR * 32 + t) * 8;
      float w[8], b[8];
      load_weight<VEC, T>(a.w, w32, c, a.width, w);
      if (a.b) load_weight<VEC, T>(a.b, w32, c, a.width, b);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float xh = (v[p][i] - mean) * rstd;
        v[p][i] = a.rms ? xh * (1.f + w[i]) : (a.b ? xh * w[i] + b[i] : xh * w[i]);
      }
      store_chunk<VEC>(y, c, a.width, v[p]);
    }
  }
}

template <typename T, int WPR, int NV, bool VEC>
__global__ void __launch_bounds__(Block<WPR>::THREADS) norm_bwd_kernel(NormArgs a) {
  grid_dep_wait();
  grid_dep_trigger();
  constexpr int G = Block<WPR>::GROUPS;
  __shared__ float2 red[G][WPR];
  __shared__ float comb[G > 1 ? Block<WPR>::THREADS * 8 : 1];
  const int grp = threadIdx.x / (WPR * 32), t = threadIdx.x % (WPR * 32), wr = t >> 5;
  const int w32 = a.wtype == ELEM_FP32;
  const float inv = 1.f / a.width;
  float dw[NV][8] = {}, db[NV][8] = {};
  for (int64_t row = (int64_t)blockIdx.x * G + grp; row < a.rows; row += (int64_t)gridDim.x * G) {
    const T* x = reinterpret_cast<const T*>(a.x) + row * a.ldx;
    const T* dy = reinterpret_cast<const T*>(a.dy) + row * a.width;
    const float rstd = a.rstd[row], mean = a.rms ? 0.f : a.mean[row];
    float xh[NV][8], v[NV][8];
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int p = 0; p < NV; ++p) {
      const int c = (p * WPR * 32 + t) * 8;
      load_chunk<VEC>(x, c, a.width, xh[p]);
      load_chunk<VEC>(dy, c, a.width, v[p]);
    }
#pragma unroll
    for (int p = 0; p < NV; ++p) {
      const int c = (p * WPR * 32 + t) * 8;
      float w[8];
      load_weight<VEC, T>(a.w, w32, c, a.width, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = v[p][i], h = (xh[p][i] - mean) * rstd;  // past the row's end d and so v are 0
        dw[p][i] += d * h;
        db[p][i] += d;
        xh[p][i] = h;
        v[p][i] = c + i < a.width ? d * (a.rms ? 1.f + w[i] : w[i]) : 0.f;
        s.x += v[p][i] * h;
        s.y += v[p][i];
      }
    }
    if (a.dx) {
      s = row_sum2<WPR>(s, red[grp], wr, 1 + grp);
      const float m1 = s.x * inv, m0 = a.rms ? 0.f : s.y * inv;
      T* dx = reinterpret_cast<T*>(a.dx) + row * a.width;
#pragma unroll
      for (int p = 0; p < NV; ++p) {
        float o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = rstd * (v[p][i] - m0 - xh[p][i] * m1);
        store_chunk<VEC>(dx, (p * WPR * 32 + t) * 8, a.width, o);
      }
    }
  }
  if (!a.dw && !a.db) return;
  float* out = a.partial + (int64_t)blockIdx.x * 2 * a.width;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float(*acc)[8] = k ? db : dw;
#pragma unroll
    for (int p = 0; p < NV; ++p) {
      const int c = (p * WPR * 32 + t) * 8;
      if constexpr (G > 1) {  // the CTA's row groups, in order
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) comb[(i * G + grp) * WPR * 32 + t] = acc[p][i];
        __syncthreads();
        if (grp == 0) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float f = 0.f;
#pragma unroll
            for (int j = 0; j < G; ++j) f += comb[(i * G + j) * WPR * 32 + t];
            acc[p][i] = f;
          }
        }
      }
      if (grp == 0) store_chunk<false>(out + k * a.width, c, a.width, acc[p]);
    }
  }
}

// column sums of the partial rows: CTA of 32 columns x 8 row lanes
template <typename T>
__global__ void __launch_bounds__(256) norm_reduce_kernel(const float* __restrict__ part, int n, int width,
                                                          void* __restrict__ dw, void* __restrict__ db, int w32) {
  grid_dep_wait();
  __shared__ float red[8][33];
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + cx;  // over [dw | db]
  float s = 0.f;
  if (col < 2 * width)
    for (int r = ry; r < n; r += 8) s += part[(int64_t)r * 2 * width + col];
  red[ry][cx] = s;
  __syncthreads();
  if (ry || col >= 2 * width) return;
  float f = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) f += red[j][cx];
  void* out = col < width ? dw : db;
  const int c = col < width ? col : col - width;
  if (!out) return;
  if (w32) reinterpret_cast<float*>(out)[c] = f;
  else reinterpret_cast<T*>(out)[c] = from_f<T>(f);
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
static bool vec_ok(const NormArgs& a) {
  return a.width % 8 == 0 && a.ldx % 8 == 0 && aligned16(a.x) && aligned16(a.y) && aligned16(a.w) && aligned16(a.b) &&
         aligned16(a.dy) && aligned16(a.dx);
}

struct Shape {
  int wpr, nv;
};
// warps per row and chunks per lane: at most 4 chunks (32 elements) a lane, so a backward row and its two sums stay
// in registers
static Shape shape_of(const NormArgs& a) {
  const int chunks = (a.width + 7) / 8;
  int wpr = 1;
  while (wpr < 16 && chunks > wpr * 32 * 4) wpr *= 2;
  int nv = (chunks + wpr * 32 - 1) / (wpr * 32);
  if (!vec_ok(a)) nv = 4;  // one unaligned variant for each row size
  return {wpr, nv};
}
static int grid_of(const NormArgs& a, const Shape& s, int num_sms, int per_sm) {
  const int groups = s.wpr > 8 ? 1 : 8 / s.wpr;
  const int64_t blocks = (a.rows + groups - 1) / groups;
  return (int)std::max<int64_t>(1, std::min<int64_t>(blocks, (int64_t)num_sms * per_sm));
}
constexpr int FWD_PER_SM = 8, BWD_PER_SM = 2;

template <typename T, int WPR, int NV, bool VEC>
static int run_fwd(const NormArgs& a, int grid, cudaStream_t st) {
  return launch_pdl(norm_fwd_kernel<T, WPR, NV, VEC>, dim3(grid), dim3(Block<WPR>::THREADS), 0, st, a);
}
template <typename T, int WPR, int NV, bool VEC>
static int run_bwd(const NormArgs& a, int grid, cudaStream_t st) {
  return launch_pdl(norm_bwd_kernel<T, WPR, NV, VEC>, dim3(grid), dim3(Block<WPR>::THREADS), 0, st, a);
}

template <typename T, bool BWD>
static int dispatch(const NormArgs& a, int num_sms, cudaStream_t st) {
  const Shape s = shape_of(a);
  const int grid = grid_of(a, s, num_sms, BWD ? BWD_PER_SM : FWD_PER_SM);
  const bool vec = vec_ok(a);
#define AFB_NORM(W, N, V) \
  if (s.wpr == W && s.nv == N && vec == V) return BWD ? run_bwd<T, W, N, V>(a, grid, st) : run_fwd<T, W, N, V>(a, grid, st);
  AFB_NORM(1, 1, true)
  AFB_NORM(1, 2, true)
  AFB_NORM(1, 3, true)
  AFB_NORM(1, 4, true)
  AFB_NORM(2, 3, true)
  AFB_NORM(2, 4, true)
  AFB_NORM(4, 3, true)
  AFB_NORM(4, 4, true)
  AFB_NORM(8, 3, true)
  AFB_NORM(8, 4, true)
  AFB_NORM(16, 3, true)
  AFB_NORM(16, 4, true)
  AFB_NORM(1, 4, false)
  AFB_NORM(2, 4, false)
  AFB_NORM(4, 4, false)
  AFB_NORM(8, 4, false)
  AFB_NORM(16, 4, false)
#undef AFB_NORM
  return 3;
}

static bool valid(const NormArgs& a) {
  return a.width >= 1 && a.width <= NORM_MAX_WIDTH && a.rows >= 0 && a.dtype >= 0 && a.dtype <= 2 &&
         (a.wtype == ELEM_FP32 || a.wtype == a.dtype);
}

}  // namespace norm

int norm_bwd_partials(const NormArgs& a, int num_sms) {
  return norm::grid_of(a, norm::shape_of(a), num_sms, norm::BWD_PER_SM);
}

int norm_fwd(const NormArgs& a, int num_sms, cudaStream_t st) {
  if (!norm::valid(a)) return 3;
  if (a.rows == 0) return 0;
  if (a.dtype == ELEM_BF16) return norm::dispatch<__nv_bfloat16, false>(a, num_sms, st);
  if (a.dtype == ELEM_FP16) return norm::dispatch<__half, false>(a, num_sms, st);
  return norm::dispatch<float, false>(a, num_sms, st);
}

int norm_bwd(const NormArgs& a, int num_sms, cudaStream_t st) {
  if (!norm::valid(a)) return 3;
  if (a.rows == 0) return 0;  // the caller zeroes dw and db
  int rc;
  if (a.dtype == ELEM_BF16) rc = norm::dispatch<__nv_bfloat16, true>(a, num_sms, st);
  else if (a.dtype == ELEM_FP16) rc = norm::dispatch<__half, true>(a, num_sms, st);
  else rc = norm::dispatch<float, true>(a, num_sms, st);
  if (rc || (!a.dw && !a.db)) return rc;
  const dim3 grid((2 * a.width + 31) / 32);
  const int n = norm_bwd_partials(a, num_sms), w32 = a.wtype == ELEM_FP32;
  if (a.dtype == ELEM_BF16)
    return launch_pdl(norm::norm_reduce_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, (const float*)a.partial, n,
                      a.width, a.dw, a.db, w32);
  if (a.dtype == ELEM_FP16)
    return launch_pdl(norm::norm_reduce_kernel<__half>, grid, dim3(256), 0, st, (const float*)a.partial, n, a.width,
                      a.dw, a.db, w32);
  return launch_pdl(norm::norm_reduce_kernel<float>, grid, dim3(256), 0, st, (const float*)a.partial, n, a.width,
                    a.dw, a.db, w32);
}

}  // namespace afb
