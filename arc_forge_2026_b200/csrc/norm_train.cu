// LayerNorm and zero-centred RMSNorm with trainable weights, forward and backward (dx, dw, db):
//
//   layer  y = xh w + b, xh = (x - mean) rstd      rms  y = xh (1 + w), xh = x rstd
//   v = dy w (or dy (1 + w)); dx = rstd (v - mean(v) - xh mean(v xh))   (rms: without mean(v))
//   dw = sum_rows dy xh, db = sum_rows dy
//
// Memory bounds both directions (forward 2, backward 3 row transfers), and some 45 KB have to be on the way to an SM at
// any time to use it. CTAs stay and walk the rows; bulk copies bring the next rows of x (and dy) into a ring in shared
// memory, several rows ahead. A group of warps takes a row into registers, NV chunks of 8 elements a lane, so it is read
// once: the variance is the mean square about the mean already known, not a difference of two sums. A thread owns the
// same columns in every row, so the weights are read once and dw and db add up in registers. Each CTA writes one row of
// partial sums of dw and db and a second kernel adds those in a fixed order (no atomics: results are bitwise
// reproducible).
//
// Measured (one B200): 16,383 x 2,048 fp32 forward 43 us (6.3 TB/s), backward 72 (5.6) + 4 for the sums;
// 5,633 x 4,608 bf16 29 (3.6), 36 (4.3) + 4. 16-bit rows have twice the elements a byte, some 11 instructions each
// forward and 17 backward: neither memory (24 % and 42 % busy with reads and writes of DRAM) nor the issue slots (44 % and
// 53 %) bound them, but the twelve warps an SM that the registers leave, which wait for their own shuffles and results.
// Rows that leave an SM one CTA (past 4,608 columns backward, 8,192 forward) are slower: 4,096 x 8,192 bf16 40 and 50 us,
// 2,048 x 16,384 40 and 144.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "ffn.h"

namespace afb {
namespace norm {

template <typename T>
AFB_DEV T from_f(float v) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return __float2bfloat16(v);
  else if constexpr (std::is_same<T, __half>::value) return __float2half(v);
  else return v;
}
// 8 elements as they lie in memory
template <typename T>
struct alignas(16) Raw {
  T v[8];
};
template <typename T>
AFB_DEV void unpack(const Raw<T>& r, float* f) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = r.v[i];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 p;
      if constexpr (std::is_same<T, __half>::value) p = __half22float2(reinterpret_cast<const __half2*>(&r)[i]);
      else p = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162*>(&r)[i]);
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  }
}
template <typename T>
AFB_DEV Raw<T> pack(const float* f) {
  Raw<T> r;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = f[i];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      reinterpret_cast<uint32_t*>(&r)[i] = std::is_same<T, __half>::value ? pack_f16x2(f[2 * i], f[2 * i + 1])
                                                                           : pack_bf16x2(f[2 * i], f[2 * i + 1]);
  }
  return r;
}
// a CTA's rows at a time: `groups` groups of `wpr` warps
struct Group {
  int wpr, lanes, idx, t;  // warps and threads of a group, this thread's group and its place in it
  AFB_DEV explicit Group(int wpr_) : wpr(wpr_), lanes(wpr_ * 32), idx(threadIdx.x / lanes), t(threadIdx.x - idx * lanes) {}
};
// Column of element i of a lane's chunk p; V elements are accessed at a time. 8 (width and every row start are
// multiples of 16 bytes): eight in a row, so a chunk is whole or absent. Else by pairs (16-bit rows of even width that
// start on 4 bytes) or one by one, across the lanes, so that a warp's accesses are contiguous.
template <int V>
AFB_DEV int col_of(const Group& g, int p, int i) {
  if (V == 8) return (p * g.lanes + g.t) * 8 + i;
  if (V == 2) return ((p * 4 + (i >> 1)) * g.lanes + g.t) * 2 + (i & 1);
  return (p * 8 + i) * g.lanes + g.t;
}
// elements past the row's end read 0
template <int V, typename T>
AFB_DEV Raw<T> load_chunk(const T* row, const Group& g, int p, int width) {
  Raw<T> r;
  if constexpr (V == 8) {
    const int c = col_of<8>(g, p, 0);
    if (c < width) {
      if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(&r)[0] = reinterpret_cast<const float4*>(row + c)[0];
        reinterpret_cast<float4*>(&r)[1] = reinterpret_cast<const float4*>(row + c)[1];
      } else {
        *reinterpret_cast<uint4*>(&r) = *reinterpret_cast<const uint4*>(row + c);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) r.v[i] = from_f<T>(0.f);
    }
  } else if constexpr (V == 2 && sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = col_of<2>(g, p, 2 * i);
      reinterpret_cast<uint32_t*>(&r)[i] = c < width ? *reinterpret_cast<const uint32_t*>(row + c) : 0u;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = col_of<V>(g, p, i);
      r.v[i] = c < width ? row[c] : from_f<T>(0.f);
    }
  }
  return r;
}
template <int V, typename T>
AFB_DEV void store_chunk(T* row, const Group& g, int p, int width, const float* f) {
  if constexpr (V == 8) {
    const int c = col_of<8>(g, p, 0);
    if (c < width) {
      Raw<T> r = pack<T>(f);
      if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(row + c)[0] = reinterpret_cast<float4*>(&r)[0];
        reinterpret_cast<float4*>(row + c)[1] = reinterpret_cast<float4*>(&r)[1];
      } else {
        *reinterpret_cast<uint4*>(row + c) = *reinterpret_cast<uint4*>(&r);
      }
    }
  } else if constexpr (V == 2 && sizeof(T) == 2) {
    const Raw<T> r = pack<T>(f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = col_of<2>(g, p, 2 * i);
      if (c < width) *reinterpret_cast<uint32_t*>(row + c) = reinterpret_cast<const uint32_t*>(&r)[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = col_of<V>(g, p, i);
      if (c < width) row[c] = from_f<T>(f[i]);
    }
  }
}
// weights (fp32 or the rows' type) as factors, 0 past the row's end
template <int V, typename T>
AFB_DEV void load_weight(const void* w, int w32, const Group& g, int p, int width, float* f) {
  if (w32) unpack(load_chunk<V>(reinterpret_cast<const float*>(w), g, p, width), f);
  else unpack(load_chunk<V>(reinterpret_cast<const T*>(w), g, p, width), f);
}
template <int V, typename T>
AFB_DEV void load_factor(const NormArgs& a, const Group& g, int p, float* f) {
  load_weight<V, T>(a.w, a.wtype == ELEM_FP32, g, p, a.width, f);
  if (a.rms) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = col_of<V>(g, p, i) < a.width ? 1.f + f[i] : 0.f;
  }
}

constexpr int MAX_WPR = 32;
// two sums over the warps of a row. Each warp leaves its sums in a slot and after one barrier adds up all of them;
// two sets of slots in turn (`ph`) make a second barrier unnecessary: a warp that writes a set again has passed the
// barrier of the other one, which every warp reaches after its last read of this one.
struct Slots {
  float2 v[2][MAX_WPR];
};
AFB_DEV float row_sum(float v, Slots& slots, const Group& g, int& ph) {
  v = warp_sum(v);
  if (g.wpr > 1) {
    const int lane = threadIdx.x & 31;
    if (lane == 0) slots.v[ph][g.t >> 5].x = v;
    named_bar_sync(1 + g.idx, g.lanes);
    v = warp_sum(lane < g.wpr ? slots.v[ph][lane].x : 0.f);
    ph ^= 1;
  }
  return v;
}
AFB_DEV float2 row_sum2(float2 v, Slots& slots, const Group& g, int& ph) {
  v.x = warp_sum(v.x);
  v.y = warp_sum(v.y);
  if (g.wpr > 1) {
    const int lane = threadIdx.x & 31;
    if (lane == 0) slots.v[ph][g.t >> 5] = v;
    named_bar_sync(1 + g.idx, g.lanes);
    v = lane < g.wpr ? slots.v[ph][lane] : make_float2(0.f, 0.f);
    v.x = warp_sum(v.x);
    v.y = warp_sum(v.y);
    ph ^= 1;
  }
  return v;
}

// The ring of a group: `depth` slots, a row of x (and of dy) each. A row is copied as the 16-byte blocks that hold it
// (none of them is without a byte of the row, so none lies outside the allocation).
constexpr int MAX_DEPTH = 8;
struct RingShape {
  int depth, part;  // slots; bytes of one row in a slot: the row rounded up to 16, and 16 more for its offset
};
// 16-byte blocks of `bytes` bytes at p
AFB_DEV uint32_t span(const uint8_t* p, int bytes) {
  return (uint32_t)(((reinterpret_cast<uintptr_t>(p) & 15) + bytes + 15) & ~uintptr_t(15));
}
AFB_DEV const void* block_of(const uint8_t* p) {
  return reinterpret_cast<const void*>(reinterpret_cast<uintptr_t>(p) & ~uintptr_t(15));
}
// What every thread of a group keeps of its ring: the slot of the row at hand and that slot's parity; and the thread
// that fetches: the next row to fetch and its place. Counted, not divided: a division would cost as much as an element's
// arithmetic does.
template <int PARTS>
struct Ring {
  uint8_t *base, *slot;
  uint64_t *full0, *full;
  int slot_bytes, part, depth, at;
  uint32_t parity;
  const uint8_t *x, *dy;  // the row at hand (PARTS 1: x alone)
  int64_t x_step, dy_step;
  int bytes;
  uint32_t* status;

  AFB_DEV void fetch(uint8_t* dst, uint64_t* bar, const uint8_t* xs, const uint8_t* ds) const {
    const uint32_t nx = span(xs, bytes), nd = PARTS > 1 ? span(ds, bytes) : 0u;
    mbar_arrive_expect_tx(bar, nx + nd);
    bulk_load_1d(dst, block_of(xs), nx, bar);
    if (PARTS > 1) bulk_load_1d(dst + part, block_of(ds), nd, bar);
  }
  AFB_DEV void start(int n) const {  // one thread: the first rows
    for (int k = 0; k < min(n, depth); ++k)
      fetch(base + k * slot_bytes, full0 + k, x + k * x_step, PARTS > 1 ? dy + k * dy_step : nullptr);
  }
  AFB_DEV bool wait() const { return mbar_wait(full, parity, status); }
  AFB_DEV void refill() const {  // one thread: the row `depth` further into the slot at hand
    fetch(slot, full, x + depth * x_step, PARTS > 1 ? dy + depth * dy_step : nullptr);
  }
  AFB_DEV void next() {
    x += x_step;
    if (PARTS > 1) dy += dy_step;
    slot += slot_bytes;
    ++full;
    if (++at == depth) at = 0, slot = base, full = full0, parity ^= 1;
  }
};

// A group's threads leave together: one that gave up waiting says at which row before that row's barrier (a later row's
// number does not stop a warp that has yet to look: it meets the others at that row's barrier)
AFB_DEV void group_sync(const Group& g) {
  if (g.wpr > 1) named_bar_sync(1 + g.idx, g.lanes);
  else __syncwarp();
}

template <typename T, int NV, int V, int MAXT>
__global__ void __launch_bounds__(MAXT) norm_fwd_kernel(NormArgs a, int wpr, int groups, RingShape rs) {
  extern __shared__ __align__(16) uint8_t ring_smem[];
  __shared__ Slots slots_s[8];
  __shared__ uint64_t full_s[8][MAX_DEPTH];
  __shared__ int bad_s[8];
  const Group g(wpr);
  Slots& slots = slots_s[g.idx];
  volatile int* bad = &bad_s[g.idx];
  if (g.t == 0) {
    for (int i = 0; i < rs.depth; ++i) mbar_init(&full_s[g.idx][i], 1);
    fence_mbar_init();
    fence_proxy_async_smem();
    *bad = INT32_MAX;
  }
  __syncthreads();
  grid_dep_wait();
  grid_dep_trigger();
  int ph = 0;
  const float inv = 1.f / a.width;
  const int64_t stride = (int64_t)gridDim.x * groups, row0 = (int64_t)blockIdx.x * groups + g.idx;
  const int n = row0 < a.rows ? (int)((a.rows - 1 - row0) / stride) + 1 : 0;  // rows of this group
  Ring<1> ring;
  ring.part = ring.slot_bytes = rs.part, ring.depth = rs.depth, ring.at = 0, ring.parity = 0, ring.status = a.status;
  ring.base = ring.slot = ring_smem + (size_t)g.idx * rs.depth * rs.part;
  ring.full0 = ring.full = full_s[g.idx];
  ring.bytes = a.width * (int)sizeof(T);
  ring.x = reinterpret_cast<const uint8_t*>(reinterpret_cast<const T*>(a.x) + row0 * a.ldx);
  ring.x_step = stride * a.ldx * (int64_t)sizeof(T);
  if (g.t == 0) ring.start(n);
  float m[NV][8], b[NV][8];
#pragma unroll
  for (int p = 0; p < NV; ++p) {
    load_factor<V, T>(a, g, p, m[p]);
    if (a.b) {
      load_weight<V, T>(a.b, a.wtype == ELEM_FP32, g, p, a.width, b[p]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) b[p][i] = 0.f;
    }
  }
  T* y = reinterpret_cast<T*>(a.y) + row0 * a.width;
  int k = 0;
  for (; k < n; ++k, ring.next(), y += stride * a.width) {
    if (!ring.wait()) *bad = k;
    const T* x = reinterpret_cast<const T*>(ring.slot + (V == 8 ? 0 : reinterpret_cast<uintptr_t>(ring.x) & 15));
    float v[NV][8];
#pragma unroll
    for (int p = 0; p < NV; ++p) unpack(load_chunk<V>(x, g, p, a.width), v[p]);
    group_sync(g);  // the slot has been read
    if (*bad <= k) break;
    if (g.t == 0 && k + rs.depth < n) ring.refill();
    float mean = 0.f;
    if (!a.rms) {
      float s = 0.f;
#pragma unroll
      for (int p = 0; p < NV; ++p)
#pragma unroll
        for (int i = 0; i < 8; ++i) s += v[p][i];
      mean = row_sum(s, slots, g, ph) * inv;
#pragma unroll
      for (int p = 0; p < NV; ++p)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[p][i] -= mean;
    }
    float q = 0.f;
#pragma unroll
    for (int p = 0; p < NV; ++p) {
      if (V == 8 && col_of<V>(g, p, 0) >= a.width) continue;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (V == 8 || col_of<V>(g, p, i) < a.width) q += v[p][i] * v[p][i];
    }
    const float rstd = rsqrtf(row_sum(q, slots, g, ph) * inv + a.eps);
    if (g.t == 0) {
      if (a.mean) a.mean[row0 + k * stride] = mean;
      if (a.rstd) a.rstd[row0 + k * stride] = rstd;
    }
#pragma unroll
    for (int p = 0; p < NV; ++p) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[p][i] = v[p][i] * rstd * m[p][i] + b[p][i];
      store_chunk<V>(y, g, p, a.width, v[p]);
    }
  }
  if (k < n && g.t == 0)  // after a failed wait: the copies in flight land first
    for (int j = k; j < min(n, k + rs.depth); ++j, ring.next()) ring.wait();
}

template <typename T, int NV, int V, int MAXT, int MINB = 1>
__global__ void __launch_bounds__(MAXT, MINB) norm_bwd_kernel(NormArgs a, int wpr, int groups, RingShape rs) {
  extern __shared__ __align__(16) uint8_t ring_smem[];
  __shared__ Slots slots_s[8];
  __shared__ uint64_t full_s[8][MAX_DEPTH];
  __shared__ int bad_s[8];
  __shared__ float comb[256 * 8];  // more than one group: 256 threads at most
  const Group g(wpr);
  Slots& slots = slots_s[g.idx];
  volatile int* bad = &bad_s[g.idx];
  if (g.t == 0) {
    for (int i = 0; i < rs.depth; ++i) mbar_init(&full_s[g.idx][i], 1);
    fence_mbar_init();
    fence_proxy_async_smem();
    *bad = INT32_MAX;
  }
  __syncthreads();
  grid_dep_wait();
  grid_dep_trigger();
  int ph = 0;
  const float inv = 1.f / a.width;
  const int lane = threadIdx.x & 31;
  float dw[NV][8] = {}, db[NV][8] = {};
  const int64_t stride = (int64_t)gridDim.x * groups, row0 = (int64_t)blockIdx.x * groups + g.idx;
  const int n = row0 < a.rows ? (int)((a.rows - 1 - row0) / stride) + 1 : 0;
  Ring<2> ring;
  ring.part = rs.part, ring.slot_bytes = 2 * rs.part, ring.depth = rs.depth, ring.at = 0, ring.parity = 0;
  ring.base = ring.slot = ring_smem + (size_t)g.idx * rs.depth * rs.part * 2;
  ring.full0 = ring.full = full_s[g.idx];
  ring.bytes = a.width * (int)sizeof(T), ring.status = a.status;
  ring.x = reinterpret_cast<const uint8_t*>(reinterpret_cast<const T*>(a.x) + row0 * a.ldx);
  ring.dy = reinterpret_cast<const uint8_t*>(reinterpret_cast<const T*>(a.dy) + row0 * a.width);
  ring.x_step = stride * a.ldx * (int64_t)sizeof(T);
  ring.dy_step = stride * a.width * (int64_t)sizeof(T);
  if (g.t == 0) ring.start(n);
  float m[NV][8];
#pragma unroll
  for (int p = 0; p < NV; ++p) load_factor<V, T>(a, g, p, m[p]);
  float my_rstd = 0.f, my_mean = 0.f;  // of 32 rows, one a lane
  T* dx = reinterpret_cast<T*>(a.dx) + row0 * a.width;
  int k = 0;
  for (; k < n; ++k, ring.next(), dx += stride * a.width) {
    if ((k & 31) == 0 && k + lane < n) {
      my_rstd = a.rstd[row0 + (k + lane) * stride];
      if (!a.rms) my_mean = a.mean[row0 + (k + lane) * stride];
    }
    if (!ring.wait()) *bad = k;
    const T* x = reinterpret_cast<const T*>(ring.slot + (V == 8 ? 0 : reinterpret_cast<uintptr_t>(ring.x) & 15));
    const T* dy = reinterpret_cast<const T*>(ring.slot + rs.part + (V == 8 ? 0 : reinterpret_cast<uintptr_t>(ring.dy) & 15));
    float h[NV][8], v[NV][8];
#pragma unroll
    for (int p = 0; p < NV; ++p) {
      unpack(load_chunk<V>(x, g, p, a.width), h[p]);
      unpack(load_chunk<V>(dy, g, p, a.width), v[p]);
    }
    group_sync(g);  // the slot has been read
    if (*bad <= k) break;
    if (g.t == 0 && k + rs.depth < n) ring.refill();
    const float r = __shfl_sync(0xffffffffu, my_rstd, k & 31), mu = __shfl_sync(0xffffffffu, my_mean, k & 31);
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int p = 0; p < NV; ++p)
#pragma unroll
      for (int i = 0; i < 8; ++i) {  // past the row's end dy and the factor are 0, and so is what they enter
        h[p][i] = (h[p][i] - mu) * r;
        dw[p][i] += v[p][i] * h[p][i];
        db[p][i] += v[p][i];
        v[p][i] *= m[p][i];
        s.x += v[p][i] * h[p][i];
        s.y += v[p][i];
      }
    if (a.dx) {
      s = row_sum2(s, slots, g, ph);
      const float m1 = s.x * inv, m0 = a.rms ? 0.f : s.y * inv;
#pragma unroll
      for (int p = 0; p < NV; ++p) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[p][i] = r * (v[p][i] - m0 - h[p][i] * m1);
        store_chunk<V>(dx, g, p, a.width, v[p]);
      }
    }
  }
  if (k < n && g.t == 0)  // after a failed wait: the copies in flight land first
    for (int j = k; j < min(n, k + rs.depth); ++j, ring.next()) ring.wait();
  if (!a.dw && !a.db) return;
  float* out = a.partial + (int64_t)blockIdx.x * 2 * a.width;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float(*acc)[8] = k ? db : dw;
#pragma unroll
    for (int p = 0; p < NV; ++p) {
      if (groups > 1) {  // the CTA's row groups, in order
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) comb[(i * groups + g.idx) * g.lanes + g.t] = acc[p][i];
        __syncthreads();
        if (g.idx == 0) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float f = 0.f;
            for (int j = 0; j < groups; ++j) f += comb[(i * groups + j) * g.lanes + g.t];
            acc[p][i] = f;
          }
        }
      }
      if (g.idx == 0) store_chunk<V>(out + k * a.width, g, p, a.width, acc[p]);
    }
  }
}

// column sums of the partial rows: CTA of 32 columns x 32 row lanes
template <typename T>
__global__ void __launch_bounds__(1024) norm_reduce_kernel(const float* __restrict__ part, int n, int width,
                                                          void* __restrict__ dw, void* __restrict__ db, int w32) {
  grid_dep_wait();
  __shared__ float red[32][33];
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + cx;  // over [dw | db]
  float s = 0.f;
  if (col < 2 * width)
    for (int r = ry; r < n; r += 32) s += part[(int64_t)r * 2 * width + col];
  red[ry][cx] = s;
  __syncthreads();
  if (ry || col >= 2 * width) return;
  float f = 0.f;
#pragma unroll
  for (int j = 0; j < 32; ++j) f += red[j][cx];
  void* out = col < width ? dw : db;
  const int c = col < width ? col : col - width;
  if (!out) return;
  if (w32) reinterpret_cast<float*>(out)[c] = f;
  else reinterpret_cast<T*>(out)[c] = from_f<T>(f);
}

static bool aligned(const void* p, int to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
// elements accessed at a time (col_of): of the rows and of the weights, which are read the same way (fp32 weights by
// pairs one by one) and may start at any element of a flat buffer
static int access_of(const NormArgs& a) {
  auto rows = [&](int to) { return aligned(a.x, to) && aligned(a.y, to) && aligned(a.dy, to) && aligned(a.dx, to); };
  auto weights = [&](int to) { return aligned(a.w, to) && aligned(a.b, to); };
  if (a.width % 8 == 0 && a.ldx % 8 == 0 && rows(16) && weights(16) && aligned(a.partial, 16)) return 8;
  return a.dtype != ELEM_FP32 && a.width % 2 == 0 && a.ldx % 2 == 0 && rows(4) && weights(4) ? 2 : 1;
}

struct Shape {
  int nv, wpr, groups, grid;
  RingShape ring;
  int smem;
};
using Kernel = void (*)(NormArgs, int, int, RingShape);

template <typename T, int NV, int MAXT>
static Kernel fwd_kernel(int v) {
  if constexpr (sizeof(T) == 2)
    if (v == 2) return norm_fwd_kernel<T, NV, 2, MAXT>;
  return v == 8 ? norm_fwd_kernel<T, NV, 8, MAXT> : norm_fwd_kernel<T, NV, 1, MAXT>;
}
template <typename T, int NV, int MAXT, int MINB = 1>
static Kernel bwd_kernel(int v) {
  if constexpr (sizeof(T) == 2)
    if (v == 2) return norm_bwd_kernel<T, NV, 2, MAXT, MINB>;
  return v == 8 ? norm_bwd_kernel<T, NV, 8, MAXT, MINB> : norm_bwd_kernel<T, NV, 1, MAXT, MINB>;
}
// the chunks and warps that plan() chooses
template <typename T, bool BWD>
static Kernel kernel_of(int nv, int v, int wpr) {
  if constexpr (BWD) {
    if (nv == 1) return bwd_kernel<T, 1, 256>(v);
    if (nv == 2) return wpr > 8 ? bwd_kernel<T, 2, 512>(v) : bwd_kernel<T, 2, 256>(v);
    if (nv == 3) return bwd_kernel<T, 3, 192, 2>(v);  // registers for two CTAs an SM
    return bwd_kernel<T, 4, 512>(v);
  } else {
    if (nv == 1) return fwd_kernel<T, 1, 256>(v);
    if (nv == 2) return fwd_kernel<T, 2, 256>(v);
    if (nv == 3) return fwd_kernel<T, 3, 256>(v);
    return wpr > 8 ? fwd_kernel<T, 4, 512>(v) : fwd_kernel<T, 4, 256>(v);
  }
}

constexpr int RING_SMEM = 160 * 1024;  // of an SM; four CTAs' static shared memory (13 KB each) fits beside it
constexpr int RING_AHEAD = 96 * 1024;  // of that, what the CTAs of an SM keep on the way

// Chunks a lane, warps a row, rows a CTA, CTAs, ring. Forward, the instructions a row takes decide the first two: some 8
// an element and 75 a warp for its sums, so few warps with much each, as far as the lanes' last chunks are not left
// idle (5,632 rows of 1,152 in bf16: three chunks 11 us, one 14, two 15, four 14). Backward, two chunks a lane (16,384
// rows of 2,048 in bf16: 46 us; one chunk 61, for the sums of twice the warps; three 49 and four 65, for want of
// registers), one where a row is 512 columns or less, and four where it passes 8,192. Where two would take more than six
// warps they leave an SM one CTA, and three, up to the six warps of which two CTAs fit, are better in 16 bits and alike in
// fp32 (10,485 rows of 3,200 in bf16 58 us, two 72; 8,192 of 4,096 49 and 59; 7,281 of 4,608 45 and 66; in fp32 4,096 of
// 4,096 42 and 43). From 4,609 columns the backward pass has one CTA an SM (7,269 of 4,616 in bf16 67 us, 4,096 of 8,192
// 50), the forward pass from 8,193.
// CTAs: as many as are resident (a second wave would wait for the first). The rings of an SM's CTAs keep 96 KB on
// the way: more makes the memory slower, not faster (96 and 160 KB: 16,383 rows of 2,048 in fp32 42.6 and 47.8 us forward,
// 71.5 and 74.5 backward, 16,384 of 2,048 in bf16 24.8 and 26.4, 44.5 and 46.1; 64 KB: 24.7 and 44.0, but 5,633 of 4,608
// backward 39.0 where this takes 35.7). A CTA alone on its SM has two slots at least (4,096 rows of 8,192 in fp32, backward:
// 78 us with one, 70 with two).
template <typename T, bool BWD>
static int plan(const NormArgs& a, int num_sms, Shape& s, Kernel& kern) {
  const int chunks = (a.width + 7) / 8;
  auto warps_of = [&](int nv) { return (chunks + 32 * nv - 1) / (32 * nv); };
  if (BWD) {
    s.nv = chunks <= 64 ? 1 : warps_of(2) > 6 && warps_of(3) <= 6 ? 3 : warps_of(2) <= 16 ? 2 : 4;
  } else {
    int best = INT32_MAX;
    for (int nv = warps_of(4) > 8 ? 4 : 1; nv <= 4; ++nv) {  // (four past 8,192 columns, where a CTA has 512 threads)
      const int cost = warps_of(nv) * (nv * 8 * 8 + 75);
      if (warps_of(nv) <= 8 + 8 * (nv == 4) && cost < best) best = cost, s.nv = nv;
    }
  }
  s.wpr = warps_of(s.nv);
  s.groups = std::max(1, 4 / s.wpr);
  const int warps = s.groups * s.wpr;
  const int v = access_of(a);
  kern = kernel_of<T, BWD>(s.nv, v, s.wpr);
  // resident CTAs by registers, asked for once a kernel and CTA size
  static std::atomic<int> resident[4][9][17];
  std::atomic<int>& r = resident[s.nv - 1][v][warps];
  int per_sm = r.load(std::memory_order_relaxed);
  if (!per_sm) {
    cudaError_t e = cudaFuncSetAttribute((const void*)kern, cudaFuncAttributeMaxDynamicSharedMemorySize, RING_SMEM);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, warps * 32, 0);
    if (e != cudaSuccess) return (int)e;
    per_sm = std::max(1, std::min(per_sm, BWD ? 4 : 8));
    r.store(per_sm, std::memory_order_relaxed);
  }
  const int64_t blocks = (a.rows + s.groups - 1) / s.groups;
  s.ring.part = (a.width * (int)sizeof(T) + 15) / 16 * 16 + 16;
  const int slot = s.ring.part * (BWD ? 2 : 1) * s.groups;
  per_sm = std::max(1, std::min(per_sm, RING_SMEM / slot));
  s.grid = (int)std::max<int64_t>(1, std::min(blocks, (int64_t)num_sms * per_sm));
  const int least = per_sm == 1 ? std::min(2, RING_SMEM / slot) : 1;
  s.ring.depth = std::max(least, std::min(MAX_DEPTH, RING_AHEAD / per_sm / slot));
  // all of a CTA's share is asked for: CTAs that start while the kernel before still holds SMs spread evenly only if an SM
  // cannot take more of them than planned (16,383 rows of 2,048 in fp32, both ways in a stream: 159 us without this, 120
  // with it)
  s.smem = std::max(s.ring.depth * slot, RING_SMEM / per_sm / 128 * 128);
  return 0;
}

template <typename T, bool BWD>
static int dispatch(const NormArgs& a, int num_sms, cudaStream_t st) {
  Shape s;
  Kernel kern;
  if (const int e = plan<T, BWD>(a, num_sms, s, kern)) return e;
  static std::atomic<uint64_t> devs[4][9][17];
  if (const int e = smem_attr_once(devs[s.nv - 1][access_of(a)][s.groups * s.wpr], (const void*)kern, RING_SMEM)) return e;
  return launch_pdl(kern, dim3(s.grid), dim3(s.groups * s.wpr * 32), s.smem, st, a, s.wpr, s.groups, s.ring);
}
template <typename T>
static int partials(const NormArgs& a, int num_sms) {
  Shape s;
  Kernel kern;
  return plan<T, true>(a, num_sms, s, kern) ? 0 : s.grid;
}

static bool valid(const NormArgs& a) {
  return a.width >= 1 && a.width <= NORM_MAX_WIDTH && a.rows >= 0 && a.dtype >= 0 && a.dtype <= 2 &&
         (a.wtype == ELEM_FP32 || a.wtype == a.dtype);
}

}  // namespace norm

int norm_bwd_partials(const NormArgs& a, int num_sms) {
  if (a.dtype == ELEM_BF16) return norm::partials<__nv_bfloat16>(a, num_sms);
  return a.dtype == ELEM_FP16 ? norm::partials<__half>(a, num_sms) : norm::partials<float>(a, num_sms);
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
  if ((a.dw || a.db) && a.partials != norm_bwd_partials(a, num_sms)) return 4;
  int rc;
  if (a.dtype == ELEM_BF16) rc = norm::dispatch<__nv_bfloat16, true>(a, num_sms, st);
  else if (a.dtype == ELEM_FP16) rc = norm::dispatch<__half, true>(a, num_sms, st);
  else rc = norm::dispatch<float, true>(a, num_sms, st);
  if (rc || (!a.dw && !a.db)) return rc;
  const dim3 grid((2 * a.width + 31) / 32);
  const int n = a.partials, w32 = a.wtype == ELEM_FP32;
  if (a.dtype == ELEM_BF16)
    return launch_pdl(norm::norm_reduce_kernel<__nv_bfloat16>, grid, dim3(1024), 0, st, (const float*)a.partial, n,
                      a.width, a.dw, a.db, w32);
  if (a.dtype == ELEM_FP16)
    return launch_pdl(norm::norm_reduce_kernel<__half>, grid, dim3(1024), 0, st, (const float*)a.partial, n, a.width,
                      a.dw, a.db, w32);
  return launch_pdl(norm::norm_reduce_kernel<float>, grid, dim3(1024), 0, st, (const float*)a.partial, n, a.width,
                    a.dw, a.db, w32);
}

}  // namespace afb
