// Gated feed-forward block of the trainers, forward and backward, on tcgen05:
//
//   g = x Wg^T, u = x Wu^T, h = act(g) u      one kernel: a 128 x 256 accumulator tile is 128 gate columns beside the
//                                             same 128 up columns, so a thread of the epilogue holds both of a pair
//   y = h W2^T (+ residual)
//   dh = dy W2, dg = dh u act'(g), du = dh act(g)   one kernel, the activation's gradient in the epilogue
//   dx = [dg | du] [Wg; Wu]
//   dW13 = [dg | du]^T x, dW2 = dy^T h        both operands of these have the reduced index (the rows) outermost
//
// The five products share one kernel, templated on which operand has K contiguous (K-major) and which has M or N
// contiguous (MN-major; read in place through the MN-major form of the shared-memory descriptor, so nothing is ever
// transposed in memory), and on the epilogue. Sums are fp32 in TMEM. h and [dg | du] are rounded once to the element
// type because the tensor cores take them as operands; g and u are kept in fp32 for the backward pass, since a
// second rounding there would show in dx and dW13. Split-K partial sums are fp32 and added in a fixed order: every
// result is bitwise reproducible.
#include <algorithm>

#include "common.cuh"
#include "ffn.h"
#include "gemm.h"

namespace afb {
namespace ffn {

constexpr int BM = 128, BN = 256, BK = 64, STAGES = 4;
constexpr uint32_t A_BYTES = BM * BK * 2, B_BYTES = BN * BK * 2;
constexpr uint32_t BAR_OFF = STAGES * (A_BYTES + B_BYTES);
constexpr uint32_t SMEM = BAR_OFF + (2 * STAGES + 1) * 8 + 16 + 1024;

enum Epi { STORE = 0, PARTIAL = 1, DUAL = 2, DACT = 3 };
enum Layout { NT = 0, NN = 1, TN = 2 };  // A K-major B K-major | A K-major B MN-major | both MN-major

struct Args {
  int64_t M = 0;  // rows of the result
  int N = 0;      // columns of the result (DUAL: F)
  int64_t K = 0;
  int F = 0;      // DUAL / DACT: columns of one half of w13
  int act = 0;
  void* out = nullptr;  // STORE: result; DUAL: h; DACT: dgu
  int64_t ldo = 0;
  const void* residual = nullptr;  // STORE
  int64_t ldr = 0;
  float* f32 = nullptr;  // PARTIAL: [splits, M, N]; DUAL: gu or null; DACT: gu
};

template <bool F16>
AFB_DEV uint32_t pack2(float a, float b) {
  return F16 ? pack_f16x2(a, b) : pack_bf16x2(a, b);
}
template <bool F16>
AFB_DEV float2 unpack2(uint32_t v) {
  if (F16) return __half22float2(*reinterpret_cast<__half2*>(&v));
  return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v));
}

// act(x) and its derivative
AFB_DEV void act_grad(float x, int act, float& a, float& d) {
  if (act == 0) {
    const float s = 1.f / (1.f + __expf(-x));
    a = x * s;
    d = s * (1.f + x * (1.f - s));
  } else if (act == 1) {
    const float c = 0.7978845608028654f, x2 = x * x;
    const float t = tanhf(c * x * (1.f + 0.044715f * x2));
    a = 0.5f * x * (1.f + t);
    d = 0.5f * (1.f + t) + 0.5f * x * (1.f - t * t) * c * (1.f + 0.134145f * x2);
  } else {
    const float p = 0.5f * (1.f + erff(x * 0.7071067811865476f));
    a = x * p;
    d = p + x * 0.3989422804014327f * __expf(-0.5f * x * x);
  }
}
AFB_DEV float act_only(float x, int act) {
  float a, d;
  act_grad(x, act, a, d);
  return a;
}

template <int LAYOUT, int EPI, bool F16>
__global__ void __launch_bounds__(192, 1)
    ffn_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, Args g,
                    uint32_t* status) {
  constexpr bool A_MN = LAYOUT == TN, B_MN = LAYOUT != NT;
  constexpr int TN_COLS = EPI == DUAL ? BN / 2 : BN;  // result columns per tile
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * A_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + BAR_OFF);
  uint64_t* empty = full + STAGES;
  uint64_t* done = empty + STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t m0 = (int64_t)blockIdx.x * BM;
  const int n0 = blockIdx.y * TN_COLS;
  const int kb_total = (int)((g.K + BK - 1) / BK);
  const int kb_per = (kb_total + gridDim.z - 1) / gridDim.z;
  const int kb0 = blockIdx.z * kb_per;
  const int num_kb = max(0, min(kb_total, kb0 + kb_per) - kb0);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc(tmem_slot, BN);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_dep_wait();
  if (threadIdx.x == 0) grid_dep_trigger();

  if (warp == 0) {
    if (lane == 0) {
      prefetch_tmap(&tmA);
      prefetch_tmap(&tmB);
      int issued = 0;
      for (int i = 0; i < num_kb; ++i) {
        const int s = i % STAGES;
        if (i >= STAGES && !mbar_wait(&empty[s], ((i / STAGES) & 1) ^ 1, status)) break;
        mbar_arrive_expect_tx(&full[s], A_BYTES + B_BYTES);
        uint8_t* a = sA + s * A_BYTES;
        uint8_t* b = sB + s * B_BYTES;
        const int k = (kb0 + i) * BK;
        if constexpr (A_MN) {
#pragma unroll
          for (int j = 0; j < BM / 64; ++j) tma_load_2d(a + j * 8192, &tmA, &full[s], (int)m0 + j * 64, k);
        } else {
          tma_load_2d(a, &tmA, &full[s], k, (int)m0);
        }
        if constexpr (B_MN) {
#pragma unroll
          for (int j = 0; j < BN / 64; ++j) tma_load_2d(b + j * 8192, &tmB, &full[s], n0 + j * 64, k);
        } else {  // two boxes of 128 rows: gate and up rows of w13 (DUAL), or consecutive rows
          tma_load_2d(b, &tmB, &full[s], k, n0);
          tma_load_2d(b + B_BYTES / 2, &tmB, &full[s], k, EPI == DUAL ? g.F + n0 : n0 + 128);
        }
        ++issued;
      }
      for (int i = max(0, issued - STAGES); i < issued; ++i) mbar_wait(&full[i % STAGES], (i / STAGES) & 1, status);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc =
          idesc_f16(128, BN, F16 ? 0 : 1) | ((uint32_t)A_MN << 15) | ((uint32_t)B_MN << 16);
      for (int i = 0; i < num_kb; ++i) {
        const int s = i % STAGES;
        if (!mbar_wait(&full[s], (i / STAGES) & 1, status)) break;
        tc_fence_after();
        const uint32_t a = smem_u32(sA + s * A_BYTES), b = smem_u32(sB + s * B_BYTES);
#pragma unroll
        for (int kk = 0; kk < BK / 16; ++kk) {
          const uint64_t da = A_MN ? sw128_desc_mn(a + kk * 2048, 8192, 1024) : sw128_desc(a) + 2 * kk;
          const uint64_t db = B_MN ? sw128_desc_mn(b + kk * 2048, 8192, 1024) : sw128_desc(b) + 2 * kk;
          umma_f16(tmem, da, db, idesc, (i | kk) != 0);
        }
        umma_commit(&empty[s]);
      }
      umma_commit(done);
    }
  } else {
    const int quad = warp & 3;
    const bool ok = mbar_wait(done, 0, status);
    tc_fence_after();
    const int64_t row = m0 + quad * 32 + lane;
    const uint32_t taddr = tmem + ((uint32_t)(quad * 32) << 16);
#pragma unroll 1
    for (int c = 0; c < TN_COLS; c += 32) {
      float v[32];
      tmem_ld32(taddr + c, v);
      float w[EPI == DUAL ? 32 : 1];
      if constexpr (EPI == DUAL) tmem_ld32(taddr + 128 + c, w);
      tmem_ld_wait();
      const int col0 = n0 + c;
      if (!ok || row >= g.M || col0 >= g.N) continue;
      if (num_kb == 0) {  // an empty split-K slice contributes zeros
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = 0.f;
      }
      if constexpr (EPI == PARTIAL) {
        float* o = g.f32 + ((int64_t)blockIdx.z * g.M + row) * g.N + col0;
#pragma unroll
        for (int j = 0; j < 32; j += 4)
          if (col0 + j < g.N) *reinterpret_cast<float4*>(o + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
      } else if constexpr (EPI == DUAL) {
        if (g.f32) {
          float* o = g.f32 + row * 2 * g.F + col0;
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            if (col0 + j < g.N) {
              *reinterpret_cast<float4*>(o + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
              *reinterpret_cast<float4*>(o + g.F + j) = make_float4(w[j], w[j + 1], w[j + 2], w[j + 3]);
            }
        }
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = act_only(v[j], g.act) * w[j];
      } else if constexpr (EPI == DACT) {
        const float* gp = g.f32 + row * 2 * g.F + col0;
        uint16_t* o = reinterpret_cast<uint16_t*>(g.out) + row * 2 * g.F + col0;
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
          if (col0 + j >= g.N) break;
          uint32_t dg[4], du[4];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const float2 gv = *reinterpret_cast<const float2*>(gp + j + 2 * t);
            const float2 uv = *reinterpret_cast<const float2*>(gp + g.F + j + 2 * t);
            float a0, d0, a1, d1;
            act_grad(gv.x, g.act, a0, d0);
            act_grad(gv.y, g.act, a1, d1);
            dg[t] = pack2<F16>(v[j + 2 * t] * uv.x * d0, v[j + 2 * t + 1] * uv.y * d1);
            du[t] = pack2<F16>(v[j + 2 * t] * a0, v[j + 2 * t + 1] * a1);
          }
          *reinterpret_cast<uint4*>(o + j) = make_uint4(dg[0], dg[1], dg[2], dg[3]);
          *reinterpret_cast<uint4*>(o + g.F + j) = make_uint4(du[0], du[1], du[2], du[3]);
        }
      }
      if constexpr (EPI == STORE || EPI == DUAL) {
        if (EPI == STORE && g.residual) {
          const uint16_t* r = reinterpret_cast<const uint16_t*>(g.residual) + row * g.ldr + col0;
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            if (col0 + j >= g.N) break;
            const uint4 q = *reinterpret_cast<const uint4*>(r + j);
            const uint32_t qq[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              const float2 f = unpack2<F16>(qq[t]);
              v[j + 2 * t] += f.x;
              v[j + 2 * t + 1] += f.y;
            }
          }
        }
        uint16_t* o = reinterpret_cast<uint16_t*>(g.out) + row * g.ldo + col0;
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
          if (col0 + j >= g.N) break;
          *reinterpret_cast<uint4*>(o + j) =
              make_uint4(pack2<F16>(v[j], v[j + 1]), pack2<F16>(v[j + 2], v[j + 3]), pack2<F16>(v[j + 4], v[j + 5]),
                         pack2<F16>(v[j + 6], v[j + 7]));
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, BN);
  }
}

// Fixed-order sum of the split-K partials [splits, M, N] -> out
template <bool F16>
__global__ void __launch_bounds__(256) ffn_reduce_kernel(const float* __restrict__ part, int splits, int64_t M, int N,
                                                         void* __restrict__ out, int64_t ldo) {
  grid_dep_wait();
  const int64_t total = M * N, idx = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * 8;
  if (idx >= total) return;
  float v[8] = {};
  for (int s = 0; s < splits; ++s) {
    const float4 a = *reinterpret_cast<const float4*>(part + s * total + idx);
    const float4 b = *reinterpret_cast<const float4*>(part + s * total + idx + 4);
    v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
    v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
  }
  const int64_t row = idx / N;
  *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(out) + row * ldo + idx % N) =
      make_uint4(pack2<F16>(v[0], v[1]), pack2<F16>(v[2], v[3]), pack2<F16>(v[4], v[5]), pack2<F16>(v[6], v[7]));
}

// splits of a result with few tiles (the weight gradients: K is the row count): as many as fill the SMs once, each
// of at least 16 K blocks
static int plan_splits(int64_t M, int N, int64_t K, int num_sms) {
  const int64_t tiles = ((M + BM - 1) / BM) * ((N + BN - 1) / BN), kb = (K + BK - 1) / BK;
  if (tiles < 1 || tiles * 2 > num_sms) return 1;
  return (int)max((int64_t)1, min((int64_t)(num_sms / tiles), kb / 16));
}

template <int LAYOUT, int EPI, bool F16>
static int launch(const void* A, int64_t lda, const void* B, int64_t ldb, int64_t b_rows, int splits, const Args& g,
                  uint32_t* status, cudaStream_t st) {
  constexpr bool A_MN = LAYOUT == TN, B_MN = LAYOUT != NT;
  CUtensorMap ta, tb;
  int rc = A_MN ? make_tmap_2d(&ta, A, 2, g.M, g.K, lda * 2, 64, BK, 1)
                : make_tmap_2d(&ta, A, 2, g.K, g.M, lda * 2, BK, BM, 1);
  if (rc) return 1000 + rc;
  rc = B_MN ? make_tmap_2d(&tb, B, 2, b_rows, g.K, ldb * 2, 64, BK, 1)
            : make_tmap_2d(&tb, B, 2, g.K, b_rows, ldb * 2, BK, 128, 1);
  if (rc) return 2000 + rc;
  auto kern = ffn_gemm_kernel<LAYOUT, EPI, F16>;
  static std::atomic<uint64_t> devs{0};
  if (const int e = smem_attr_once(devs, (const void*)kern, SMEM)) return e;
  constexpr int cols = EPI == DUAL ? BN / 2 : BN;
  const dim3 grid((unsigned)((g.M + BM - 1) / BM), (g.N + cols - 1) / cols, splits);
  return launch_pdl(kern, grid, dim3(192), SMEM, st, ta, tb, g, status);
}

// C [M, N] = A B in LAYOUT, rounded to the element type, split over K where that pays
template <int LAYOUT, bool F16>
static int product(const void* A, int64_t lda, const void* B, int64_t ldb, Args g, float* scratch, int num_sms,
                   uint32_t* status, cudaStream_t st) {
  const int splits = g.residual ? 1 : plan_splits(g.M, g.N, g.K, num_sms);
  if (splits == 1) return launch<LAYOUT, STORE, F16>(A, lda, B, ldb, g.N, 1, g, status, st);
  g.f32 = scratch;
  int rc = launch<LAYOUT, PARTIAL, F16>(A, lda, B, ldb, g.N, splits, g, status, st);
  if (rc) return rc;
  const int64_t n8 = g.M * g.N / 8;
  return launch_pdl(ffn_reduce_kernel<F16>, dim3((unsigned)((n8 + 255) / 256)), dim3(256), 0, st,
                    (const float*)scratch, splits, g.M, g.N, g.out, g.ldo);
}

static size_t product_scratch(int64_t M, int N, int64_t K, int num_sms) {
  const int s = plan_splits(M, N, K, num_sms);
  return s > 1 ? (size_t)s * M * N : 0;
}

template <bool F16>
static int fwd(const FfnShape& s, const void* x, int64_t ldx, const void* w13, const void* w2, const void* residual,
               int64_t ldr, void* h, float* gu, void* y, float* scratch, int num_sms, uint32_t* status,
               cudaStream_t st) {
  Args g;
  g.M = s.T, g.N = s.F, g.K = s.H, g.F = s.F, g.act = s.act, g.out = h, g.ldo = s.F, g.f32 = gu;
  int rc = launch<NT, DUAL, F16>(x, ldx, w13, s.H, 2 * s.F, 1, g, status, st);
  if (rc) return rc;
  g = Args();
  g.M = s.T, g.N = s.N, g.K = s.F, g.out = y, g.ldo = s.N, g.residual = residual, g.ldr = ldr;
  return product<NT, F16>(h, s.F, w2, s.F, g, scratch, num_sms, status, st);
}

template <bool F16>
static int bwd(const FfnShape& s, const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w13,
               const void* w2, const void* h, const float* gu, void* dgu, void* dx, void* dw13, void* dw2,
               float* scratch, int num_sms, uint32_t* status, cudaStream_t st) {
  int rc = 0;
  Args g;
  if (dw2) {
    g.M = s.N, g.N = s.F, g.K = s.T, g.out = dw2, g.ldo = s.F;
    if ((rc = product<TN, F16>(dy, lddy, h, s.F, g, scratch, num_sms, status, st))) return rc;
  }
  if (!dx && !dw13) return 0;
  g = Args();
  g.M = s.T, g.N = s.F, g.K = s.N, g.F = s.F, g.act = s.act, g.out = dgu, g.f32 = const_cast<float*>(gu);
  if ((rc = launch<NN, DACT, F16>(dy, lddy, w2, s.F, s.F, 1, g, status, st))) return rc;
  if (dx) {
    g = Args();
    g.M = s.T, g.N = s.H, g.K = 2 * s.F, g.out = dx, g.ldo = s.H;
    if ((rc = product<NN, F16>(dgu, 2 * s.F, w13, s.H, g, scratch, num_sms, status, st))) return rc;
  }
  if (dw13) {
    g = Args();
    g.M = 2 * s.F, g.N = s.H, g.K = s.T, g.out = dw13, g.ldo = s.H;
    if ((rc = product<TN, F16>(dgu, 2 * s.F, x, ldx, g, scratch, num_sms, status, st))) return rc;
  }
  return 0;
}

static bool valid(const FfnShape& s) {
  return s.T >= 0 && s.H > 0 && s.F > 0 && s.N > 0 && !(s.H % 8) && !(s.F % 8) && !(s.N % 8) && s.act >= 0 &&
         s.act <= 2;
}

}  // namespace ffn

size_t ffn_fwd_scratch(const FfnShape& s, int num_sms) {
  return ffn::product_scratch(s.T, s.N, s.F, num_sms);
}
size_t ffn_bwd_scratch(const FfnShape& s, int num_sms) {
  return std::max({ffn::product_scratch(s.N, s.F, s.T, num_sms), ffn::product_scratch(s.T, s.H, 2 * s.F, num_sms),
                   ffn::product_scratch(2 * s.F, s.H, s.T, num_sms)});
}

int ffn_fwd(const FfnShape& s, const void* x, int64_t ldx, const void* w13, const void* w2, const void* residual,
            int64_t ldr, void* h, float* gu, void* y, float* scratch, int num_sms, uint32_t* status, cudaStream_t st) {
  if (!ffn::valid(s)) return 3;
  if (s.T == 0) return 0;
  return (s.fp16 ? ffn::fwd<true> : ffn::fwd<false>)(s, x, ldx, w13, w2, residual, ldr, h, gu, y, scratch, num_sms,
                                                     status, st);
}

int ffn_bwd(const FfnShape& s, const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w13,
            const void* w2, const void* h, const float* gu, void* dgu, void* dx, void* dw13, void* dw2, float* scratch,
            int num_sms, uint32_t* status, cudaStream_t st) {
  if (!ffn::valid(s)) return 3;
  if (s.T == 0) return 0;  // the caller zeroes the weight gradients
  return (s.fp16 ? ffn::bwd<true> : ffn::bwd<false>)(s, dy, lddy, x, ldx, w13, w2, h, gu, dgu, dx, dw13, dw2, scratch,
                                                     num_sms, status, st);
}

}  // namespace afb
