// Gated feed-forward block of the trainers, forward and backward, on tcgen05:
//
//   g = x Wg^T, u = x Wu^T, h = act(g) u      one kernel: a 256-column accumulator tile is 128 gate columns beside
//                                             the same 128 up columns, so an epilogue thread holds both of a pair
//   y = h W2^T (+ residual)
//   dh = dy W2, dg = dh p, du = dh q          one kernel; p = u act'(g) and q = act(g) come from the forward epilogue
//   dx = [dg | du] [Wg; Wu]
//   dW13 = [dg | du]^T x, dW2 = dy^T h        both operands of these have the reduced index (the rows) outermost
//
// The five products share one kernel, templated on which operand has K contiguous (K-major) and which has M or N
// contiguous (MN-major; read in place through the MN-major form of the shared-memory descriptor, so nothing is ever
// transposed in memory), and on the epilogue. Sums are fp32 in TMEM. h and [dg | du] are rounded once to the element
// type because the tensor cores take them as operands; p and q are kept in fp32 for the backward pass, since a second
// rounding there would show in dx and dW13. Split-K partial sums are fp32 and added in a fixed order: every result is
// bitwise reproducible. Few rows have forward kernels of their own (below).
//
// Measured (one B200, kernels alone, TFLOP/s of 1,646 measured for a library GEMM): 4,100 x 2,048 x 6,144 forward DUAL
// 155 us (1,330) and y 77 (1,340), backward DACT 93 (1,110), dx 145 (1,420), the weight gradients 230 (1,350); a product
// of 8,192^3 735 (1,496). What is lost: the last wave of tiles (8 % on average there) and some 5 us a launch.
#include <algorithm>
#include <type_traits>

#include "ffn.h"
#include "gemm.h"
#include "tc_pair.cuh"

namespace afb {
namespace ffn {

// A pair of CTAs computes a 256 x 256 accumulator tile: each holds 128 rows of A and 128 of the 256 rows of B
constexpr int BM = 256, BN = 256, BK = 64;
constexpr uint32_t OP_BYTES = 128 * BK * 2;  // one operand of one CTA and stage
constexpr int EPI_WARPS = 8, THREADS = 64 + 32 * EPI_WARPS;

enum Epi { STORE = 0, PARTIAL = 1, DUAL = 2, DACT = 3 };
// A K-major B K-major | A K-major B MN-major | both MN-major | dx (NN) and the weight gradients (TN) in one launch
enum Layout { NT = 0, NN = 1, TN = 2, GRADS = 3 };

constexpr int STAGES = 6;
constexpr uint32_t EPI_OFF = STAGES * 2 * OP_BYTES;
constexpr uint32_t EPI_BYTES = 4096;  // staging of an epilogue warp: 32 rows of 128 bytes
constexpr uint32_t BAR_OFF = EPI_OFF + EPI_WARPS * EPI_BYTES;
constexpr uint32_t SMEM = BAR_OFF + (2 * STAGES + 4) * 8 + 16 + 1024;

// The backward products after DACT in one launch: dx [T, H] (2F / 64 K blocks a tile), dW13 [2F, H] and dW2 [N, F] (T / 64
// K blocks a tile). Alone each of them ends in a wave that leaves pairs idle; together the tiles with fewer K blocks
// fill in behind those with more: pair p of P takes long tiles p, p + P, ..., then x short ones where it had one long
// tile more than the others, y otherwise (x <= y).
struct Grads {
  uint32_t tiles[3] = {}, mt[3] = {}, nt[3] = {}, kb[3] = {};  // dx, dW13, dW2
  int M[3] = {}, N[3] = {};
  uint32_t dx_long = 0;            // the long tiles are dx's (else the weight gradients')
  uint32_t longs = 0, shorts = 0;  // tiles of the two kinds
  uint32_t x = 0, y = 0;
};
struct Args {
  int64_t M = 0;  // rows of the result
  int N = 0;      // columns of the result (DUAL: F)
  int64_t K = 0;
  int F = 0;      // DUAL, DACT: columns of one half of w13
  int act = 0;
  int splits = 1;                  // PARTIAL
  const void* residual = nullptr;  // STORE, optional
  int64_t ldr = 0;
  Grads grads;           // GRADS
  float* f32 = nullptr;  // PARTIAL: sums [splits, M in whole tiles, N]; DUAL: p and q (at_gu) or null; DACT: p and q
};
// tensor maps: operands; the 16-bit result (STORE, DUAL h, DACT dg), and DACT's du; GRADS: of each product
template <int LAYOUT>
struct Maps {
  CUtensorMap a[LAYOUT == GRADS ? 3 : 1], b[LAYOUT == GRADS ? 3 : 1], out[LAYOUT == GRADS ? 3 : 2];
};

// p and q are kept as the epilogue's threads hold them, 32 rows x 8 columns (32 bytes a row) at a time: a warp's access
// is 1 KB in one piece. (Row-major, a warp's 32-byte pieces of 32 rows cost four times the L1 cycles, which the MMAs'
// operands need too: 187 against 152 us for the forward product at 4,100 x 2,048 x 6,144.)
AFB_DEV int64_t at_gu(int64_t row, int col, int F, int half) {
  return ((row >> 5) * 2 + half) * F * 32 + (int64_t)(col >> 3) * 256 + (row & 31) * 8 + (col & 7);
}

template <bool F16>
AFB_DEV uint32_t pack2(float a, float b) {
  return F16 ? pack_f16x2(a, b) : pack_bf16x2(a, b);
}
template <bool F16>
AFB_DEV float2 unpack2(uint32_t v) {
  if (F16) return __half22float2(*reinterpret_cast<__half2*>(&v));
  return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v));
}

// act(x) and its derivative. The quotients are __fdividef (2 units in the last place; 0 for a divisor past 2^126, where
// the quotient is below the smallest normal number); tanh(z) = 1 - 2 / (exp(2 z) + 1) is used as 1 + t and 1 - t^2,
// where its absolute error of some 1e-7 is what counts.
// The choice is a template parameter of the loops over a thread's values: a branch a value would leave their quotients'
// latencies one after the other (DACT at 4,100 x 6,144: 135 us with it).
template <int ACT>
AFB_DEV void act_grad(float x, float& a, float& d) {
  if constexpr (ACT == 0) {
    const float s = __fdividef(1.f, 1.f + __expf(-x));
    a = x * s;
    d = s * (1.f + x * (1.f - s));
  } else if constexpr (ACT == 1) {
    const float c = 0.7978845608028654f, x2 = x * x;
    const float t = 1.f - __fdividef(2.f, 1.f + __expf(2.f * c * x * (1.f + 0.044715f * x2)));
    a = 0.5f * x * (1.f + t);
    d = 0.5f * (1.f + t) + 0.5f * x * (1.f - t * t) * c * (1.f + 0.134145f * x2);
  } else {
    const float p = 0.5f * (1.f + erff(x * 0.7071067811865476f));
    a = x * p;
    d = p + x * 0.3989422804014327f * __expf(-0.5f * x * x);
  }
}
template <int ACT>
AFB_DEV float act_only(float x) {
  float a, d;
  act_grad<ACT>(x, a, d);
  return a;
}
template <typename F>
AFB_DEV void with_act(int act, F&& f) {
  if (act == 0) f(std::integral_constant<int, 0>());
  else if (act == 1) f(std::integral_constant<int, 1>());
  else f(std::integral_constant<int, 2>());
}

struct Tile {
  int m, n, split;  // row tile, column tile, K split (GRADS: product)
  uint32_t kb0, kb1;
};
// tile order: bands of 8 row tiles, down the band first, so that the tiles in flight share both operands in L2.
// 32-bit: the tile count is checked on the host, and a 64-bit division costs the producer some 200 cycles.
AFB_DEV Tile tile_at(uint32_t t, uint32_t mt, uint32_t nt) {
  Tile r;
  const uint32_t per = mt * nt;
  r.split = t / per;
  t -= r.split * per;
  const uint32_t band = t / (8u * nt), in = t - band * 8u * nt, rows = min(8u, mt - band * 8u), n = in / rows;
  r.m = band * 8u + in - n * rows;
  r.n = n;
  return r;
}
// the k-th tile of pair p of P; false behind its last one
AFB_DEV bool grads_tile(const Grads& g, uint32_t k, uint32_t p, uint32_t P, Tile& r) {
  const uint32_t more = g.longs % P, nl = g.longs / P + (p < more);
  uint32_t i;
  bool dx;
  if (k < nl) {
    i = k * P + p;
    dx = g.dx_long;
  } else {
    const uint32_t j = k - nl;
    if (j >= (p < more ? g.x : g.y)) return false;
    i = j < g.x ? j * P + p : g.x * P + (j - g.x) * (P - more) + (p - more);
    if (i >= g.shorts) return false;
    dx = !g.dx_long;
  }
  const uint32_t q = dx ? 0 : i < g.tiles[1] ? 1 : 2;
  if (q == 2) i -= g.tiles[1];
  r = tile_at(i, g.mt[q], g.nt[q]);
  r.split = q;
  r.kb0 = 0;
  r.kb1 = g.kb[q];
  return true;
}

AFB_DEV void st32(void* p, const uint32_t* r) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
AFB_DEV void ld32(const void* p, uint32_t* r) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "l"(p)
               : "memory");
}
AFB_DEV void st_gu(float* p, const float* v) { st32(p, reinterpret_cast<const uint32_t*>(v)); }
AFB_DEV void ld_gu(const float* p, float* v) { ld32(p, reinterpret_cast<uint32_t*>(v)); }

// a 16-bit row of 64 columns (or fp32 of 32) -> a 128-byte swizzled staging row; of 32 columns -> a 64-byte one
AFB_DEV void put_row(uint8_t* buf, int row, const uint32_t* w) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    *reinterpret_cast<uint4*>(buf + sw128_offset(row, j)) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
}
AFB_DEV void put_half_row(uint8_t* buf, int row, const uint32_t* w) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    *reinterpret_cast<uint4*>(buf + row * 64 + ((j ^ ((row >> 1) & 3)) << 4)) =
        make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
}

// Persistent: pair p of the grid takes tiles p, p + pairs, ... Each CTA: warp 0 loads its halves of the operands by
// TMA into a STAGES-deep ring, one thread of the leader's warp 1 issues the MMAs of both CTAs into one of two TMEM
// accumulators, and 8 epilogue warps drain the other one (two warps a lane quadrant, half of the columns each) through
// swizzled staging rows and TMA stores, so the tensor cores work through the next tile meanwhile. A K block takes 600
// cycles where its MMAs take 512, more ring stages do not change that (5 and 6 are equal), and every line an epilogue
// moves through L1 or shared memory adds to it: by all signs shared memory's bandwidth bounds the tiles (a K block moves
// 80 KB of it a CTA). So the epilogue is kept to whole 128-byte lines.
template <int LAYOUT, int EPI, bool F16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    ffn_gemm_kernel(const __grid_constant__ Maps<LAYOUT> maps, Args g, uint32_t* status) {
  constexpr bool B_MN = LAYOUT != NT;
  constexpr int TN_COLS = EPI == DUAL ? BN / 2 : BN;  // result columns per tile
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + BAR_OFF);  // leader's: both CTAs' operands have landed
  uint64_t* empty = full + STAGES;                               // the pair's MMAs of the stage are done
  uint64_t* acc_full = empty + STAGES;                           // [2] accumulator complete
  uint64_t* acc_empty = acc_full + 2;                            // [2] leader's: drained by both CTAs' epilogues
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_cta_rank();
  const uint32_t mt = (uint32_t)((g.M + BM - 1) / BM), nt = (g.N + TN_COLS - 1) / TN_COLS, tiles = mt * nt * g.splits;
  const uint32_t pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const uint32_t kb_total = (uint32_t)((g.K + BK - 1) / BK);
  // the k-th tile of this pair
  auto tile = [&](uint32_t k, Tile& r) {
    if constexpr (LAYOUT == GRADS) return grads_tile(g.grads, k, pair, pairs, r);
    const uint32_t t = pair + k * pairs;
    if (t >= tiles) return false;
    r = tile_at(t, mt, nt);
    r.kb0 = 0;
    r.kb1 = kb_total;
    if constexpr (EPI == PARTIAL) {  // at most 32 splits of 2^25 blocks
      r.kb0 = kb_total * r.split / (uint32_t)g.splits;
      r.kb1 = kb_total * (r.split + 1) / (uint32_t)g.splits;
    }
    return true;
  };
  auto a_mn = [](const Tile& r) { return LAYOUT == TN || (LAYOUT == GRADS && r.split > 0); };
  auto q_of = [](const Tile& r) { return LAYOUT == GRADS ? r.split : 0; };  // the product's maps

  if (threadIdx.x >= 32 && threadIdx.x < 32 + (LAYOUT == GRADS ? 3 : 1)) {
    prefetch_tmap(&maps.a[threadIdx.x - 32]);
    prefetch_tmap(&maps.b[threadIdx.x - 32]);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&acc_full[s], 1);
      mbar_init(&acc_empty[s], 2 * EPI_WARPS);
    }
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc_pair(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_dep_wait();
  if (threadIdx.x == 0) grid_dep_trigger();

  if (warp == 0) {
    if (lane == 0) {
      uint32_t i = 0, s = 0, ph = 1;  // stages issued, the ring's next stage and its empty barrier's parity
      bool ok = true;
      Tile tl;
      for (uint32_t n = 0; ok && tile(n, tl); ++n) {
        const CUtensorMap *tm_a = &maps.a[q_of(tl)], *tm_b = &maps.b[q_of(tl)];
        const int ma = tl.m * BM + (int)rank * 128;
        const int nb = EPI == DUAL ? (int)rank * g.F + tl.n * TN_COLS : tl.n * TN_COLS + (int)rank * 128;
        for (uint32_t kb = tl.kb0; kb < tl.kb1; ++kb, ++i) {
          if (!mbar_wait(&empty[s], ph, status)) {  // (passes at once in the ring's first round)
            ok = false;
            break;
          }
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 4 * OP_BYTES);
          const uint32_t bar = cluster_addr(&full[s], 0);
          uint8_t* a = smem + s * 2 * OP_BYTES;
          uint8_t* b = a + OP_BYTES;
          const int k = (int)kb * BK;
          if (a_mn(tl)) {
            tma_load_2d_pair(a, tm_a, bar, ma, k);
            tma_load_2d_pair(a + 8192, tm_a, bar, ma + 64, k);
          } else {
            tma_load_2d_pair(a, tm_a, bar, k, ma);
          }
          if constexpr (B_MN) {
            tma_load_2d_pair(b, tm_b, bar, nb, k);
            tma_load_2d_pair(b + 8192, tm_b, bar, nb + 64, k);
          } else {
            tma_load_2d_pair(b, tm_b, bar, k, nb);
          }
          if (++s == STAGES) s = 0, ph ^= 1;
        }
      }
      // every stage issued has been read (so its copies have landed) before the CTA may leave
      for (uint32_t j = i > STAGES ? i - STAGES : 0; j < i; ++j)
        mbar_wait(&empty[j % STAGES], (j / STAGES) & 1, status);
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      uint32_t n = 0, s = 0, ph = 0;  // tiles of this pair; ring stage and its full barrier's parity
      bool ok = true;
      Tile tl;
      for (; ok && tile(n, tl); ++n) {
        const bool am = a_mn(tl);
        const uint32_t idesc = idesc_f16(BM, BN, F16 ? 0 : 1) | ((uint32_t)am << 15) | ((uint32_t)B_MN << 16);
        const uint32_t kb0 = tl.kb0, kb1 = tl.kb1;
        const uint32_t acc = tmem + (n & 1) * BN;
        if (!mbar_wait(&acc_empty[n & 1], ((n >> 1) & 1) ^ 1, status)) break;
        tc_fence_after();
        for (uint32_t kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(&full[s], ph, status)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a = smem_u32(smem + s * 2 * OP_BYTES), b = a + OP_BYTES;
#pragma unroll
          for (int kk = 0; kk < BK / 16; ++kk) {
            const uint64_t da = am ? sw128_desc_mn(a + kk * 2048, 8192, 1024) : sw128_desc(a) + 2 * kk;
            const uint64_t db = B_MN ? sw128_desc_mn(b + kk * 2048, 8192, 1024) : sw128_desc(b) + 2 * kk;
            umma_f16_pair(acc, da, db, idesc, kb > kb0 || kk > 0);
          }
          umma_commit_pair(&empty[s]);
          if (++s == STAGES) s = 0, ph ^= 1;
        }
        umma_commit_pair(&acc_full[n & 1]);
      }
    }
  } else {
    const int quad = warp & 3, half = (warp - 2) >> 2;
    uint8_t* buf = smem + EPI_OFF + (warp - 2) * EPI_BYTES;
    const uint32_t drained[2] = {cluster_addr(&acc_empty[0], 0), cluster_addr(&acc_empty[1], 0)};
    constexpr int HALF = TN_COLS / 2;  // result columns of a warp
    const int warp_row = (int)rank * 128 + quad * 32, lane_col = half * HALF;
    // the staging rows are free once the last store has read them; written, they go to the async proxy
    auto begin_put = [&] {
      if (lane == 0) bulk_wait_read<0>();
      __syncwarp();
    };
    auto end_put = [&] {
      fence_proxy_async_smem();
      __syncwarp();
    };
    // DACT: p and q of 16 columns, two chunks ahead of their use
    float gq[2][EPI == DACT ? 16 : 1], uq[2][EPI == DACT ? 16 : 1];
    struct GuTile {
      const float *g, *u;  // this lane's first column of the tile, or null where its row is outside the result
      int col;
    };
    auto gu_tile = [&](uint32_t k) {
      GuTile r{nullptr, nullptr, 0};
      Tile tl;
      if (EPI != DACT || !tile(k, tl)) return r;
      const int64_t row = (int64_t)tl.m * BM + warp_row + lane;
      r.col = tl.n * TN_COLS + lane_col;
      if (row < g.M) r.g = g.f32 + at_gu(row, r.col, g.F, 0), r.u = g.f32 + at_gu(row, r.col, g.F, 1);
      return r;
    };
    auto load_gu = [&](const GuTile& p, int c, float* gp, float* up) {
      if (!p.g) return;
#pragma unroll
      for (int j = 0; j < 16; j += 8)
        if (p.col + c * 16 + j < g.N) {  // 8 columns further is 256 floats further
          ld_gu(p.g + (c * 16 + j) * 32, gp + j);
          ld_gu(p.u + (c * 16 + j) * 32, up + j);
        }
    };
    GuTile gu_now = gu_tile(0);
    if constexpr (EPI == DACT) {
      load_gu(gu_now, 0, gq[0], uq[0]);
      load_gu(gu_now, 1, gq[1], uq[1]);
    }
    uint32_t n = 0;  // tiles of this pair
    Tile tl;
    for (; tile(n, tl); ++n) {
      const int row0 = tl.m * BM + warp_row, col0 = tl.n * TN_COLS + lane_col;
      const int64_t row = (int64_t)row0 + lane, M = LAYOUT == GRADS ? g.grads.M[q_of(tl)] : g.M;
      const int N = LAYOUT == GRADS ? g.grads.N[q_of(tl)] : g.N;
      const bool live = row < M, any = row0 < M;  // this lane's row, one of the warp's
      // one answer for the warp
      if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[n & 1], (n >> 1) & 1, status))) break;
      tc_fence_after();
      const uint32_t acc = tmem + (n & 1) * BN + ((uint32_t)(quad * 32) << 16) + half * HALF;
      // the accumulator is free as soon as this warp's last column is in registers
      bool told = false;
      auto tell = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote_relaxed(drained[n & 1]);
        told = true;
      };
      if constexpr (EPI == STORE) {
#pragma unroll 1
        for (int c = 0; c < HALF && any; c += 64) {
          const int col = col0 + c;
          if (col >= N) break;
          float v[64];
          tmem_ld32(acc + c, v);
          tmem_ld32(acc + c + 32, v + 32);
          tmem_ld_wait();
          if (c + 64 >= HALF) tell();
          if (g.residual && live) {
            const uint16_t* rp = reinterpret_cast<const uint16_t*>(g.residual) + row * g.ldr + col;
#pragma unroll
            for (int j = 0; j < 64; j += 8)
              if (col + j < N) {
                const uint4 q = *reinterpret_cast<const uint4*>(rp + j);
                const uint32_t r[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float2 f = unpack2<F16>(r[i]);
                  v[j + 2 * i] += f.x;
                  v[j + 2 * i + 1] += f.y;
                }
              }
          }
          uint32_t w[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) w[j] = pack2<F16>(v[2 * j], v[2 * j + 1]);
          begin_put();
          put_row(buf, lane, w);
          end_put();
          if (lane == 0) {
            tma_store_2d(&maps.out[q_of(tl)], buf, col, row0);
            bulk_commit();
          }
        }
      } else if constexpr (EPI == PARTIAL) {
#pragma unroll 1
        for (int c = 0; c < HALF && any; c += 32) {
          const int col = col0 + c;
          if (col >= g.N) break;
          float v[32];
          tmem_ld32(acc + c, v);
          tmem_ld_wait();
          if (c + 32 >= HALF) tell();
          begin_put();
          put_row(buf, lane, reinterpret_cast<const uint32_t*>(v));
          end_put();
          if (lane == 0) {
            tma_store_2d(&maps.out[0], buf, col, tl.split * (int)mt * BM + row0);
            bulk_commit();
          }
        }
      } else if constexpr (EPI == DUAL) {
        if (any && col0 < g.N) {
          uint32_t h[32];
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            float v[32], w[32];
            tmem_ld32(acc + q * 32, v);
            tmem_ld32(acc + BN / 2 + q * 32, w);
            tmem_ld_wait();
            if (q == 1) tell();
            if (g.f32) {
              with_act(g.act, [&](auto A) {
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                  float a0, d0, a1, d1;
                  act_grad<A.value>(v[j], a0, d0);
                  act_grad<A.value>(v[j + 1], a1, d1);
                  h[q * 16 + j / 2] = pack2<F16>(a0 * w[j], a1 * w[j + 1]);
                  w[j] *= d0, w[j + 1] *= d1;
                  v[j] = a0, v[j + 1] = a1;
                }
              });
#pragma unroll
              for (int j = 0; j < 32; j += 8) {
                const int col = col0 + q * 32 + j;
                if (live && col < g.N) {
                  st_gu(g.f32 + at_gu(row, col, g.F, 0), w + j);
                  st_gu(g.f32 + at_gu(row, col, g.F, 1), v + j);
                }
              }
            } else {
              with_act(g.act, [&](auto A) {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                  h[q * 16 + j] = pack2<F16>(act_only<A.value>(v[2 * j]) * w[2 * j],
                                             act_only<A.value>(v[2 * j + 1]) * w[2 * j + 1]);
              });
            }
          }
          begin_put();
          put_row(buf, lane, h);
          end_put();
          if (lane == 0) {
            tma_store_2d(&maps.out[0], buf, col0, row0);
            bulk_commit();
          }
        }
      } else {  // DACT
        constexpr int CH = HALF / 16;
        const GuTile gu_next = gu_tile(n + 1);
        uint32_t dg[16], du[16];  // 32 columns
        auto chunk = [&](int c, float* gp, float* up, uint32_t* dgp, uint32_t* dup) {
          float v[16];
          tmem_ld16(acc + c * 16, v);
          tmem_ld_wait();
          if (c == CH - 1) tell();
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            dgp[j] = pack2<F16>(v[2 * j] * gp[2 * j], v[2 * j + 1] * gp[2 * j + 1]);
            dup[j] = pack2<F16>(v[2 * j] * up[2 * j], v[2 * j + 1] * up[2 * j + 1]);
          }
          load_gu(c + 2 < CH ? gu_now : gu_next, (c + 2) % CH, gp, up);
        };
#pragma unroll 1
        for (int c = 0; c < CH; c += 2) {
          chunk(c, gq[0], uq[0], dg, du);
          chunk(c + 1, gq[1], uq[1], dg + 8, du + 8);
          const int col = col0 + c * 16;
          if (!any || col >= g.N) continue;
          begin_put();
          put_half_row(buf, lane, dg);
          put_half_row(buf + 2048, lane, du);
          end_put();
          if (lane == 0) {
            tma_store_2d(&maps.out[0], buf, col, row0);
            tma_store_2d(&maps.out[1], buf + 2048, col, row0);
            bulk_commit();
          }
        }
        gu_now = gu_next;
      }
      if (!told) tell();
    }
    if (lane == 0) bulk_wait<0>();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// Fixed-order sum of the split-K partials [splits, rows, N] (+ residual, rows ldr apart) -> out [M, N]
template <bool F16>
__global__ void __launch_bounds__(256) ffn_reduce_kernel(const float* __restrict__ part, int splits, int64_t rows,
                                                         int64_t M, int N, void* __restrict__ out,
                                                         const uint16_t* __restrict__ residual, int64_t ldr) {
  grid_dep_wait();
  grid_dep_trigger();
  const int64_t idx = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * 8;
  if (idx >= M * N) return;
  float v[8] = {};
  for (int s = 0; s < splits; ++s) {
    const float4 a = *reinterpret_cast<const float4*>(part + s * rows * N + idx);
    const float4 b = *reinterpret_cast<const float4*>(part + s * rows * N + idx + 4);
    v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
    v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
  }
  if (residual) {  // (N is a multiple of 8: the eight elements are of one row)
    const uint4 q = *reinterpret_cast<const uint4*>(residual + idx / N * ldr + idx % N);
    const uint32_t r[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2<F16>(r[i]);
      v[2 * i] += f.x;
      v[2 * i + 1] += f.y;
    }
  }
  *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(out) + idx) =
      make_uint4(pack2<F16>(v[0], v[1]), pack2<F16>(v[2], v[3]), pack2<F16>(v[4], v[5]), pack2<F16>(v[6], v[7]));
}

// K splits of a product: those that minimise waves of tiles x K blocks of a tile (0.37 us each at the rate the products
// reach), plus the fp32 partials written and read again (about 4 TB/s through L2) and the second launch (3 us).
// `us`: the estimate.
constexpr double KB_US = 0.37;
static int plan_splits(int64_t M, int N, int64_t K, int num_sms, double* us = nullptr) {
  const int64_t tiles = ((M + BM - 1) / BM) * ((N + BN - 1) / BN), kb = (K + BK - 1) / BK, pairs = num_sms / 2;
  int best = 1;
  double cost = 1e300;
  for (int s = 1; s <= 32 && s * 4 <= std::max<int64_t>(kb, 4) && (s == 1 || tiles < pairs); ++s) {
    const double waves = (double)((tiles * s + pairs - 1) / pairs);
    const double c = waves * (double)((kb + s - 1) / s) * KB_US +
                     (s > 1 ? 3. + 8. * s * (double)M * N / 4e6 : 0.);
    if (c < cost * 0.98) best = s, cost = c;
  }
  if (us) *us = cost;
  return best;
}

struct Ptr {  // a row-major matrix
  const void* p;
  int64_t ld;
};

// maps of A [M, K] and B [n, K] (K-major: K innermost) or of their transposes as they lie (MN-major)
static int operand_maps(CUtensorMap* a, CUtensorMap* b, bool a_mn, bool b_mn, Ptr A, Ptr B, int64_t M, int64_t n,
                        int64_t K) {
  int rc = a_mn ? make_tmap_2d(a, A.p, 2, M, K, A.ld * 2, 64, BK, 1)
                : make_tmap_2d(a, A.p, 2, K, M, A.ld * 2, BK, 128, 1);
  if (rc) return 1000 + rc;
  rc = b_mn ? make_tmap_2d(b, B.p, 2, n, K, B.ld * 2, 64, BK, 1) : make_tmap_2d(b, B.p, 2, K, n, B.ld * 2, BK, 128, 1);
  return rc ? 2000 + rc : 0;
}

template <int LAYOUT, int EPI, bool F16>
static int launch(Ptr A, Ptr B, int64_t b_rows, Maps<LAYOUT>& maps, const Args& g, int num_sms, uint32_t* status,
                  cudaStream_t st) {
  const int rc = operand_maps(&maps.a[0], &maps.b[0], LAYOUT == TN, LAYOUT != NT, A, B, g.M, b_rows, g.K);
  if (rc) return rc;
  auto kern = ffn_gemm_kernel<LAYOUT, EPI, F16>;
  static std::atomic<uint64_t> devs{0};
  if (const int e = smem_attr_once(devs, (const void*)kern, SMEM)) return e;
  constexpr int cols = EPI == DUAL ? BN / 2 : BN;
  const int64_t tiles = ((g.M + BM - 1) / BM) * ((g.N + cols - 1) / cols) * g.splits;
  if (tiles >= (1 << 30)) return 5;
  const int pairs = (int)std::min<int64_t>(tiles, std::max(1, num_sms / 2));
  return launch_pdl(kern, dim3(2 * pairs), dim3(THREADS), SMEM, st, maps, g, status);
}

// map of a result: boxes of 32 rows x 128 (or 64) bytes
static int row_map(CUtensorMap* m, const void* p, int bytes, int64_t cols, int64_t rows, int64_t ld, int row_bytes) {
  const int rc = make_tmap_2d(m, p, bytes, cols, rows, ld * bytes, row_bytes / bytes, 32, row_bytes);
  return rc ? 3000 + rc : 0;
}

// out [M, N] = A B in LAYOUT (+ residual), rounded to the element type, split over K where that pays
template <int LAYOUT, bool F16>
static int product(Ptr A, Ptr B, int64_t M, int N, int64_t K, void* out, Ptr residual, float* scratch, int num_sms,
                   uint32_t* status, cudaStream_t st) {
  Maps<LAYOUT> maps;
  Args g;
  g.M = M, g.N = N, g.K = K, g.residual = residual.p, g.ldr = residual.ld;
  g.splits = plan_splits(M, N, K, num_sms);
  const int64_t rows = (M + BM - 1) / BM * BM;  // of a split's partial sums: whole tiles
  int rc = g.splits == 1 ? row_map(&maps.out[0], out, 2, N, M, N, 128)
                         : row_map(&maps.out[0], scratch, 4, N, rows * g.splits, N, 128);
  if (rc) return rc;
  if (g.splits == 1) return launch<LAYOUT, STORE, F16>(A, B, N, maps, g, num_sms, status, st);
  rc = launch<LAYOUT, PARTIAL, F16>(A, B, N, maps, g, num_sms, status, st);
  if (rc) return rc;
  return launch_pdl(ffn_reduce_kernel<F16>, dim3((unsigned)((M * N / 8 + 255) / 256)), dim3(256), 0, st,
                    (const float*)scratch, g.splits, rows, M, N, out, (const uint16_t*)residual.p, residual.ld);
}

// ------------------------------------------------------------------------------------------ few rows
// With few rows the weights' bytes are the time. The weights take the M side of the MMA (128 weight rows a CTA, gate
// and up tiles side by side in TMEM for DUAL) and the rows the N side, padded to NT; the C CTAs of a cluster take a
// share of K each and add their partial sums through distributed shared memory, so no partial goes through HBM and
// there is one launch a product. h is kept as two terms (value and rounding error, rows 0.. and T.. of a [2T, F]
// buffer): the second MMA column block costs nothing here and leaves the result with its own rounding only.
constexpr int64_t PREFETCH = 48 << 20;  // of the down projection's weights, into the 126 MB of L2

static int64_t weight_bytes(const FfnShape& s) { return (2 * (int64_t)s.H + s.N) * s.F * 2; }
// Up to 32 rows an SM holds two CTAs, with more one, and clusters of a power of two leave SMs without one where there are
// many weight tiles: so the limits, each between two measured sizes. Measured with cold weights, us here and as large
// tiles. 64 rows: 2,560 x 10,240 (157 MB of weights) 51.5 and 52.0, 4,096 x 8,192 (201 MB) 52.5 and 49.7. 128 rows:
// 2,560 x 4,096 (63 MB) 29.7 and 31.1, 2,048 x 6,144 (75 MB) 34.1 and 31.9 (80 rows 31.6 and 30.7); 4,096 x 5,120
// (126 MB), whose tiles happen to fill the clusters, 43.3 and 44.8, 2,560 x 10,240 75 and 54. 256 rows: 2,048 x 2,048
// (25 MB) 23.5 and 25.8, 1,152 x 4,304 (30 MB) 28.2 and 22.9. 384 rows: 2,048 x 1,536 (19 MB) 25.2 and 25.7,
// 2,048 x 2,048 30.2 and 28.3; 512 rows of 2,048 x 1,024 23.6 and 23.5. 32 rows: 5,120 x 17,408 (535 MB) 96 and 104.
static bool few(const FfnShape& s) {
  const int64_t b = weight_bytes(s);
  return s.T <= 32 || (s.T <= 64 && b <= 180'000'000) || (s.T <= 128 && b <= 70'000'000) ||
         (s.T <= 256 && b <= 27'000'000) || (s.T <= 384 && b <= 22'000'000);
}

template <bool DUAL_, int NT>
struct Few {
  static constexpr int NA = DUAL_ ? 2 : 1, NB = DUAL_ ? NT : 2 * NT;  // weight tiles and MMA columns
  static constexpr uint32_t STAGE = NA * 16384 + NB * 128;
  static constexpr uint32_t BUDGET = NT <= 32 ? 110592 : 204800;  // two CTAs an SM up to 32 rows
  static constexpr int STAGES = BUDGET / STAGE;
  static constexpr uint32_t TOTAL = STAGES * STAGE + (2 * STAGES + 1) * 8 + 16 + 1024;
  static_assert(STAGES * STAGE >= NA * NT * 512u, "partial sums reuse the ring");
};
struct FewArgs {
  int T = 0, n = 0;  // rows; weight rows (DUAL: F)
  int chunk = 0;     // rows of a CTA (gridDim.z chunks)
  int K = 0, F = 0, act = 0;
  void* out = nullptr;             // DUAL: h [2T, F]; else y [T, n]
  float* gu = nullptr;             // DUAL: p and q (at_gu) or null
  const void* residual = nullptr;  // else: [T, n] or null
  int64_t ldr = 0;
  const void* next = nullptr;      // DUAL: the down projection's weights, `next_bytes` of them (a multiple of 16)
  int64_t next_bytes = 0;
};

template <bool DUAL_, int NT, bool F16>
__global__ void __launch_bounds__(192) ffn_few_kernel(const __grid_constant__ CUtensorMap tm_w,
                                                      const __grid_constant__ CUtensorMap tm_x, FewArgs g,
                                                      uint32_t* status) {
  using S = Few<DUAL_, NT>;
  constexpr int STAGES = S::STAGES, NB = S::NB;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * S::STAGE);
  uint64_t* empty = full + STAGES;
  uint64_t* done = empty + STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int C = gridDim.x, rank = blockIdx.x, w0 = blockIdx.y * 128;
  const int t0 = blockIdx.z * g.chunk, rows = min(g.chunk, g.T - t0);
  const int kb_total = (g.K + BK - 1) / BK, kb0 = kb_total * rank / C, num_kb = kb_total * (rank + 1) / C - kb0;
  constexpr uint32_t TMEM_COLS = 2 * NT;

  // the weights: for DUAL the previous kernel in the stream may have written them (prefetched into L2, which is never
  // stale); for the down projection it is the DUAL kernel, which waited for everything before it, so they are loaded
  auto load_w = [&](int i) {
    uint8_t* a = smem + (i % STAGES) * S::STAGE;
    uint64_t* bar = &full[i % STAGES];
    mbar_arrive_expect_tx(bar, S::STAGE);
    tma_load_2d(a, &tm_w, bar, (kb0 + i) * BK, w0);
    if constexpr (DUAL_) tma_load_2d(a + 16384, &tm_w, bar, (kb0 + i) * BK, g.F + w0);
  };
  auto load_x = [&](int i) {
    uint8_t* b = smem + (i % STAGES) * S::STAGE + S::NA * 16384;
    tma_load_2d(b, &tm_x, &full[i % STAGES], (kb0 + i) * BK, t0);
    if constexpr (!DUAL_) tma_load_2d(b + NT * 128, &tm_x, &full[i % STAGES], (kb0 + i) * BK, g.T + t0);
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    fence_mbar_init();
    fence_proxy_async_smem();
    if constexpr (DUAL_) {
      for (int i = 0; i < min(num_kb, STAGES); ++i) {
        tma_prefetch_l2_2d(&tm_w, (kb0 + i) * BK, w0);
        tma_prefetch_l2_2d(&tm_w, (kb0 + i) * BK, g.F + w0);
      }
    } else {
      for (int i = 0; i < min(num_kb, STAGES); ++i) load_w(i);
    }
  }
  if (warp == 1) tmem_alloc(tmem_slot, TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_dep_wait();
  if (threadIdx.x == 0) grid_dep_trigger();

  if (warp == 0) {
    if (lane == 0) {
      int issued = 0;
      for (int i = 0; i < num_kb; ++i) {
        if (i >= STAGES && !mbar_wait(&empty[i % STAGES], ((i / STAGES) & 1) ^ 1, status)) break;
        if (DUAL_ || i >= STAGES) load_w(i);
        load_x(i);
        ++issued;
      }
      if constexpr (DUAL_) {
        // this CTA's share of the next kernel's weights into L2: HBM works on through the sums and the epilogue
        const int64_t ctas = (int64_t)gridDim.x * gridDim.y * gridDim.z;
        const int64_t id = ((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x;
        const int64_t each = (g.next_bytes / 16 + ctas - 1) / ctas * 16, end = min(g.next_bytes, (id + 1) * each);
        for (int64_t at = id * each; at < end; at += 16384)
          bulk_prefetch_l2(reinterpret_cast<const uint8_t*>(g.next) + at, (uint32_t)min((int64_t)16384, end - at));
      }
      for (int i = max(0, issued - STAGES); i < issued; ++i) mbar_wait(&full[i % STAGES], (i / STAGES) & 1, status);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_f16(128, NB, F16 ? 0 : 1);
      for (int i = 0; i < num_kb; ++i) {
        const int s = i % STAGES;
        if (!mbar_wait(&full[s], (i / STAGES) & 1, status)) break;
        tc_fence_after();
        const uint32_t a = smem_u32(smem + s * S::STAGE), b = a + S::NA * 16384;
#pragma unroll
        for (int kk = 0; kk < BK / 16; ++kk) {
          umma_f16(tmem, sw128_desc(a) + 2 * kk, sw128_desc(b) + 2 * kk, idesc, (i | kk) != 0);
          if constexpr (DUAL_)
            umma_f16(tmem + NT, sw128_desc(a + 16384) + 2 * kk, sw128_desc(b) + 2 * kk, idesc, (i | kk) != 0);
        }
        umma_commit(&empty[s]);
      }
      umma_commit(done);
    }
  } else {
    // partial sums to shared memory (the ring is free: every MMA has read it): [NA][rows][128]
    const int quad = warp & 3;
    mbar_wait(done, 0, status);  // (a wait that gives up is in the status word)
    tc_fence_after();
    const uint32_t taddr = tmem + ((uint32_t)(quad * 32) << 16);
    float* p = reinterpret_cast<float*>(smem) + quad * 32 + lane;
    constexpr int CW = NT < 32 ? NT : 32;  // columns at a time
#pragma unroll 1
    for (int c = 0; c < rows; c += CW) {
      float v[CW], w[CW];
      if constexpr (CW == 16) {
        tmem_ld16(taddr + c, v);
        tmem_ld16(taddr + NT + c, w);  // DUAL: up; else the second term of h
      } else {
        tmem_ld32(taddr + c, v);
        tmem_ld32(taddr + NT + c, w);
      }
      tmem_ld_wait();
      const int n = rows - c;
#pragma unroll
      for (int j = 0; j < CW; ++j) {
        if constexpr (DUAL_) {
          if (j < n) p[(c + j) * 128] = v[j], p[(rows + c + j) * 128] = w[j];
        } else {
          if (j < n) p[(c + j) * 128] = v[j] + w[j];
        }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  cluster_sync();
  {
    uint32_t part[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) part[c] = cluster_addr(smem, min(c, C - 1));
    // four weight rows of one row: the cluster's partial sums in their order, all on the way at once
    auto sum = [&](uint32_t off) {
      float4 q[8];
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (c < C) q[c] = ld_cluster_f4(part[c] + off);
      float4 s = q[0];
#pragma unroll
      for (int c = 1; c < 8; ++c)
        if (c < C) s.x += q[c].x, s.y += q[c].y, s.z += q[c].z, s.w += q[c].w;
      return s;
    };
    const int quads = rows * 32;  // (row, four weight rows), dealt to the cluster's threads
#pragma unroll 1
    for (int e = rank * 192 + threadIdx.x; e < quads; e += C * 192) {
      const int r = e >> 5, t = t0 + r, f = (e & 31) * 4, col = w0 + f;
      if (col >= g.n) continue;
      float4 a = sum((r * 128 + f) * 4);
      if constexpr (DUAL_) {
        const float4 u = sum(((rows + r) * 128 + f) * 4);
        float4 d;
        with_act(g.act, [&](auto A) {
          act_grad<A.value>(a.x, a.x, d.x);
          act_grad<A.value>(a.y, a.y, d.y);
          act_grad<A.value>(a.z, a.z, d.z);
          act_grad<A.value>(a.w, a.w, d.w);
        });
        if (g.gu) {
          *reinterpret_cast<float4*>(g.gu + at_gu(t, col, g.F, 0)) = make_float4(u.x * d.x, u.y * d.y, u.z * d.z, u.w * d.w);
          *reinterpret_cast<float4*>(g.gu + at_gu(t, col, g.F, 1)) = a;
        }
        a = make_float4(a.x * u.x, a.y * u.y, a.z * u.z, a.w * u.w);
        const uint2 hi = make_uint2(pack2<F16>(a.x, a.y), pack2<F16>(a.z, a.w));
        const float2 r0 = unpack2<F16>(hi.x), r1 = unpack2<F16>(hi.y);
        const uint2 lo = make_uint2(
            pack2<F16>(isfinite(r0.x) ? a.x - r0.x : 0.f, isfinite(r0.y) ? a.y - r0.y : 0.f),
            pack2<F16>(isfinite(r1.x) ? a.z - r1.x : 0.f, isfinite(r1.y) ? a.w - r1.y : 0.f));
        uint16_t* h = reinterpret_cast<uint16_t*>(g.out) + (int64_t)t * g.F + col;
        *reinterpret_cast<uint2*>(h) = hi;
        *reinterpret_cast<uint2*>(h + (int64_t)g.T * g.F) = lo;
      } else {
        if (g.residual) {
          const uint2 q = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(g.residual) + t * g.ldr + col);
          const float2 r0 = unpack2<F16>(q.x), r1 = unpack2<F16>(q.y);
          a.x += r0.x, a.y += r0.y, a.z += r1.x, a.w += r1.y;
        }
        *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(g.out) + (int64_t)t * g.n + col) =
            make_uint2(pack2<F16>(a.x, a.y), pack2<F16>(a.z, a.w));
      }
    }
  }
  cluster_sync();  // no CTA leaves while another reads its partial sums
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

// CTAs of a cluster: as many of 8, 4, 2 or 1 as leave each two K blocks and all clusters resident at once (a cluster that
// has to wait for another costs the kernel's time again: at 64 rows 48 clusters of 4 take 25 us, 48 of 2 take 18). How
// many are resident is asked for once a kernel, size and device. Negative: an error.
template <bool DUAL_, int NT, bool F16>
static int few_cluster(int clusters, int kb) {
  auto kern = ffn_few_kernel<DUAL_, NT, F16>;
  static std::atomic<uint64_t> devs{0};
  if (const int e = smem_attr_once(devs, (const void*)kern, Few<DUAL_, NT>::TOTAL)) return -e;
  static std::atomic<int> resident[64][4];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return -(int)e;
  for (int i = 3; i > 0; --i) {
    if (kb / (1 << i) < 2) continue;
    int most = resident[dev & 63][i].load(std::memory_order_relaxed);
    if (!most) {
      cudaLaunchConfig_t cfg = {};
      cudaLaunchAttribute at;
      at.id = cudaLaunchAttributeClusterDimension;
      at.val.clusterDim = {1u << i, 1, 1};
      cfg.gridDim = dim3(1 << i), cfg.blockDim = dim3(192), cfg.dynamicSmemBytes = Few<DUAL_, NT>::TOTAL;
      cfg.attrs = &at, cfg.numAttrs = 1;
      e = cudaOccupancyMaxActiveClusters(&most, kern, &cfg);
      if (e != cudaSuccess) return -(int)e;
      most = std::max(most * (NT <= 32 ? 2 : 1), 1);  // (counted at one CTA an SM)
      resident[dev & 63][i].store(most, std::memory_order_relaxed);
    }
    if (clusters <= most) return 1 << i;
  }
  return 1;
}

template <bool DUAL_, int NT, bool F16>
static int launch_few(Ptr w, int64_t w_rows, Ptr x, int64_t x_rows, FewArgs g, int chunks, int C, uint32_t* status,
                      cudaStream_t st) {
  using S = Few<DUAL_, NT>;
  CUtensorMap tw, tx;
  int rc = make_tmap_2d(&tw, w.p, 2, g.K, w_rows, w.ld * 2, BK, 128, 1);
  if (!rc) rc = make_tmap_2d(&tx, x.p, 2, g.K, x_rows, x.ld * 2, BK, NT, 1);
  if (rc) return 5000 + rc;
  g.chunk = (g.T + chunks - 1) / chunks;
  if (g.chunk > NT) return 6;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(C, (g.n + 127) / 128, chunks);
  cfg.blockDim = dim3(192);
  cfg.dynamicSmemBytes = S::TOTAL;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {(unsigned)C, 1, 1};
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, ffn_few_kernel<DUAL_, NT, F16>, tw, tx, g, status);
  return e == cudaSuccess ? (int)cudaGetLastError() : (int)e;
}

// The rows go as chunks of NT, or of half of that (and half again, to 32) where that costs the clusters no CTA: the partial
// sums that a cluster exchanges are halved (80 rows at 2,560 x 640: 16.5 us in one chunk, 14.5 in two; 128 rows at
// 256 x 136: 13.6 in two chunks, 10.1 in four). Chunks of 32 only if there are twice as many (80 rows at 2,560 x 640 in
// three: 14.7; chunks of 16: 64 rows at 2,048 x 512 11.6, of 32 10.9).
template <bool DUAL_, int NT, bool F16>
static int few_rows(Ptr w, int64_t w_rows, Ptr x, int64_t x_rows, const FewArgs& g, uint32_t* status, cudaStream_t st) {
  const int tiles = (g.n + 127) / 128, kb = (g.K + BK - 1) / BK, chunks = (g.T + NT - 1) / NT;
  const int C = few_cluster<DUAL_, NT, F16>(chunks * tiles, kb);
  if (C < 0) return -C;
  if constexpr (NT > 32) {
    const int chunks2 = (g.T + NT / 2 - 1) / (NT / 2);
    if (NT > 64 || chunks2 == 2 * chunks) {
      const int C2 = few_cluster<DUAL_, NT / 2, F16>(chunks2 * tiles, kb);
      if (C2 < 0) return -C2;
      if (C2 >= C) return few_rows<DUAL_, NT / 2, F16>(w, w_rows, x, x_rows, g, status, st);
    }
  }
  return launch_few<DUAL_, NT, F16>(w, w_rows, x, x_rows, g, chunks, C, status, st);
}

template <int NT, bool F16>
static int fwd_few(const FfnShape& s, Ptr x, Ptr w13, Ptr w2, Ptr residual, void* h, float* gu, void* y, uint32_t* status,
                   cudaStream_t st) {
  FewArgs g;
  g.T = (int)s.T, g.n = s.F, g.K = s.H, g.F = s.F, g.act = s.act, g.out = h, g.gu = gu;
  g.next = w2.p, g.next_bytes = std::min<int64_t>((int64_t)s.N * s.F * 2, PREFETCH);
  const int rc = few_rows<true, NT, F16>(w13, 2 * (int64_t)s.F, x, s.T, g, status, st);
  if (rc) return rc;
  g = FewArgs();
  g.T = (int)s.T, g.n = s.N, g.K = s.F, g.out = y, g.residual = residual.p, g.ldr = residual.ld;
  return few_rows<false, NT, F16>(w2, s.N, {h, s.F}, 2 * s.T, g, status, st);
}

// ------------------------------------------------------------------------------------------ one to 32 rows
// Here a launch's latency counts beside the weights' bytes, and the kernels above have a ring to fill, TMEM to allocate
// and read and two cluster barriers. These read the weights straight into registers and add a CTA's partial sums, one
// share of K a warp, through shared memory. h goes from the first to the second in two terms, as above.
//
// One row: dot products on the CUDA cores, whose FMAs keep pace with HBM (2,048 x 6,144: some 3 us of them beside 11.5 us
// of loads). A CTA takes two columns of h (four weight rows) or two of y; its four warps take chunks of 256 elements, so
// every load is 512 bytes of a row in one piece. Small CTAs, many an SM, keep enough loads on the way (eight warps and
// four columns a CTA: 18.5 us where this takes 14.8).
//
// More rows: mma.sync, for a lane can load 16 bytes of "its" weight row as they lie and hand them on as fragments. K may
// come in any order if weights and rows agree, so lane 4 r + c takes elements 8 c .. 8 c + 7 of a block of 32 of row r:
// two MMAs' worth. A CTA takes 8 columns of h (its MMA's 16 weight rows are the 8 gate and the 8 up rows, so a
// thread ends with both of a pair) or 16 of y. FMAs instead, with the rows' values in registers: 2 rows 18.4 us at
// 2,048 x 6,144 and 14.3 at 1,152 x 4,304, 4 rows 27 and 15; this 18.3 and 10.7, 18.8 and 11.0.
//
// Measured with cold weights, us here and in the kernels above; the limits lie between two measured sizes. One row:
// 2,048 x 6,144 15 and 20.6, 5,120 x 17,408 86 and 93 (6.2 TB/s and 5.7), 2,048 x 512 4.7 and 8.7. Eight rows:
// 2,048 x 512 5.5 and 8.8, 2,048 x 2,048 7.8 and 11.9, 2,048 x 6,144 (75 MB of weights) 21.0 and 22.2, 2,560 x 6,144
// (94 MB) 29.9 and 24.6 (rows of 2,560 take a second round of the warps' blocks for a quarter of it: 2,560 x 2,560 16.7
// and 15.1), 5,120 x 17,408 (535 MB) 129 and 92, for a row's 64 bytes at a time are less than HBM wants. Sixteen rows:
// 2,048 x 512 5.4 and 8.9, 2,048 x 2,048 (25 MB) 11.0 and 12.4, 1,152 x 4,304 (30 MB) 16.4 and 14.1. 32 rows:
// 2,048 x 512 (6 MB) 8.2 and 9.9, 256 x 136 6.6 and 10, 2,560 x 640 (10 MB) 13.9 and 11.5.
static bool tokens(const FfnShape& s) {
  return s.T == 1 || (s.T <= 8 && weight_bytes(s) <= 85'000'000) || (s.T <= 16 && weight_bytes(s) <= 27'000'000) ||
         (s.T <= 32 && weight_bytes(s) <= 7'000'000);
}

// not by way of L1, which another kernel on the SM may have filled before the weights were written
AFB_DEV uint4 ld_weights(const void* p) {
  uint4 v;
  asm volatile("ld.global.cg.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}
AFB_DEV void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

struct TokenArgs {
  int T = 0, n = 0, K = 0, act = 0;  // rows; columns of the result (DUAL: F)
  const void* w = nullptr;           // [n or 2 n, K]
  const void* x = nullptr;           // DUAL: [T, K]; else h [2T, K]
  int64_t ldx = 0;
  void* out = nullptr;             // DUAL: h [2T, F]; else y [T, n]
  float* gu = nullptr;             // DUAL: p and q (at_gu) or null
  const void* residual = nullptr;  // else: [T, n] or null
  int64_t ldr = 0;
};
// from the sums of one element (DUAL: gate a and up u; else a) to what is stored
template <bool DUAL_, bool F16>
AFB_DEV void finish(const TokenArgs& g, int t, int col, float a, float u) {
  uint16_t* out = reinterpret_cast<uint16_t*>(g.out) + (int64_t)t * g.n + col;
  if constexpr (DUAL_) {
    float d;
    with_act(g.act, [&](auto A) { act_grad<A.value>(a, a, d); });
    if (g.gu) {
      g.gu[at_gu(t, col, g.n, 0)] = u * d;
      g.gu[at_gu(t, col, g.n, 1)] = a;
    }
    const float h = a * u;
    const uint32_t hi = pack2<F16>(h, 0.f);
    const float f = unpack2<F16>(hi).x;
    out[0] = (uint16_t)hi;
    out[(int64_t)g.T * g.n] = (uint16_t)pack2<F16>(isfinite(f) ? h - f : 0.f, 0.f);
  } else {
    if (g.residual) a += unpack2<F16>(reinterpret_cast<const uint16_t*>(g.residual)[t * g.ldr + col]).x;
    out[0] = (uint16_t)pack2<F16>(a, 0.f);
  }
}

// Sums of V values over a warp's lanes, each left in the lanes whose top bits are its index: a step exchanges half of
// the values that are left
template <int V>
AFB_DEV float warp_sums(float* v) {
  const int lane = threadIdx.x & 31;
  int bit = 16;
#pragma unroll
  for (int n = V / 2; n > 0; n >>= 1, bit >>= 1) {
    const bool up = lane & bit;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float give = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, bit);
    }
  }
#pragma unroll
  for (; bit > 0; bit >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], bit);
  return v[0];
}
template <bool F16>
AFB_DEV void unpack8(const uint4& q, float* f) {
  const uint32_t r[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = unpack2<F16>(r[i]);
    f[2 * i] = v.x, f[2 * i + 1] = v.y;
  }
}

constexpr int ROW_WARPS = 4, ROW_COLS = 2;

template <bool DUAL_, bool F16>
__global__ void __launch_bounds__(32 * ROW_WARPS) ffn_row_kernel(TokenArgs g) {
  // weight rows; chunks a warp has on the way at a time (half of them: 17.0 us at 2,048 x 6,144 and 12.3 at 1,152 x 4,304,
  // where these take 14.8 and 9.0)
  constexpr int WR = DUAL_ ? 2 * ROW_COLS : ROW_COLS, U = DUAL_ ? 2 : 4, STEP = ROW_WARPS * 256;
  __shared__ float red[ROW_WARPS][WR];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n0 = blockIdx.x * ROW_COLS, first = warp * 256 + lane * 8;
  const uint16_t* w = reinterpret_cast<const uint16_t*>(g.w) + (int64_t)n0 * g.K;
  auto row_of = [&](int r) { return w + (int64_t)(r < ROW_COLS ? r : g.n + r - ROW_COLS) * g.K; };
  uint4 q[U][WR];
  auto load = [&](int k0) {  // this lane's 8 elements of a weight row and chunk
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k0 + u * STEP < g.K) {
#pragma unroll
        for (int r = 0; r < WR; ++r) q[u][r] = ld_weights(row_of(r) + k0 + u * STEP);
      }
  };
  // as above: W2 may be read before the wait, W13 only brought nearer
  if constexpr (!DUAL_) {
    load(first);
  } else if ((lane & 7) == 0) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (first + u * STEP < g.K) {
#pragma unroll
        for (int r = 0; r < WR; ++r) prefetch_l2(row_of(r) + first + u * STEP);
      }
  }
  grid_dep_wait();
  grid_dep_trigger();
  float acc[WR] = {};
  for (int k0 = first; k0 < g.K; k0 += U * STEP) {
    if (DUAL_ || k0 != first) load(k0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * STEP;
      if (k < g.K) {
        const uint16_t* xp = reinterpret_cast<const uint16_t*>(g.x) + k;
        float x[8], f[8];
        unpack8<F16>(*reinterpret_cast<const uint4*>(xp), x);
        if constexpr (!DUAL_) {  // h in two terms
          unpack8<F16>(*reinterpret_cast<const uint4*>(xp + g.ldx), f);
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] += f[i];
        }
#pragma unroll
        for (int r = 0; r < WR; ++r) {
          unpack8<F16>(q[u][r], f);
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[r] += f[i] * x[i];
        }
      }
    }
  }
  const float s = warp_sums<WR>(acc);
  if (lane % (32 / WR) == 0) red[warp][lane / (32 / WR)] = s;
  __syncthreads();
  const int r = threadIdx.x;
  if (r >= ROW_COLS) return;
  float a = 0.f, u = 0.f;
#pragma unroll
  for (int i = 0; i < ROW_WARPS; ++i) {
    a += red[i][r];
    if (DUAL_) u += red[i][WR - ROW_COLS + r];
  }
  finish<DUAL_, F16>(g, 0, n0 + r, a, u);
}

template <bool F16>
AFB_DEV void mma_rows(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    mma_bf16(c, a0, a1, a2, a3, b0, b1);
}

constexpr int TOK_WARPS = 16;

// NG: groups of 8 rows (one past the last is computed as the last and left out)
template <bool DUAL_, int NG, bool F16>
__global__ void __launch_bounds__(32 * TOK_WARPS) ffn_tokens_kernel(TokenArgs g) {
  // terms of the rows' values, blocks of 64 elements at a time, columns of the result
  constexpr int TERMS = DUAL_ ? 1 : 2, U = DUAL_ ? 2 : 4, STEP = TOK_WARPS * 64, COLS = DUAL_ ? 8 : 16;
  __shared__ float red[TOK_WARPS][8 * NG][16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, gc = (lane & 3) * 8, first = warp * 64;
  const int n0 = blockIdx.x * COLS;
  const uint16_t* wp[2];  // rows gr and gr + 8 of the MMA
#pragma unroll
  for (int i = 0; i < 2; ++i)
    wp[i] = reinterpret_cast<const uint16_t*>(g.w) +
            (int64_t)(DUAL_ ? i * g.n + n0 + gr : min(n0 + i * 8 + gr, g.n - 1)) * g.K;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  uint4 q[U][2][2];
  auto load = [&](int kb) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int k = kb + u * STEP + j * 32 + gc;
#pragma unroll
        for (int i = 0; i < 2; ++i) q[u][i][j] = k < g.K ? ld_weights(wp[i] + k) : zero;
      }
  };
  if constexpr (!DUAL_) {
    load(first);
  } else if (gc == 0) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (first + u * STEP < g.K) prefetch_l2(wp[0] + first + u * STEP), prefetch_l2(wp[1] + first + u * STEP);
  }
  grid_dep_wait();
  grid_dep_trigger();
  float acc[NG][4] = {};
  const uint16_t* xp[NG];
#pragma unroll
  for (int i = 0; i < NG; ++i) xp[i] = reinterpret_cast<const uint16_t*>(g.x) + min(i * 8 + gr, g.T - 1) * g.ldx;
  for (int kb = first; kb < g.K; kb += U * STEP) {
    if (DUAL_ || kb != first) load(kb);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (kb + u * STEP < g.K) {
        uint4 x[2][NG][TERMS];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int k = kb + u * STEP + j * 32 + gc;
#pragma unroll
          for (int i = 0; i < NG; ++i)
#pragma unroll
            for (int t = 0; t < TERMS; ++t)
              x[j][i][t] = k < g.K ? *reinterpret_cast<const uint4*>(xp[i] + t * g.T * g.ldx + k) : zero;
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < NG; ++i)
#pragma unroll
            for (int t = 0; t < TERMS; ++t) {
              const uint4 &a = q[u][0][j], &b = q[u][1][j], &v = x[j][i][t];
              mma_rows<F16>(acc[i], a.x, b.x, a.y, b.y, v.x, v.y);
              mma_rows<F16>(acc[i], a.z, b.z, a.w, b.w, v.z, v.w);
            }
      }
  }
  // of the MMA's result a lane holds weight rows gr and gr + 8 of rows 2 (lane % 4) and the next
#pragma unroll
  for (int i = 0; i < NG; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) red[warp][i * 8 + (lane & 3) * 2 + (e & 1)][gr + (e >> 1) * 8] = acc[i][e];
  __syncthreads();
  const int t = threadIdx.x / COLS, r = threadIdx.x % COLS;
  static_assert(8 * NG * COLS <= 32 * TOK_WARPS, "a thread has one element at most");
  if (t >= g.T || n0 + r >= g.n) return;
  float a = 0.f, u = 0.f;
#pragma unroll
  for (int i = 0; i < TOK_WARPS; ++i) {
    a += red[i][t][r];
    if (DUAL_) u += red[i][t][r + 8];
  }
  finish<DUAL_, F16>(g, t, n0 + r, a, u);
}

template <bool F16>
static int fwd_tokens(const FfnShape& s, Ptr x, Ptr w13, Ptr w2, Ptr residual, void* h, float* gu, void* y,
                      cudaStream_t st) {
  auto run = [&](auto dual, const TokenArgs& g) {
    constexpr bool D = decltype(dual)::value;
    if (s.T == 1) return launch_pdl(ffn_row_kernel<D, F16>, dim3(g.n / ROW_COLS), dim3(32 * ROW_WARPS), 0, st, g);
    auto kern = s.T <= 8 ? ffn_tokens_kernel<D, 1, F16> : s.T <= 16 ? ffn_tokens_kernel<D, 2, F16> : ffn_tokens_kernel<D, 4, F16>;
    return launch_pdl(kern, dim3(D ? g.n / 8 : (g.n + 15) / 16), dim3(32 * TOK_WARPS), 0, st, g);
  };
  TokenArgs g;
  g.T = (int)s.T, g.n = s.F, g.K = s.H, g.act = s.act, g.w = w13.p, g.x = x.p, g.ldx = x.ld, g.out = h, g.gu = gu;
  const int rc = run(std::true_type(), g);
  if (rc) return rc;
  g = TokenArgs();
  g.T = (int)s.T, g.n = s.N, g.K = s.F, g.w = w2.p, g.x = h, g.ldx = s.F, g.out = y, g.residual = residual.p;
  g.ldr = residual.ld;
  return run(std::false_type(), g);
}

static size_t product_scratch(int64_t M, int N, int64_t K, int num_sms) {
  const int s = plan_splits(M, N, K, num_sms);
  return s > 1 ? (size_t)s * ((M + BM - 1) / BM * BM) * N : 0;
}

template <bool F16>
static int fwd(const FfnShape& s, Ptr x, Ptr w13, Ptr w2, Ptr residual, void* h, float* gu, void* y, float* scratch,
               int num_sms, uint32_t* status, cudaStream_t st) {
  if (tokens(s)) return fwd_tokens<F16>(s, x, w13, w2, residual, h, gu, y, st);
  if (few(s)) {
    auto f = s.T <= 16 ? fwd_few<16, F16> : s.T <= 32 ? fwd_few<32, F16> : s.T <= 64 ? fwd_few<64, F16> : fwd_few<128, F16>;
    return f(s, x, w13, w2, residual, h, gu, y, status, st);
  }
  Maps<NT> maps;
  Args g;
  g.M = s.T, g.N = s.F, g.K = s.H, g.F = s.F, g.act = s.act, g.f32 = gu;
  int rc = row_map(&maps.out[0], h, 2, s.F, s.T, s.F, 128);
  if (!rc) rc = launch<NT, DUAL, F16>(x, w13, 2 * (int64_t)s.F, maps, g, num_sms, status, st);
  if (rc) return rc;
  return product<NT, F16>({h, s.F}, w2, s.T, s.N, s.F, y, residual, scratch, num_sms, status, st);
}

// Tiles of the products after DACT, and whether one launch of all of them is expected to take less time than a launch
// (5 us beside its tiles) for each. A K block takes some 15% more there, for tiles of different products in flight
// share less of L2. Measured, together against apart: 1,237 x 1,152 x 4,304 56 and 85 us, 16,384 x 2,048 x 512 114 and
// 136; 4,100 x 2,048 x 6,144, whose tiles fill their waves, 383 and 362; and dx of few tiles and many K blocks has to
// be split.
static bool plan_grads(const FfnShape& s, bool dw13, bool dw2, int num_sms, Grads& g) {
  const int64_t M[3] = {s.T, dw13 ? 2 * (int64_t)s.F : 0, dw2 ? s.N : 0}, K[3] = {2 * (int64_t)s.F, s.T, s.T};
  const int N[3] = {s.H, s.H, s.F};
  const int64_t P = num_sms / 2;
  double apart = 0;
  int64_t units = 0;
  for (int q = 0; q < 3; ++q) {
    if (!M[q]) continue;
    const int64_t mt = (M[q] + BM - 1) / BM, nt = (N[q] + BN - 1) / BN;
    if (mt * nt >= (1 << 28)) return false;
    g.M[q] = (int)M[q], g.N[q] = N[q], g.mt[q] = (uint32_t)mt, g.nt[q] = (uint32_t)nt, g.tiles[q] = (uint32_t)(mt * nt);
    g.kb[q] = (uint32_t)((K[q] + BK - 1) / BK);
    units += (int64_t)g.tiles[q] * g.kb[q];
    double us = 0;
    plan_splits(M[q], N[q], K[q], num_sms, &us);
    apart += us + 5.;
  }
  const int64_t kt = std::max(g.kb[1], g.kb[2]), weights = (int64_t)g.tiles[1] + g.tiles[2];
  g.dx_long = g.kb[0] >= kt;
  g.longs = (uint32_t)(g.dx_long ? g.tiles[0] : weights), g.shorts = (uint32_t)(g.dx_long ? weights : g.tiles[0]);
  const int64_t kl = g.dx_long ? g.kb[0] : kt, ks = g.dx_long ? kt : g.kb[0];
  const int64_t each = g.longs / P, more = g.longs % P;
  // the least load of a pair that holds all short tiles
  int64_t load = std::max((each + (more > 0)) * kl, (units + P - 1) / P);
  for (;; ++load) {
    g.x = more ? (uint32_t)((load - (each + 1) * kl) / ks) : 0;
    g.y = (uint32_t)((load - each * kl) / ks);
    if (more * g.x + (P - more) * (int64_t)g.y >= g.shorts) break;
  }
  return load * KB_US * 1.15 + 5. < apart;
}

template <bool F16>
static int bwd(const FfnShape& s, Ptr dy, Ptr x, Ptr w13, Ptr w2, const void* h, const float* gu, void* dgu, void* dx,
               void* dw13, void* dw2, float* scratch, int num_sms, uint32_t* status, cudaStream_t st) {
  const Ptr none{nullptr, 0}, d{dgu, 2 * (int64_t)s.F};
  int rc = 0;
  Args gr;
  const bool together = dx && (dw13 || dw2) && plan_grads(s, dw13, dw2, num_sms, gr.grads);
  if (dw2 && !together && (rc = product<TN, F16>(dy, {h, s.F}, s.N, s.F, s.T, dw2, none, scratch, num_sms, status, st)))
    return rc;
  if (!dx && !dw13) return 0;
  Maps<NN> maps;
  Args g;
  g.M = s.T, g.N = s.F, g.K = s.N, g.F = s.F, g.act = s.act, g.f32 = const_cast<float*>(gu);
  uint16_t* o = reinterpret_cast<uint16_t*>(dgu);
  rc = row_map(&maps.out[0], o, 2, s.F, s.T, d.ld, 64);
  if (!rc) rc = row_map(&maps.out[1], o + s.F, 2, s.F, s.T, d.ld, 64);
  if (!rc) rc = launch<NN, DACT, F16>(dy, w2, s.F, maps, g, num_sms, status, st);
  if (rc) return rc;
  if (together) {
    Maps<GRADS> m;
    rc = operand_maps(&m.a[0], &m.b[0], false, true, d, w13, s.T, s.H, 2 * (int64_t)s.F);
    if (!rc) rc = row_map(&m.out[0], dx, 2, s.H, s.T, s.H, 128);
    if (!rc && dw13) rc = operand_maps(&m.a[1], &m.b[1], true, true, d, x, 2 * (int64_t)s.F, s.H, s.T);
    if (!rc && dw13) rc = row_map(&m.out[1], dw13, 2, s.H, 2 * (int64_t)s.F, s.H, 128);
    if (!rc && dw2) rc = operand_maps(&m.a[2], &m.b[2], true, true, dy, {h, s.F}, s.N, s.F, s.T);
    if (!rc && dw2) rc = row_map(&m.out[2], dw2, 2, s.F, s.N, s.F, 128);
    if (rc) return rc;
    if (!dw13) m.a[1] = m.a[0], m.b[1] = m.b[0], m.out[1] = m.out[0];  // not read, but fetched ahead
    if (!dw2) m.a[2] = m.a[0], m.b[2] = m.b[0], m.out[2] = m.out[0];
    auto kern = ffn_gemm_kernel<GRADS, STORE, F16>;
    static std::atomic<uint64_t> devs{0};
    if ((rc = smem_attr_once(devs, (const void*)kern, SMEM))) return rc;
    return launch_pdl(kern, dim3(2 * (num_sms / 2)), dim3(THREADS), SMEM, st, m, gr, status);
  }
  if (dx && (rc = product<NN, F16>(d, w13, s.T, s.H, 2 * (int64_t)s.F, dx, none, scratch, num_sms, status, st)))
    return rc;
  if (dw13) rc = product<TN, F16>(d, x, 2 * (int64_t)s.F, s.H, s.T, dw13, none, scratch, num_sms, status, st);
  return rc;
}

static bool valid(const FfnShape& s) {
  return s.T >= 0 && s.H > 0 && s.F > 0 && s.N > 0 && !(s.H % 8) && !(s.F % 8) && !(s.N % 8) && s.act >= 0 &&
         s.act <= 2;
}

}  // namespace ffn

size_t ffn_fwd_scratch(const FfnShape& s, int num_sms) {
  return ffn::few(s) ? 0 : ffn::product_scratch(s.T, s.N, s.F, num_sms);
}
int64_t ffn_h_rows(const FfnShape& s) { return ffn::few(s) ? 2 * s.T : s.T; }
size_t ffn_bwd_scratch(const FfnShape& s, int num_sms) {
  return std::max({ffn::product_scratch(s.N, s.F, s.T, num_sms), ffn::product_scratch(s.T, s.H, 2 * s.F, num_sms),
                   ffn::product_scratch(2 * s.F, s.H, s.T, num_sms)});
}

int ffn_fwd(const FfnShape& s, const void* x, int64_t ldx, const void* w13, const void* w2, const void* residual,
            int64_t ldr, void* h, float* gu, void* y, float* scratch, int num_sms, uint32_t* status, cudaStream_t st) {
  if (!ffn::valid(s)) return 3;
  if (s.T == 0) return 0;
  return (s.fp16 ? ffn::fwd<true> : ffn::fwd<false>)(s, {x, ldx}, {w13, s.H}, {w2, s.F}, {residual, ldr}, h, gu, y,
                                                     scratch, num_sms, status, st);
}

int ffn_bwd(const FfnShape& s, const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w13,
            const void* w2, const void* h, const float* gu, void* dgu, void* dx, void* dw13, void* dw2, float* scratch,
            int num_sms, uint32_t* status, cudaStream_t st) {
  if (!ffn::valid(s)) return 3;
  if (s.T == 0) return 0;  // the caller zeroes the weight gradients
  return (s.fp16 ? ffn::bwd<true> : ffn::bwd<false>)(s, {dy, lddy}, {x, ldx}, {w13, s.H}, {w2, s.F}, h, gu, dgu, dx,
                                                     dw13, dw2, scratch, num_sms, status, st);
}

}  // namespace afb
