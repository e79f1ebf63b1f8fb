// Matrix products of the dense operators on tcgen05, for 16-bit operands (bf16, fp16) and for 4-bit ones with a
// scale per 32 elements.  Two kernels:
//
//   pair_gemm    D[256 x 256], D[256 x 192] or D[256 x 128] tiles on pairs of CTAs.
//   stream_gemm  the weights are the M operand (128 rows a tile), up to 192 tokens the N operand, and a cluster of
//                up to eight CTAs shares the k axis of a tile: for few tokens, where every byte of the weights is
//                read once and that read has to be spread over all SMs.
//
// Both accumulate in fp32 in TMEM over the whole of a CTA's k range; stream_gemm adds the CTAs' partial sums in the
// order of their ranks, so a call gives the same bits each time.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "dense_types.h"
#include "ptx_cluster.cuh"

namespace fdmoe {
namespace dense {

// ------------------------------------------------------------- bounded waits
// Every wait ends: after `limit_ns` it records what it waited for, raises the CTA's abort flag, and all roles leave.
// The warps that issue copies and MMAs run their loops with all lanes and let one elected lane issue: inside a branch
// on the lane the compiler cannot tell that one thread is active, and instructions whose operands have to be uniform
// cost several times as much (the pair kernel's k block took 684 cycles so, whatever the tile's width).  Their lanes
// come together after every wait: a lane that fell behind by a whole ring of stages would look at a parity that had
// flipped twice, and wait for a phase that does not come.  For that all lanes make the same number of steps, also after
// a wait that ran out, which stops the waits and the issuing only.
struct Waiter {
  volatile uint32_t* abort_flag;
  uint32_t* status;
  uint64_t limit_ns;

  __device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, uint32_t code) const {
    if (ptx::mbar_try_wait(bar, parity)) return true;
    return slow(bar, parity, code);
  }
  // The same by a whole warp that goes on together.
  __device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, uint32_t code) const {
    return __all_sync(0xffffffffu, wait(bar, parity, code));
  }
  // The same by the lanes of a warp that issues, each with its own answer; `ok`: none of this lane's has run out yet.
  // One vote where all find the phase complete: without it 64 tokens of a 1024 x 2048 training step took 38.6 us, not 37.6.
  __device__ __forceinline__ bool wait_together(uint64_t* bar, uint32_t parity, uint32_t code, bool ok) const {
    if (__all_sync(0xffffffffu, ok && ptx::mbar_try_wait(bar, parity))) return true;
    if (ok) ok = wait(bar, parity, code);
    __syncwarp();
    return ok;
  }
  __device__ __noinline__ bool slow(uint64_t* bar, uint32_t parity, uint32_t code) const {
    const uint64_t t0 = ptx::globaltimer_ns();
    for (;;) {
      for (int i = 0; i < 64; ++i)
        if (ptx::mbar_try_wait(bar, parity)) return true;
      if (*abort_flag) return false;
      if (ptx::globaltimer_ns() - t0 > limit_ns) {
        atomicCAS_system(status, 0u, code);
        *abort_flag = 1;
        return false;
      }
    }
  }
  // After an abort: copies and MMAs that were issued before it end within microseconds; the CTA's shared memory and
  // TMEM are given back two milliseconds later.
  __device__ __forceinline__ void drain() const {
    if (!*abort_flag) return;
    const uint64_t t0 = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
  }
};

// --------------------------------------------------------------- arithmetic
__device__ __forceinline__ uint32_t pack2(float lo, float hi, bool bf16) {
  uint32_t r;
  if (bf16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ void unpack2(uint32_t v, bool bf16, float& lo, float& hi) {
  if (bf16) {
    lo = __uint_as_float(v << 16);
    hi = __uint_as_float(v & 0xFFFF0000u);
  } else {
    asm("{\n\t.reg .f16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}"
        : "=f"(lo), "=f"(hi)
        : "r"(v));
  }
}
// Two values at a time: the epilogues are bound by instruction issue, and one instruction multiplies or adds both.
struct F2 {
  unsigned long long v;
  __device__ __forceinline__ F2() {}
  __device__ __forceinline__ F2(float lo, float hi) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi)); }
  __device__ __forceinline__ void get(float& lo, float& hi) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
};
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ uint32_t pack2(F2 a, bool bf16) {
  float lo, hi;
  a.get(lo, hi);
  return pack2(lo, hi, bf16);
}
__device__ __forceinline__ F2 as_f2(uint32_t lo, uint32_t hi) { return F2(__uint_as_float(lo), __uint_as_float(hi)); }
// 1 / (1 + 2^(-g log2 e)); an exponential that overflows gives 0.  The exponential is off by 2^-22 of itself and, for the
// rounding of its argument, by |g| 2^-23; the sum and the reciprocal by 2^-24 and 2^-23.
__device__ __forceinline__ F2 sigmoid(F2 g) {
  float lo, hi;
  (g * F2(-1.44269504f, -1.44269504f)).get(lo, hi);
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(lo));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(hi));
  lo += 1.0f;
  hi += 1.0f;
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(lo));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(hi));
  return F2(lo, hi);
}
__device__ __forceinline__ F2 gate(F2 g, F2 u) { return g * sigmoid(g) * u; }

// The projections g and u are kept for the backward pass in 24 bits, an fp32 number without its last eight (cut, so
// that a NaN stays one): in the 16 bits of the operands their rounding would be as large an error of dx and dw13 as the
// rounding of dg and du (relative error in bf16: 3.0e-3 instead of 2.4e-3).  The upper 16 bits of g and u lie in
// [T, 2I], the eight that follow of both in one word of [T, I].
__device__ __forceinline__ uint32_t upper16(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7632); }
__device__ __forceinline__ uint32_t next8(uint32_t g0, uint32_t u0, uint32_t g1, uint32_t u1) {
  return __byte_perm(__byte_perm(g0, u0, 0x0051), __byte_perm(g1, u1, 0x0051), 0x5410);
}
// Two neighbouring values from a word of upper halves and a word of lower bytes (which = 0: g, 1: u); the last eight
// bits are of no consequence.
template <int which>
__device__ __forceinline__ F2 from24(uint32_t upper, uint32_t lower) {
  return as_f2(__byte_perm(upper, lower, which ? 0x1055 : 0x1044), __byte_perm(upper, lower, which ? 0x3277 : 0x3266));
}

// Eight columns of a row: the activation from both projections, what is kept of them, and their gradients from dh.
template <bool BF16>
__device__ __forceinline__ uint4 gate8(const uint32_t* g, const uint32_t* u) {
  uint32_t h[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) h[q] = pack2(gate(as_f2(g[2 * q], g[2 * q + 1]), as_f2(u[2 * q], u[2 * q + 1])), BF16);
  return make_uint4(h[0], h[1], h[2], h[3]);
}
__device__ __forceinline__ void keep8(const uint32_t* g, const uint32_t* u, uint4& upper_g, uint4& upper_u, uint4& lower) {
  upper_g = make_uint4(upper16(g[0], g[1]), upper16(g[2], g[3]), upper16(g[4], g[5]), upper16(g[6], g[7]));
  upper_u = make_uint4(upper16(u[0], u[1]), upper16(u[2], u[3]), upper16(u[4], u[5]), upper16(u[6], u[7]));
  lower = make_uint4(next8(g[0], u[0], g[1], u[1]), next8(g[2], u[2], g[3], u[3]), next8(g[4], u[4], g[5], u[5]),
                     next8(g[6], u[6], g[7], u[7]));
}
template <bool BF16>
__device__ __forceinline__ void gradient8(uint4 upper_g, uint4 upper_u, uint4 lower, const uint32_t* d, uint4& grad_g,
                                          uint4& grad_u) {
  const uint32_t gw[4] = {upper_g.x, upper_g.y, upper_g.z, upper_g.w}, uw[4] = {upper_u.x, upper_u.y, upper_u.z, upper_u.w};
  const uint32_t lw[4] = {lower.x, lower.y, lower.z, lower.w};
  uint32_t dg[4], du[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const F2 g = from24<0>(gw[q], lw[q]), u = from24<1>(uw[q], lw[q]);
    const F2 dh = as_f2(d[2 * q], d[2 * q + 1]);
    const F2 sg = sigmoid(g), silu = g * sg;
    // silu' = s + g s (1 - s)
    const F2 slope = fma2(silu, fma2(sg, F2(-1.0f, -1.0f), F2(1.0f, 1.0f)), sg);
    dg[q] = pack2(dh * u * slope, BF16);
    du[q] = pack2(dh * silu, BF16);
  }
  grad_g = make_uint4(dg[0], dg[1], dg[2], dg[3]);
  grad_u = make_uint4(du[0], du[1], du[2], du[3]);
}

// -------------------------------------------------------------- pair kernel
// A pair of CTAs works on D[256 x tile_n] tiles: CTA r holds rows [128 r, 128 r + 128) of A, of D, and half of the
// rows of B (gated: CTA 0 the gate projection's, CTA 1 the up projection's, so that D holds tile_n / 2 columns of
// each), and the even CTA issues MMAs of 256 x tile_n x 16 (64 for 4-bit operands) that read both.  With tile_n = 256
// 32 KB per stage and CTA (64 k of 16-bit operands, 256 k of 4-bit ones) serve 512 cycles of MMA, which is what one
// CTA's tile of 128 x 256 needs 48 KB for.  Two rules make it fit few tiles (MakePairPlan): a smaller tile_n, and a
// cluster of two or four pairs that share the k axis of a tile and add their partial sums through shared memory.
constexpr int kPairThreads = 384;
constexpr int kStageOperand = 16384;  // 128 rows of 128 bytes
constexpr int kScaleBlock = 512;      // scales of 128 rows and 128 k

template <bool MX4, int EPI>
struct PairShape {
  // Results leave through shared memory in boxes of 32 rows of 128 bytes (boxes of half the width took twice the
  // time: the copy engine works by rows), two per epilogue warp.  Fewer stages for more boxes did not pay: with four
  // stages the 4096 x 6144 x 2048 gated product took 162 us instead of 149.
  static constexpr int kBoxes = MX4 ? 1 : 2;
  static constexpr int kStaging = kBoxes * 4096;
  static constexpr int kStages = 5;
  static constexpr int kAccs = MX4 ? 1 : 2;  // 256 columns each; 4-bit operands' scales need columns too
  static constexpr int kScales = MX4 ? 6 * kScaleBlock : 0;  // per stage: A 2 blocks, B 4
  static constexpr int kBarriers = 256 + FDMOE_PAIR_LIST * 4;  // and the list of tiles
  static constexpr int kSmem =
      kStages * (2 * kStageOperand + kScales) + 8 * kStaging + kBarriers + 1024;  // 1024: alignment of the base
  static_assert(kSmem > 196 * 1024, "takes all columns of an SM's TMEM: no other kernel that takes some may fit beside it");
};

struct PairTile {
  int m, n;
};
// Tiles in groups of eight row tiles, so that the tiles in flight share operands in L2.
__device__ __forceinline__ PairTile pair_tile(int tile, int tiles_m, int tiles_n) {
  const int per_group = 8 * tiles_n, g = tile / per_group, r = tile - g * per_group;
  const int rows = min(8, tiles_m - g * 8);
  return {g * 8 + r % rows, r / rows};
}

// Writes 16 bytes (chunk `j` of eight) of a row of a box of 32 rows of 128 bytes, in the 128-byte swizzle.
__device__ __forceinline__ void stage16(uint8_t* box, int lane, int j, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  *reinterpret_cast<uint4*>(box + lane * 128 + ((j ^ (lane & 7)) << 4)) = make_uint4(a, b, c, d);
}

template <bool MX4, int EPI, bool BF16>
__global__ void __launch_bounds__(kPairThreads, 1) pair_gemm(const __grid_constant__ FdmoePairParams p) {
  using S = PairShape<MX4, EPI>;
  constexpr bool kGated = EPI == FDMOE_EPI_GATED || EPI == FDMOE_EPI_GATED_SAVE || EPI == FDMOE_EPI_GATED_F32;
  constexpr bool kF32 = EPI == FDMOE_EPI_F32 || EPI == FDMOE_EPI_GATED_F32;
  constexpr bool kMany = !MX4 && EPI == FDMOE_EPI_HALF;  // launches may have several products
  constexpr int kAccCols = 256;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (ptx::smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t* stages = smem;
  uint8_t* scales = stages + S::kStages * 2 * kStageOperand;
  uint8_t* staging = scales + S::kStages * S::kScales;
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + 8 * S::kStaging);
  uint64_t* empty = full + S::kStages;
  uint64_t* acc_full = empty + S::kStages;
  uint64_t* acc_empty = acc_full + S::kAccs;
  uint64_t* gu_full = acc_empty + S::kAccs;  // gradient: one per epilogue warp
  uint64_t* sums_full = gu_full + 8;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sums_full + 1);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  uint32_t* list = tmem_slot + 2;  // [0]: how many; product << 28 | tile

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // A cluster is `split` pairs, which share the k axis of a tile.
  const uint32_t cta = ptx::cluster_rank(), rank = cta & 1, leader = cta & ~1u, part = cta >> 1;
  const int split = p.split;
  const int shift = split >> 1;  // log2
  const int first = blockIdx.x >> (1 + shift), step = gridDim.x >> (1 + shift);
  const Waiter wt{abort_flag, p.status, p.timeout_ns};

  // What comes before the first load is a fixed cost of every launch, and most of it is the fetching of instructions
  // that run once: barriers are set up by the lanes of a warp, and the first tile is looked up (its divisions) while
  // another warp waits for the tensor memory.
  if (warp == 1) {
    constexpr int kEmptyAcc = 2 * S::kStages + S::kAccs, kCount = kEmptyAcc + S::kAccs + 8 + 1;
    static_assert(kCount <= 32, "one barrier per lane");
    // an accumulator is given back by the epilogue warps of both CTAs
    if (lane < kCount) ptx::mbar_init(full + lane, lane >= kEmptyAcc && lane < kEmptyAcc + S::kAccs ? 16 : 1);
    if (lane == 0) *abort_flag = 0;
    ptx::fence_mbar_init();
    __syncwarp();
    if (lane == 0 && split > 1)
      ptx::mbar_expect_tx(sums_full, (p.product[0].tile_n * 512 >> shift) * (split - 1));  // the other pairs'
  }
  if (warp == 0 && ptx::elect_one()) {
    ptx::prefetch_tmap(&p.product[0].a);
    ptx::prefetch_tmap(&p.product[0].b);
  }
  if (warp == 2) {
    ptx::tmem_alloc_pair(tmem_slot, 512);
    ptx::tmem_relinquish_pair();
  }
  if constexpr (kMany) {
    // The tiles of several products in this pair's order: rounds over the pairs, each taking part as long as it has
    // tiles of the product left, so that the tiles in work at a time are neighbours.
    if (warp == 3 && p.products > 1) {
      uint32_t n = 0;
      for (int g = 0; g < p.products; ++g) {
        uint32_t have[FDMOE_PAIR_MOST / 32], tile = 0;
#pragma unroll
        for (int i = 0; i < FDMOE_PAIR_MOST / 32; ++i) have[i] = i * 32 + lane < step ? p.count[g][i * 32 + lane] : 0;
        for (uint32_t r = 0; r < p.count[g][first]; ++r) {
          uint32_t before = 0, all = 0;
#pragma unroll
          for (int i = 0; i < FDMOE_PAIR_MOST / 32; ++i) {
            const uint32_t in = __ballot_sync(0xffffffffu, have[i] > r);
            all += __popc(in);
            if (first >= i * 32) before += __popc(first >= i * 32 + 32 ? in : in & ((1u << (first - i * 32)) - 1u));
          }
          if (lane == 0 && n < FDMOE_PAIR_LIST - 3) list[1 + n] = (uint32_t)g << 28 | (tile + before);
          tile += all;
          ++n;
        }
      }
      if (lane == 0) list[0] = min(n, (uint32_t)FDMOE_PAIR_LIST - 3);
    }
  }
  // The i-th tile of this pair (cluster) and its product.
  const auto tile_at = [&](int i, int& g, PairTile& t) {
    g = 0;
    int tile = first + i * step;
    if (kMany && p.products > 1) {
      if (i >= (int)list[0]) return false;
      g = list[1 + i] >> 28;
      tile = list[1 + i] & 0x0FFFFFFF;
    } else if (tile >= p.product[0].tiles_m * p.product[0].tiles_n) {
      return false;
    }
    t = pair_tile(tile, p.product[g].tiles_m, p.product[g].tiles_n);
    return true;
  };
  int g;
  PairTile t;
  const bool listed = kMany && p.products > 1;
  bool have = !listed && tile_at(0, g, t);
  ptx::tcgen05_fence_before();
  __syncthreads();
  ptx::cluster_sync_relaxed();  // all CTAs' barriers are set up
  ptx::tcgen05_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (listed) have = tile_at(0, g, t);
  ptx::grid_wait_dependency();  // nothing of global memory is touched before this
  ptx::grid_launch_dependents();

  if (warp == 0) {
    // ---- loads: both CTAs fill their own stages; the bytes are counted on the even CTA's barriers
    {
      const bool elected = ptx::elect_one();
      int stage = 0;
      uint32_t parity = 1;
      bool ok = true;
      for (int i = 0; have; have = tile_at(++i, g, t)) {
        const FdmoePairProduct& pr = p.product[g];
        const int half_n = pr.tile_n >> 1;  // rows of B per CTA; gated: columns of each projection
        const int kb0 = pr.kblocks * (int)part >> shift, kb1 = pr.kblocks * ((int)part + 1) >> shift;
        // rows along N come in boxes of 64, the second of which may be used in part
        const uint32_t b_bytes = pr.b_mn && half_n > 64 ? kStageOperand : half_n * 128;
        const int ax = t.m * 256 + (int)rank * 128;
        const int bx = kGated ? t.n * half_n + (int)rank * p.up_row : t.n * pr.tile_n + (int)rank * half_n;
        for (int kb = kb0; kb < kb1; ++kb) {
          const int s = stage;
          ok = wt.wait_together(empty + s, parity, FDMOE_DENSE_TIMEOUT_EMPTY, ok);
          if (++stage == S::kStages) stage = 0, parity ^= 1;
          if (!ok || p.stall || !elected) continue;
          if (rank == 0) ptx::mbar_expect_tx(full + s, 2 * (kStageOperand + b_bytes + S::kScales));
          const uint32_t bar = ptx::map_rank(ptx::smem_u32(full + s), leader);
          const uint32_t sa = ptx::smem_u32(stages + s * 2 * kStageOperand), sb = sa + kStageOperand;
          if (MX4) {
            // 128 bytes of a row are 256 elements
            ptx::tma_load_2d_pair(sa, &pr.a, bar, kb * 128, ax);
            ptx::tma_load_2d_pair(sb, &pr.b, bar, kb * 128, bx);
            const uint32_t sf = ptx::smem_u32(scales + s * S::kScales);
            ptx::tma_load_2d_pair(sf, &p.sfa, bar, 0, (t.m * 2 + (int)rank) * p.sf_chunks + kb * 2);
            // both CTAs need the scales of all 256 rows of B
            const int b0 = kGated ? t.n : t.n * 2, b1 = kGated ? p.sf_up_block + t.n : t.n * 2 + 1;
            ptx::tma_load_2d_pair(sf + 2 * kScaleBlock, &p.sfb, bar, 0, b0 * p.sf_chunks + kb * 2);
            ptx::tma_load_2d_pair(sf + 4 * kScaleBlock, &p.sfb, bar, 0, b1 * p.sf_chunks + kb * 2);
          } else {
            if (pr.a_mn) {
              ptx::tma_load_2d_pair(sa, &pr.a, bar, ax, kb * 64);
              ptx::tma_load_2d_pair(sa + 8192, &pr.a, bar, ax + 64, kb * 64);
            } else {
              ptx::tma_load_2d_pair(sa, &pr.a, bar, kb * 64, ax);
            }
            if (pr.b_mn) {
              ptx::tma_load_2d_pair(sb, &pr.b, bar, bx, kb * 64);
              if (half_n > 64) ptx::tma_load_2d_pair(sb + 8192, &pr.b, bar, bx + 64, kb * 64);
            } else {
              ptx::tma_load_2d_pair(sb, &pr.b, bar, kb * 64, bx);
            }
          }
        }
      }
    }
  } else if (warp == 1) {
    // ---- MMAs: one thread of the even CTA
    if (rank == 0) {
      const bool elected = ptx::elect_one();
      int stage = 0;
      uint32_t parity = 0;
      bool ok = true;
      for (int n = 0; have; have = tile_at(++n, g, t)) {
        const FdmoePairProduct& pr = p.product[g];
        const int kb0 = pr.kblocks * (int)part >> shift, kb1 = pr.kblocks * ((int)part + 1) >> shift;
        const uint32_t idesc = ptx::make_idesc_f16(256, pr.tile_n, BF16, pr.a_mn, pr.b_mn);
        // 16 k further: 32 bytes along a row, or 16 rows of 128 bytes
        const uint32_t a_step = pr.a_mn ? 2048 >> 4 : 32 >> 4, b_step = pr.b_mn ? 2048 >> 4 : 32 >> 4;
        const uint32_t a_lead = pr.a_mn ? 8192 : 16, b_lead = pr.b_mn ? 8192 : 16;
        const int acc = n % S::kAccs;
        const uint32_t aph = (n / S::kAccs) & 1;
        ok = wt.wait_together(acc_empty + acc, aph ^ 1, FDMOE_DENSE_TIMEOUT_ACC, ok);
        ptx::tcgen05_fence_after();
        const uint32_t d = tmem + acc * kAccCols;
        for (int kb = kb0; kb < kb1; ++kb) {
          const int s = stage;
          ok = wt.wait_together(full + s, parity, FDMOE_DENSE_TIMEOUT_FULL, ok);
          if (++stage == S::kStages) stage = 0, parity ^= 1;
          ptx::tcgen05_fence_after();
          if (!ok || !elected) continue;
          const uint32_t sa = ptx::smem_u32(stages + s * 2 * kStageOperand), sb = sa + kStageOperand;
          if (MX4) {
            const uint32_t sf = ptx::smem_u32(scales + s * S::kScales);
            // scales have TMEM columns of their own per stage: A 2 x 4, B 2 x 8 (k block, row block)
            const uint32_t ta = tmem + kAccCols + s * 24, tb = ta + 8;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              ptx::tmem_copy_scales_pair(ta + c * 4, ptx::smem_desc_scales(sf + c * kScaleBlock));
              ptx::tmem_copy_scales_pair(tb + c * 8, ptx::smem_desc_scales(sf + (2 + c) * kScaleBlock));
              ptx::tmem_copy_scales_pair(tb + c * 8 + 4, ptx::smem_desc_scales(sf + (4 + c) * kScaleBlock));
            }
            const uint64_t da = ptx::smem_desc_sw128(sa, 16), db = ptx::smem_desc_sw128(sb, 16);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              ptx::umma_mx4_pair(d, da + k * 2, db + k * 2, ptx::make_idesc_mx4(256, 256, (k & 1) * 2),
                                 ta + (k >> 1) * 4, tb + (k >> 1) * 8, kb != kb0 || k != 0);
          } else {
            const uint64_t da = ptx::smem_desc_sw128(sa, a_lead), db = ptx::smem_desc_sw128(sb, b_lead);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              ptx::umma_f16_pair(d, da + k * a_step, db + k * b_step, idesc, kb != kb0 || k != 0);
          }
          ptx::umma_commit_pair(empty + s, leader);
        }
        if (ok && elected) ptx::umma_commit_pair(acc_full + acc, leader);
      }
    }
  } else if (warp >= 4) {
    // ---- epilogue: warps w and w + 4 read the same 32 lanes and take turns with the groups of columns
    const bool elected = ptx::elect_one();
    const int w = warp - 4, quad = warp & 3;
    uint8_t* buf = staging + w * S::kStaging;
    const uint32_t sbuf = ptx::smem_u32(buf);
    // Box i: 32 rows (quarter i & 3 of the CTA's, which are the warp's own lanes) of a group of columns (i >> 2).
    constexpr int kGroup = kF32 ? 32 : 64;
    constexpr int kMost = (kGated ? 128 : 256) / kGroup / 2;  // boxes of a warp
    const auto box_at = [&](int j) { return w + 8 * j; };
    // Gradient: the boxes first take the upper halves of g and u of a group of columns, which dg and du then replace;
    // the lower bytes of this lane's row come straight into registers.
    uint32_t gu_count = 0;
    uint4 lower[8];
    auto fetch_gu = [&](const PairTile& t, int box) {
      const FdmoePairProduct& pr = p.product[0];
      const int y = t.m * 256 + (int)rank * 128 + (box & 3) * 32, x = t.n * pr.tile_n + (box >> 2) * 64;
      const int row = y + lane, col = x;
      const uint16_t* at = static_cast<const uint16_t*>(p.lower) + (int64_t)row * pr.cols + col;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        lower[j] = row < pr.rows && col + 8 * j < pr.cols ? ptx::ld_global_u32x4(at + 8 * j) : make_uint4(0, 0, 0, 0);
      if (elected) {
        ptx::bulk_wait_group_read0();
        ptx::mbar_expect_tx(gu_full + w, 8192);
        ptx::tma_load_2d(buf, &p.gu[0], gu_full + w, x, y);
        ptx::tma_load_2d(buf + 4096, &p.gu[1], gu_full + w, x, y);
      }
    };
    for (int n = 0; have; have = tile_at(++n, g, t)) {
      const FdmoePairProduct& pr = p.product[g];
      const int half_n = pr.tile_n >> 1, tile_cols = kGated ? half_n : pr.tile_n, boxes = tile_cols / kGroup * 4;
      const int acc = n % S::kAccs;
      if constexpr (EPI == FDMOE_EPI_GATED_GRAD)
        if (split == 1 && box_at(0) < boxes) fetch_gu(t, box_at(0));
      const bool done = wt.wait_warp(acc_full + acc, (n / S::kAccs) & 1, FDMOE_DENSE_TIMEOUT_DONE);
      ptx::tcgen05_fence_after();
      const uint32_t d = tmem + acc * kAccCols + (uint32_t(quad * 32) << 16);
      const int tile_row = t.m * 256 + (int)rank * 128;
      const int col0 = t.n * tile_cols;
      if (split > 1) {
        // The k axis is shared, and this is the cluster's only tile.  Every pair stores its partial sums of a box into
        // the shared memory of the box's owner, [box of the owner][pair][part][column / 4][row][4], where the stages
        // were: all MMAs have read theirs once every CTA has arrived at the cluster's barrier.
        constexpr int kParts = kGated ? 2 : 1, kBoxSums = kGroup * 128;  // bytes
        // Each of the owner's eight warps then adds them, in the order of the pairs, for eight rows of a box at a time:
        // eight lanes write 128 bytes of a row (a lane per row took eight times the stores' cycles, and whole boxes
        // through the copy engine left most warps idle).  A row's place in its 512 bytes is turned by the eighth of
        // the box's columns, so that such lanes read from different banks.
        constexpr int kCols = kF32 ? 4 : 8;  // of a lane: 16 bytes of a result
        const int quarters = boxes >> shift << 2, eighth = lane & 7;
        int row, col;  // this lane's first row; the second is four further
        const auto place = [&](int i) {
          const int box = ((i >> 2) << shift) + (int)part;
          row = tile_row + (box & 3) * 32 + (i & 3) * 8 + (lane >> 3), col = col0 + (box >> 2) * kGroup + eighth * kCols;
        };
        uint4 gu[3][2];
        const auto fetch = [&](int i) {  // gradient: g, u and their lower bytes
          place(i);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const bool in = i < quarters && row + 4 * k < pr.rows && col < pr.cols;
            const int64_t at = (int64_t)(row + 4 * k) * pr.cols, at2 = 2 * at + col;
            gu[0][k] = in ? ptx::ld_global_u32x4(static_cast<const uint16_t*>(p.from[0]) + at2) : uint4();
            gu[1][k] = in ? ptx::ld_global_u32x4(static_cast<const uint16_t*>(p.from[1]) + at2) : uint4();
            gu[2][k] = in ? ptx::ld_global_u32x4(static_cast<const uint16_t*>(p.lower) + at + col) : uint4();
          }
        };
        if constexpr (EPI == FDMOE_EPI_GATED_GRAD) fetch(w);
        ptx::cluster_sync_relaxed();
        if (done)
          for (int c = w >> 2; c < pr.tile_n >> 5; c += 2) {
            uint32_t v[32];
            ptx::tmem_ld_32x32(d + c * 32, v);
            const int q = kGated && c * 32 >= half_n, column = c * 32 - q * half_n, box = column / kGroup * 4 + quad;
            const uint32_t owner = box & (split - 1);
            const uint32_t at = (((box >> shift << shift) + part) * kParts + q) * kBoxSums + (column % kGroup) * 128;
            const uint32_t to = ptx::map_rank(ptx::smem_u32(stages) + at, 2 * owner + rank);
            const uint32_t bar = ptx::map_rank(ptx::smem_u32(sums_full), 2 * owner + rank);
            ptx::tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const uint32_t on = j * 512 + (lane ^ (kF32 ? j : (column % kGroup) / 8 + j / 2)) * 16;
              if (owner == part)
                *reinterpret_cast<uint4*>(stages + at + on) = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
              else
                ptx::st_async_u32x4(to + on, v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3], bar);
            }
          }
        ptx::epilogue_sync();
        if (!done || !wt.wait_warp(sums_full, 0, FDMOE_DENSE_TIMEOUT_DONE)) break;
        for (int i = w; i < quarters; i += 8) {
          if (EPI == FDMOE_EPI_GATED_GRAD && i != w) fetch(i);
          place(i);
          uint32_t v[kParts][2][kCols];
          const uint32_t from = ptx::smem_u32(stages) + ((i >> 2) << shift) * kParts * kBoxSums + eighth * kCols * 128;
          const int turned = ((i & 3) * 8 + (lane >> 3)) ^ eighth;  // the second row, four further: bit 2 the other way
          for (int r = 0; r < split; ++r)
#pragma unroll
            for (int q = 0; q < kParts; ++q)
#pragma unroll
              for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int j = 0; j < kCols; j += 4) {
                  const float4 f =
                      ptx::ld_shared_f32x4(from + (r * kParts + q) * kBoxSums + j * 128 + (turned ^ (4 * k)) * 16);
                  const float add[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
                  for (int e = 0; e < 4; ++e)
                    v[q][k][j + e] = __float_as_uint(r == 0 ? add[e] : __uint_as_float(v[q][k][j + e]) + add[e]);
                }
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint32_t* const v0 = v[0][k];
            const uint32_t* const v1 = v[kParts - 1][k];
            const auto put = [&](void* to, int width, uint4 x) {  // 16 bytes; `to` has `width` times the columns
              const int64_t at = (int64_t)(row + 4 * k) * pr.cols * width + col;
              if (row + 4 * k < pr.rows && col < pr.cols)
                *reinterpret_cast<uint4*>(static_cast<uint8_t*>(to) + at * (kF32 ? 4 : 2)) = x;
            };
            if constexpr (kF32) {
              float y[4];
#pragma unroll
              for (int e = 0; e < 4; e += 2) {
                const F2 a = as_f2(v0[e], v0[e + 1]);
                (kGated ? gate(a, as_f2(v1[e], v1[e + 1])) : a).get(y[e], y[e + 1]);
              }
              put(p.to[0], 1, make_uint4(__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]),
                                         __float_as_uint(y[3])));
            } else if constexpr (kGated) {
              put(p.to[0], 1, gate8<BF16>(v0, v1));
              if constexpr (EPI == FDMOE_EPI_GATED_SAVE) {
                uint4 x[3];
                keep8(v0, v1, x[0], x[1], x[2]);
                put(p.to[1], 2, x[0]);
                put(p.to[2], 2, x[1]);
                put(p.lower, 1, x[2]);
              }
            } else if constexpr (EPI == FDMOE_EPI_GATED_GRAD) {
              uint4 x[2];
              gradient8<BF16>(gu[0][k], gu[1][k], gu[2][k], v0, x[0], x[1]);
              put(p.to[0], 2, x[0]);
              put(p.to[1], 2, x[1]);
            } else {
              uint32_t h[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) h[e] = pack2(as_f2(v0[2 * e], v0[2 * e + 1]), BF16);
              put(p.to[0], 1, make_uint4(h[0], h[1], h[2], h[3]));
            }
          }
        }
        break;
      }
      if (!done) break;
      // 32 columns (from `column` of part q on) of a box from the accumulator
      auto load = [&](int box, int q, int column, uint32_t (&v)[32]) {
        ptx::tmem_ld_32x32(d + q * half_n + (box >> 2) * kGroup + column, v);
      };
      auto release = [&]() {  // this warp has read its part of the accumulator
        ptx::tcgen05_fence_before();
        __syncwarp();
        if (elected) ptx::mbar_arrive_cluster(ptx::map_rank(ptx::smem_u32(acc_empty + acc), leader));
      };
      // Waits until this warp's boxes may be written again (its last stores have read them).
      auto boxes_free = [&]() {
        if (elected) ptx::bulk_wait_group_read0();
        __syncwarp();
      };
      auto boxes_written = [&]() {
        ptx::fence_proxy_async_shared();
        __syncwarp();
      };
      // Sends buffer b, which all lanes have written, to where `box` lies in result `map`.
      auto send = [&](int map, int b, int box) {
        const int row = tile_row + (box & 3) * 32, col = col0 + (box >> 2) * kGroup;
        if (elected && row < pr.rows && col < pr.cols) ptx::tma_store_2d(&pr.out[map], sbuf + b * 4096, col, row);
      };
      if constexpr (EPI == FDMOE_EPI_HALF) {
        // All of the warp's columns are read, rounded and the accumulator given back before the first is stored.
        uint32_t w[kMost][32];
#pragma unroll
        for (int j = 0; j < kMost; ++j) {
          const int box = box_at(j);
          if (box >= boxes) break;
          uint32_t v[2][32];
          load(box, 0, 0, v[0]);
          load(box, 0, 32, v[1]);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) w[j][i] = pack2(as_f2(v[i >> 4][(2 * i) & 31], v[i >> 4][(2 * i + 1) & 31]), BF16);
        }
        release();
        if constexpr (S::kBoxes >= kMost) boxes_free();
#pragma unroll
        for (int j = 0; j < kMost; ++j) {
          const int box = box_at(j), b = S::kBoxes >= kMost ? j : 0;
          if (box >= boxes) break;
          if constexpr (S::kBoxes < kMost) boxes_free();
#pragma unroll
          for (int i = 0; i < 8; ++i)
            stage16(buf + b * 4096, lane, i, w[j][4 * i], w[j][4 * i + 1], w[j][4 * i + 2], w[j][4 * i + 3]);
          boxes_written();
          send(0, b, box);
          if (elected) ptx::bulk_commit_group();
        }
      } else if constexpr (EPI == FDMOE_EPI_F32) {
        uint32_t v[kMost][32];
#pragma unroll
        for (int j = 0; j < kMost; ++j)
          if (box_at(j) < boxes) load(box_at(j), 0, 0, v[j]);
        ptx::tmem_ld_wait();
        release();
#pragma unroll
        for (int j = 0; j < kMost; ++j) {
          const int box = box_at(j);
          if (box >= boxes) break;
          boxes_free();
#pragma unroll
          for (int i = 0; i < 8; ++i) stage16(buf, lane, i, v[j][4 * i], v[j][4 * i + 1], v[j][4 * i + 2], v[j][4 * i + 3]);
          boxes_written();
          send(0, 0, box);
          if (elected) ptx::bulk_commit_group();
        }
      } else if constexpr (EPI == FDMOE_EPI_GATED_F32) {
        uint32_t g[kMost][32], u[kMost][32];
#pragma unroll
        for (int j = 0; j < kMost; ++j)
          if (box_at(j) < boxes) {
            load(box_at(j), 0, 0, g[j]);
            load(box_at(j), 1, 0, u[j]);
          }
        ptx::tmem_ld_wait();
        release();
#pragma unroll
        for (int j = 0; j < kMost; ++j) {
          const int box = box_at(j);
          if (box >= boxes) break;
          boxes_free();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float y[4];
            gate(as_f2(g[j][4 * i], g[j][4 * i + 1]), as_f2(u[j][4 * i], u[j][4 * i + 1])).get(y[0], y[1]);
            gate(as_f2(g[j][4 * i + 2], g[j][4 * i + 3]), as_f2(u[j][4 * i + 2], u[j][4 * i + 3])).get(y[2], y[3]);
            stage16(buf, lane, i, __float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]),
                    __float_as_uint(y[3]));
          }
          boxes_written();
          send(0, 0, box);
          if (elected) ptx::bulk_commit_group();
        }
      } else if constexpr (kGated) {
        // One box of 64 columns, 32 at a time; 4-bit operands have one accumulator, which is given back before the
        // activation is computed.
        const int box = box_at(0);
        uint32_t g[MX4 ? 2 : 1][32], u[MX4 ? 2 : 1][32];
        if (MX4 && box < boxes) {
#pragma unroll
          for (int i = 0; i < (MX4 ? 2 : 1); ++i) {
            load(box, 0, i * 32, g[i]);
            load(box, 1, i * 32, u[i]);
          }
        }
        if constexpr (MX4) {
          ptx::tmem_ld_wait();
          release();
        }
        if (box < boxes) {
          boxes_free();
          uint32_t up[EPI == FDMOE_EPI_GATED_SAVE ? 32 : 1];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t(&gi)[32] = g[MX4 ? i : 0];
            uint32_t(&ui)[32] = u[MX4 ? i : 0];
            if constexpr (!MX4) {
              load(box, 0, i * 32, gi);
              load(box, 1, i * 32, ui);
              ptx::tmem_ld_wait();
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {  // eight columns
              const uint4 h = gate8<BF16>(gi + 8 * j, ui + 8 * j);
              stage16(buf, lane, i * 4 + j, h.x, h.y, h.z, h.w);
              if constexpr (EPI == FDMOE_EPI_GATED_SAVE) {
                uint4 upper_g, upper_u, lower;
                keep8(gi + 8 * j, ui + 8 * j, upper_g, upper_u, lower);
                stage16(buf + 4096, lane, i * 4 + j, upper_g.x, upper_g.y, upper_g.z, upper_g.w);
                up[16 * i + 4 * j] = upper_u.x, up[16 * i + 4 * j + 1] = upper_u.y;
                up[16 * i + 4 * j + 2] = upper_u.z, up[16 * i + 4 * j + 3] = upper_u.w;
                const int row = tile_row + (box & 3) * 32 + lane;
                const int col = col0 + (box >> 2) * 64 + i * 32 + j * 8;  // columns come in eights
                if (row < pr.rows && col < pr.cols)
                  *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.lower) + (int64_t)row * pr.cols + col) = lower;
              }
            }
          }
          if constexpr (!MX4) release();
          boxes_written();
          send(0, 0, box);
          if constexpr (EPI == FDMOE_EPI_GATED_SAVE) {
            if (elected) ptx::bulk_commit_group();
            send(1, 1, box);
            if (elected) {
              ptx::bulk_commit_group();
              ptx::bulk_wait_group_read1();  // h has left
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i) stage16(buf, lane, i, up[4 * i], up[4 * i + 1], up[4 * i + 2], up[4 * i + 3]);
            boxes_written();
            send(2, 0, box);
          }
          if (elected) ptx::bulk_commit_group();
        } else if constexpr (!MX4) {
          release();
        }
      } else {
#pragma unroll 1
        for (int n = 0; n < kMost; ++n) {
          const int box = box_at(n);
          if (box >= boxes) break;
          if (n > 0) fetch_gu(t, box);
          wt.wait_warp(gu_full + w, gu_count++ & 1, FDMOE_DENSE_TIMEOUT_FULL);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t v[32];
            load(box, 0, i * 32, v);
            ptx::tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 4; ++j) {  // eight columns
              uint4* const g_at = reinterpret_cast<uint4*>(buf + lane * 128 + (((i * 4 + j) ^ (lane & 7)) << 4));
              uint4* const u_at = g_at + 4096 / 16;
              uint4 dg, du;
              gradient8<BF16>(*g_at, *u_at, lower[i * 4 + j], v + 8 * j, dg, du);
              *g_at = dg;
              *u_at = du;
            }
          }
          boxes_written();
          send(0, 0, box);
          send(1, 1, box);
          if (elected) ptx::bulk_commit_group();
        }
        release();
      }
    }
    if (elected) ptx::bulk_wait_group_read0();  // the boxes stay until they have been read
  }
  __syncwarp();
  if (warp < 4 && split > 1) ptx::cluster_sync_relaxed();  // the epilogue warps' exchange of partial sums
  ptx::tcgen05_fence_before();
  __syncthreads();
  wt.drain();
  ptx::cluster_sync_relaxed();  // neither CTA leaves while the other may still read its operands or arrive on its barriers
  ptx::tcgen05_fence_after();
  if (warp == 2) ptx::tmem_dealloc_pair(tmem, 512);
}

// ------------------------------------------------------------ stream kernel
// One CTA: D[128 weight rows x tile_tokens] (gated: two such accumulators, gate and up) over its part of the k axis.
// The cluster's partial sums meet in shared memory: CTA r adds those of every split-th group of four tokens.
constexpr int kStreamThreads = 320;  // 8 epilogue warps (4 took 10 % longer at 96 tokens of 2048 x 6144), loads, MMAs
constexpr int kStreamLoads = 8, kStreamMmas = 9;  // their warps

template <bool MX4, int EPI>
__global__ void __launch_bounds__(kStreamThreads) stream_gemm(const __grid_constant__ FdmoeStreamParams p) {
  constexpr bool kGated = EPI == FDMOE_EPI_GATED || EPI == FDMOE_EPI_GATED_F32;
  constexpr int kParts = kGated ? 2 : 1;
  constexpr int kScales = MX4 ? (kParts + 1) * 2 * kScaleBlock : 0;
  static_assert(!MX4 || FDMOE_STREAM_TOKENS_MX4 == 128, "each of several tiles of tokens is a block of scales");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (ptx::smem_u32(smem_raw) & 1023)) & 1023);
  const int nt = p.tile_tokens;
  const uint32_t stage_bytes = kParts * kStageOperand + nt * 128 + kScales;  // a multiple of 1024: nt of 16
  __shared__ uint64_t full[FDMOE_STREAM_STAGES], empty[FDMOE_STREAM_STAGES], acc_full, sums_full;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile uint32_t abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x;  // in the cluster (split, 1, 1)
  const int row0 = blockIdx.y * FDMOE_STREAM_ROWS, tok0 = blockIdx.z * nt;
  const int kb0 = rank * p.kblocks_each + min(rank, p.kblocks_more);
  const int kb1 = kb0 + p.kblocks_each + (rank < p.kblocks_more);
  const Waiter wt{&abort_flag, p.status, p.timeout_ns};

  // The first loads need no more than their barriers: they are on their way before the CTA's other warps are ready.
  const int filled = min(p.stages, kb1 - kb0);
  const bool elected = ptx::elect_one();
  auto load_weights = [&](int s, int kb) {
    uint64_t* bar = full + s;
    uint8_t* sa = smem + s * stage_bytes;
    uint8_t* sf = sa + kParts * kStageOperand + nt * 128;
    ptx::mbar_expect_tx(bar, stage_bytes);
#pragma unroll
    for (int q = 0; q < kParts; ++q) {
      ptx::tma_load_2d(sa + q * kStageOperand, &p.a, bar, kb * (MX4 ? 128 : 64), row0 + q * p.up_row);
      if (MX4)
        ptx::tma_load_2d(sf + q * 2 * kScaleBlock, &p.sfa, bar, 0,
                         ((int)blockIdx.y + q * p.sf_up_block) * p.sf_chunks + kb * 2);
    }
  };
  auto load_tokens = [&](int s, int kb) {
    uint8_t* sb = smem + s * stage_bytes + kParts * kStageOperand;
    ptx::tma_load_2d(sb, &p.b, full + s, kb * (MX4 ? 128 : 64), tok0);
    if (MX4) ptx::tma_load_2d(sb + nt * 128 + kParts * 2 * kScaleBlock, &p.sfb, full + s, 0,
                              (tok0 >> 7) * p.sf_chunks + kb * 2);
  };
  if (warp == kStreamLoads) {
    if (elected) {
      ptx::prefetch_tmap(&p.a);
      ptx::prefetch_tmap(&p.b);
    }
    if (lane < FDMOE_STREAM_STAGES) {
      ptx::mbar_init(full + lane, 1);
      ptx::mbar_init(empty + lane, 1);
    }
    ptx::fence_mbar_init();
    ptx::fence_proxy_async_shared();
    __syncwarp();
    // The weights may be read while the launch before this one still writes the tokens.
    if (p.early_weights && elected && !p.stall)
      for (int i = 0; i < filled; ++i) load_weights(i, kb0 + i);
    ptx::grid_wait_dependency();
    // Only now may the next launch start: what it reads early was written before this launch's predecessor ended.
    ptx::grid_launch_dependents();
    if (elected && !p.stall)
      for (int i = 0; i < filled; ++i) {
        if (!p.early_weights) load_weights(i, kb0 + i);
        load_tokens(i, kb0 + i);
      }
    __syncwarp();
  } else if (warp == kStreamMmas) {
    if (lane == 0) {
      ptx::mbar_init(&acc_full, 1);
      ptx::mbar_init(&sums_full, 1);
      abort_flag = 0;
      ptx::fence_mbar_init();
      // the partial sums of this CTA's groups of four tokens, from every other CTA of the cluster
      const int groups = (min(nt, p.tokens - tok0) + 3) >> 2;
      if (rank < groups && p.split > 1)
        ptx::mbar_expect_tx(&sums_full, (uint32_t)((groups - rank + p.split - 1) / p.split * (p.split - 1) * kParts * 2048));
    }
    __syncwarp();
  } else if (warp == 0) {
    ptx::tmem_alloc(&tmem_slot, p.tmem_cols);
    ptx::tmem_relinquish();
  }
  ptx::tcgen05_fence_before();
  __syncthreads();
  ptx::tcgen05_fence_after();
  const uint32_t tmem = tmem_slot;

  if (warp == kStreamLoads) {
    int s = 0;
    uint32_t parity = 0;
    bool ok = true;
    for (int kb = kb0 + filled; kb < kb1; ++kb) {
      ok = wt.wait_together(empty + s, parity, FDMOE_DENSE_TIMEOUT_EMPTY, ok);
      if (ok && elected && !p.stall) {
        load_weights(s, kb);
        load_tokens(s, kb);
      }
      if (++s == p.stages) s = 0, parity ^= 1;
    }
  } else if (warp == kStreamMmas) {
    {
      const uint32_t idesc = ptx::make_idesc_f16(128, nt, p.bf16, false, false);
      bool ok = true;
      uint32_t parity = 0;
      for (int i = 0, stage = 0; i < kb1 - kb0; ++i) {
        const int s = stage;
        ok = wt.wait_together(full + s, parity, FDMOE_DENSE_TIMEOUT_FULL, ok);
        if (++stage == p.stages) stage = 0, parity ^= 1;
        ptx::tcgen05_fence_after();
        if (!ok || !elected) continue;
        const uint32_t sa = ptx::smem_u32(smem + s * stage_bytes), sb = sa + kParts * kStageOperand;
        const uint64_t db = ptx::smem_desc_sw128(sb, 16);
        if (MX4) {
          const uint32_t sf = sb + nt * 128;
          const uint32_t tsf = tmem + kParts * nt + s * (kParts + 1) * 8;  // columns of this stage's scales
#pragma unroll
          for (int q = 0; q < 2 * (kParts + 1); ++q)
            ptx::tmem_copy_scales(tsf + q * 4, ptx::smem_desc_scales(sf + q * kScaleBlock));
          const uint32_t tsb = tsf + kParts * 8;  // a tile of tokens begins with a block of 128 rows of scales
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t id = ptx::make_idesc_mx4(128, nt, (k & 1) * 2);
#pragma unroll
            for (int q = 0; q < kParts; ++q)
              ptx::umma_mx4(tmem + q * nt, ptx::smem_desc_sw128(sa + q * kStageOperand, 16) + k * 2, db + k * 2, id,
                            tsf + q * 8 + (k >> 1) * 4, tsb + (k >> 1) * 4, (i | k) != 0);
          }
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int q = 0; q < kParts; ++q)
              ptx::umma_bf16(tmem + q * nt, ptx::smem_desc_sw128(sa + q * kStageOperand, 16) + k * 2, db + k * 2,
                             idesc, (i | k) != 0);
        }
        ptx::umma_commit(empty + s);
      }
      if (ok && elected) ptx::umma_commit(&acc_full);
    }
  } else {
    const int count = min(nt, p.tokens - tok0);
    // warps w and w + 4 read the same 32 lanes (rows) and take turns with the tokens
    const int quad = warp & 3, half = warp >> 2;
    const uint32_t d = tmem + (uint32_t(quad * 32) << 16);
    const int row = row0 + quad * 32 + lane;
    int owner = half * 4 % p.split, slot = half * 4 / p.split;  // of this warp's next group of tokens
    const int slots = (((count + 3) >> 2) - rank + p.split - 1) / p.split;  // groups that this CTA finishes
    const bool done = wt.wait_warp(&acc_full, 0, FDMOE_DENSE_TIMEOUT_DONE);
    ptx::tcgen05_fence_after();
    constexpr bool kF32 = EPI == FDMOE_EPI_F32 || EPI == FDMOE_EPI_GATED_F32;
    const bool even_ld = (p.ld & 1) == 0;
    // Four tokens' results of this row.  Several groups' are computed before the first is stored: one after the other
    // they took 800 cycles each, nearly all of it latency.
    auto results = [&](const float(&v)[kParts][4], float(&y)[4]) {
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        if constexpr (kGated)
          gate(F2(v[0][i], v[0][i + 1]), F2(v[1][i], v[1][i + 1])).get(y[i], y[i + 1]);
        else
          y[i] = v[0][i], y[i + 1] = v[0][i + 1];
      }
    };
    // Neighbouring lanes exchange two of the four, so that each stores two rows of two tokens.
    auto store = [&](int t, const float(&y)[4]) {
      const int64_t at = (int64_t)(tok0 + t) * p.ld;
      if constexpr (kF32) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (t + i < count && row < p.rows) static_cast<float*>(p.out)[at + i * p.ld + row] = y[i];
      } else {
        uint16_t* out = static_cast<uint16_t*>(p.out);
        const bool odd = lane & 1;
        const float a = __shfl_xor_sync(0xffffffffu, odd ? y[0] : y[2], 1);
        const float b = __shfl_xor_sync(0xffffffffu, odd ? y[1] : y[3], 1);
        const uint32_t w0 = odd ? pack2(a, y[2], p.bf16) : pack2(y[0], a, p.bf16);
        const uint32_t w1 = odd ? pack2(b, y[3], p.bf16) : pack2(y[1], b, p.bf16);
        const int r = row & ~1, i0 = odd ? 2 : 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (t + i0 + i >= count) break;
          const uint32_t w = i ? w1 : w0;
          uint16_t* o = out + at + (i0 + i) * p.ld + r;
          if (even_ld && r + 1 < p.rows) {
            *reinterpret_cast<uint32_t*>(o) = w;
          } else {
            if (r < p.rows) o[0] = static_cast<uint16_t>(w);
            if (r + 1 < p.rows) o[1] = static_cast<uint16_t>(w >> 16);
          }
        }
      }
    };
    if (p.split == 1) {
      if (done)
        for (int c = half * 16; c < count; c += 32) {
          uint32_t v[kParts][16];
#pragma unroll
          for (int q = 0; q < kParts; ++q) ptx::tmem_ld_32x16(d + q * nt + c, v[q]);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; i += 8) {
            if (c + i >= count) break;
            float y[2][4];
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              float f[kParts][4];
#pragma unroll
              for (int q = 0; q < kParts; ++q)
#pragma unroll
                for (int j = 0; j < 4; ++j) f[q][j] = __uint_as_float(v[q][i + 4 * g + j]);
              results(f, y[g]);
            }
            store(c + i, y[0]);
            store(c + i + 4, y[1]);
          }
        }
    } else {
      // Groups of four tokens are dealt out to the CTAs of the cluster.  Each CTA stores its partial sums of a group
      // into the owner's shared memory, [group of the owner][CTA][part][row][4 tokens], where the stages were: every
      // CTA's MMAs have read theirs once all have arrived at the cluster's barrier.  The bytes are counted on a barrier
      // of the owner, which a releasing and acquiring barrier of the cluster would take 900 cycles longer than.
      ptx::cluster_sync_relaxed();
      uint8_t* const own = smem + (quad * 32 + lane) * 16;
      const uint32_t mine = ptx::smem_u32(own);
      if (done)
        for (int c = half * 16; c < count; c += 32) {
          uint32_t v[kParts][16];
#pragma unroll
          for (int q = 0; q < kParts; ++q) ptx::tmem_ld_32x16(d + q * nt + c, v[q]);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            if (c + i < count) {
              const uint32_t at = (slot * p.split + rank) * kParts * 2048, to = ptx::map_rank(mine + at, owner);
              const uint32_t bar = ptx::map_rank(ptx::smem_u32(&sums_full), owner);
#pragma unroll
              for (int q = 0; q < kParts; ++q)
                if (owner == rank)
                  *reinterpret_cast<uint4*>(own + at + q * 2048) =
                      make_uint4(v[q][i], v[q][i + 1], v[q][i + 2], v[q][i + 3]);
                else
                  ptx::st_async_u32x4(to + q * 2048, v[q][i], v[q][i + 1], v[q][i + 2], v[q][i + 3], bar);
            }
            if (++owner == p.split) owner = 0, ++slot;
          }
          for (owner += 4; owner >= p.split; owner -= p.split) ++slot;  // the other warp's four groups
        }
      ptx::epilogue_sync();
      const bool have = slots > 0 && wt.wait_warp(&sums_full, 0, FDMOE_DENSE_TIMEOUT_DONE);
      auto finish = [&](auto groups, int slot) {
        constexpr int kGroups = decltype(groups)::value;
        float f[kGroups][kParts][4] = {}, y[kGroups][4];
#pragma unroll(4 / kGroups)
        for (int r = 0; r < p.split; ++r)
#pragma unroll
          for (int q = 0; q < kParts; ++q)
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
              const float4 v = *reinterpret_cast<const float4*>(own + (((slot + 2 * g) * p.split + r) * kParts + q) * 2048);
              f[g][q][0] += v.x;
              f[g][q][1] += v.y;
              f[g][q][2] += v.z;
              f[g][q][3] += v.w;
            }
#pragma unroll
        for (int g = 0; g < kGroups; ++g) results(f[g], y[g]);
#pragma unroll
        for (int g = 0; g < kGroups; ++g) store(((slot + 2 * g) * p.split + rank) * 4, y[g]);
      };
      slot = have ? half : slots;
      for (; slot + 2 < slots; slot += 4) finish(std::integral_constant<int, 2>(), slot);
      if (slot < slots) finish(std::integral_constant<int, 1>(), slot);
    }
  }
  __syncwarp();
  if (warp >= kStreamLoads && p.split > 1) ptx::cluster_sync_relaxed();
  ptx::tcgen05_fence_before();
  __syncthreads();
  // A CTA that has given up did not wait for the others' partial sums, which may still be on their way here: it stays
  // until every CTA of the cluster has ended (exited threads count as arrived) or has given up too.
  if (p.split > 1 && abort_flag) ptx::cluster_sync_relaxed();
  wt.drain();
  ptx::tcgen05_fence_after();
  if (warp == 0) ptx::tmem_dealloc(tmem, p.tmem_cols);
}

}  // namespace dense
}  // namespace fdmoe
