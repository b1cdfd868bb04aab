// ortho.cu -- orthogonalisation of an update by Newton-Schulz products, on the tensor cores.
//
//   X_0 = G / (|G|_F + eps)          (transposed where G has more rows than columns: X is r x c,
//   A = X X^T                         r <= c)
//   X <- (a + b A + c A^2) X          `steps` times, with (a, b, c) of each step
//
// All products run as D = P Q^T with both operands K-major, on tcgen05.mma kind::f16: A takes X twice,
// A^2 takes A twice (A is symmetric), and the last takes the polynomial and X^T, so X is kept in both
// orders.  Polynomials of A are symmetric: only tiles that touch the lower triangle are computed, and
// each block of 32 x 32 below the diagonal is stored at (i, j) and turned around at (j, i).  Flops of a
// step: r^2 c + r^3 + 2 r^2 c.  With long rows several steps form a group that goes through X once (the
// enums below).
//
// Precision: 3 x fp16.  An operand v is kept as v * 2^k = hi + lo, hi = fp16(v 2^k) and
// lo = fp16(v 2^k - hi), and P Q^T = hi hi^T + hi lo^T + lo hi^T in fp32: 22 bits of each operand,
// which is what fp32 products of long sums deliver.  (Why not plain fp16 or bf16: the iteration
// multiplies small singular values by 3.4 in each step, and the rounding of X with them; one
// rounding to 8 or 11 bits in the first steps is a few percent of the result.)  fp16 has the range
// for it because the spectrum is bounded: |X_0|_2 <= |X_0|_F <= 1, and |X_{k+1}|_2 <= the maximum of
// |a s + b s^3 + c s^5| over [0, bound_k], a bound on every entry of X; those of A and B follow.
// The scales 2^k put each matrix's bound just below 2^15; scale_table() works them out, on the host for
// |X_0|_F = 1 and on the device for a matrix that is no larger than eps, so that none needs a host round
// trip.  Powers of two, so scaling adds no error.
//
// The tensor core truncates each addition to its fp32 accumulator, so a long sum of one sign comes out
// low by half a unit per MMA: 1.8e-5 of the result at a depth of 2601.  So an accumulator takes a
// run of slices only, and the epilogue warps add these partial sums in registers, rounded to nearest.
// The products with lo, two thirds of the MMAs but 2^-11 of the sum, go to an accumulator of their own
// where there is room for one.  fp32 results: products of up to 3 slices add up every slice, those of up to 24
// every second, longer ones every third.  Errors (and the fp32 library products'), with runs of three throughout and
// with these: 2601 x 1001 4.1e-6 and 2.8e-6 (3.3e-6) in 383 and 418 us, 365 x 1135 3.7e-6 and 2.7e-6 (2.3e-6) in
// 245 and 275, 120 x 834 3.2e-6 and 1.9e-6 (1.5e-6) in 142 and 158, 130 x 4000 2.9e-6 and 1.8e-6 (1.3e-6) in 247
// and 261.  fp16 and bf16 results, whose own rounding is far larger, take 1024 and 2048 values.
//
// Kernel: one launch runs the whole iteration (cooperative, one CTA per SM).  A product's tiles are
// shared out over the CTA pairs; each CTA counts itself in when its part is stored, and the loads of
// the next product wait until all have.  A launch for each product took 11 us from one to the next on a
// batch of four of 256 x 256; this takes 7.2.  Warp 0 loads operand slices by TMA (64 deep, 128-byte
// swizzle, hi and lo of both operands) into a ring of stages; warp 1 issues 3 x 4 MMAs per stage into one
// of the TMEM accumulators; warps 4..11 read the others, apply the epilogue and store.  All
// on CTA pairs (cta_group::2), tiles of 256 x 256, 128 or 64: a CTA of the pair loads its 128 rows of P
// and half of the tile's rows of Q, for 256 x 256 two thirds of what a single CTA's 128 x 256 tile
// takes.  That counts: an SM takes in about 64 bytes a cycle, so narrower tiles wait for their
// operands.  No multicast.
// Every mbarrier wait is bounded, as in rbf_fwd_tc.cu.
#include <cuda.h>

#include <algorithm>

#define RBF_WAIT_INLINE  // a call would tie up registers across the register split below
#include "lm_common.cuh"
#include "lm_kernels.cuh"

namespace rbf {
namespace lm {
namespace {

constexpr int kTileRows = 256;                 // of a CTA pair's tile, 128 rows per CTA
constexpr int BK = 64;                         // operand depth of a stage: 128 bytes of fp16
constexpr int kEpiWarps = 8;
constexpr int kThreads = 32 * (4 + kEpiWarps);  // a warpgroup for the loads and MMAs, two for the epilogue
// Registers per thread: launched with kRegs each, then the first warpgroup passes most of its own to
// the other two, which hold 128 partial sums each (kRegsLow + 2 kRegsHigh = 3 kRegs).
constexpr int kRegs = 168, kRegsLow = 40, kRegsHigh = 232;
static_assert(kRegsLow + 2 * kRegsHigh <= 3 * kRegs && kThreads == 384, "register split");
constexpr size_t kSmemMax = 232448;
constexpr int kTurnWords = 32 * 32;             // an epilogue warp's block in shared memory

enum { kSymmetric = 0, kBoth = 1, kFinal = 2 };

// The matrices of an iteration, and the products D = P Q^T it is made of.  A group of steps is
//   A = X X^T,  Q = a + b A + c A^2                                     kGram, kSquare
//   and for every further step of the group, with P the last polynomial (P = Q at first):
//     T = A P,  A = T P                     (the next X X^T)            kTimes, kAgain
//     P = a + b A + c A^2,  Q = P Q                                     kSquare, kChain
//   X = Q X                                                             kApply
// For fp32 results every step is a group, Q leaves the identity out (Q = b A + c A^2) and X = a X + Q X:
// in the full polynomial the terms of Q X cancel, whose rounding is 3 times the fp32 library product's
// error, and 1 / 50 of what rounding the result to 16 bits takes.
enum { mX, mXT0, mXT1, mA, mT, mP, mQ0, mQ1, kMatrices };
enum { kGram, kSquare, kTimes, kAgain, kChain, kApply };
constexpr int kMaxSteps = 32;
constexpr int kMaxOps = 4 * kMaxSteps;  // 11 products for a group of three steps, 3 for a single one
constexpr int kNone = kMatrices;        // no addend

// hi and lo of one matrix per batch entry, row-major.
struct Split {
  __half* hi;
  __half* lo;
  int64_t rows, cols, ld, matrix;  // strides of rows (a multiple of 32) and of matrices, in elements
};

struct Op {
  uint8_t kind, p, q, d, t, add;  // matrices: the operands, where D and its transpose go, what is added
  uint8_t out_kind;
  uint8_t run;                    // slices that share a TMEM accumulator
  int tiles;                      // of one matrix of the batch
};

// Factors of one product of one batch entry: D = acc * (accumulator) + add * addend + diagonal * I.
struct Scale {
  float acc, add, diagonal;
};

struct IterArgs {
  CUtensorMap as_p[kMatrices][2], as_q[kMatrices][2];  // hi, lo; boxes of a CTA's rows of either operand
  Split mat[kMatrices];
  Op op[kMaxOps];
  int ops, batch;
  int out_dtype;
  void* out;                      // of the last product: out[column * ld_out + row]
  int64_t ld_out, out_matrix;
  const Scale* scale;             // [batch][ops]
  unsigned* arrived;              // CTAs that have finished a product, counted over all products
  int* status;
  unsigned long long timeout_ns;
  int debug_skip_first_load;
};

// Wait (bounded) until `want` CTAs have arrived; what they wrote before is visible after it.
__device__ __forceinline__ bool wait_arrived(const unsigned* arrived, unsigned want, int* status,
                                             unsigned long long timeout_ns) {
  const unsigned long long t0 = ptx::globaltimer();
  while (true) {
    unsigned v;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(arrived) : "memory");
    if (v >= want) return true;
    if (ptx::globaltimer() - t0 > timeout_ns) {
      atomicExch(status, 7);
      return false;
    }
  }
}

// Tile t of a matrix.  Symmetric products: only tiles with a row >= their first column, so
// `per` more column tiles for each further row tile.
template <int BN>
__device__ __forceinline__ void tile_of(int t, int out_kind, int tiles_m, int tiles_n, int& tm, int& tn) {
  if (out_kind != kSymmetric) {
    // Bands of 8 row tiles, so that the tiles in flight share both operands in L2.
    constexpr int band = 8;
    const int bi = t / (band * tiles_n);
    const int in = t - bi * band * tiles_n;
    const int rows = min(tiles_m - bi * band, band);
    tn = in / rows;
    tm = bi * band + in - tn * rows;
    return;
  }
  constexpr int per = kTileRows / BN;
  int row = 0, left = t;
  while (true) {
    const int n = min(per * (row + 1), tiles_n);
    if (left < n) break;
    left -= n;
    ++row;
  }
  tm = row;
  tn = left;
}

// Eight (hi, lo) pairs as eight hi and eight lo.
__device__ __forceinline__ void unzip(const uint32_t* w, uint4& hi, uint4& lo) {
  hi = make_uint4(__byte_perm(w[0], w[1], 0x5410), __byte_perm(w[2], w[3], 0x5410),
                  __byte_perm(w[4], w[5], 0x5410), __byte_perm(w[6], w[7], 0x5410));
  lo = make_uint4(__byte_perm(w[0], w[1], 0x7632), __byte_perm(w[2], w[3], 0x7632),
                  __byte_perm(w[4], w[5], 0x7632), __byte_perm(w[6], w[7], 0x7632));
}

__device__ __forceinline__ void split_f16(float x, __half& hi, __half& lo) {
  hi = __float2half_rn(x);
  lo = __float2half_rn(x - __half2float(hi));
}

template <int BN>
struct Plan {
  static constexpr int BROWS = BN / 2;   // rows of Q each CTA loads
  static constexpr uint32_t A_BYTES = 128 * BK * 2;
  static constexpr uint32_t B_BYTES = BROWS * BK * 2;
  static constexpr uint32_t STAGE = 2 * (A_BYTES + B_BYTES);
  static constexpr size_t FIXED = 1024 + 256 + sizeof(uint32_t) * kEpiWarps * kTurnWords;
  static constexpr int STAGES = (int)((kSmemMax - FIXED) / STAGE);
  static constexpr size_t SMEM = FIXED + (size_t)STAGES * STAGE;
  // NACC accumulators of ACC columns, so that the MMAs go on while the epilogue reads.  Where TMEM (512
  // columns) holds it, the hi x lo products have a part of their own (column BN on): see the truncation above.
  static constexpr bool APART = BN <= 128;
  static constexpr uint32_t ACC = APART ? 2 * BN : BN, TCOLS = 512;
  static constexpr int NACC = TCOLS / ACC;
  static_assert(STAGES >= 2 && SMEM <= kSmemMax, "stages");
};

template <int BN>
__global__ void __launch_bounds__(kThreads, 1) ortho_kernel(const __grid_constant__ IterArgs it) {
  using P = Plan<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + P::STAGES * P::STAGE);  // [STAGES] TMA -> MMA
  uint64_t* empty = full + P::STAGES;                                         // [STAGES] MMA -> TMA
  uint64_t* acc_full = empty + P::STAGES;                                     // [NACC] MMA -> epilogue
  uint64_t* acc_empty = acc_full + P::NACC;                                   // [NACC] epilogue -> MMA
  uint64_t* begun = acc_empty + P::NACC;                                      // TMA -> epilogue: a product may begin
  uint64_t* drain = begun + 1;                                                // MMA teardown
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  unsigned* stored = tmem_slot + 1;                                           // epilogue warps, over all products

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = ptx::cluster_ctarank();
  const bool leader = rank == 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < P::STAGES; ++s) {
      ptx::mbar_init(&full[s], 1);
      ptx::mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < P::NACC; ++b) {
      ptx::mbar_init(&acc_full[b], 1);
      ptx::mbar_init(&acc_empty[b], 2 * kEpiWarps);
    }
    ptx::mbar_init(begun, 1);
    ptx::mbar_init(drain, 1);
    *stored = 0;
    ptx::fence_mbar_init();
  }
  if (warp == 0 && lane < kMatrices) {
    for (int h = 0; h < 2; ++h) {
      ptx::prefetch_tensormap(&it.as_p[lane][h]);
      ptx::prefetch_tensormap(&it.as_q[lane][h]);
    }
  }
  ptx::cluster_sync();  // the peer's barriers exist before any remote arrive
  if (warp == 1) {
    ptx::tmem_alloc_pair(tmem_slot, P::TCOLS);
    ptx::tmem_relinquish_pair();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int unit = blockIdx.x >> 1;
  const int units = gridDim.x >> 1;
  const int products = it.ops;

  if (warp < 4) {
    ptx::regs_shrink<kRegsLow>();
    if (warp == 0) {
      // ------------------------------------------------------------ TMA producer
      if (lane == 0) {
        int stage = 0;
        uint32_t phase = 0, issued = 0, last = 0;
        bool ok = true, skipped = false;
        for (int p = 0; p < products && ok; ++p) {
          const Op op = it.op[p];
          const CUtensorMap *mp = it.as_p[op.p], *mq = it.as_q[op.q];
          const int tiles = op.tiles, out_kind = op.out_kind, total = tiles * it.batch;
          const int num_kc = (int)((it.mat[op.p].cols + BK - 1) / BK);
          const int tiles_m = (int)((it.mat[op.p].rows + kTileRows - 1) / kTileRows);
          const int tiles_n = (int)((it.mat[op.q].rows + BN - 1) / BN);
          // The operands come from the other CTAs' epilogues: plain stores, read here by TMA.  This thread
          // alone polls for them and passes it on to its CTA's epilogue: with nine pollers a CTA, 1024 x 4096 took
          // 317 us in place of 301 and 2601 x 1001 fp32 417 in place of 405 (four of 256 x 256: 132, 136).
          if (p > 0) {
            ok = wait_arrived(it.arrived, (unsigned)p * gridDim.x, it.status, it.timeout_ns);
            if (!ok) break;
            ptx::mbar_arrive(begun);
          }
          ptx::fence_proxy_async_global();
          for (int t = unit; t < total && ok; t += units) {
            const int z = t / tiles;
            int tm, tn;
            tile_of<BN>(t - z * tiles, out_kind, tiles_m, tiles_n, tm, tn);
            const int i0 = tm * kTileRows + (int)rank * 128;
            const int j0 = tn * BN + (int)rank * P::BROWS;
            for (int kc = 0; kc < num_kc; ++kc) {
              if (!ptx::mbar_wait_bounded(&empty[stage], phase ^ 1, it.status, it.timeout_ns)) { ok = false; break; }
              if (it.debug_skip_first_load && !skipped && blockIdx.x == 0) {
                skipped = true;  // test hook: this stage never fills, so its consumer times out
              } else {
                uint8_t* s = smem + stage * P::STAGE;
                if (leader) ptx::mbar_arrive_expect_tx(&full[stage], 2 * P::STAGE);
                const uint32_t fc = ptx::map_to_rank(&full[stage], 0);
                ptx::tma_load_3d_pair(s, mp, kc * BK, i0, z, fc);
                ptx::tma_load_3d_pair(s + P::A_BYTES, mp + 1, kc * BK, i0, z, fc);
                ptx::tma_load_3d_pair(s + 2 * P::A_BYTES, mq, kc * BK, j0, z, fc);
                ptx::tma_load_3d_pair(s + 2 * P::A_BYTES + P::B_BYTES, mq + 1, kc * BK, j0, z, fc);
                if (leader) {
                  issued |= 1u << stage;
                  last = (last & ~(1u << stage)) | (phase << stage);
                }
              }
              if (++stage == P::STAGES) {
                stage = 0;
                phase ^= 1;
              }
            }
          }
        }
        // The leader's commits arrive here too: none may be on its way when this CTA's shared memory goes, so
        // every stage is awaited once more.
        for (int s = 0; s < P::STAGES && ok; ++s) {
          ok = ptx::mbar_wait_bounded(&empty[stage], phase ^ 1, it.status, it.timeout_ns);
          if (++stage == P::STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
        // Error path: let every load issued land before the CTA exits (the leader's barriers count
        // both CTAs' bytes, and the final cluster barrier holds the peer until then).
        if (!ok)
          for (int s = 0; s < P::STAGES; ++s)
            if (issued >> s & 1u) ptx::mbar_wait_bounded(&full[s], (last >> s) & 1u, it.status, it.timeout_ns);
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------ MMA issuer (the whole warp)
      if (leader) {
        constexpr uint32_t idesc = ptx::idesc_f16(kTileRows, BN);
        const uint32_t elected = ptx::elect_one();
        const uint64_t base = ptx::smem_desc(ptx::smem_u32(smem), 16, 1024, 2);
        int stage = 0, acc = 0;
        uint32_t phase = 0, acc_phase = 0;
        bool ok = true;
        for (int p = 0; p < products && ok; ++p) {
          const Op op = it.op[p];
          const int num_kc = (int)((it.mat[op.p].cols + BK - 1) / BK), total = op.tiles * it.batch;
          // A unit of work is one run of op.run stages of a tile: each has an accumulator of its own.
          const int runs = (num_kc + op.run - 1) / op.run;
          for (int t = unit; t < total && ok; t += units) {
            for (int run = 0; run < runs && ok; ++run) {
              if (!ptx::mbar_wait_bounded(&acc_empty[acc], acc_phase ^ 1, it.status, it.timeout_ns)) { ok = false; break; }
              ptx::tc_fence_after();
              const uint32_t d = tmem + (uint32_t)acc * P::ACC;
              const int depth = min((int)op.run, num_kc - run * op.run);
              for (int kc = 0; kc < depth; ++kc) {
                if (!ptx::mbar_wait_bounded(&full[stage], phase, it.status, it.timeout_ns)) { ok = false; break; }
                ptx::tc_fence_after();
                // Descriptors of the stage's four operands: the address field counts 16 bytes.
                const uint64_t phi = base + (uint32_t)stage * (P::STAGE >> 4);
                const uint64_t plo = phi + (P::A_BYTES >> 4);
                const uint64_t qhi = phi + (2 * P::A_BYTES >> 4);
                const uint64_t qlo = phi + ((2 * P::A_BYTES + P::B_BYTES) >> 4);
#pragma unroll
                for (int k = 0; k < BK / 16; ++k) {  // 16 fp16 are 32 bytes along the swizzled row
                  ptx::mma_f16_ss_pair(d, phi + 2 * k, qhi + 2 * k, idesc, (kc | k) != 0, elected);
                  ptx::mma_f16_ss_pair(P::APART ? d + BN : d, phi + 2 * k, qlo + 2 * k, idesc, !P::APART || (kc | k) != 0, elected);
                  ptx::mma_f16_ss_pair(P::APART ? d + BN : d, plo + 2 * k, qhi + 2 * k, idesc, 1, elected);
                }
                if (elected) ptx::mma_commit_pair(&empty[stage]);
                __syncwarp();
                if (++stage == P::STAGES) {
                  stage = 0;
                  phase ^= 1;
                }
              }
              if (!ok) break;
              if (elected) ptx::mma_commit_pair(&acc_full[acc]);
              __syncwarp();
              if (++acc == P::NACC) {
                acc = 0;
                acc_phase ^= 1;
              }
            }
          }
        }
        if (elected) ptx::mma_commit_pair(drain);
        __syncwarp();
      }
    }
  } else {
    ptx::regs_grow<kRegsHigh>();
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3;           // TMEM lane quadrant this warp may access
    const int h = (warp - 4) >> 2;    // half of the tile's columns
    uint32_t* turn = reinterpret_cast<uint32_t*>(smem + P::STAGES * P::STAGE + 256) + (warp - 4) * kTurnWords;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int p = 0; p < products && ok; ++p) {
      const Op op = it.op[p];
      const int64_t M = it.mat[op.p].rows, N = it.mat[op.q].rows;
      const int num_kc = (int)((it.mat[op.p].cols + BK - 1) / BK);
      const int tiles_m = (int)((M + kTileRows - 1) / kTileRows), tiles_n = (int)((N + BN - 1) / BN);
      const int total = op.tiles * it.batch;
      const int runs = (num_kc + op.run - 1) / op.run;
      const bool sym = op.out_kind == kSymmetric;
      const bool adds = op.add != kNone;
      const Split d = it.mat[op.d], dt = it.mat[op.t], add = it.mat[adds ? op.add : mA];
      // The addend too comes from other CTAs, and a CTA counts itself in for this product only once
      // the last one is complete.
      if (p > 0 && !ptx::mbar_wait_bounded(begun, (p - 1) & 1, it.status, it.timeout_ns)) break;
      for (int t = unit; t < total; t += units) {
        const int z = t / op.tiles;
        int tm, tn;
        tile_of<BN>(t - z * op.tiles, op.out_kind, tiles_m, tiles_n, tm, tn);
        const int64_t i0 = (int64_t)tm * kTileRows + rank * 128 + q * 32;
        const int64_t i = i0 + lane;
        const Scale sc = it.scale[(int64_t)z * it.ops + p];
        const int64_t col0 = (int64_t)tn * BN + h * (BN / 2);
        const int sub = lane >> 2, part = (lane & 3) * 8;
        // The addend of a block of 32 x 32, four lanes a row; a block's is fetched while the one before
        // it is worked on, the first one's while the accumulator fills.  (Row pitches are multiples of
        // 32, so a block's columns lie inside their row.)
        uint4 add_hi[4], add_lo[4];
        auto fetch = [&](int g) {
          const int64_t j = col0 + g * 32;
          if (!adds || j >= N || (sym && j > i0)) return;
          const int64_t at = z * add.matrix + (i0 + sub) * add.ld + j + part;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (i0 + sub + 8 * k < M) {
              add_hi[k] = *reinterpret_cast<const uint4*>(add.hi + at + 8 * k * add.ld);
              add_lo[k] = *reinterpret_cast<const uint4*>(add.lo + at + 8 * k * add.ld);
            }
        };
        if (runs == 1) fetch(0);
        // All runs but the last are added up in registers; the last one's accumulator takes the
        // total, so that the stores below go over it a few columns at a time.
        const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(h * (BN / 2));
        float sum[BN / 2];
        for (int run = 0; run < runs; ++run) {
          if (!ptx::mbar_wait_bounded(&acc_full[acc], acc_phase, it.status, it.timeout_ns)) { ok = false; break; }
          ptx::tc_fence_after();
          if (runs == 1) break;
#pragma unroll
          for (int c = 0; c < BN / 64; ++c) {
            uint32_t v[32];
            const uint32_t at = lanes + (uint32_t)acc * P::ACC + c * 32;
            ptx::tmem_ld32(at, v);
            if constexpr (P::APART) {
              uint32_t x[32];
              ptx::tmem_ld32(at + BN, x);
              ptx::tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) + __uint_as_float(x[e]));
            } else {
              ptx::tmem_wait_ld();
            }
#pragma unroll
            for (int e = 0; e < 32; ++e)
              sum[c * 32 + e] = run == 0 ? __uint_as_float(v[e]) : sum[c * 32 + e] + __uint_as_float(v[e]);
            if (run + 1 == runs) {
#pragma unroll
              for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(sum[c * 32 + e]);
              ptx::tmem_st32(at, v);
            }
          }
          if (run + 1 == runs) {
            ptx::tmem_wait_st();
            break;
          }
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive_cluster(ptx::map_to_rank(&acc_empty[acc], 0));
          if (++acc == P::NACC) {
            acc = 0;
            acc_phase ^= 1;
          }
        }
        if (!ok) break;
        if (runs > 1) fetch(0);  // (not next to the partial sums: registers)
        // Blocks of 32 x 32, in a loop that is not unrolled: instructions that run for the first time
        // in a launch are fetched from L2, and took most of a small product's time when this was
        // straight-line.  A block goes through shared memory, so that four lanes read or write 64
        // bytes of a row: with a row a lane every access touched 32 lines.
#pragma unroll 1
        for (int g = 0; g < BN / 64; ++g) {
          const int64_t j0 = col0 + g * 32;
          // Below the diagonal, on it, or above it: the same for the whole warp, like the bounds.
          const bool inside = j0 < N && i0 < M && !(sym && j0 > i0);
          const int64_t d_at = z * d.matrix + (i0 + sub) * d.ld + j0 + part;
          uint32_t v[32];
          __syncwarp();  // the TMEM load is a whole warp's; the last block's reads of `turn` are done
          ptx::tmem_ld32(lanes + (uint32_t)acc * P::ACC + g * 32, v);
          if (P::APART && runs == 1) {
            uint32_t x[32];
            ptx::tmem_ld32(lanes + (uint32_t)acc * P::ACC + BN + g * 32, x);
            ptx::tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) + __uint_as_float(x[e]));
          } else {
            ptx::tmem_wait_ld();
          }
          if (g == BN / 64 - 1) {  // the accumulator goes back before the last stores
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive_cluster(ptx::map_to_rank(&acc_empty[acc], 0));
          }
          if (!inside) continue;
          // Word (row, column) of the block is at row * 32 + (column ^ row): rows, columns and the
          // runs of eight below are all read and written without bank conflicts.
#pragma unroll
          for (int e = 0; e < 32; ++e) turn[lane * 32 + (e ^ lane)] = v[e];
          __syncwarp();
          const bool both = !sym || j0 < i0;  // a block on the diagonal is computed whole
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int r = sub + 8 * k;
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = sc.acc * __uint_as_float(turn[r * 32 + ((part + e) ^ r)]);
            if (adds) {
              const __half2* hi = reinterpret_cast<const __half2*>(&add_hi[k]);
              const __half2* lo = reinterpret_cast<const __half2*>(&add_lo[k]);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 x = __half22float2(hi[e]), y = __half22float2(lo[e]);
                f[2 * e] = fmaf(sc.add, x.x + y.x, f[2 * e]);
                f[2 * e + 1] = fmaf(sc.add, x.y + y.y, f[2 * e + 1]);
              }
              if (sym && j0 == i0) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  if (part + e == r) f[e] += sc.diagonal;
              }
            }
            uint32_t w[8];  // fp32, or hi in the low half and lo in the high half
            if (op.out_kind == kFinal) {
#pragma unroll
              for (int e = 0; e < 8; ++e) w[e] = __float_as_uint(f[e]);
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                __half hi, lo;
                split_f16(f[e], hi, lo);
                w[e] = (uint32_t)__half_as_ushort(hi) | (uint32_t)__half_as_ushort(lo) << 16;
              }
              if (i0 + r < M) {
                uint4 hi, lo;
                unzip(w, hi, lo);
                *reinterpret_cast<uint4*>(d.hi + d_at + 8 * k * d.ld) = hi;
                *reinterpret_cast<uint4*>(d.lo + d_at + 8 * k * d.ld) = lo;
              }
            }
            if (both) {
#pragma unroll
              for (int e = 0; e < 8; ++e) turn[r * 32 + ((part + e) ^ r)] = w[e];
            }
          }
          if (g + 1 < BN / 64) fetch(g + 1);
          if (!both) continue;
          __syncwarp();
          if (op.out_kind == kFinal) {
            if (i < M) {
              for (int e = 0; e < 32 && j0 + e < N; ++e)
                store_as(it.out, z * it.out_matrix + (j0 + e) * it.ld_out + i, it.out_dtype, __uint_as_float(turn[lane * 32 + (e ^ lane)]));
            }
            continue;
          }
          // The other order: four lanes write a column's 32 rows.
          const int64_t t_at = z * dt.matrix + (j0 + sub) * dt.ld + i0 + part;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int col = sub + 8 * k;
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = turn[(part + e) * 32 + (col ^ (part + e))];
            if (j0 + col < N) {
              uint4 hi, lo;
              unzip(w, hi, lo);
              *reinterpret_cast<uint4*>(dt.hi + t_at + 8 * k * dt.ld) = hi;
              *reinterpret_cast<uint4*>(dt.lo + t_at + 8 * k * dt.ld) = lo;
            }
          }
        }
        if (++acc == P::NACC) {
          acc = 0;
          acc_phase ^= 1;
        }
      }
      if (!ok) break;
      // This warp's part of the product is in memory, and the CTA's once all warps have said so (a
      // count, not a barrier: a warp that gives up on a wait leaves the others to give up on theirs).
      // TMA reads it in other CTAs: every thread's stores pass the proxy fence before the count.
      ptx::fence_proxy_async_global();
      __syncwarp();
      if (lane == 0) {
        __threadfence_block();
        if (atomicAdd(stored, 1u) == (unsigned)(p + 1) * kEpiWarps - 1) {
          // The fence takes in the other warps' stores and gives them out with the count.
          asm volatile("fence.acq_rel.gpu;" ::: "memory");
          asm volatile("red.relaxed.gpu.global.add.u32 [%0], 1;" ::"l"(it.arrived) : "memory");
        }
      }
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  // Every MMA issued finishes before TMEM is freed, and the leader's last commit, which arrives in both CTAs,
  // has arrived here before this CTA may leave.
  if (warp == 1) ptx::mbar_wait_bounded(drain, 0, it.status, it.timeout_ns);
  ptx::cluster_sync();  // neither CTA leaves before both are done with each other's memory
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc_pair(tmem, P::TCOLS);
  }
}

// ---- the norm, the scales and the first X ---------------------------------------------------

constexpr int kNormThreads = 256;

struct PrepArgs {
  const void* g;
  int64_t rows, cols, row_stride, matrix_stride;  // of G; its rows are contiguous
  int parts, ops;
  int whole;               // Q with the identity
  float eps;
  float coef[kMaxSteps][3];
  uint8_t kind[kMaxOps];   // of the iteration's products
  double* part;            // [batch][parts] sums of squares
  Scale* scale;            // [batch][ops]
  __half* g_hi;            // G's order: [rows, ld_g]
  __half* g_lo;
  __half* t_hi;            // the other order: [cols, ld_t]
  __half* t_lo;
  int64_t ld_g, ld_t, g_matrix, t_matrix;
  int* status;             // [0] status word, [1] arrivals of the products' CTAs
  Scale usual[kMaxOps];    // the factors for |X_0|_F = 1
};

// Sums of squares in 64 bits: an update of any magnitude has a norm.  A warp takes pieces of
// kNormPiece packs a lane of one row.
constexpr int kNormPiece = 4;

template <typename T, int VEC>
__global__ void __launch_bounds__(kNormThreads) ortho_norm_kernel(const PrepArgs a) {
  __shared__ double red[kNormThreads / 32];
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const int64_t z = blockIdx.y;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (z == 0 && blockIdx.x == 0 && threadIdx.x == 0) {
    a.status[0] = 0;
    a.status[1] = 0;  // the arrival counter
  }
  constexpr int piece = 32 * kNormPiece * VEC;
  const int64_t per_row = (a.cols + piece - 1) / piece, items = per_row * a.rows;
  const int64_t warps = (int64_t)a.parts * (kNormThreads / 32);
  double s = 0.0;
  for (int64_t it = (int64_t)blockIdx.x * (kNormThreads / 32) + warp; it < items; it += warps) {
    const int64_t i = it / per_row;
    const int64_t j0 = (it - i * per_row) * piece + lane * VEC;
    const T* row = static_cast<const T*>(a.g) + z * a.matrix_stride + i * a.row_stride;
    Pack<T, VEC> p[kNormPiece];
#pragma unroll
    for (int u = 0; u < kNormPiece; ++u) {
      const int64_t j = j0 + u * 32 * VEC;
      if (j < a.cols) {
        p[u] = *reinterpret_cast<const Pack<T, VEC>*>(row + j);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) p[u].v[e] = from_f32<T>(0.f);
      }
    }
#pragma unroll
    for (int u = 0; u < kNormPiece; ++u)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const double v = to_f32(p[u].v[e]);
        s = fma(v, v, s);
      }
  }
  s = warp_sum(s);
  if (lane == 0) red[warp] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kNormThreads / 32; ++w) s += red[w];
    a.part[z * a.parts + blockIdx.x] = s;
  }
}

// 2^k that brings values of at most `bound` below 2^15 (bounds past 2^+-100 keep the last scale:
// what is smaller does not count next to the rest, what is larger has diverged).
__host__ __device__ inline double pow2_scale(double bound) {
  int e = 0;
  if (bound > 0.0 && isfinite(bound)) e = ilogb(bound) + 1;
  e = e < -100 ? -100 : e > 100 ? 100 : e;
  return ldexp(1.0, 15 - e);
}

// max |f| over [0, top] of f = s^k (c0 + c1 u + c2 u^2): at the ends, or where f' = 0, a quadratic in u.
// With u = s (k = 0 or 1) or u = s^2 (k = 1, `odd`: the polynomial of a step).
__host__ __device__ inline double max_on(double top, int k, bool odd, double c0, double c1, double c2) {
  auto f = [&](double s) {
    const double u = odd ? s * s : s;
    return fabs((k == 1 ? s : 1.0) * (c0 + u * (c1 + u * c2)));
  };
  double m = fmax(f(0.0), f(top));
  const double last = odd ? top * top : top;
  auto at = [&](double u) {
    if (u > 0.0 && u < last) m = fmax(m, f(odd ? sqrt(u) : u));
  };
  // f' is proportional to A u^2 + B u + C.
  const double A = k == 0 ? 0.0 : odd ? 5.0 * c2 : 3.0 * c2, B = k == 0 ? 2.0 * c2 : odd ? 3.0 * c1 : 2.0 * c1;
  const double C = k == 0 ? c1 : c0;
  const double disc = B * B - 4.0 * A * C;
  if (A == 0.0) {
    if (B != 0.0) at(-C / B);
  } else if (disc >= 0.0) {
    at((-B + sqrt(disc)) / (2.0 * A));
    at((-B - sqrt(disc)) / (2.0 * A));
  }
  return m;
}

constexpr double kSlack = 1.0 + 1e-3;  // on the bounds, for rounding along the way

__host__ __device__ inline double first_scale(double rho) { return pow2_scale(rho * kSlack); }

// The factors of every product for one matrix; rho is |X_0|_F.  x bounds |X|_2; A, T, P and Q are
// polynomials in the eigenvalues of X X^T, whose bounds follow; sx ... sq are the matrices' scales.
__host__ __device__ inline void scale_table(double rho, const PrepArgs& a, Scale* out) {
  double x = rho * kSlack, u = 0.0, q = 0.0, next = 0.0;
  double sx = first_scale(rho), sa = 1.0, st = 1.0, sp = 1.0, sq = 1.0;
  int step = 0;
  bool chained = false;  // Q is the last polynomial itself
  for (int i = 0; i < a.ops; ++i) {
    const double c0 = a.coef[step][0], c1 = a.coef[step][1], c2 = a.coef[step][2];
    double acc = 0.0, add = 0.0, diagonal = 0.0;
    switch (a.kind[i]) {
      case kGram:
        u = x * x;
        sa = pow2_scale(u);
        acc = sa / (sx * sx);
        chained = false;
        break;
      case kSquare: {
        const double p = max_on(u, 0, false, a.whole ? c0 : 0.0, c1, c2) * kSlack;
        sp = pow2_scale(p);
        acc = c2 * sp / (sa * sa);
        add = c1 * sp / sa;
        diagonal = a.whole ? c0 * sp : 0.0;
        next = max_on(x, 1, true, c0, c1, c2) * kSlack;
        if (!chained) {
          q = p;
          sq = sp;
        } else {
          q *= p;
        }
        break;
      }
      case kTimes:
        st = pow2_scale(max_on(u, 1, false, c0, c1, c2) * kSlack);
        acc = st / (sa * sp);
        break;
      case kAgain: {
        x = next;
        u = x * x;
        const double to = pow2_scale(u);
        acc = to / (st * sp);
        sa = to;
        chained = true;
        ++step;
        break;
      }
      case kChain: {
        const double to = pow2_scale(q * kSlack);
        acc = to / (sp * sq);
        sq = to;
        break;
      }
      default: {  // kApply
        x = next;
        const double to = i + 1 == a.ops ? 1.0 : pow2_scale(x);
        acc = to / (sq * sx);
        add = c0 * to / sx;  // unless Q is whole
        sx = to;
        ++step;
      }
    }
    out[i] = {(float)acc, (float)add, (float)diagonal};
  }
}

constexpr int kTile = 64;
constexpr int kTilePitch = kTile + 1;

// X_0 in both orders, a 64 x 64 tile of G per CTA; the first CTA of a matrix writes its factors.
static_assert(kMaxOps <= 256, "a thread copies one");
template <typename T, int VEC>
__global__ void __launch_bounds__(256) ortho_split_kernel(const PrepArgs a) {
  __shared__ uint32_t tile[kTile * kTilePitch];  // hi in the low half, lo in the high half
  __shared__ double s_factor, s_rho;
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const int64_t z = blockIdx.z;
  const int64_t i0 = (int64_t)blockIdx.y * kTile, j0 = (int64_t)blockIdx.x * kTile;
  // 8 columns of two rows a thread, on their way while the norm's partial sums are added.
  const int cx = (threadIdx.x & 7) * 8, ry = threadIdx.x >> 3;
  Pack<T, 8> p[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int64_t i = i0 + ry + 32 * u;
    const T* row = static_cast<const T*>(a.g) + z * a.matrix_stride + i * a.row_stride;
#pragma unroll
    for (int e = 0; e < 8; e += VEC) {
      const int64_t j = j0 + cx + e;
      if (i < a.rows && j < a.cols) {
        const Pack<T, VEC> q = *reinterpret_cast<const Pack<T, VEC>*>(row + j);
#pragma unroll
        for (int k = 0; k < VEC; ++k) p[u].v[e + k] = q.v[k];
      } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) p[u].v[e + k] = from_f32<T>(0.f);
      }
    }
  }
  if (threadIdx.x < 32) {
    double t = 0.0;
    for (int k = threadIdx.x; k < a.parts; k += 32) t += a.part[z * a.parts + k];
    t = warp_sum(t);
    if (threadIdx.x == 0) {
      const double norm = sqrt(t), den = norm + (double)a.eps;
      // |X_0|_F is 1 unless the update is no larger than eps; only then are the factors worked out here (6 us
      // for 15 products).
      const double rho = den > 0.0 ? norm / den : 0.0;
      s_rho = rho > 0.5 ? 1.0 : rho;
      s_factor = first_scale(s_rho) / den;
    }
  }
  __syncthreads();
  if (blockIdx.x == 0 && blockIdx.y == 0) {
    Scale* out = a.scale + z * a.ops;
    if (s_rho == 1.0) {
      if (threadIdx.x < a.ops) out[threadIdx.x] = a.usual[threadIdx.x];
    } else if (threadIdx.x == 0) {
      scale_table(s_rho, a, out);
    }
  }
  const double factor = s_factor;
  // In fp32 where the factor has its full precision there (one more rounding, the same for all).
  const bool wide = !(fabs(factor) > 1e-30 && fabs(factor) < 1e30);
  const float narrow = (float)factor;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int64_t i = i0 + ry + 32 * u;
    uint32_t both[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float g = to_f32(p[u].v[e]);
      __half hi, lo;
      split_f16(wide ? (float)((double)g * factor) : g * narrow, hi, lo);
      both[e] = (uint32_t)__half_as_ushort(hi) | (uint32_t)__half_as_ushort(lo) << 16;
      tile[(ry + 32 * u) * kTilePitch + cx + e] = both[e];
    }
    if (i < a.rows && j0 + cx < a.cols) {  // up to the pitch, a multiple of 32
      uint4 hi, lo;
      unzip(both, hi, lo);
      const int64_t at = z * a.g_matrix + i * a.ld_g + j0 + cx;
      *reinterpret_cast<uint4*>(a.g_hi + at) = hi;
      *reinterpret_cast<uint4*>(a.g_lo + at) = lo;
    }
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int64_t j = j0 + ry + 32 * u;
    if (j < a.cols && i0 + cx < a.rows) {
      uint32_t w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = tile[(cx + e) * kTilePitch + ry + 32 * u];
      uint4 hi, lo;
      unzip(w, hi, lo);
      const int64_t at = z * a.t_matrix + j * a.ld_t + i0 + cx;
      *reinterpret_cast<uint4*>(a.t_hi + at) = hi;
      *reinterpret_cast<uint4*>(a.t_lo + at) = lo;
    }
  }
}

// ---- host side ----------------------------------------------------------------------------

// Steps that a group may hold.  Carrying A over (two products of r^3 in place of going through X: r^2 c + 2
// r^2 c) saves (1.5 c / r - 1.5) r^3 a step, at one product more.  Up to three steps, which leaves the
// error where it was: an error of A grows by a^2 a step; four steps and more let it show (8 times, for an
// update with a few strong directions).
int group_size(const float* coef, int step, int steps) {
  const int left = steps - step, groups = (left + 2) / 3;
  const int n = (left + groups - 1) / groups;
  double growth = 1.0;
  for (int k = 0; k + 1 < n; ++k) {
    growth *= (double)coef[3 * (step + k)] * coef[3 * (step + k)];
    if (growth > 200.0) return k + 1;
  }
  return n;
}

// The products of an iteration.
int list_ops(bool tall, bool whole, bool grouped, const float* coef, int steps, Op* op) {
  int n = 0, xt = mXT0;
  auto put = [&](int kind, int p, int q, int d, int t, int out_kind, int add = kNone) {
    op[n++] = Op{(uint8_t)kind, (uint8_t)p, (uint8_t)q, (uint8_t)d, (uint8_t)t, (uint8_t)add, (uint8_t)out_kind, 0, 0};
  };
  for (int step = 0; step < steps;) {
    const int size = grouped ? group_size(coef, step, steps) : 1;
    int last = mQ0, q = mQ0;  // the last polynomial, and the product of the group's
    put(kGram, mX, mX, mA, mA, kSymmetric);
    put(kSquare, mA, mA, mQ0, mQ0, kSymmetric, mA);
    for (int k = 1; k < size; ++k) {
      put(kTimes, mA, last, mT, mT, kSymmetric);
      put(kAgain, mT, last, mA, mA, kSymmetric);
      put(kSquare, mA, mA, mP, mP, kSymmetric, mA);
      const int to = q == mQ0 ? mQ1 : mQ0;
      put(kChain, mP, q, to, to, kSymmetric);
      last = mP;
      q = to;
    }
    step += size;
    if (step < steps) {
      const int to = xt == mXT0 ? mXT1 : mXT0;
      put(kApply, q, xt, mX, to, kBoth, whole ? kNone : mX);  // X in place: a thread reads what it replaces
      xt = to;
    } else if (tall) {
      // The last product runs in the order that lets the lanes of a warp write the result's rows.
      put(kApply, q, xt, mX, mX, kFinal, whole ? kNone : mX);
    } else {
      put(kApply, xt, q, mX, mX, kFinal, whole ? kNone : xt);
    }
  }
  return n;
}

struct Layout {
  int64_t r, c;  // X is r x c, r <= c
  int64_t ld_c, ld_r;
  size_t status, part, scale, mat[kMatrices], end;
  int parts;
  bool may_group;
};

Layout layout_of(int64_t batch, int64_t rows, int64_t cols, int steps) {
  Layout L;
  L.r = std::min(rows, cols);
  L.c = std::max(rows, cols);
  L.ld_c = round_up(L.c, 32);
  L.ld_r = round_up(L.r, 32);
  L.may_group = 4 * L.c >= 5 * L.r && steps > 1;
  // About 8 K values for each CTA of the norm, and no more CTAs than give each SM four.
  const int64_t want = std::min<int64_t>(ceil_div(rows * cols, 8192), ceil_div(4 * kSmCount, batch > 0 ? batch : 1));
  L.parts = (int)std::max<int64_t>(1, want);
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t o = off;
    off = (size_t)round_up((int64_t)(off + bytes), (int64_t)kAlign);
    return o;
  };
  L.status = take(64);
  L.part = take(sizeof(double) * batch * L.parts);
  L.scale = take(sizeof(Scale) * batch * kMaxOps);
  const size_t x = sizeof(__half) * 2 * batch * L.r * L.ld_c, xt = sizeof(__half) * 2 * batch * L.c * L.ld_r;
  const size_t sq = sizeof(__half) * 2 * batch * L.r * L.ld_r;
  for (int m = 0; m < kMatrices; ++m) {
    const bool used = m <= mA || m == mQ0 || L.may_group;  // the others belong to groups of steps
    L.mat[m] = !used ? L.mat[mA] : take(m == mX ? x : m <= mXT1 ? xt : sq);
  }
  L.end = off;
  return L;
}

int64_t tiles_of(int64_t M, int64_t N, int bn, int out_kind) {
  const int64_t m = ceil_div(M, kTileRows), n = ceil_div(N, bn);
  if (out_kind != kSymmetric) return m * n;
  int64_t t = 0;
  for (int64_t i = 0; i < m; ++i) t += std::min<int64_t>((kTileRows / bn) * (i + 1), n);
  return t;
}

template <int BN>
cudaError_t launch_iteration(IterArgs& it, cudaStream_t stream) {
  using PL = Plan<BN>;
  auto k = ortho_kernel<BN>;
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PL::SMEM);
  if (e != cudaSuccess) return e;
  // The register split must fit into what the block is launched with, or it would wait for ever.
  static const int regs = [&] {
    cudaFuncAttributes fa{};
    return cudaFuncGetAttributes(&fa, k) == cudaSuccess ? fa.numRegs : 0;
  }();
  if (regs < kRegs) return cudaErrorInvalidConfiguration;
  for (int m = 0; m < kMatrices; ++m) {
    const Split& s = it.mat[m];
    for (int h = 0; h < 2; ++h) {
      const __half* base = h == 0 ? s.hi : s.lo;
      if (!make_tmap_f16(&it.as_p[m][h], base, s.cols, s.rows, it.batch, s.ld, s.matrix, BK, 128) ||
          !make_tmap_f16(&it.as_q[m][h], base, s.cols, s.rows, it.batch, s.ld, s.matrix, BK, PL::BROWS))
        return cudaErrorInvalidValue;
    }
  }
  int64_t most = 0;
  for (int i = 0; i < it.ops; ++i) {
    Op& op = it.op[i];
    const int64_t tiles = tiles_of(it.mat[op.p].rows, it.mat[op.q].rows, BN, op.out_kind);
    if (tiles * it.batch >= (int64_t(1) << 30)) return cudaErrorInvalidConfiguration;
    op.tiles = (int)tiles;
    most = std::max(most, tiles * it.batch);
  }
  // A cooperative launch: the CTAs wait for one another between products, so all must be resident.
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = PL::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeCooperative;
  attr[1].val.cooperative = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3((unsigned)device_sm_count());
  static int resident[64];  // clusters, by device
  int dev = 0;
  if ((e = cudaGetDevice(&dev)) != cudaSuccess) return e;
  int clusters = dev < 64 ? resident[dev] : 0;
  if (clusters == 0) {
    if ((e = cudaOccupancyMaxActiveClusters(&clusters, k, &cfg)) != cudaSuccess) return e;
    if (clusters < 1) return cudaErrorCooperativeLaunchTooLarge;
    if (dev < 64) resident[dev] = clusters;
  }
  cfg.gridDim = dim3(2 * (unsigned)std::min<int64_t>(most, clusters));
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, k, it);
}

// Estimated time of the products with tiles of width bn, in cycles.  A slice of 64 costs a pair the larger
// of its 12 MMAs (6 bn cycles) and its operands' way into shared memory (64 bytes a cycle and CTA: 1024, 768
// and 640 for bn = 256, 128 and 64; 850 for 128 with every SM at it).  A product ends with what nothing
// hides, the epilogue of a tile and the wait for the other CTAs: 3700 + 130 bn.  Measured for 64, 128
// and 256: four of 256 x 256: 128, 204 and 361 us; 2048 x 4096 bf16: 921, 799 and 1089, grouped 734, 671 and 1049;
// 4096 x 8192: 6.9, 5.4 and 5.0 ms, grouped 5.3, 4.2 and 4.0.
int64_t estimate(const IterArgs& it, const Op* op, int ops, int bn) {
  const int64_t pairs = device_sm_count() / 2, slice = bn == 256 ? 1536 : bn == 128 ? 850 : 640;
  int64_t cost = 0;
  for (int i = 0; i < ops; ++i) {
    const Split &p = it.mat[op[i].p], &q = it.mat[op[i].q];
    cost += ceil_div(tiles_of(p.rows, q.rows, bn, op[i].out_kind) * it.batch, pairs) * ceil_div(p.cols, BK) * slice + 3700 + 130 * bn;
  }
  return cost;
}

// Slices that share an accumulator, of a product of `slices`: see the truncation above.
int run_of(int dtype, int64_t slices) {
  if (dtype != LM_F32) return dtype == LM_F16 ? 16 : 32;
  return slices <= 3 ? 1 : slices <= 24 ? 2 : 3;
}

// The products and the tile width with the least estimated time.
int plan(IterArgs& it, bool tall, bool whole, bool may_group, const float* coef, int steps) {
  Op op[kMaxOps];
  int best = 0;
  int64_t least = 0;
  for (int grouped = 0; grouped <= (whole && may_group ? 1 : 0); ++grouped) {
    const int ops = list_ops(tall, whole, grouped != 0, coef, steps, op);
    for (const int bn : {256, 128, 64}) {
      const int64_t cost = estimate(it, op, ops, bn);
      if (best == 0 || cost < least) {
        best = bn;
        least = cost;
        it.ops = ops;
        std::copy(op, op + ops, it.op);
      }
    }
  }
  return best;
}

}  // namespace

size_t ortho_workspace_bytes(int64_t batch, int64_t rows, int64_t cols, int steps) {
  return layout_of(batch, rows, cols, steps).end;
}

int ortho_max_steps() { return kMaxSteps; }

cudaError_t launch_orthogonalize(const OrthoArgs& o, const WaitConfig& wc, cudaStream_t stream) {
  if (o.batch == 0 || o.rows == 0 || o.cols == 0) return cudaSuccess;
  const Layout L = layout_of(o.batch, o.rows, o.cols, o.steps);
  const bool tall = o.rows > o.cols;
  int* status = ws_at<int>(o.workspace, L.status);
  IterArgs it{};
  for (int m = 0; m < kMatrices; ++m) {
    Split& s = it.mat[m];
    s.rows = m == mXT0 || m == mXT1 ? L.c : L.r;
    s.cols = m == mX ? L.c : L.r;
    s.ld = m == mX ? L.ld_c : L.ld_r;
    s.matrix = s.rows * s.ld;
    s.hi = ws_at<__half>(o.workspace, L.mat[m]);
    s.lo = s.hi + o.batch * s.matrix;
  }
  const bool whole = o.dtype != LM_F32;
  it.batch = (int)o.batch;
  const int bn = plan(it, tall, whole, L.may_group, o.coefficients, o.steps);

  PrepArgs p{};
  p.g = o.update;
  p.rows = o.rows;
  p.cols = o.cols;
  p.row_stride = o.row_stride;
  p.matrix_stride = o.matrix_stride;
  p.parts = L.parts;
  p.ops = it.ops;
  p.whole = whole;
  p.eps = o.eps;
  for (int k = 0; k < o.steps; ++k)
    for (int e = 0; e < 3; ++e) p.coef[k][e] = o.coefficients[3 * k + e];
  for (int i = 0; i < it.ops; ++i) p.kind[i] = it.op[i].kind;
  scale_table(1.0, p, p.usual);
  p.part = ws_at<double>(o.workspace, L.part);
  p.scale = ws_at<Scale>(o.workspace, L.scale);
  const Split& g = it.mat[tall ? mXT0 : mX];
  const Split& t = it.mat[tall ? mX : mXT0];
  p.g_hi = g.hi;
  p.g_lo = g.lo;
  p.ld_g = g.ld;
  p.g_matrix = g.matrix;
  p.t_hi = t.hi;
  p.t_lo = t.lo;
  p.ld_t = t.ld;
  p.t_matrix = t.matrix;
  p.status = status;
  auto prep = [&](auto norm, auto split) {
    cudaError_t e = launch_kernel(norm, dim3(L.parts, (unsigned)o.batch), dim3(kNormThreads), 0, stream, p);
    if (e != cudaSuccess) return e;
    return launch_kernel(split, dim3((unsigned)ceil_div(o.cols, kTile), (unsigned)ceil_div(o.rows, kTile), (unsigned)o.batch),
                         dim3(256), 0, stream, p);
  };
  const int64_t es = (int64_t)elem_bytes(o.dtype);
  const bool packs = (o.cols * es) % 16 == 0 && (o.row_stride * es) % 16 == 0 &&
                     (o.batch == 1 || (o.matrix_stride * es) % 16 == 0) &&
                     reinterpret_cast<uintptr_t>(o.update) % 16 == 0;
  auto by_pack = [&](auto x) {
    using T = decltype(x);
    constexpr int V = 16 / sizeof(T);
    return packs ? prep(ortho_norm_kernel<T, V>, ortho_split_kernel<T, V>)
                 : prep(ortho_norm_kernel<T, 1>, ortho_split_kernel<T, 1>);
  };
  cudaError_t e = o.dtype == LM_F32 ? by_pack(float{}) : o.dtype == LM_BF16 ? by_pack(__nv_bfloat16{}) : by_pack(__half{});
  if (e != cudaSuccess) return e;

  for (int i = 0; i < it.ops; ++i) it.op[i].run = (uint8_t)run_of(o.dtype, ceil_div(it.mat[it.op[i].p].cols, BK));
  it.out = o.out;
  it.ld_out = o.cols;
  it.out_matrix = o.rows * o.cols;
  it.out_dtype = o.dtype;
  it.scale = p.scale;
  it.arrived = reinterpret_cast<unsigned*>(status + 1);
  it.status = status;
  it.timeout_ns = wc.timeout_ns;
  it.debug_skip_first_load = wc.debug_skip_first_load;
  e = bn == 256 ? launch_iteration<256>(it, stream) : bn == 128 ? launch_iteration<128>(it, stream) : launch_iteration<64>(it, stream);
  if (e != cudaSuccess) return e;
  note_launches(3);
  return cudaGetLastError();
}

}  // namespace lm
}  // namespace rbf
