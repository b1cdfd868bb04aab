// ortho.cu -- orthogonalisation of an update by Newton-Schulz products, on the tensor cores.
//
//   X_0 = G / (|G|_F + eps)          (transposed where G has more rows than columns: X is r x c,
//   A = X X^T,  B = b A + c A^2       r <= c)
//   X <- a X + B X                    `steps` times, with (a, b, c) of each step
//
// All three products run as D = P Q^T with both operands K-major, on tcgen05.mma kind::f16: A takes
// X twice, A^2 takes A twice (A is symmetric), and B X takes B and X^T, so every step keeps X in
// both orders.  A and B are symmetric: only tiles that touch the lower triangle are computed, and
// each block of 32 x 32 below the diagonal is stored at (i, j) and turned around at (j, i).  Flops of a step: r^2 c + r^3 + 2 r^2 c.
//
// Precision: 3 x fp16.  An operand v is kept as v * 2^k = hi + lo, hi = fp16(v 2^k) and
// lo = fp16(v 2^k - hi), and P Q^T = hi hi^T + hi lo^T + lo hi^T in fp32: 22 bits of each operand,
// which is what fp32 products of long sums deliver.  (Why not plain fp16 or bf16: the iteration
// multiplies small singular values by 3.4 in each step, and the rounding of X with them; one
// rounding to 8 or 11 bits in the first steps is a few percent of the result.)  fp16 has the range
// for it because the spectrum is bounded: |X_0|_2 <= |X_0|_F <= 1, and |X_{k+1}|_2 <= the maximum of
// |a s + b s^3 + c s^5| over [0, bound_k], a bound on every entry of X; those of A and B follow.
// The scales 2^k put each matrix's bound just below 2^15; scale_table() works them out per matrix
// on the device, so zero, tiny and diverging updates need no host round trip.  Powers of two, so
// scaling adds no error.
//
// The tensor core truncates each addition to its fp32 accumulator, so a long sum of one sign comes out
// low by half a unit per MMA: 1.8e-5 of the result at a depth of 2601.  So an accumulator takes a
// run of slices only, and the epilogue warps add these partial sums in registers, rounded to nearest.
// A run is 256 deep for fp32 results (error 4.8e-6 there, the fp32 library product's is 3.3e-6), 1024
// for fp16 and 2048 for bf16, whose own rounding is far larger: short runs cost up to 9% of the time.
//
// Kernel: one launch runs the whole iteration (cooperative, one CTA per SM).  A product's tiles are
// shared out over the CTA pairs; each CTA counts itself in when its part is stored, and the loads of
// the next product wait until all have.  Against a launch for each product, which the next one's
// start had to follow, (11 us from one to the next) this takes 8 us for a batch of four of 256 x 256.  Warp 0 loads operand slices by TMA (64 deep, 128-byte swizzle, hi and lo of
// both operands) into a ring of stages; warp 1 issues 3 x 4 MMAs per stage into one of
// two TMEM accumulators; warps 4..11 read the other one, apply the epilogue and store.  All
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

// Scale factors of one step of one matrix (see scale_table).
struct StepScale {
  float gram;             // A      from the accumulator of X X^T
  float square, linear;   // B      from the accumulator of A^2, and from A
  float product, keep;    // X_next from the accumulator of B X, and from X
};

enum { kSymmetric = 0, kBoth = 1, kFinal = 2 };

// One product D = P Q^T of every matrix of the batch.
struct GemmArgs {
  int64_t M, N;             // D [M, N] per matrix
  int tiles;                // of one matrix
  int tiles_m, tiles_n;
  int num_kc;               // slices of the depth
  int out_kind;             // kSymmetric, kBoth, kFinal
  int kind;                 // of the scales: 0 gram, 1 square, 2 product
  int out_dtype;
  // D = alpha * accumulator + beta * (add_hi + add_lo), alpha and beta from the scale table
  const __half* add_hi;     // row-major [M, ld_d] (NULL: no addend)
  const __half* add_lo;
  __half* d_hi;             // row-major [M, ld_d]
  __half* d_lo;
  __half* t_hi;             // transposed [N, ld_t]; pitches are multiples of 32
  __half* t_lo;
  int64_t ld_d, ld_t, d_matrix, t_matrix;  // strides of rows and of matrices, in elements
  void* out;                // kFinal: out[col * ld_out + row], type out_dtype
  int64_t ld_out, out_matrix;
};

// The whole iteration: for each step gram, square and one of the two products (X^T alternates
// between two buffers), the last step's being `final`.
enum { kGram = 0, kSquare = 1, kProduct = 2, kLast = 4, kProducts = 5 };
struct IterArgs {
  CUtensorMap map[kProducts][4];  // P hi, P lo, Q hi, Q lo
  GemmArgs gemm[kProducts];
  const StepScale* scale;         // [batch][steps]
  unsigned* arrived;              // CTAs that have finished a product, counted over all products
  int* status;
  unsigned long long timeout_ns;
  int steps, batch;
  int run;                        // slices that share a TMEM accumulator
  int debug_skip_first_load;
};
static_assert(sizeof(IterArgs) <= 4096, "kernel parameters");

__device__ __forceinline__ int product_index(int p, int steps) {
  const int step = p / 3, w = p - 3 * step;
  if (w < 2) return w;
  return step + 1 == steps ? kLast : kProduct + (step & 1);
}

// Wait (bounded) until `want` CTAs have arrived; what they wrote before is visible after it.
// `pause`: between polls, where nothing hangs on the first moment.
template <bool pause>
__device__ __forceinline__ bool wait_arrived(const unsigned* arrived, unsigned want, int* status,
                                             unsigned long long timeout_ns) {
  const unsigned long long t0 = ptx::globaltimer();
  while (true) {
    unsigned v;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(arrived) : "memory");
    if (v >= want) return true;
    if (pause) __nanosleep(64);
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
  static constexpr uint32_t TCOLS = 2 * BN;
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
  uint64_t* acc_full = empty + P::STAGES;                                     // [2] MMA -> epilogue
  uint64_t* acc_empty = acc_full + 2;                                         // [2] epilogue -> MMA
  uint64_t* drain = acc_empty + 2;                                            // MMA teardown
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
    for (int b = 0; b < 2; ++b) {
      ptx::mbar_init(&acc_full[b], 1);
      ptx::mbar_init(&acc_empty[b], 2 * kEpiWarps);
    }
    ptx::mbar_init(drain, 1);
    *stored = 0;
    ptx::fence_mbar_init();
  }
  if (warp == 0 && lane < 4)
    for (int p = 0; p < kProducts; ++p) ptx::prefetch_tensormap(&it.map[p][lane]);
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
  const int products = 3 * it.steps;

  if (warp < 4) {
    ptx::regs_shrink<kRegsLow>();
    if (warp == 0) {
      // ------------------------------------------------------------ TMA producer
      if (lane == 0) {
        int stage = 0;
        uint32_t phase = 0, issued = 0, last = 0;
        bool ok = true, skipped = false;
        for (int p = 0; p < products && ok; ++p) {
          const int pi = product_index(p, it.steps);
          const CUtensorMap* map = it.map[pi];
          const int tiles = it.gemm[pi].tiles, num_kc = it.gemm[pi].num_kc, out_kind = it.gemm[pi].out_kind;
          const int tiles_m = it.gemm[pi].tiles_m, tiles_n = it.gemm[pi].tiles_n;
          const int total = tiles * it.batch;
          for (int t = unit; t < total && ok; t += units) {
            const int z = t / tiles;
            int tm, tn;
            tile_of<BN>(t - z * tiles, out_kind, tiles_m, tiles_n, tm, tn);
            const int i0 = tm * kTileRows + (int)rank * 128;
            const int j0 = tn * BN + (int)rank * P::BROWS;
            if (t == unit && p > 0) {
              // The operands come from the other CTAs' epilogues: plain stores, read here by TMA.
              ok = wait_arrived<false>(it.arrived, (unsigned)p * gridDim.x, it.status, it.timeout_ns);
              if (!ok) break;
            }
            if (t == unit) ptx::fence_proxy_async();
            for (int kc = 0; kc < num_kc; ++kc) {
              if (!ptx::mbar_wait_bounded(&empty[stage], phase ^ 1, it.status, it.timeout_ns)) { ok = false; break; }
              if (it.debug_skip_first_load && !skipped && blockIdx.x == 0) {
                skipped = true;  // test hook: this stage never fills, so its consumer times out
              } else {
                uint8_t* s = smem + stage * P::STAGE;
                if (leader) ptx::mbar_arrive_expect_tx(&full[stage], 2 * P::STAGE);
                const uint32_t fc = ptx::map_to_rank(&full[stage], 0);
                ptx::tma_load_3d_pair(s, map, kc * BK, i0, z, fc);
                ptx::tma_load_3d_pair(s + P::A_BYTES, map + 1, kc * BK, i0, z, fc);
                ptx::tma_load_3d_pair(s + 2 * P::A_BYTES, map + 2, kc * BK, j0, z, fc);
                ptx::tma_load_3d_pair(s + 2 * P::A_BYTES + P::B_BYTES, map + 3, kc * BK, j0, z, fc);
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
          const int pi = product_index(p, it.steps);
          const int num_kc = it.gemm[pi].num_kc, total = it.gemm[pi].tiles * it.batch;
          // A unit of work is one run of it.run stages of a tile: each has an accumulator of its own.
          const int runs = (num_kc + it.run - 1) / it.run;
          for (int t = unit; t < total && ok; t += units) {
            for (int run = 0; run < runs && ok; ++run) {
              if (!ptx::mbar_wait_bounded(&acc_empty[acc], acc_phase ^ 1, it.status, it.timeout_ns)) { ok = false; break; }
              ptx::tc_fence_after();
              const uint32_t d = tmem + (uint32_t)(acc * BN);
              const int depth = min(it.run, num_kc - run * it.run);
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
                  ptx::mma_f16_ss_pair(d, phi + 2 * k, qlo + 2 * k, idesc, 1, elected);
                  ptx::mma_f16_ss_pair(d, plo + 2 * k, qhi + 2 * k, idesc, 1, elected);
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
              if (++acc == 2) {
                acc = 0;
                acc_phase ^= 1;
              }
            }
          }
        }
        if (elected) ptx::mma_commit_pair(drain);  // every MMA issued so far finishes before TMEM is freed
        __syncwarp();
        ptx::mbar_wait_bounded(drain, 0, it.status, it.timeout_ns);
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
      const GemmArgs a = it.gemm[product_index(p, it.steps)];  // in registers: its index is not constant
      const int total = a.tiles * it.batch;
      const int runs = (a.num_kc + it.run - 1) / it.run;
      const bool sym = a.out_kind == kSymmetric;
      // The addend too comes from other CTAs, and a CTA counts itself in for this product only once
      // the last one is complete.
      if (p > 0) {
        int in = 1;
        if (lane == 0) in = wait_arrived<true>(it.arrived, (unsigned)p * gridDim.x, it.status, it.timeout_ns);
        ok = __shfl_sync(0xffffffffu, in, 0) != 0;
        if (!ok) break;
      }
      for (int t = unit; t < total; t += units) {
        const int z = t / a.tiles;
        int tm, tn;
        tile_of<BN>(t - z * a.tiles, a.out_kind, a.tiles_m, a.tiles_n, tm, tn);
        const int64_t i0 = (int64_t)tm * kTileRows + rank * 128 + q * 32;
        const int64_t i = i0 + lane;
        const StepScale sc = it.scale[(int64_t)z * it.steps + p / 3];
        const float alpha = a.kind == 0 ? sc.gram : a.kind == 1 ? sc.square : sc.product;
        const float beta = a.kind == 0 ? 0.f : a.kind == 1 ? sc.linear : sc.keep;
        const int64_t col0 = (int64_t)tn * BN + h * (BN / 2);
        const int sub = lane >> 2, part = (lane & 3) * 8;
        // The addend of a block of 32 x 32, four lanes a row; a block's is fetched while the one before
        // it is worked on, the first one's while the accumulator fills.  (Row pitches are multiples of
        // 32, so a block's columns lie inside their row.)
        uint4 add_hi[4], add_lo[4];
        auto fetch = [&](int g) {
          const int64_t j = col0 + g * 32;
          if (a.add_hi == nullptr || j >= a.N || (sym && j > i0)) return;
          const int64_t at = z * a.d_matrix + (i0 + sub) * a.ld_d + j + part;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (i0 + sub + 8 * k < a.M) {
              add_hi[k] = *reinterpret_cast<const uint4*>(a.add_hi + at + 8 * k * a.ld_d);
              add_lo[k] = *reinterpret_cast<const uint4*>(a.add_lo + at + 8 * k * a.ld_d);
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
            const uint32_t at = lanes + (uint32_t)(acc * BN + c * 32);
            ptx::tmem_ld32(at, v);
            ptx::tmem_wait_ld();
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
          if (++acc == 2) {
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
          const bool inside = j0 < a.N && i0 < a.M && !(sym && j0 > i0);
          const int64_t d_at = z * a.d_matrix + (i0 + sub) * a.ld_d + j0 + part;
          uint32_t v[32];
          __syncwarp();  // the TMEM load is a whole warp's; the last block's reads of `turn` are done
          ptx::tmem_ld32(lanes + (uint32_t)(acc * BN + g * 32), v);
          ptx::tmem_wait_ld();
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
            for (int e = 0; e < 8; ++e) f[e] = alpha * __uint_as_float(turn[r * 32 + ((part + e) ^ r)]);
            if (a.add_hi != nullptr) {
              const __half2* hi = reinterpret_cast<const __half2*>(&add_hi[k]);
              const __half2* lo = reinterpret_cast<const __half2*>(&add_lo[k]);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 x = __half22float2(hi[e]), y = __half22float2(lo[e]);
                f[2 * e] = fmaf(beta, x.x + y.x, f[2 * e]);
                f[2 * e + 1] = fmaf(beta, x.y + y.y, f[2 * e + 1]);
              }
            }
            uint32_t w[8];  // fp32, or hi in the low half and lo in the high half
            if (a.out_kind == kFinal) {
#pragma unroll
              for (int e = 0; e < 8; ++e) w[e] = __float_as_uint(f[e]);
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                __half hi, lo;
                split_f16(f[e], hi, lo);
                w[e] = (uint32_t)__half_as_ushort(hi) | (uint32_t)__half_as_ushort(lo) << 16;
              }
              if (i0 + r < a.M) {
                uint4 hi, lo;
                unzip(w, hi, lo);
                *reinterpret_cast<uint4*>(a.d_hi + d_at + 8 * k * a.ld_d) = hi;
                *reinterpret_cast<uint4*>(a.d_lo + d_at + 8 * k * a.ld_d) = lo;
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
          if (a.out_kind == kFinal) {
            if (i < a.M) {
              for (int e = 0; e < 32 && j0 + e < a.N; ++e)
                store_as(a.out, z * a.out_matrix + (j0 + e) * a.ld_out + i, a.out_dtype, __uint_as_float(turn[lane * 32 + (e ^ lane)]));
            }
            continue;
          }
          // The other order: four lanes write a column's 32 rows.
          __half* th = sym ? a.d_hi : a.t_hi;
          __half* tl = sym ? a.d_lo : a.t_lo;
          const int64_t ld = sym ? a.ld_d : a.ld_t;
          const int64_t t_at = z * (sym ? a.d_matrix : a.t_matrix) + (j0 + sub) * ld + i0 + part;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int col = sub + 8 * k;
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = turn[(part + e) * 32 + (col ^ (part + e))];
            if (j0 + col < a.N) {
              uint4 hi, lo;
              unzip(w, hi, lo);
              *reinterpret_cast<uint4*>(th + t_at + 8 * k * ld) = hi;
              *reinterpret_cast<uint4*>(tl + t_at + 8 * k * ld) = lo;
            }
          }
        }
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1;
        }
      }
      if (!ok) break;
      // This warp's part of the product is in memory, and the CTA's once all warps have said so (a
      // count, not a barrier: a warp that gives up on a wait leaves the others to give up on theirs).
      __syncwarp();
      if (lane == 0) {
        __threadfence_block();
        if (atomicAdd(stored, 1u) == (unsigned)(p + 1) * kEpiWarps - 1) {
          __threadfence();
          asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(it.arrived) : "memory");
        }
      }
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::cluster_sync();  // neither CTA leaves before both are done with each other's memory
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc_pair(tmem, P::TCOLS);
  }
}

// ---- the norm, the scales and the first X ---------------------------------------------------

constexpr int kMaxSteps = 32;
constexpr int kNormThreads = 256;

struct PrepArgs {
  const void* g;
  int64_t rows, cols, row_stride, matrix_stride;  // of G; its rows are contiguous
  int dtype, tall, parts, steps;
  float eps;
  float coef[kMaxSteps][3];
  double* part;            // [batch][parts] sums of squares
  StepScale* scale;        // [batch][steps]
  __half* g_hi;            // G's order: [rows, ld_g]
  __half* g_lo;
  __half* t_hi;            // the other order: [cols, ld_t]
  __half* t_lo;
  int64_t ld_g, ld_t, g_matrix, t_matrix;
  int* status;             // [0] status word, [1] arrivals of the products' CTAs
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
__device__ double pow2_scale(double bound) {
  int e = 0;
  if (bound > 0.0 && isfinite(bound)) e = ilogb(bound) + 1;
  e = e < -100 ? -100 : e > 100 ? 100 : e;
  return ldexp(1.0, 15 - e);
}

__device__ double max_on(double top, double c1, double c3, double c5) {
  // max of |c1 s + c3 s^3 + c5 s^5| over [0, top]: at the end, or where c1 + 3 c3 u + 5 c5 u^2 = 0, u = s^2
  auto p = [&](double s) { return fabs(s * (c1 + s * s * (c3 + s * s * c5))); };
  double m = p(top);
  auto at = [&](double u) {
    if (u > 0.0 && u < top * top) m = fmax(m, p(sqrt(u)));
  };
  const double A = 5.0 * c5, B = 3.0 * c3, disc = B * B - 4.0 * A * c1;
  if (A == 0.0) {
    if (B != 0.0) at(-c1 / B);
  } else if (disc >= 0.0) {
    at((-B + sqrt(disc)) / (2.0 * A));
    at((-B - sqrt(disc)) / (2.0 * A));
  }
  return m;
}

constexpr double kSlack = 1.0 + 1e-3;  // on the bounds, for rounding along the way

__device__ double first_scale(double rho) { return pow2_scale(rho * kSlack); }

// The scales of every step of one matrix; rho is |X_0|_F.
__device__ void scale_table(double rho, const PrepArgs& a, StepScale* out) {
  double bound = rho * kSlack;
  double sx = first_scale(rho);
  for (int k = 0; k < a.steps; ++k) {
    const double ca = a.coef[k][0], cb = a.coef[k][1], cc = a.coef[k][2];
    const double u = bound * bound;
    const double sa = pow2_scale(u);
    // |b u + c u^2| over [0, bound^2]
    double mb = fabs(u * (cb + cc * u));
    if (cc != 0.0) {
      const double peak = -cb / (2.0 * cc);
      if (peak > 0.0 && peak < u) mb = fmax(mb, fabs(peak * (cb + cc * peak)));
    }
    const double sb = pow2_scale(mb * kSlack);
    const double next = max_on(bound, ca, cb, cc) * kSlack;
    const double sn = k + 1 == a.steps ? 1.0 : pow2_scale(next);
    out[k].gram = (float)(sa / (sx * sx));
    out[k].square = (float)(cc * sb / (sa * sa));
    out[k].linear = (float)(cb * sb / sa);
    out[k].product = (float)(sn / (sb * sx));
    out[k].keep = (float)(ca * sn / sx);
    bound = next;
    sx = sn;
  }
}

constexpr int kTile = 64;
constexpr int kTilePitch = kTile + 1;

// X_0 in both orders, a 64 x 64 tile of G per CTA; the first CTA of a matrix writes its scales.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) ortho_split_kernel(const PrepArgs a) {
  __shared__ uint32_t tile[kTile * kTilePitch];  // hi in the low half, lo in the high half
  __shared__ double s_factor;
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const int64_t z = blockIdx.z;
  const int64_t i0 = (int64_t)blockIdx.y * kTile, j0 = (int64_t)blockIdx.x * kTile;
  // 8 columns of two rows a thread; the loads do not wait for the norm.
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
      const bool first = blockIdx.x == 0 && blockIdx.y == 0;
      const double rho = den > 0.0 ? norm / den : 0.0;
      s_factor = first_scale(rho) / den;
      if (first) scale_table(rho, a, a.scale + z * a.steps);
    }
  }
  __syncthreads();
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

// One matrix kept as hi and lo in both halves of a buffer.
struct Split {
  __half* hi;
  __half* lo;
  int64_t rows, cols, ld, matrix;
};

struct Layout {
  int64_t r, c;                 // X is r x c, r <= c
  int64_t ld_c, ld_r;
  size_t status, part, scale, x, xt0, xt1, a, b, end;
  int parts;
};

Layout layout_of(int64_t batch, int64_t rows, int64_t cols, int steps) {
  Layout L;
  L.r = std::min(rows, cols);
  L.c = std::max(rows, cols);
  L.ld_c = round_up(L.c, 32);
  L.ld_r = round_up(L.r, 32);
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
  L.scale = take(sizeof(StepScale) * batch * steps);
  const size_t x = sizeof(__half) * 2 * batch * L.r * L.ld_c, xt = sizeof(__half) * 2 * batch * L.c * L.ld_r;
  const size_t sq = sizeof(__half) * 2 * batch * L.r * L.ld_r;
  L.x = take(x);
  L.xt0 = take(xt);
  L.xt1 = take(xt);
  L.a = take(sq);
  L.b = take(sq);
  L.end = off;
  return L;
}

Split split_at(void* ws, size_t off, int64_t batch, int64_t rows, int64_t cols, int64_t ld) {
  Split s;
  s.hi = ws_at<__half>(ws, off);
  s.lo = s.hi + batch * rows * ld;
  s.rows = rows;
  s.cols = cols;
  s.ld = ld;
  s.matrix = rows * ld;
  return s;
}

int64_t tiles_of(int64_t M, int64_t N, int bn, int out_kind) {
  const int64_t m = ceil_div(M, kTileRows), n = ceil_div(N, bn);
  if (out_kind != kSymmetric) return m * n;
  int64_t t = 0;
  for (int64_t i = 0; i < m; ++i) t += std::min<int64_t>((kTileRows / bn) * (i + 1), n);
  return t;
}

// One product D = P Q^T of the iteration, apart from where D goes.
struct Operands {
  const Split* p;
  const Split* q;
};

template <int BN>
cudaError_t launch_iteration(IterArgs& it, const Operands* op, cudaStream_t stream) {
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
  int64_t most = 0;
  for (int p = 0; p < kProducts; ++p) {
    GemmArgs& a = it.gemm[p];
    const Split &l = *op[p].p, &r = *op[p].q;
    if (!make_tmap_f16(&it.map[p][0], l.hi, l.cols, l.rows, it.batch, l.ld, l.matrix, BK, 128) ||
        !make_tmap_f16(&it.map[p][1], l.lo, l.cols, l.rows, it.batch, l.ld, l.matrix, BK, 128) ||
        !make_tmap_f16(&it.map[p][2], r.hi, r.cols, r.rows, it.batch, r.ld, r.matrix, BK, PL::BROWS) ||
        !make_tmap_f16(&it.map[p][3], r.lo, r.cols, r.rows, it.batch, r.ld, r.matrix, BK, PL::BROWS))
      return cudaErrorInvalidValue;
    a.M = l.rows;
    a.N = r.rows;
    a.num_kc = (int)ceil_div(l.cols, BK);
    a.tiles_m = (int)ceil_div(a.M, kTileRows);
    a.tiles_n = (int)ceil_div(a.N, BN);
    const int64_t tiles = tiles_of(a.M, a.N, BN, a.out_kind);
    if (tiles * it.batch >= (int64_t(1) << 30)) return cudaErrorInvalidConfiguration;
    a.tiles = (int)tiles;
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

// The tile width with the least estimated time.  A slice of 64 costs a pair the larger of its 12 MMAs
// (6 BN cycles) and its operands' way into shared memory (64 bytes a cycle and CTA: 1024, 768 and 640
// cycles for BN = 256, 128 and 64); a product ends with an epilogue that nothing hides.
int tile_width(const IterArgs& it, const Operands* op) {
  const int64_t pairs = device_sm_count() / 2;
  int best = 0;
  int64_t least = 0;
  for (const int bn : {256, 128, 64}) {
    const int64_t slice = bn == 256 ? 1536 : bn == 128 ? 768 : 640;
    int64_t cost = 0;
    for (const int p : {kGram, kSquare, kProduct})
      cost += ceil_div(tiles_of(op[p].p->rows, op[p].q->rows, bn, it.gemm[p].out_kind) * it.batch, pairs) *
                  ceil_div(op[p].p->cols, BK) * slice + 32 * bn;
    if (best == 0 || cost < least) {
      best = bn;
      least = cost;
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
  StepScale* scale = ws_at<StepScale>(o.workspace, L.scale);
  const Split x = split_at(o.workspace, L.x, o.batch, L.r, L.c, L.ld_c);
  const Split xt = split_at(o.workspace, L.xt0, o.batch, L.c, L.r, L.ld_r);
  const Split xt_next = split_at(o.workspace, L.xt1, o.batch, L.c, L.r, L.ld_r);
  const Split ma = split_at(o.workspace, L.a, o.batch, L.r, L.r, L.ld_r);
  const Split mb = split_at(o.workspace, L.b, o.batch, L.r, L.r, L.ld_r);

  PrepArgs p{};
  p.g = o.update;
  p.rows = o.rows;
  p.cols = o.cols;
  p.row_stride = o.row_stride;
  p.matrix_stride = o.matrix_stride;
  p.dtype = o.dtype;
  p.tall = tall;
  p.parts = L.parts;
  p.steps = o.steps;
  p.eps = o.eps;
  for (int k = 0; k < o.steps; ++k)
    for (int e = 0; e < 3; ++e) p.coef[k][e] = o.coefficients[3 * k + e];
  p.part = ws_at<double>(o.workspace, L.part);
  p.scale = scale;
  const Split& g = tall ? xt : x;
  const Split& t = tall ? x : xt;
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
  auto by_pack = [&](auto t) {
    using T = decltype(t);
    constexpr int V = 16 / sizeof(T);
    return packs ? prep(ortho_norm_kernel<T, V>, ortho_split_kernel<T, V>)
                 : prep(ortho_norm_kernel<T, 1>, ortho_split_kernel<T, 1>);
  };
  cudaError_t e = o.dtype == LM_F32 ? by_pack(float{}) : o.dtype == LM_BF16 ? by_pack(__nv_bfloat16{}) : by_pack(__half{});
  if (e != cudaSuccess) return e;
  note_launches(2);

  IterArgs it{};
  it.scale = scale;
  it.arrived = reinterpret_cast<unsigned*>(status + 1);
  it.status = status;
  it.timeout_ns = wc.timeout_ns;
  it.steps = o.steps;
  it.batch = (int)o.batch;
  it.run = o.dtype == LM_F32 ? 4 : o.dtype == LM_F16 ? 16 : 32;
  it.debug_skip_first_load = wc.debug_skip_first_load;
  auto to = [](GemmArgs& a, int out_kind, int kind, const Split& d) {
    a.out_kind = out_kind;
    a.kind = kind;
    a.d_hi = d.hi;
    a.d_lo = d.lo;
    a.ld_d = d.ld;
    a.d_matrix = d.matrix;
  };
  auto add = [](GemmArgs& a, const Split& s) {
    a.add_hi = s.hi;
    a.add_lo = s.lo;
  };
  const Split xts[2] = {xt, xt_next};
  Operands op[kProducts];
  op[kGram] = {&x, &x};
  to(it.gemm[kGram], kSymmetric, 0, ma);
  op[kSquare] = {&ma, &ma};
  to(it.gemm[kSquare], kSymmetric, 1, mb);
  add(it.gemm[kSquare], ma);
  for (int b = 0; b < 2; ++b) {
    // X in place (each value is read by the thread that replaces it), X^T into the other buffer.
    GemmArgs& a = it.gemm[kProduct + b];
    op[kProduct + b] = {&mb, &xts[b]};
    to(a, kBoth, 2, x);
    add(a, x);
    a.t_hi = xts[1 - b].hi;
    a.t_lo = xts[1 - b].lo;
    a.ld_t = xts[1 - b].ld;
    a.t_matrix = xts[1 - b].matrix;
  }
  // The last product runs in the order that lets the lanes of a warp write the result's rows.
  const Split& last = xts[(o.steps - 1) & 1];
  GemmArgs& f = it.gemm[kLast];
  op[kLast] = tall ? Operands{&mb, &last} : Operands{&last, &mb};
  to(f, kFinal, 2, tall ? x : last);
  add(f, tall ? x : last);
  f.out = o.out;
  f.ld_out = o.cols;
  f.out_matrix = o.rows * o.cols;
  f.out_dtype = o.dtype;
  const int bn = tile_width(it, op);
  e = bn == 256 ? launch_iteration<256>(it, op, stream) : bn == 128 ? launch_iteration<128>(it, op, stream)
                                                                    : launch_iteration<64>(it, op, stream);
  if (e != cudaSuccess) return e;
  note_launches(1);
  return cudaGetLastError();
}

}  // namespace lm
}  // namespace rbf
