// Shared projection with low-rank adapters of many requests:
//   y[m] = [residual +] [gate *] act( W x[m] + bias + scale_a B_a (A_a x[m]) ),  a = ids(m)
// (rows whose id is outside [0, adapters) take the projection alone).  The
// projection is the reference's Linear::forward / ops::mul_mat_add
// (crate/runtime/nn_blocks.rs:82,179-195) with the element-wise ops of its
// blocks; the adapters have no counterpart there.
//
// Two launches.  shrink_kernel (shrink_tc_kernel for many rows) forms
// t[m] = scale_a A_a x[m] in f32 and stores it as two bf16 parts.
// lora_gemm_kernel then runs one product whose K axis is x's, followed by the
// ranks of the adapters that occur in a 128-row tile, 16 at a time: a slot multiplies the 128 x 16 piece of t, zero in the
// rows of other adapters, by the BN x 16 piece of B_a.  The zeros add nothing,
// so a row's result does not depend on its neighbours; and each B_a is read
// once per tile however many rows use it, which is all that a row-by-row
// batch has to read.
//
// lora_gemm_kernel is persistent, one block per SM, 128 x BN tiles, K in steps
// of 64 through a ring of shared-memory stages:
//   warp 0       TMA: x and W tiles (128B swizzle); in the slot stages the
//                B_a pieces (32-byte rows, 32B swizzle), up to four per stage;
//   warp 1       tcgen05.mma (M 128, N BN, K 16) into a double-buffered TMEM
//                accumulator;
//   warps 2..5   one row per thread: the tile's list of distinct adapters, and
//                the t pieces of the slot stages, written to shared memory;
//   warps 6..13  epilogue: TMEM lane quarter = warp % 4, half of the columns
//                each; bias, activation, gated residual, store.
// It is launched while shrink_kernel still runs (its x W^T part does not need
// t); the t warps wait for it.  Every mbarrier wait is bounded (%globaltimer,
// 2 s); on expiry the block records an error in the device's status word,
// stops issuing work and still releases its TMEM.
#include <type_traits>

#include "act.cuh"
#include "common.cuh"
#include "epilogue.cuh"
#include "tc.cuh"

namespace l3d {
namespace lora {

using namespace l3d::tc;

struct Params {
  int M, N, K, R, A;
  const __nv_bfloat16 *x, *a;
  int64_t x_ld, y_ld, res_ld;
  const float* scale;     // [A]
  const int32_t* ranks;   // [A] or null (= R)
  const void* ids;        // row m has id ids[m / per]
  int ids64, per;
  int x_rows;             // rows of an x tile that are loaded
  const void* bias;
  int bias_dtype, bias_vec;
  const void* gate;
  int gate_dtype;
  const void* res;
  int res_vec;
  void* y;
  int y_dtype, y_vec, act;
  __nv_bfloat16* t;       // [PARTS, M, R] scale_a A_a x[m] and its rounding error
  uint64_t wait_ns;
};

// t enters the second product as the sum of two bf16 numbers: one alone would
// be off by up to 2^-8 of B_a t, as much as the rounding of a bf16 y; the pair
// is off by 2^-16 and costs one more K-16 product per slot (4% at rank 64 and
// K = 1536).
constexpr int PARTS = 2;
// An infinite v, or one that bf16 rounds to infinity, has to leave the second part
// with no infinity of the other sign (or inf - inf): the first part ends at bf16's
// largest value, the second takes the rest (NaN and infinity among it).
__device__ __forceinline__ void split(float v, float& hi, float& lo) {
  constexpr float MOST = 0x1.fep127f;
  hi = __bfloat162float(__float2bfloat16_rn(fminf(fmaxf(v, -MOST), MOST)));
  lo = v - hi;
}

__device__ int g_lora_status;
constexpr int ST_TIMEOUT = 5;

__device__ __forceinline__ int adapter_of(const Params& p, int m) {
  const int g = m / p.per;
  const int64_t id = p.ids64 ? static_cast<const int64_t*>(p.ids)[g] : static_cast<const int32_t*>(p.ids)[g];
  return id >= 0 && id < p.A ? int(id) : -1;
}
// Rank of adapter a, and the slots of 16 ranks that it takes.  t is 0 in the ranks
// past its own: A's are 0 there, and 0 times an infinite x would be NaN.
__device__ __forceinline__ int rank_of(const Params& p, int a) {
  return p.ranks ? min(max(p.ranks[a], 0), p.R) : p.R;
}
__device__ __forceinline__ int slots_of(const Params& p, int a) { return (rank_of(p, a) + 15) / 16; }

// --------------------------------------------------------------------- shrink
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// t for a group of 16 rows: eight warps share K, interleaved in chunks of 32,
// and add up through shared memory in a fixed order.  A lane loads 8
// consecutive k of a row at once and uses them as the operands of two K-16
// products: both operands permute k alike, so the sums are the same and every
// load is 16 bytes.  blockIdx.y strides over the distinct adapters of the
// group, blockIdx.z over their ranks, 32 at a time.
__global__ void __launch_bounds__(256, 1) shrink_kernel(const Params p) {
  constexpr int ROWS = 16, NT = 4, RB = 32, WK = 8;
  __shared__ float red[WK][ROWS][RB + 4];
  __shared__ int s_id[ROWS], s_list[ROWS], s_wcount[8];
  asm volatile("griddepcontrol.launch_dependents;");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const int m0 = blockIdx.x * ROWS;
  // The distinct adapters of the group, in the order of their first rows.
  const int mine = tid < ROWS && m0 + tid < p.M ? adapter_of(p, m0 + tid) : -1;
  if (tid < ROWS) s_id[tid] = mine;
  __syncthreads();
  bool first = mine >= 0;
  for (int q = 0; first && q < tid; ++q) first = s_id[q] != mine;
  const uint32_t firsts = __ballot_sync(0xffffffffu, first);
  if (lane == 0) s_wcount[warp] = __popc(firsts);
  __syncthreads();
  int before = 0, count = 0;
#pragma unroll
  for (int w = 0; w < (ROWS + 31) / 32; ++w) {
    if (w < warp) before += s_wcount[w];
    count += s_wcount[w];
  }
  if (first) s_list[before + __popc(firsts & ((1u << lane) - 1))] = mine;
  __syncthreads();
  const __nv_bfloat16* xr[2];
  bool xok[2];
#pragma unroll
  for (int hf = 0; hf < 2; ++hf) {
    const int m = m0 + hf * 8 + g;
    xok[hf] = m < p.M;
    xr[hf] = p.x + int64_t(xok[hf] ? m : 0) * p.x_ld + 8 * t4;
  }
  const int chunks = (p.K + 31) / 32;
  for (int d = blockIdx.y; d < count; d += gridDim.y) {
    const int a = s_list[d];
    const int own = rank_of(p, a), rank = (own + 15) / 16 * 16;
    for (int r0 = blockIdx.z * RB; r0 < rank; r0 += gridDim.z * RB) {
      const int nt = min((rank - r0) / 8, NT);  // 8-rank tiles
      float c[NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) c[j][e] = 0.f;
      const __nv_bfloat16* ar = p.a + (int64_t(a) * p.R + r0 + g) * p.K + 8 * t4;
#pragma unroll 4
      for (int kc = warp; kc < chunks; kc += WK) {
        const int k = kc * 32;
        const bool kok = k + 8 * t4 < p.K;
        uint4 xv[2], av[NT];
        const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
          xv[hf] = kok && xok[hf] ? __ldg(reinterpret_cast<const uint4*>(xr[hf] + k)) : zero;
#pragma unroll
        for (int j = 0; j < NT; ++j)
          av[j] = kok && j < nt ? __ldg(reinterpret_cast<const uint4*>(ar + int64_t(8 * j) * p.K + k)) : zero;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          if (j < nt) {
            mma_16816(c[j], xv[0].x, xv[1].x, xv[0].y, xv[1].y, av[j].x, av[j].y);
            mma_16816(c[j], xv[0].z, xv[1].z, xv[0].w, xv[1].w, av[j].z, av[j].w);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int col = j * 8 + 2 * t4;
        *reinterpret_cast<float2*>(&red[warp][g][col]) = make_float2(c[j][0], c[j][1]);
        *reinterpret_cast<float2*>(&red[warp][g + 8][col]) = make_float2(c[j][2], c[j][3]);
      }
      __syncthreads();
      const float sc = p.scale[a];
      for (int e = tid; e < ROWS * RB; e += 256) {
        const int row = e / RB, col = e % RB;
        if (s_id[row] != a || r0 + col >= rank) continue;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < WK; ++w) v += red[w][row][col];
        v = r0 + col < own ? v * sc : 0.f;
        const int64_t at = int64_t(m0 + row) * p.R + r0 + col;
        float hi, lo;
        split(v, hi, lo);
        p.t[at] = __float2bfloat16_rn(hi);
        p.t[int64_t(p.M) * p.R + at] = __float2bfloat16_rn(lo);
      }
      __syncthreads();
    }
  }
}

// t for many rows, on the 5th-generation tensor cores: a block per 128-row tile,
// two blocks per SM, and for each distinct adapter of the tile one product of
// the tile with A_a (M 128, N R, K in steps of 64 by TMA).  31569 x 1536, rank
// 64: about 20 us, and 70 by mma.sync (its loads, straight to registers, are the limit).
//   warp 0 TMA, warp 1 MMA, warps 2..5 the tile's adapters and the epilogue
struct ShrinkTc {
  int stages, tmem;
};
constexpr int SHRINK_THREADS = 6 * 32;
__device__ __forceinline__ void umma_f16_rt(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
      : "memory");
}

__global__ void __launch_bounds__(SHRINK_THREADS, 2)
    shrink_tc_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_a,
                     const Params p, const ShrinkTc sc) {
  constexpr int BM = 128, BK = 64, X_BYTES = BM * BK * 2;
  int* const status = &g_lora_status;
  extern __shared__ __align__(1024) uint8_t smem[];  // no static shared memory: 1024-byte aligned
  const int a_bytes = p.R * BK * 2, stage_bytes = X_BYTES + a_bytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + sc.stages * stage_bytes);
  uint64_t* full = bars;                 // [stages]
  uint64_t* empty = full + sc.stages;    // [stages]
  uint64_t* acc_full = empty + sc.stages;
  uint64_t* acc_free = acc_full + 1;
  uint64_t* drain = acc_free + 1;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(drain + 1);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1) + 1;
  int* ids = reinterpret_cast<int*>(bars + 32);  // [BM]
  int* list = ids + BM;                          // [BM] the distinct adapters, by their first rows
  int* firsts = list + BM;                       // [4]
  asm volatile("griddepcontrol.launch_dependents;");
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int m0 = blockIdx.x * BM, kblocks = (p.K + BK - 1) / BK;
  if (threadIdx.x == 0) {
    for (int s = 0; s < sc.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(acc_free, 4);
    mbar_init(drain, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(sc.tmem));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  const int r = threadIdx.x - 64;  // row of warps 2..5
  int mine = -1, place = 0;
  bool first = false;
  if (warp >= 2) {
    mine = m0 + r < p.M ? adapter_of(p, m0 + r) : -1;
    ids[r] = mine;
  }
  __syncthreads();
  if (warp >= 2) {
    const uint32_t same = __match_any_sync(0xffffffffu, mine);
    first = mine >= 0 && (same & ((1u << lane) - 1)) == 0;
    for (int q = 0; first && q < (r & ~31); ++q) first = ids[q] != mine;
    const uint32_t mask = __ballot_sync(0xffffffffu, first);
    place = __popc(mask & ((1u << lane) - 1));
    if (lane == 0) firsts[warp - 2] = __popc(mask);
  }
  __syncthreads();
  int count = 0;
  for (int w = 0; w < 4; ++w) {
    if (w < warp - 2) place += firsts[w];
    count += firsts[w];
  }
  if (first) list[place] = mine;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  auto wait_warp = [&](uint64_t* bar, uint32_t parity) {
    const bool got = __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status, ST_TIMEOUT, p.wait_ns)) != 0;
    __syncwarp();
    return got;
  };
  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      for (int d = 0; ok && d < count; ++d)
        for (int kb = 0; kb < kblocks; ++kb, ++it) {
          const int s = it % sc.stages;
          if (it >= sc.stages &&
              !mbar_wait(&empty[s], (it / sc.stages - 1) & 1, abort_flag, status, ST_TIMEOUT, p.wait_ns)) {
            ok = false;
            break;
          }
          mbar_expect_tx(&full[s], uint32_t(stage_bytes));
          tma_load_2d(smem + s * stage_bytes, &map_x, &full[s], kb * BK, m0);
          tma_load_2d(smem + s * stage_bytes + X_BYTES, &map_a, &full[s], kb * BK, list[d] * p.R);
        }
    }
  } else if (warp == 1) {
    const bool leader = elect_one();
    const uint32_t idesc = make_idesc(BM, p.R);
    int it = 0;
    bool ok = true;
    for (int d = 0; ok && d < count; ++d) {
      if (d > 0) ok = wait_warp(acc_free, (d - 1) & 1);
      tc_fence_after();
      for (int kb = 0; ok && kb < kblocks; ++kb, ++it) {
        const int s = it % sc.stages;
        ok = wait_warp(&full[s], (it / sc.stages) & 1);
        if (!ok) break;
        tc_fence_after();
        const uint64_t da = smem_desc_sw128(smem + s * stage_bytes);
        const uint64_t db = smem_desc_sw128(smem + s * stage_bytes + X_BYTES);
        if (leader) {
#pragma unroll
          for (int k = 0; k < BK / 16; ++k)
            umma_f16_rt(tmem_base, da + uint64_t(2 * k), db + uint64_t(2 * k), idesc, (kb | k) ? 1u : 0u);
          umma_commit(&empty[s]);
        }
      }
      if (ok && leader) umma_commit(acc_full);
    }
  } else {
    const int quarter = warp & 3, row = quarter * 32 + lane, m = m0 + row;
    const int a_row = ids[row];
    for (int d = 0; d < count; ++d) {
      if (!wait_warp(acc_full, d & 1)) break;
      tc_fence_after();
      const int a = list[d], rank = rank_of(p, a);
      const float scale = p.scale[a];
      for (int c = 0; c < rank; c += 16) {
        float v[16];
        tmem_ld16(tmem_base + (uint32_t(quarter * 32) << 16) + uint32_t(c), v);
        if (a_row == a) {
          uint4 u[PARTS][2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float hi[8], lo[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) split(c + 8 * h + e < rank ? v[8 * h + e] * scale : 0.f, hi[e], lo[e]);
            u[0][h] = pack(hi, __nv_bfloat16());
            u[1][h] = pack(lo, __nv_bfloat16());
          }
#pragma unroll
          for (int part = 0; part < PARTS; ++part) {
            uint4* dst = reinterpret_cast<uint4*>(p.t + (int64_t(part) * p.M + m) * p.R + c);
            dst[0] = u[part][0];
            dst[1] = u[part][1];
          }
        }
        __syncwarp();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_free);
    }
  }
  // Teardown: after an abort, wait (bounded) for the MMAs this block issued,
  // and give TMA loads still in flight 1 ms to land.
  tc_fence_before();
  __syncthreads();
  if (*abort_flag && warp == 1 && elect_one()) {
    umma_commit(drain);
    mbar_drain(drain, 0, p.wait_ns);
    const uint64_t t0 = globaltimer();
    while (globaltimer() - t0 < 1000000ull) {
    }
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(sc.tmem));
  }
}

// ----------------------------------------------------------------------- gemm
constexpr int BM = 128, BK = 64;
constexpr int A_BYTES = BM * BK * 2;
constexpr int SLOT_A = BM * 32;          // a t piece: 128 rows of 32 bytes
constexpr int THREADS = 14 * 32;

template <int BN>
struct Cfg {
  // Blocks of 64 along K per stage: two for the narrow tiles of few rows, which
  // wait for memory (whole 256-byte pieces of a weight row, half the barriers):
  // 16 x 2048 -> 2048 10.1 us, one 12.4; 64 x 2048 -> 8192 27.3 us, one 30.4.
  static constexpr int KS = BN <= 64 ? 2 : 1;
  static constexpr int A_STAGE = KS * A_BYTES;
  static constexpr int B_BYTES = BN * BK * 2;
  static constexpr int B_STAGE = KS * B_BYTES;
  static constexpr int SLOT_B = BN * 32;
  static constexpr int PER_STAGE = A_STAGE / (PARTS * SLOT_A);  // slots of a stage
  static constexpr int NST = BN == 256 || BN == 64 ? 4 : BN == 128 ? 6 : 5;
  static constexpr int LISTS = 2 * (2 * BM + 1) * 4 + BM * 4 + 64;
  static constexpr int STG = 8 * 32 * 17 * 4;  // per epilogue warp: 32 rows x 16 columns, padded
  static constexpr int SMEM = NST * (A_STAGE + B_STAGE) + 512 + LISTS + STG;
  static constexpr int TMEM = 2 * BN < 32 ? 32 : 2 * BN;  // a power of two
  static_assert(SMEM <= 227 * 1024, "shared memory budget");
  static_assert((4 * NST + 9) * 8 + 16 <= 512, "barrier area");
};

// K-major operand of 32-byte rows, 32B-swizzled: 8-row groups 256 B apart.
__device__ __forceinline__ uint64_t smem_desc_sw32(const void* tile) {
  const uint64_t addr = smem_u32(tile);
  uint64_t d = 0;
  d |= (addr >> 4) & 0x3fffull;
  d |= uint64_t(1) << 16;
  d |= uint64_t(256 >> 4) << 32;
  d |= uint64_t(1) << 46;
  d |= uint64_t(6) << 61;                // SWIZZLE_32B
  return d;
}

// RES: there is a residual (kept out of the registers of the other form, which
// would spill).  Bound for few rows by one block's chain of steps: 64 x 2048 ->
// 8192 takes 13.6 us without adapters (the weight alone 5 us at the copy rate), 28
// with 32 of them, since the slot stages, some 17 here, each fetch their pieces of t
// from L2 after a wait for a free stage, and begin when shrink_kernel (9 us) is done;
// for many rows by the loads of a K step, 48 KB from L2 for 512 clocks of products: the
// tensor pipe is 64% busy, which is 63 bytes per clock and SM.  31569 x 1536 -> 8192,
// rank 64 takes 701 to 711 us in all by graph replay after a pause (1145 TFLOP/s, 69% of
// a plain product's rate), 780 to 830 in a loop, at the clock that the power limit leaves.
template <int BN, bool RES>
__global__ void __launch_bounds__(THREADS, 1)
    lora_gemm_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                     const __grid_constant__ CUtensorMap map_b, const Params p) {
  using C = Cfg<BN>;
  constexpr int NST = C::NST, PER_STAGE = C::PER_STAGE;
  constexpr uint32_t IDESC = make_idesc(BM, BN);
  int* const status = &g_lora_status;
  extern __shared__ __align__(1024) uint8_t smem[];  // no static shared memory: 1024-byte aligned
  uint8_t* sa = smem;
  uint8_t* sb = sa + NST * C::A_STAGE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sb + NST * C::B_STAGE);
  uint64_t* full = bars;                 // [NST] TMA landed
  uint64_t* empty = full + NST;          // [NST] MMA has read the stage
  uint64_t* tgo = empty + NST;           // [NST] the stage is free for t pieces
  uint64_t* tfull = tgo + NST;           // [NST] the t pieces of a slot stage are written
  uint64_t* acc_full = tfull + NST;      // [2]
  uint64_t* acc_empty = acc_full + 2;    // [2]
  uint64_t* list_full = acc_empty + 2;   // [2]
  uint64_t* list_empty = list_full + 2;  // [2]
  uint64_t* drain = list_empty + 2;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(drain + 1);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1) + 1;
  // Adapters of the rows of the tile; per tile parity the distinct ones, in the
  // order of their first rows, the end of each one's slots, and their number.
  int* ids = reinterpret_cast<int*>(bars + 64);
  int* list_id = ids + BM;               // [2][BM]
  int* list_end = list_id + 2 * BM;      // [2][BM] slots up to and with this adapter
  int* total = list_end + 2 * BM;        // [2]
  int* wsum = total + 2;                 // [8] per-warp sums of the list builders
  float* stg = reinterpret_cast<float*>(wsum + 8);  // [8][32][17] epilogue staging

  // (The shuffle tells the compiler that the role is the same in all lanes.)
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int num_n = (p.N + BN - 1) / BN;
  const int tiles = ((p.M + BM - 1) / BM) * num_n;
  const int kblocks = (p.K + C::KS * BK - 1) / (C::KS * BK);
  if (threadIdx.x == 0) {
    for (int s = 0; s < NST; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
      mbar_init(&tgo[s], 1);
      mbar_init(&tfull[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 8);
      mbar_init(&list_full[i], 4);
      mbar_init(&list_empty[i], 2);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(C::TMEM));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    return mbar_wait(bar, parity, abort_flag, status, ST_TIMEOUT, p.wait_ns);
  };

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      int it = 0;  // ring position
      bool ok = true;
      int nt = 0;
      const uint32_t x_bytes = uint32_t(p.x_rows) * (BK * 2);
      for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x, ++nt) {
        const int m0 = (tile / num_n) * BM, n0 = (tile % num_n) * BN;
        for (int kb = 0; kb < kblocks; ++kb, ++it) {
          const int s = it % NST;
          if (it >= NST && !wait(&empty[s], (it / NST - 1) & 1)) { ok = false; break; }
          mbar_expect_tx(&full[s], C::KS * (x_bytes + C::B_BYTES));
#pragma unroll
          for (int i = 0; i < C::KS; ++i) {  // (blocks past K read as zero)
            const int k = (kb * C::KS + i) * BK;
            tma_load_2d(sb + s * C::B_STAGE + i * C::B_BYTES, &map_w, &full[s], k, n0);
            tma_load_2d(sa + s * C::A_STAGE + i * A_BYTES, &map_x, &full[s], k, m0);
          }
        }
        const int lb = nt & 1;
        if (!ok || !wait(&list_full[lb], (nt >> 1) & 1)) break;
        const int slots = total[lb];
        int d = 0, first = 0;  // adapter of the slot, its first slot
        for (int q0 = 0; q0 < slots; q0 += PER_STAGE, ++it) {
          const int s = it % NST, n = min(PER_STAGE, slots - q0);
          if (it >= NST && !wait(&empty[s], (it / NST - 1) & 1)) { ok = false; break; }
          mbar_arrive(&tgo[s]);
          mbar_expect_tx(&full[s], n * C::SLOT_B);
          for (int q = q0; q < q0 + n; ++q) {
            while (q >= list_end[lb * BM + d]) first = list_end[lb * BM + d++];
            tma_load_3d(sb + s * C::B_STAGE + (q - q0) * C::SLOT_B, &map_b, &full[s], (q - first) * 16,
                        n0, list_id[lb * BM + d]);
          }
        }
        mbar_arrive(&list_empty[lb]);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA
    // The whole warp keeps step and one elected lane issues, so that loop state
    // and descriptors stay in uniform registers.
    const bool leader = elect_one();
    auto wait_warp = [&](uint64_t* bar, uint32_t parity) {
      return __all_sync(0xffffffffu, wait(bar, parity)) != 0;
    };
    int it = 0, nt = 0;
    uint32_t tph = 0;  // parity of each stage's next tfull phase
    bool ok = true;
    for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x, ++nt) {
      const int acc = nt & 1;
      if (nt >= 2 && !wait_warp(&acc_empty[acc], (nt / 2 - 1) & 1)) break;
      tc_fence_after();
      const uint32_t d = tmem_base + uint32_t(acc * BN);
      for (int kb = 0; kb < kblocks; ++kb, ++it) {
        const int s = it % NST;
        if (!wait_warp(&full[s], (it / NST) & 1)) { ok = false; break; }
        tc_fence_after();
        const uint64_t da = smem_desc_sw128(sa + s * C::A_STAGE), db = smem_desc_sw128(sb + s * C::B_STAGE);
        if (leader) {
#pragma unroll
          for (int k = 0; k < C::KS * BK / 16; ++k)
            umma_f16<IDESC>(d, da + uint64_t((k >> 2) * (A_BYTES >> 4) + 2 * (k & 3)),
                            db + uint64_t((k >> 2) * (C::B_BYTES >> 4) + 2 * (k & 3)), (kb | k) ? 1u : 0u);
          umma_commit(&empty[s]);
        }
      }
      if (!ok || !wait_warp(&list_full[acc], (nt >> 1) & 1)) break;
      const int slots = total[acc];
      __syncwarp();
      if (leader) mbar_arrive(&list_empty[acc]);
      for (int q0 = 0; q0 < slots; q0 += PER_STAGE, ++it) {
        const int s = it % NST, n = min(PER_STAGE, slots - q0);
        ok = wait_warp(&full[s], (it / NST) & 1) && wait_warp(&tfull[s], (tph >> s) & 1);
        if (!ok) break;
        tph ^= 1u << s;
        tc_fence_after();
        if (leader) {
          for (int q = 0; q < n; ++q) {
            const uint64_t db = smem_desc_sw32(sb + s * C::B_STAGE + q * C::SLOT_B);
#pragma unroll
            for (int part = 0; part < PARTS; ++part)
              umma_f16<IDESC>(d, smem_desc_sw32(sa + s * C::A_STAGE + (q * PARTS + part) * SLOT_A), db, 1u);
          }
          umma_commit(&empty[s]);
        }
      }
      if (ok && leader) umma_commit(&acc_full[acc]);
    }
  } else if (warp < 6) {
    // -------------------------------------- adapter lists and t pieces
    const int r = threadIdx.x - 64;  // row of the tile
    // (The stage of a t piece is signalled by the producer: a wait on `empty`
    // from here could be more than one phase ahead of it.)
    int it = 0, nt = 0;
    uint32_t tph = 0;  // parity of each stage's next tgo phase
    bool ok = true, arrived = false;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++nt) {
      const int m = (tile / num_n) * BM + r, lb = nt & 1;
      const int a = m < p.M ? adapter_of(p, m) : -1;
      if (nt >= 2) ok = wait(&list_empty[lb], (nt / 2 - 1) & 1) && ok;
      ids[r] = a;
      // The first row of each adapter takes a place; ends are running sums.
      const uint32_t same = __match_any_sync(0xffffffffu, a);
      // All four warps leave together when a wait of any has run out.
      uint32_t all_ok;
      asm volatile(
          "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
          "bar.red.and.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
          : "=r"(all_ok)
          : "r"(uint32_t(ok))
          : "memory");
      if (!all_ok) break;
      bool first = a >= 0 && (same & ((1u << lane) - 1)) == 0;
      for (int q = 0; first && q < (r & ~31); ++q) first = ids[q] != a;
      const uint32_t mask = __ballot_sync(0xffffffffu, first);
      int n = first ? slots_of(p, a) : 0;
      int sum = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
      }
      if (lane == 31) {
        wsum[warp - 2] = sum;
        wsum[4 + warp - 2] = __popc(mask);
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
      int base = 0, place = __popc(mask & ((1u << lane) - 1)), all = 0;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        if (w < warp - 2) { base += wsum[w]; place += wsum[4 + w]; }
        all += wsum[w];
      }
      if (first) {
        list_id[lb * BM + place] = a;
        list_end[lb * BM + place] = base + sum;
      }
      if (r == 0) total[lb] = all;
      // The adapters of this lane's rows, read before the four warps part: one that
      // has no slot stage of this tile goes on and writes the next tile's ids.
      int ad[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) ad[i] = ids[lane + 32 * i];
      asm volatile("bar.sync 1, 128;" ::: "memory");
      if (lane == 0) mbar_arrive(&list_full[lb]);
      it += kblocks;
      if (all > 0 && !arrived) {
        asm volatile("griddepcontrol.wait;" ::: "memory");  // shrink_kernel's t
        arrived = true;
      }
      // Stage s belongs to warp 2 + s % 4, which writes all rows of its t pieces
      // (four per lane): four stages' loads of t are in flight at once, and a
      // warp meets the phases of its stages' tgo in order.
      const int m0 = (tile / num_n) * BM, rows = min(p.M - m0, BM);
      int d = 0, start = 0;
      for (int q0 = 0; q0 < all; q0 += PER_STAGE, ++it) {
        const int s = it % NST, cnt = min(PER_STAGE, all - q0);
        const uint32_t ph = (tph >> s) & 1;
        tph ^= 1u << s;
        if ((s & 3) != warp - 2) {
          for (int q = q0; q < q0 + cnt; ++q)
            while (q >= list_end[lb * BM + d]) start = list_end[lb * BM + d++];
          continue;
        }
        if (ok) ok = __all_sync(0xffffffffu, wait(&tgo[s], ph)) != 0;
        if (!ok) continue;
        for (int q = 0; q < cnt; ++q) {
          while (q0 + q >= list_end[lb * BM + d]) start = list_end[lb * BM + d++];
          const int a_q = list_id[lb * BM + d], c_q = (q0 + q - start) * 16;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = lane + 32 * i;
            if (row >= rows) continue;  // (rows past M: their products are not stored)
            const int sw = ((row >> 2) & 1) << 4;
#pragma unroll
            for (int part = 0; part < PARTS; ++part) {
              uint8_t* dst = sa + s * C::A_STAGE + (q * PARTS + part) * SLOT_A + row * 32;
              if (ad[i] == a_q) {
                const __nv_bfloat16* src = p.t + (int64_t(part) * p.M + m0 + row) * p.R + c_q;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst + sw)), "l"(src) : "memory");
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst + (16 ^ sw))), "l"(src + 8)
                             : "memory");
              } else {
                *reinterpret_cast<uint4*>(dst) = make_uint4(0, 0, 0, 0);
                *reinterpret_cast<uint4*>(dst + 16) = make_uint4(0, 0, 0, 0);
              }
            }
          }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&tfull[s]);
      }
    }
    // Where no row has an adapter nothing above has waited: without this, the end of
    // this kernel would not say that shrink_kernel has read ids (and x) to the end.
    if (!arrived) asm volatile("griddepcontrol.wait;" ::: "memory");
  } else {
    // ------------------------------------------------------------- epilogue
    const int quarter = warp & 3, half = (warp - 6) >> 2;
    // 32-column chunks of this warp: [c_lo, c_hi).
    const int c_lo = BN >= 64 ? half * (BN / 2) : half * 32;
    const int c_hi = BN >= 64 ? c_lo + BN / 2 : min(c_lo + 32, BN);
    const bool vec = p.y_vec && (!RES || p.res_vec);
    int nt = 0;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++nt) {
      const int m0 = (tile / num_n) * BM, n0 = (tile % num_n) * BN, acc = nt & 1;
      // The residual of the tile is brought to L2 while the products run.
      const int row = m0 + quarter * 32 + lane;
      if (RES && row < p.M) {
        const int es = p.y_dtype == L3D_BF16 ? 2 : 4;
        const char* rr = static_cast<const char*>(p.res) + (int64_t(row) * p.res_ld + n0) * es;
        const int end = min(c_hi, p.N - n0) * es;
        for (int b = c_lo * es; b < end; b += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(rr + b));
      }
      if (!__all_sync(0xffffffffu, mbar_wait_idle(&acc_full[acc], (nt / 2) & 1, abort_flag, status,
                                                   ST_TIMEOUT, p.wait_ns)))
        break;
      __syncwarp();
      tc_fence_after();
      const uint32_t ta = tmem_base + uint32_t(acc * BN) + (uint32_t(quarter * 32) << 16);
#pragma unroll 1
      for (int c = c_lo; c < c_hi; c += 32) {
        const int col0 = n0 + c;
        if (col0 >= p.N) break;
        const bool whole = vec && col0 + 32 <= p.N, bf = p.y_dtype == L3D_BF16;
        // The residual is read before the accumulator, without branches between
        // its loads: its latency is that of one load.
        uint4 u[4];
        if (RES && whole && bf && row < p.M) {
          const uint4* src = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.res) +
                                                            int64_t(row) * p.res_ld + col0);
#pragma unroll
          for (int q = 0; q < 4; ++q) u[q] = src[q];
        }
        __syncwarp();  // the load from tensor memory is the whole warp's
        float v[32];
        tmem_ld32(ta + uint32_t(c), v);
        if (p.bias) gemm::add_bias<32>(p, col0, v);
        if (p.act) gemm::epi_act<32, true>(p.act, bf, v);
        if (whole) {
          // Aligned rows: 64 (or 128) consecutive bytes of a row per thread.
          if (RES && p.gate) gemm::mul_gate<32>(p, col0, v);
          if (row < p.M) {
            if (bf) {
              __nv_bfloat16* yr = static_cast<__nv_bfloat16*>(p.y) + int64_t(row) * p.y_ld + col0;
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                float (&f)[8] = *reinterpret_cast<float(*)[8]>(&v[8 * q]);
                if constexpr (RES) {
                  float r[8];
                  unpack(u[q], r, __nv_bfloat16());
#pragma unroll
                  for (int e = 0; e < 8; ++e) f[e] += r[e];
                }
                *reinterpret_cast<uint4*>(yr + q * 8) = pack(f, __nv_bfloat16());
              }
            } else {
              float* yr = static_cast<float*>(p.y) + int64_t(row) * p.y_ld + col0;
              if constexpr (RES) {
                const float4* src = reinterpret_cast<const float4*>(static_cast<const float*>(p.res) +
                                                                    int64_t(row) * p.res_ld + col0);
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                  const float4 t = src[q];
                  v[4 * q] += t.x; v[4 * q + 1] += t.y; v[4 * q + 2] += t.z; v[4 * q + 3] += t.w;
                }
              }
#pragma unroll
              for (int q = 0; q < 8; ++q)
                *reinterpret_cast<float4*>(yr + q * 4) =
                    make_float4(v[q * 4], v[q * 4 + 1], v[q * 4 + 2], v[q * 4 + 3]);
            }
          }
        } else {
          // Any alignment, and the last columns: through shared memory, so that
          // a half warp reads and writes 16 consecutive elements of a row.
          // (Places outside the matrix read its last element: no branches.)
          float* st = stg + (warp - 6) * (32 * 17);
#pragma unroll
          for (int hc = 0; hc < 32; hc += 16) {
            const int col = col0 + hc + (lane & 15), cc = min(col, p.N - 1);
            auto row_of = [&](int i) { return m0 + quarter * 32 + 2 * i + (lane >> 4); };
            float r[16];
            if (RES && bf) {
#pragma unroll
              for (int i = 0; i < 16; ++i)
                r[i] = to_f(static_cast<const __nv_bfloat16*>(p.res)[int64_t(min(row_of(i), p.M - 1)) * p.res_ld + cc]);
            } else if (RES) {
#pragma unroll
              for (int i = 0; i < 16; ++i)
                r[i] = static_cast<const float*>(p.res)[int64_t(min(row_of(i), p.M - 1)) * p.res_ld + cc];
            }
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 16; ++e) st[lane * 17 + e] = v[hc + e];
            __syncwarp();
            if (col >= p.N) continue;
            const float g = !RES || !p.gate ? 1.f
                            : p.gate_dtype == L3D_F32
                                ? static_cast<const float*>(p.gate)[col]
                                : __bfloat162float(static_cast<const __nv_bfloat16*>(p.gate)[col]);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int m = row_of(i);
              if (m >= p.M) continue;
              float o = st[(2 * i + (lane >> 4)) * 17 + (lane & 15)];
              if (RES) o = fmaf(g, o, r[i]);
              if (bf) static_cast<__nv_bfloat16*>(p.y)[int64_t(m) * p.y_ld + col] = __float2bfloat16_rn(o);
              else static_cast<float*>(p.y)[int64_t(m) * p.y_ld + col] = o;
            }
          }
        }
        __syncwarp();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[acc]);
    }
  }

  // Teardown: after an abort, wait (bounded) for the MMAs this block issued,
  // and give TMA loads still in flight 1 ms to land.
  tc_fence_before();
  __syncthreads();
  if (*abort_flag && warp == 1 && elect_one()) {  // the lane that issued
    umma_commit(drain);
    mbar_drain(drain, 0, p.wait_ns);
    const uint64_t t0 = globaltimer();
    while (globaltimer() - t0 < 1000000ull) {
    }
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base),
                 "r"(C::TMEM));
  }
}

// ------------------------------------------------------------------------ host
// bf16 [rows, cols], row stride ld elements; box 64 columns x box_rows, 128B swizzle.
static bool make_map2(CUtensorMap* m, const void* base, uint64_t rows, uint64_t cols, uint64_t ld,
                      uint32_t box_rows) {
  auto fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {cols, rows};
  const cuuint64_t strides[1] = {ld * 2};
  const cuuint32_t box[2] = {uint32_t(BK), box_rows};
  const cuuint32_t es[2] = {1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, es,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// lora_b [A, n, R]: box 16 ranks x box_rows x 1, 32B swizzle (rows past n read as zero).
static bool make_map_b(CUtensorMap* m, const void* base, uint64_t A, uint64_t n, uint64_t R,
                       uint32_t box_rows) {
  auto fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[3] = {R, n, A};
  const cuuint64_t strides[2] = {R * 2, n * R * 2};
  const cuuint32_t box[3] = {16u, box_rows, 1u};
  const cuuint32_t es[3] = {1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, es,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_32B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int BN, bool RES>
static cudaError_t launch_gemm(const CUtensorMap& mx, const void* w, int64_t w_ld, const void* b,
                               const Params& p, cudaStream_t s) {
  auto k = lora_gemm_kernel<BN, RES>;
  cudaError_t e = set_smem_limit(reinterpret_cast<const void*>(k), Cfg<BN>::SMEM);
  if (e != cudaSuccess) return e;
  CUtensorMap mw, mb;
  if (!make_map2(&mw, w, uint64_t(p.N), uint64_t(p.K), uint64_t(w_ld), BN) ||
      !make_map_b(&mb, b, uint64_t(p.A), uint64_t(p.N), uint64_t(p.R), BN))
    return cudaErrorInvalidValue;
  const int64_t tiles = int64_t((p.M + BM - 1) / BM) * ((p.N + BN - 1) / BN);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(tiles < sm_count() ? tiles : sm_count()));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = Cfg<BN>::SMEM;
  cfg.stream = s;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k, mx, mw, mb, p);
}

// The tile width with the least estimated time: rounds of the device x the K
// steps of a tile, each as long as its products (2 BN clocks) or its loads.
// Measured (us) for widths 32, 64, 128, 256:
//   16 x 2048 -> 2048     10.1   10.3   12.9   16.1     64 x 2048 -> 8192  42.6  27.3  28.9  35.7
//   512 x 1024 -> 4096    25.4   20.0   17.7   21.5   4098 x 2048 -> 2048  94.2  64.7  53.1  47.1
//   31569 x 1536 -> 8192  1834   1114    827    705
static int pick_bn(int64_t M, int64_t N) {
  const int sms = sm_count();
  int best = 256;
  double least = 1e300;
  for (int bn = 256; bn >= 32; bn /= 2) {
    const int64_t tiles = ((M + BM - 1) / BM) * ((N + bn - 1) / bn);
    const double rounds = double((tiles + sms - 1) / sms);
    const double step = 2.0 * bn > 200 + 1.0 * bn ? 2.0 * bn : 200 + 1.0 * bn;
    if (rounds * step < least * 0.999) {
      least = rounds * step;
      best = bn;
    }
  }
  return best;
}

cudaError_t status_read(int* status, int reset) {
  cudaError_t e = cudaMemcpyFromSymbol(status, g_lora_status, sizeof(int));
  if (e == cudaSuccess && reset) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_lora_status, &zero, sizeof(int));
  }
  return e;
}

}  // namespace lora
}  // namespace l3d

using namespace l3d;

extern "C" size_t l3d_lora_linear_workspace_size(int64_t m, int64_t r) {
  if (m < 0 || r < 0) return 0;
  return size_t(m) * size_t(r) * 4 + 256;  // A x in bf16, and its rounding error
}

extern "C" int l3d_lora_linear(const l3d_tensor* x, const l3d_tensor* weight,
                               const l3d_tensor* bias, const l3d_tensor* lora_a,
                               const l3d_tensor* lora_b, const l3d_tensor* lora_scale,
                               const l3d_tensor* ranks, const l3d_tensor* ids, int act,
                               const l3d_tensor* residual, const l3d_tensor* gate,
                               const l3d_tensor* y, void* workspace, size_t workspace_bytes,
                               l3d_stream stream) {
  using namespace l3d::lora;
  const char* op = "l3d_lora_linear";
  const struct { const l3d_tensor* t; const char* name; int ndim; } need[] = {
      {x, "x", 0}, {weight, "weight", 2}, {lora_a, "lora_a", 3}, {lora_b, "lora_b", 3},
      {lora_scale, "lora_scale", 1}, {ids, "ids", 1}, {y, "y", 0}};
  for (const auto& e : need) {
    if (!e.t) return fail(L3D_E_NULL, "%s: %s is required", op, e.name);
    if (no_data(e.t)) return fail(L3D_E_NULL, "%s: %s has a null data pointer", op, e.name);
    if (e.ndim ? e.t->ndim != e.ndim : (e.t->ndim < 1 || e.t->ndim > L3D_MAX_DIMS))
      return fail(L3D_E_SHAPE, "%s: %s has a wrong rank", op, e.name);
  }
  if (x->dtype != L3D_BF16 || weight->dtype != L3D_BF16 || lora_a->dtype != L3D_BF16 ||
      lora_b->dtype != L3D_BF16)
    return fail(L3D_E_DTYPE, "%s: x, weight, lora_a and lora_b must be BF16", op);
  if (y->dtype != L3D_BF16 && y->dtype != L3D_F32)
    return fail(L3D_E_DTYPE, "%s: y must be BF16 or F32", op);
  if (lora_scale->dtype != L3D_F32) return fail(L3D_E_DTYPE, "%s: lora_scale must be F32", op);
  if (ids->dtype != L3D_I32 && ids->dtype != L3D_I64)
    return fail(L3D_E_DTYPE, "%s: ids must be I32 or I64", op);
  const int64_t n = weight->dims[0], k = weight->dims[1];
  const int64_t A = lora_a->dims[0], R = lora_a->dims[1];
  if (n <= 0 || k <= 0) return fail(L3D_E_SHAPE, "%s: empty weight", op);
  if (A <= 0 || R <= 0 || R % 16 || R > 256)
    return fail(L3D_E_UNSUPPORTED, "%s: at least one adapter and ranks padded to a multiple of 16, at most 256", op);
  if (lora_a->dims[2] != k || lora_b->dims[0] != A || lora_b->dims[1] != n || lora_b->dims[2] != R ||
      lora_scale->dims[0] != A)
    return fail(L3D_E_SHAPE, "%s: lora_a [A, R, k], lora_b [A, n, R], lora_scale [A]", op);
  if (x->dims[x->ndim - 1] != k) return fail(L3D_E_SHAPE, "%s: x last dim != k", op);
  if (y->ndim != x->ndim || y->dims[y->ndim - 1] != n) return fail(L3D_E_SHAPE, "%s: y last dim != n", op);
  int64_t M = 1;
  for (int i = 0; i < x->ndim - 1; ++i) {
    if (x->dims[i] != y->dims[i]) return fail(L3D_E_SHAPE, "%s: x/y leading dims differ", op);
    M *= x->dims[i];
  }
  if (M > INT32_MAX / 2 || n > INT32_MAX / 2 || k > INT32_MAX / 2 || A > INT32_MAX / 2)
    return fail(L3D_E_UNSUPPORTED, "%s: dimensions exceed 2^30", op);
  // Contiguous packed operands, 16-byte aligned rows.
  const int64_t w_ld = n > 1 ? weight->strides[0] : k;
  if (k > 1 && weight->strides[1] != 1) return fail(L3D_E_ALIGN, "%s: weight rows must be contiguous", op);
  if (k % 8 || w_ld % 8 || reinterpret_cast<uintptr_t>(elem_ptr(weight)) % 16)
    return fail(L3D_E_ALIGN, "%s: k must be a multiple of 8 and weight rows 16-byte aligned", op);
  auto packed = [](const l3d_tensor* t) {
    int64_t s = 1;
    for (int i = t->ndim - 1; i >= 0; s *= t->dims[i], --i)
      if (t->dims[i] > 1 && t->strides[i] != s) return false;
    return true;
  };
  if (!packed(lora_a) || !packed(lora_b) || !packed(lora_scale) || !packed(ids))
    return fail(L3D_E_ALIGN, "%s: lora_a, lora_b, lora_scale and ids must be contiguous", op);
  if (reinterpret_cast<uintptr_t>(elem_ptr(lora_a)) % 16 || reinterpret_cast<uintptr_t>(elem_ptr(lora_b)) % 16)
    return fail(L3D_E_ALIGN, "%s: lora_a and lora_b must be 16-byte aligned", op);
  if (ranks) {
    if (no_data(ranks)) return fail(L3D_E_NULL, "%s: ranks has a null data pointer", op);
    if (ranks->dtype != L3D_I32) return fail(L3D_E_DTYPE, "%s: ranks must be I32", op);
    if (ranks->ndim != 1 || ranks->dims[0] != A || !packed(ranks))
      return fail(L3D_E_SHAPE, "%s: ranks must be contiguous [A]", op);
  }
  if (act < ACT_NONE || act > ACT_GELU_TANH) return fail(L3D_E_UNSUPPORTED, "%s: unknown activation", op);
  auto matrix = [&](const l3d_tensor* t, int64_t cols, int64_t* ld) {
    RowMap m;
    if ((cols > 1 && t->strides[t->ndim - 1] != 1) || !make_rowmap(t, t->ndim - 1, &m) || m.nd != 1)
      return false;
    *ld = M > 1 ? m.strides[0] : cols;
    return true;
  };
  int64_t x_ld = 0, y_ld = 0, res_ld = 0;
  if (!matrix(x, k, &x_ld) || !matrix(y, n, &y_ld))
    return fail(L3D_E_ALIGN, "%s: x and y must be row-major matrices (one row stride)", op);
  if (x_ld % 8 || reinterpret_cast<uintptr_t>(elem_ptr(x)) % 16)
    return fail(L3D_E_ALIGN, "%s: x rows must be 16-byte aligned", op);
  if (bias) {
    if (no_data(bias)) return fail(L3D_E_NULL, "%s: bias has no data", op);
    if (bias->dtype != L3D_F32 && bias->dtype != L3D_BF16)
      return fail(L3D_E_DTYPE, "%s: bias must be F32 or BF16", op);
    if (numel(bias) != n || !packed(bias)) return fail(L3D_E_SHAPE, "%s: bias must be contiguous [n]", op);
  }
  if (residual) {
    if (no_data(residual)) return fail(L3D_E_NULL, "%s: residual has no data", op);
    if (residual->dtype != y->dtype) return fail(L3D_E_DTYPE, "%s: residual must have y's dtype", op);
    bool same = residual->ndim == y->ndim;
    for (int i = 0; same && i < y->ndim; ++i) same = residual->dims[i] == y->dims[i];
    if (!same) return fail(L3D_E_SHAPE, "%s: residual must have y's shape", op);
    if (!matrix(residual, n, &res_ld)) return fail(L3D_E_ALIGN, "%s: residual must be a row-major matrix", op);
  }
  if (gate) {
    if (!residual) return fail(L3D_E_SHAPE, "%s: gate needs a residual", op);
    if (no_data(gate)) return fail(L3D_E_NULL, "%s: gate has no data", op);
    if (gate->dtype != L3D_F32 && gate->dtype != L3D_BF16)
      return fail(L3D_E_DTYPE, "%s: gate must be F32 or BF16", op);
    if (numel(gate) != n || !packed(gate)) return fail(L3D_E_SHAPE, "%s: gate must be contiguous [n]", op);
  }
  if (M > 0 && (ids->dims[0] <= 0 || M % ids->dims[0]))
    return fail(L3D_E_SHAPE, "%s: the rows must divide evenly among the ids", op);
  const size_t want = l3d_lora_linear_workspace_size(M, R);
  if (!workspace || workspace_bytes < want)
    return fail(L3D_E_WORKSPACE, "%s: workspace of %zu bytes required", op, want);
  if (reinterpret_cast<uintptr_t>(workspace) % 256)
    return fail(L3D_E_ALIGN, "%s: workspace must be 256-byte aligned", op);
  if (M == 0) return L3D_OK;
  Params p{};
  p.M = int(M); p.N = int(n); p.K = int(k); p.R = int(R); p.A = int(A);
  p.x = reinterpret_cast<const __nv_bfloat16*>(elem_ptr(x));
  p.a = reinterpret_cast<const __nv_bfloat16*>(elem_ptr(lora_a));
  p.x_ld = x_ld; p.y_ld = y_ld; p.res_ld = res_ld;
  p.scale = reinterpret_cast<const float*>(elem_ptr(lora_scale));
  p.ranks = ranks ? reinterpret_cast<const int32_t*>(elem_ptr(ranks)) : nullptr;
  p.ids = elem_ptr(ids);
  p.ids64 = ids->dtype == L3D_I64;
  p.per = int(M / ids->dims[0]);
  auto aligned = [](const void* q, int64_t ld_bytes) {
    return reinterpret_cast<uintptr_t>(q) % 16 == 0 && ld_bytes % 16 == 0;
  };
  const int es = dtype_size(y->dtype);
  p.bias = bias ? elem_ptr(bias) : nullptr;
  p.bias_dtype = bias ? bias->dtype : L3D_F32;
  p.bias_vec = aligned(p.bias, 0);
  p.gate = gate ? elem_ptr(gate) : nullptr;
  p.gate_dtype = gate ? gate->dtype : L3D_F32;
  p.res = residual ? elem_ptr(residual) : nullptr;
  p.res_vec = aligned(p.res, res_ld * es);
  p.y = const_cast<char*>(elem_ptr(y));
  p.y_dtype = y->dtype;
  p.y_vec = aligned(p.y, y_ld * es);
  p.act = act;
  p.t = static_cast<__nv_bfloat16*>(workspace);
  p.wait_ns = l3d::tc::WAIT_LIMIT_NS;
  // Of a tile with fewer rows only those are loaded (in groups of 8, the
  // swizzle's unit); the other rows' products are not stored.
  p.x_rows = M < BM ? int((M + 7) / 8 * 8) : BM;
  CUtensorMap mx;
  if (!make_map2(&mx, p.x, uint64_t(M), uint64_t(k), uint64_t(x_ld), uint32_t(p.x_rows)))
    return fail(L3D_E_CUDA, "%s: cuTensorMapEncodeTiled failed for x", op);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  // Few rows: 16 per block, the group's adapters and their ranks in parallel
  // blocks.  More than a device of such groups (2368 rows): the tensor-core form
  // (both take 9 us at 4098 x 2048, rank 32; at 8587 rows 18 and 9).
  const int64_t groups = (M + 15) / 16;
  if (groups <= sm_count()) {
    const int64_t most = A < 16 ? A : 16, y_blocks = most < M ? most : M, z_blocks = (R + 31) / 32;
    shrink_kernel<<<dim3(unsigned(groups), unsigned(y_blocks), unsigned(z_blocks)), 256, 0, s>>>(p);
  } else {
    ShrinkTc sc{};
    const int stage = 128 * 64 * 2 + int(R) * 64 * 2;
    sc.stages = 104 * 1024 / stage < 6 ? 104 * 1024 / stage : 6;
    for (sc.tmem = 32; sc.tmem < int(R);) sc.tmem *= 2;
    const int smem = sc.stages * stage + 256 + (128 + 128 + 4) * 4;
    CUtensorMap ma;
    if (!make_map2(&ma, p.a, uint64_t(A) * uint64_t(R), uint64_t(k), uint64_t(k), uint32_t(R)))
      return fail(L3D_E_CUDA, "%s: cuTensorMapEncodeTiled failed for lora_a", op);
    if (set_smem_limit(reinterpret_cast<const void*>(shrink_tc_kernel), 110 * 1024) != cudaSuccess)
      return fail(L3D_E_CUDA, "%s: cannot reserve shared memory", op);
    shrink_tc_kernel<<<unsigned((M + 127) / 128), SHRINK_THREADS, size_t(smem), s>>>(mx, ma, p, sc);
  }
  if (cudaGetLastError() != cudaSuccess) return fail(L3D_E_CUDA, "%s: launch failed", op);
  const void* w = elem_ptr(weight);
  const void* b = elem_ptr(lora_b);
  cudaError_t e;
  auto launch = [&](auto bn) {
    constexpr int BN = decltype(bn)::value;
    return residual ? launch_gemm<BN, true>(mx, w, w_ld, b, p, s) : launch_gemm<BN, false>(mx, w, w_ld, b, p, s);
  };
  switch (pick_bn(M, n)) {
    case 32: e = launch(std::integral_constant<int, 32>()); break;
    case 64: e = launch(std::integral_constant<int, 64>()); break;
    case 128: e = launch(std::integral_constant<int, 128>()); break;
    default: e = launch(std::integral_constant<int, 256>()); break;
  }
  if (e != cudaSuccess) return fail(L3D_E_CUDA, "%s: %s", op, cudaGetErrorString(e));
  return L3D_OK;
}
