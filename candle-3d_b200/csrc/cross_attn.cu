// Attention of packed sequences to keys of other lengths (cross attention to an encoder's states; attention of
// each of several scenes to itself, where the keys are its own rows), on the 5th-generation tensor cores:
//   out[t, h] = sum_j softmax_j(scale q[t, h] . K[j]) V[j]
// over the keys k_offsets[b] <= j < k_offsets[b + 1] of the sequence b that row t belongs to; query heads
// h G .. h G + G - 1 read key head h.  The reference's attention core is exact_sdpa_heads
// (crate/runtime/attention_math.rs:199-259); it takes one sequence after the other.
//
// An item is a tile of up to 128 rows of one sequence and key head (128 / G tokens with their G query heads) by
// all of the sequence's keys.  The grid has a block per item; two blocks run on an SM, and each, while it
// works, takes further items off the grid (cluster launch control), so that set-up is paid once and no SM waits for
// the slowest.  K and V rings run on from one item to the next, and the next item's first scores are formed while
// the last one's output is divided and stored.
//   warp 0     loads Q tiles and the ring of 64-key K tiles, warp 2 the ring of V tiles (TMA);
//   warp 1     issues S = Q K^T (two buffers of 64 columns, so that S(n + 2) is formed while softmax(n + 1) runs)
//              and O += P V (P read from tensor memory, over the scores it comes from);
//   warp 3     takes the items, one ahead of the loads, finds their rows and keys from the offsets (lengths are never
//              on the host) and lists them in shared memory for the other warps, whose code this keeps small; those
//              without keys it answers itself;
//   warps 4-7  one row per thread: S to P in registers, the running maximum and sum, O's rescaling where the
//              maximum has grown past 2^8, zeros over V rows past a sequence's end (another sequence's, or
//              anything: a masked probability is 0, but 0 x NaN is not), and the output.
// Where there are fewer items than blocks, each is cut into parts along its keys, and combine_kernel weighs the
// parts of each row; an item's parts have fixed places.  Where every sequence has as many rows, up to 16 a key head,
// decode_attn.cu takes the call instead (few_rows).
// P is rounded to the input type for the second product, as tensor memory takes it: two parts would be half as many
// products again.  Against 64 bits the error is 2.3e-3 of the output's norm where the output's type alone gives 1.7e-3
// (2 x 2049 rows, bf16).
// Every mbarrier wait is bounded (%globaltimer, 2 s; those for an item 60 s); on expiry the block records an error
// in the device's status word and stops.
// Measured: 3 x 31569 rows x 12 heads of 128 over up to 1370 keys 641 us (1063 TFLOP/s, 64% of a plain product; call
// after call, at the power limit, 744: 916); 2 x 2049 rows x 16 heads of 128 53.6 us (673 TFLOP/s); 4 x 8192 rows x 16
// heads of 64 over up to 1370 keys 194 us (522 TFLOP/s).  A 64-key tile takes an SM some 1000 clocks either way, of which
// the exponentials need 512: the softmax warps' chain, with the products' round trip (scores of 64 keys read all of Q
// from shared memory, 384 clocks for 256 of products) partly under it.
#include <type_traits>

#include "attn.cuh"
#include "common.cuh"
#include "decode_attn.cuh"
#include "tc.cuh"

namespace l3d {
namespace cross {

using namespace l3d::attn;

constexpr int BQ = 128, BKV = 64, THREADS = 256, CTAS = 2;
constexpr int ST_TIMEOUT = 5, ST_MISALIGNED = 6;
constexpr float RESCALE_LOG2 = 8.f;   // as in attn.cu
// log2 of a row's largest probability: f16 goes down to 2^-24 only, and up to 2^15 there is room.  (At 2^0 the
// weight of 255 keys of 2^-18 each beside one of 1 was off by up to 1%.)
template <typename T>
constexpr float HELD_LOG2 = std::is_same<T, __half>::value ? 7.f : 0.f;
constexpr int MAX_PARTS = 16;
// Sequences, and key heads of them all: while a block passes over items without rows or keys, its other warps wait
// for the next one, and those waits are bounded (2 s).  2^20 sequences without rows or keys x 64 heads: 110 ms.
constexpr int64_t MAX_BATCH = int64_t(1) << 20, MAX_HEADS = int64_t(1) << 26;
// Places of the list of items: the one that is looked for while up to three before it are not done with (the one
// whose last product was just issued, and two of a tile each whose scores were).
constexpr int LISTED = 4;

__device__ int g_cross_status;

template <int D>
struct Cfg {
  static constexpr int DC = D / 64;
  static constexpr int Q_BYTES = BQ * D * 2, KV_BYTES = BKV * D * 2;
  static constexpr int REST = 512;    // barriers
  // The output of a softmax warp's 32 rows on its way to memory: one place of 64 columns, or two of 32.
  static constexpr int OUT_COLS = D == 64 ? 64 : 32, OUT_BYTES = BQ * 128;
  static constexpr int BUFS = (226 * 1024 / CTAS - REST - Q_BYTES - OUT_BYTES) / KV_BYTES;
  static constexpr int KST = BUFS / 2, VST = BUFS - KST;
  static constexpr int SMEM = Q_BYTES + BUFS * KV_BYTES + OUT_BYTES + REST;
  static constexpr uint32_t COL_S = 0, COL_O = 2 * BKV, TMEM_COLS = 256;
  static_assert(COL_O + D <= TMEM_COLS && TMEM_COLS * CTAS <= 512, "TMEM budget");
  static_assert((2 * BUFS + 13 + 2 * LISTED) * 8 + 8 + 16 + LISTED * 32 <= REST, "barrier area");
  // Of 8 pairs of P, those of ex2_poly2: none at D = 128 (voxel scenes 657 us, 669 with one), one at D = 64
  // (4 x 8192 rows x 16 heads over 1370 keys: 198 us, 214 without, 200 with two).
  static constexpr int POLY = D == 64 ? 1 : 0;
};

struct Params {
  int B, G, Hkv, Tq, Tk;
  int N;                       // rows of every sequence; 0: q_offsets
  int tpt;                     // tokens of a tile
  int q_th;                    // a tile lists its tokens before its heads
  int k_hn, v_hn;              // the K / V maps list heads before rows
  int k_hm, v_hm;              // 0: heads expanded (stride 0)
  const void *q_offsets, *k_offsets;
  int q64, k64;
  void* out;
  int64_t ot, oh;              // element strides
  int o_tma, o_th;             // the output's map can be used; it lists tokens before heads
  float scale_log2;            // softmax scale * log2(e), > 0
  int parts;
  float *part_l, *part_o;      // [parts, Tq, Hq], [parts, Tq, Hq, D]
  uint64_t wait_ns;
};

// offsets[i], clamped to [0, most].
__device__ __forceinline__ int offset_at(const void* p, int is64, int i, int most) {
  const int64_t v = is64 ? static_cast<const int64_t*>(p)[i] : int64_t(static_cast<const int32_t*>(p)[i]);
  return v < 0 ? 0 : v < most ? int(v) : most;
}

struct alignas(16) Item {
  int h, part;                 // h < 0: no further item
  int row0, rows;              // the tile's first token, its tokens
  int key0, keys;              // the sequence's first key, its keys
  int t0, tiles;               // the part's first key tile and its number
};
static_assert(sizeof(Item) == 32, "two 16-byte loads");

// Finds items by their numbers, (tile, key head, part) with the part fastest.  The warp holds 32 sequences at a
// time, one per lane.
struct Finder {
  int window;
  int64_t base;                // tiles before the window
  int cnt, incl, q0, q1, k0, k1;
  __device__ __forceinline__ void load(const Params& p) {
    const int b = window * 32 + (threadIdx.x & 31);
    q0 = q1 = k0 = k1 = 0;
    if (b < p.B) {
      q0 = p.N ? b * p.N : offset_at(p.q_offsets, p.q64, b, p.Tq);
      q1 = p.N ? q0 + p.N : offset_at(p.q_offsets, p.q64, b + 1, p.Tq);
      k0 = offset_at(p.k_offsets, p.k64, b, p.Tk);
      k1 = offset_at(p.k_offsets, p.k64, b + 1, p.Tk);
    }
    cnt = q1 > q0 ? (q1 - q0 + p.tpt - 1) / p.tpt : 0;
    incl = cnt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (int(threadIdx.x & 31) >= o) incl += up;
    }
  }
  __device__ __forceinline__ void start(const Params& p) {
    base = 0;
    window = 0;
    load(p);
  }
  // False: past the last item.
  __device__ __forceinline__ bool at(const Params& p, int idx, Item& it) {
    const int per = p.Hkv * p.parts, tile = idx / per;
    if (tile < base) start(p);
    int all;
    while (tile - base >= (all = __shfl_sync(0xffffffffu, incl, 31))) {
      if ((window + 1) * 32 >= p.B) return false;
      base += all;
      ++window;
      load(p);
    }
    const int rel = int(tile - base);
    const int lane = __ffs(__ballot_sync(0xffffffffu, incl > rel)) - 1;
    const int first = rel - (__shfl_sync(0xffffffffu, incl, lane) - __shfl_sync(0xffffffffu, cnt, lane));
    const int a = __shfl_sync(0xffffffffu, q0, lane), e = __shfl_sync(0xffffffffu, q1, lane);
    it.key0 = __shfl_sync(0xffffffffu, k0, lane);
    it.keys = max(__shfl_sync(0xffffffffu, k1, lane) - it.key0, 0);
    const int rest = idx - tile * per;
    it.h = rest / p.parts;
    it.part = rest - it.h * p.parts;
    it.row0 = a + first * p.tpt;
    it.rows = min(e - it.row0, p.tpt);
    const int tiles = (it.keys + BKV - 1) / BKV, chunk = (tiles + p.parts - 1) / p.parts;
    it.t0 = min(it.part * chunk, tiles);
    it.tiles = min(chunk, tiles - it.t0);
    return true;
  }
};

// Asks for a block of the grid that has not started yet; the answer comes to 16 bytes of shared memory.
__device__ __forceinline__ void take_block(uint32_t answer, uint64_t* bar) {
  asm volatile(
      "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(answer),
      "r"(smem_u32(bar))
      : "memory");
}
// The block's number, -1: none was left.
__device__ __forceinline__ int taken_block(uint32_t answer) {
  uint32_t got, x;
  asm volatile(
      "{\n\t.reg .b128 r;\n\t.reg .pred p;\n\t"
      "ld.shared.b128 r, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "selp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n\t}"
      : "=r"(got), "=r"(x)
      : "r"(answer)
      : "memory");
  return got ? int(x) : -1;
}

__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, const void* src, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
          reinterpret_cast<uint64_t>(map)),
      "r"(smem_u32(src)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

template <typename T, int D>
__global__ void __launch_bounds__(THREADS, CTAS)
    cross_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                 const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_o, const Params p) {
  using C = Cfg<D>;
  constexpr uint32_t IDESC_S = idesc_of<T>(128, BKV);
  constexpr uint32_t IDESC_O = idesc_of<T>(128, D) | (1u << 16);  // B (V) MN-major
  int* const status = &g_cross_status;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  if (smem_u32(smem_raw) & 1023u) {
    if (threadIdx.x == 0) atomicCAS(status, 0, ST_MISALIGNED);
    return;
  }
  uint8_t* sq = smem_raw;                            // [DC][128 x 64]
  uint8_t* sk = sq + C::Q_BYTES;                     // [KST][DC][64 x 64]
  uint8_t* sv = sk + C::KST * C::KV_BYTES;           // [VST][DC][64 x 64]
  uint8_t* so = sv + C::VST * C::KV_BYTES;           // [4][32 x 64], or [4][2][32 x 32]
  uint64_t* bars = reinterpret_cast<uint64_t*>(so + C::OUT_BYTES);
  uint64_t* k_full = bars;                           // [KST]
  uint64_t* k_empty = k_full + C::KST;               // [KST]
  uint64_t* v_full = k_empty + C::KST;               // [VST]
  uint64_t* v_empty = v_full + C::VST;               // [VST]
  uint64_t* s_full = v_empty + C::VST;               // [2] (by S buffer)
  uint64_t* p_full = s_full + 2;                     // [2][2] (by half of the keys)
  uint64_t* pv_done = p_full + 4;                    // [2]
  uint64_t* q_full = pv_done + 2;
  uint64_t* q_empty = q_full + 1;
  uint64_t* mma_drain = q_empty + 1;                 // abort teardown only
  uint64_t* answered = mma_drain + 1;
  uint64_t* started = answered + 1;                  // an item's loads have begun
  uint64_t* listed = started + 1;                    // [LISTED]
  uint64_t* unlisted = listed + LISTED;              // [LISTED]
  volatile int* abort_flag = reinterpret_cast<volatile int*>(unlisted + LISTED);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(unlisted + LISTED) + 1;
  uint8_t* answer = so + C::OUT_BYTES + C::REST - 16 - LISTED * 32;
  Item* list = reinterpret_cast<Item*>(answer + 16);  // [LISTED]

  // (The shuffle tells the compiler that the role is the same in all lanes.)
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.launch_dependents;");
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::KST; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
    }
    for (int s = 0; s < C::VST; ++s) {
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[2 * i], 4);
      mbar_init(&p_full[2 * i + 1], 4);
      mbar_init(&pv_done[i], 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    mbar_init(mma_drain, 1);
    mbar_init(answered, 1);
    mbar_init(started, 1);
    for (int i = 0; i < LISTED; ++i) {
      mbar_init(&listed[i], 1);
      mbar_init(&unlisted[i], 7);  // two loading warps, the MMA warp, four softmax warps
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(C::TMEM_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    return mbar_wait(bar, parity, abort_flag, status, ST_TIMEOUT, p.wait_ns);
  };
  auto wait_warp = [&](uint64_t* bar, uint32_t parity) {  // the warp's lanes stay together
    const bool got = __all_sync(0xffffffffu, wait(bar, parity)) != 0;
    __syncwarp();  // before the warp-wide (.aligned) instructions that follow
    return got;
  };
  Item it;
  int loads = 0, q_loads = 0, asked = 0;  // of this warp's ring, of Q, for blocks (abort teardown)
  // The listed item number i (of this block); false: there is none, or a wait ran out.
  auto item = [&](int i, Item& t) {
    if (!wait_warp(&listed[i % LISTED], (i / LISTED) & 1)) return false;
    const int4* src = reinterpret_cast<const int4*>(list + i % LISTED);
    reinterpret_cast<int4*>(&t)[0] = src[0];
    reinterpret_cast<int4*>(&t)[1] = src[1];
    return t.h >= 0;
  };
  auto done_with = [&](int i) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&unlisted[i % LISTED]);
  };

  if (warp == 0 || warp == 2) {
    // ------------------------------------------------------- loads of Q and K; of V
    const bool isk = warp == 0;
    uint64_t* full = isk ? k_full : v_full;
    uint64_t* empty = isk ? k_empty : v_empty;
    uint8_t* ring = isk ? sk : sv;
    const int stages = isk ? C::KST : C::VST;
    const CUtensorMap* map = isk ? &map_k : &map_v;
    const int hn = isk ? p.k_hn : p.v_hn, hm = isk ? p.k_hm : p.v_hm;
    int s = 0, turn = 0;
    bool ok = true;
    for (int i = 0; ok && item(i, it); done_with(i++)) {
      if (isk) {
        if (lane == 0) mbar_arrive(started);
        if (q_loads > 0) ok = wait_warp(q_empty, (q_loads - 1) & 1);
        if (!ok) continue;
        if (lane == 0) {
          mbar_expect_tx(q_full, C::DC * 128 * p.tpt * p.G);
          for (int dc = 0; dc < C::DC; ++dc)
            tma_load_3d(sq + dc * (BQ * 128), &map_q, q_full, dc * 64, p.q_th ? it.row0 : it.h * p.G,
                        p.q_th ? it.h * p.G : it.row0);
        }
        ++q_loads;
      }
      const int hh = it.h * hm;
      for (int j = 0; j < it.tiles; ++j) {
        if (turn > 0) ok = wait_warp(&empty[s], (turn - 1) & 1);
        if (!ok) break;
        if (lane == 0) {
          const int row = it.key0 + (it.t0 + j) * BKV;
          mbar_expect_tx(&full[s], C::KV_BYTES);
          for (int dc = 0; dc < C::DC; ++dc)
            tma_load_4d(ring + s * C::KV_BYTES + dc * (BKV * 128), map, &full[s], dc * 64, hn ? hh : row, hn ? row : hh, 0);
        }
        ++loads;
        if (++s == stages) {
          s = 0;
          ++turn;
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA
    // The whole warp keeps step and one elected lane issues.  Scores run two tiles ahead of P V, across the
    // ends of items.
    const bool leader = elect_one();
    auto commit = [&](uint64_t* bar) {
      if (leader) umma_commit(bar);
    };
    const uint32_t t_s = tmem_base + C::COL_S, t_o = tmem_base + C::COL_O;
    int ns = 0, js = 0, ks = 0, kturn = 0, items = 0;  // of the next scores: number, tile of its item, K slot, Q
    int is = 0, tiles_s = 0;                           // its item's number and tiles
    bool ok = true;
    auto next_s = [&] {
      Item t;
      const bool got = item(is, t);
      tiles_s = t.tiles;
      return got;
    };
    bool more = next_s();
    auto issue_s = [&] {
      if (js == 0) ok = wait_warp(q_full, items & 1);
      ok = ok && wait_warp(&k_full[ks], kturn & 1);
      if (!ok) return;
      tc_fence_after();
      const uint64_t da = smem_desc_sw128(sq), db = smem_desc_sw128(sk + ks * C::KV_BYTES);
      if (leader) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          umma_f16<IDESC_S>(t_s + (ns & 1) * BKV, da + uint64_t((k >> 2) * (BQ * 128 >> 4) + 2 * (k & 3)),
                            db + uint64_t((k >> 2) * (BKV * 128 >> 4) + 2 * (k & 3)), k ? 1u : 0u);
      }
      commit(&s_full[ns & 1]);
      commit(&k_empty[ks]);
      if (++ks == C::KST) {
        ks = 0;
        ++kturn;
      }
      ++ns;
      if (++js == tiles_s) {
        commit(q_empty);
        js = 0;
        ++items;
        ++is;
        more = next_s();
      }
    };
    int n = 0, vs = 0, vturn = 0;
    for (int i = 0; i < 2 && ok && more; ++i) issue_s();
    for (int i = 0; ok && item(i, it); done_with(i++)) {
      for (int j = 0; ok && j < it.tiles; ++j) {
        // (P of an item's first tile comes after the last item's output was read: O is free.)
        const uint64_t db = smem_desc_sw128_mn(sv + vs * C::KV_BYTES, BKV * 128);
        ok = wait_warp(&v_full[vs], vturn & 1);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          ok = ok && wait_warp(&p_full[2 * (n & 1) + half], (n >> 1) & 1);
          if (!ok) break;
          tc_fence_after();
          if (leader) {
#pragma unroll
            for (int k = 2 * half; k < 2 * half + 2; ++k)
              umma_f16_ts<IDESC_O>(t_o, t_s + (n & 1) * BKV + uint32_t(k * 8), db + uint64_t(k * (16 * 128 >> 4)),
                                   (j | k) ? 1u : 0u);
          }
        }
        if (!ok) break;
        commit(&v_empty[vs]);
        commit(&pv_done[n & 1]);  // the last commit of all: the block waits for it
        if (++vs == C::VST) {
          vs = 0;
          ++vturn;
        }
        ++n;
        if (more) issue_s();  // over the P that the product before it has read
      }
    }
  } else if (warp == 3) {
    // ---------------------------------------------------------------- items
    // (An item can take longer than any wait for a tile: the waits here are bounded by 30 times as long.)
    auto wait_item = [&](uint64_t* bar, uint32_t parity) {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status, ST_TIMEOUT, 30 * p.wait_ns)) != 0;
    };
    Finder find;
    find.start(p);
    int idx = int(blockIdx.x), i = 0;
    bool ok = true;
    while (ok && idx >= 0) {
      if (find.at(p, idx, it)) {
        if (it.tiles > 0) {
          if (i >= LISTED) ok = wait_item(&unlisted[i % LISTED], ((i / LISTED) - 1) & 1);
          if (!ok) break;
          if (lane == 0) {
            list[i % LISTED] = it;
            mbar_arrive(&listed[i % LISTED]);
          }
          ok = wait_item(started, i & 1);
          ++i;
        } else if (p.parts > 1) {
          for (int x = lane; x < it.rows * p.G; x += 32)
            p.part_l[(int64_t(it.part) * p.Tq + it.row0 + x / p.G) * (p.Hkv * p.G) + it.h * p.G + x % p.G] = -INFINITY;
        } else {  // no keys: zeros
          for (int x = lane; x < it.rows * p.G * (D / 8); x += 32) {
            const int r = x / (D / 8);
            T* dst = static_cast<T*>(p.out) + (it.row0 + r / p.G) * p.ot + int64_t(it.h * p.G + r % p.G) * p.oh;
            *reinterpret_cast<uint4*>(dst + x % (D / 8) * 8) = make_uint4(0, 0, 0, 0);
          }
        }
      }
      if (!ok) break;
      if (lane == 0) {
        mbar_expect_tx(answered, 16);
        take_block(smem_u32(answer), answered);
      }
      ++asked;
      ok = wait_warp(answered, (asked - 1) & 1);
      if (ok) idx = taken_block(smem_u32(answer));
      // (The answer's place is written again by the async proxy.)
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
    }
    if (ok && i >= LISTED) ok = wait_item(&unlisted[i % LISTED], ((i / LISTED) - 1) & 1);
    if (ok && lane == 0) {
      list[i % LISTED].h = -1;
      mbar_arrive(&listed[i % LISTED]);
    }
  } else {
    // ------------------------------------------------------ softmax / epilogue
    const int r = (warp & 3) * 32 + lane;
    const uint32_t lane_off = uint32_t((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem_base + C::COL_S + lane_off, t_o = tmem_base + C::COL_O + lane_off;
    // This thread's row of a tile: token i, query head g of the key head's.
    const int i = p.q_th ? r % p.tpt : r / p.G, g = p.q_th ? r / p.tpt : r - i * p.G;
    const float2 sc2 = f2(p.scale_log2);
    int n = 0, vs = 0, vturn = 0;
    bool ok = true;
    for (int at = 0; ok && item(at, it); done_with(at++)) {
      const bool valid = i < it.rows && g < p.G;
      const bool active = __any_sync(0xffffffffu, valid);  // the warp holds rows
      float m = -INFINITY;                         // running max less HELD_LOG2, log2 units
      float2 l2 = f2(0.f);                         // running row sum (two parts)
      for (int j = 0; j < it.tiles; ++j, ++n) {
        ok = wait_warp(&s_full[n & 1], (n >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        // V rows past the sequence's keys may hold anything: zero them, once the tile has landed.
        const int held = it.keys - (it.t0 + j) * BKV;
        if (held < BKV) {
          ok = wait_warp(&v_full[vs], vturn & 1);
          if (!ok) break;
          const int vrow = r & (BKV - 1);
          if (vrow >= held) {
            uint8_t* vr = sv + vs * C::KV_BYTES + vrow * 128;
#pragma unroll
            for (int x = 0; x < D / 16; ++x) {
              const int c = (r / BKV) * (D / 16) + x;
              *reinterpret_cast<uint4*>(vr + (c >> 3) * (BKV * 128) + ((c & 7) << 4)) = make_uint4(0, 0, 0, 0);
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
        }
        if (++vs == C::VST) {
          vs = 0;
          ++vturn;
        }
        if (!active) {  // no rows: keep the other warps' pace
          if (lane == 0) {
            mbar_arrive(&p_full[2 * (n & 1)]);
            mbar_arrive(&p_full[2 * (n & 1) + 1]);
          }
          continue;
        }
        const uint32_t t_sn = t_s + (n & 1) * BKV;
        float s[BKV];
        tmem_ld64(t_sn, s);
        if (held < BKV) {
#pragma unroll
          for (int e = 0; e < BKV; ++e)
            if (e >= held) s[e] = -INFINITY;
        }
        __syncwarp();
        float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int e = 4; e < BKV; e += 2) mx[(e >> 1) & 3] = max_nan(mx[(e >> 1) & 3], s[e], s[e + 1]);
        const float mxs = max_nan(max_nan(mx[0], mx[1], mx[2]), mx[3]) * p.scale_log2;  // scale > 0
        const bool grow = !(mxs <= m + (RESCALE_LOG2 + HELD_LOG2<T>));  // always on the first key a row sees
        const float m_new = grow ? mxs - HELD_LOG2<T> : m;
        const float alpha = grow ? ex2f(m - m_new) : 1.f;   // 0 on the first
        if (j > 0 && __any_sync(0xffffffffu, grow)) {
          ok = wait_warp(&pv_done[(n - 1) & 1], ((n - 1) >> 1) & 1);  // O is stable
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {  // (s is live: few columns at a time)
            float o[16];
            tmem_ld16(t_o + uint32_t(c), o);
            uint32_t u[16];
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              const float2 v = mul2(make_float2(o[e], o[e + 1]), f2(alpha));
              u[e] = __float_as_uint(v.x);
              u[e + 1] = __float_as_uint(v.y);
            }
            tmem_st16u(t_o + uint32_t(c), u);
          }
        }
        // P = exp2(s * scale * log2 e - m); all scores of -inf so far: subtract 0, so that P = 0.
        const float2 nm2 = f2(m_new == -INFINITY ? 0.f : minus_max(m_new));
        l2 = mul2(l2, f2(alpha));
#pragma unroll
        for (int c = 0; c < BKV; c += 32) {
          uint32_t u[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float2 x = fma2(make_float2(s[c + e], s[c + e + 1]), sc2, nm2);
            const float2 pr = ((e >> 1) & 7) < C::POLY ? ex2_poly2(x) : make_float2(ex2f(x.x), ex2f(x.y));
            l2 = add2(l2, pr);
            u[e >> 1] = pack_pair<T>(pr.x, pr.y);
          }
          tmem_st16u(t_sn + uint32_t(c / 2), u);
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[2 * (n & 1) + c / 32]);
        }
        m = m_new;
      }
      // The output, or this part's O / l and log2 sum, after the item's last P V.
      if (ok) ok = wait_warp(&pv_done[(n - 1) & 1], ((n - 1) >> 1) & 1);
      tc_fence_after();
      if (!ok || !active) continue;
      float l = l2.x + l2.y;
      if (m == -INFINITY && l == l) l = 0.f;  // (ex2_poly2 gives 1e-42 for -inf, not 0)
      const float inv = l > 0.f ? 1.f / l : l == l ? 0.f : l;  // no keys: zeros; NaN stays
      const int64_t token = it.row0 + i;
      const int64_t pr = (int64_t(it.part) * p.Tq + token) * (p.Hkv * p.G) + it.h * p.G + g;
      if (p.parts > 1 && valid) p.part_l[pr] = l > 0.f ? m + log2f(l) : l == l ? -INFINITY : l;
      T* orow = static_cast<T*>(p.out) + token * p.ot + int64_t(it.h * p.G + g) * p.oh;
      __syncwarp();  // the loads from tensor memory are the whole warp's
      const uint32_t rows = __ballot_sync(0xffffffffu, valid);
      if (p.parts > 1) {  // 16 columns at a time through shared memory, 64 bytes of eight rows per store
        uint8_t* stage = so + (warp & 3) * (32 * 128);
        float* prow = p.part_o + pr * D;
#pragma unroll 1
        for (int c = 0; c < D; c += 16) {
          float o[16];
          tmem_ld16(t_o + uint32_t(c), o);
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<float4*>(stage + lane * 64 + ((q ^ (lane >> 1 & 3)) << 4)) =
                make_float4(o[4 * q] * inv, o[4 * q + 1] * inv, o[4 * q + 2] * inv, o[4 * q + 3] * inv);
          __syncwarp();
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int row = 8 * x + (lane >> 2);
            float* dst = reinterpret_cast<float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(prow), row));
            const float4 v = *reinterpret_cast<const float4*>(stage + row * 64 + (((lane & 3) ^ (row >> 1 & 3)) << 4));
            if (rows >> row & 1) *reinterpret_cast<float4*>(dst + c + (lane & 3) * 4) = v;
          }
          __syncwarp();
        }
        continue;
      }
      // OC columns of the warp's 32 rows at a time through shared memory, at D = 128 two places in turn, then a TMA
      // store; or, where some of the rows are no part of the sequence, whole lines of several rows per store.  (Each
      // thread storing its own row took 7,400 clocks an item of 18 tiles, of 33,000; one place of 64 columns at
      // D = 128 3 to 4% of the whole.)
      constexpr int OC = C::OUT_COLS, ROW = OC * 2, CHUNKS = OC / 8;
      auto place = [&](int row, int j) { return row * ROW + ((j ^ (OC == 64 ? row & 7 : row >> 1 & 3)) << 4); };
      const bool box = p.o_tma && rows == 0xffffffffu;
      const int t_box = it.row0 + (warp & 3) * 32 / p.G, h_box = it.h * p.G;
#pragma unroll 1
      for (int c = 0; c < D; c += OC) {
        uint8_t* stage = so + (warp & 3) * (32 * 128) + (OC == 64 ? 0 : (c & 32) * 64);
        if (lane == 0) {  // the last store from this place has read it
          if constexpr (OC == 64) bulk_wait_read0();
          else bulk_wait_read1();
        }
        __syncwarp();
#pragma unroll
        for (int x = 0; x < OC / 32; ++x) {
          float o[32];
          tmem_ld32(t_o + uint32_t(c + 32 * x), o);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = o[8 * q + e] * inv;
            *reinterpret_cast<uint4*>(stage + place(lane, 4 * x + q)) = pack(v, T());
          }
        }
        if (box) {
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) tma_store_3d(&map_o, stage, c, p.o_th ? t_box : h_box, p.o_th ? h_box : t_box);
        } else {
          __syncwarp();
#pragma unroll
          for (int x = 0; x < CHUNKS; ++x) {
            const int row = 32 / CHUNKS * x + lane / CHUNKS, j = lane % CHUNKS;
            T* dst = reinterpret_cast<T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(orow), row));
            const uint4 v = *reinterpret_cast<const uint4*>(stage + place(row, j));
            if (rows >> row & 1) *reinterpret_cast<uint4*>(dst + c + j * 8) = v;
          }
          __syncwarp();
        }
        if (lane == 0) bulk_commit();  // (an empty group where nothing was stored: the places take turns)
      }
    }
    if (lane == 0) bulk_wait0();
  }

  // Teardown, as in attn.cu: after an abort nothing the block started may still be running when it frees TMEM
  // and exits.
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    if (warp == 1 && elect_one()) {  // the lane that issued
      umma_commit(mma_drain);
      mbar_drain(mma_drain, 0, p.wait_ns);
    }
    if (warp == 3 && lane == 0 && asked > 0) mbar_drain(answered, uint32_t(asked - 1) & 1u, p.wait_ns);
    if ((warp == 0 || warp == 2) && lane == 0) {  // the newest load of each slot, and of Q
      const int stages = warp == 0 ? C::KST : C::VST;
      for (int i = max(loads - stages, 0); i < loads; ++i)
        mbar_drain(warp == 0 ? &k_full[i % stages] : &v_full[i % stages], uint32_t(i / stages) & 1u, p.wait_ns);
      if (q_loads > 0) mbar_drain(q_full, uint32_t(q_loads - 1) & 1u, p.wait_ns);
    }
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base),
                 "r"(C::TMEM_COLS));
  }
}

// The parts of each row weighed by 2^(their log2 sum - the largest), a warp per row of a sequence.
template <typename T, int D>
__global__ void __launch_bounds__(128) combine_kernel(const Params p) {
  constexpr int E = D / 32;
  using Vec = typename std::conditional<E == 4, float4, float2>::type;
  const int lane = threadIdx.x & 31, Hq = p.Hkv * p.G;
  const int64_t rows = int64_t(p.Tq) * Hq, row = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int64_t token = row / Hq;
  const bool none = !p.N && (token < offset_at(p.q_offsets, p.q64, 0, p.Tq) || token >= offset_at(p.q_offsets, p.q64, p.B, p.Tq));
  asm volatile("griddepcontrol.wait;" ::: "memory");  // (of rows of no sequence too: the kernel ends after the one before)
  if (none) return;
  float w = lane < p.parts ? p.part_l[lane * rows + row] : -INFINITY, mx = w;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  w = w == -INFINITY ? 0.f : exp2f(w - mx);
  float sum = w;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  alignas(16) float acc[E] = {};
  for (int k = 0; k < p.parts; ++k) {
    const float wk = __shfl_sync(0xffffffffu, w, k);
    if (wk == 0.f) continue;
    const Vec v = reinterpret_cast<const Vec*>(p.part_o + (k * rows + row) * D)[lane];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = fmaf(wk, reinterpret_cast<const float*>(&v)[e], acc[e]);
  }
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
  T* orow = static_cast<T*>(p.out) + token * p.ot + (row - token * Hq) * p.oh + lane * E;
  alignas(8) T o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = from_f<T>(acc[e] * inv);
  if constexpr (E == 4) *reinterpret_cast<uint2*>(orow) = *reinterpret_cast<const uint2*>(o);
  else *reinterpret_cast<uint32_t*>(orow) = *reinterpret_cast<const uint32_t*>(o);
}

// Parts of an item: as many as two rounds of the device take, for an item's time is that of its keys (some 0.7 us a
// tile) however few items there are; of four key tiles at least by the keys' average.  (2 x up to 1273 rows x 16 / 4
// heads of 64 over up to 3299 keys: 41 us whole, 32 in two parts.)
static int parts_for(int64_t B, int64_t Tq, int64_t Tk, int64_t G, int64_t Hkv) {
  const int64_t tpt = BQ / G, items = Hkv * (Tq / tpt + B), tiles = (Tk / B + BKV - 1) / BKV;
  int64_t parts = 2 * CTAS * int64_t(sm_count()) / items;
  if (parts > tiles / 4) parts = tiles / 4;
  return int(parts < 1 ? 1 : parts > MAX_PARTS ? MAX_PARTS : parts);
}

// Single rows (or a few) of every sequence: their work is reading the keys.  us here and in the kernel above: 32 x 16
// heads of 64, up to 1370 keys: 1 row 26.9 and 37.9, 8 28.6 and 37.4, 12 32.6 and 37.5, 16 40.8 and 37.8, 32 59.8 and
// 38.1; 64 x 4 heads of 128, 1029 keys: 8 24.3 and 27.5, 16 32.9 and 27.9; 2 x 2 heads of 64, 600 keys: 16 8.5 and
// 11.6, 128 8.9 and 10.9.  Up to 16 rows (two columns of 8) the forms are near each other, and this one keeps two parts
// of each probability.
// (The last two: what decode_attn.cu takes, and counts in 32 bits.)
static bool few_rows(int64_t B, int64_t N, int64_t G, int64_t Tk) {
  return N > 0 && N * G <= 16 && B <= decode::MAX_BATCH && B * (Tk / 16 + 1) <= int64_t(1) << 30;
}

cudaError_t status_read(int* status, int reset) {
  cudaError_t e = cudaMemcpyFromSymbol(status, g_cross_status, sizeof(int));
  if (e == cudaSuccess && reset) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_cross_status, &zero, sizeof(int));
  }
  return e;
}

template <typename T, int D>
static cudaError_t launch(const CUtensorMap (&maps)[4], const Params& p, int64_t items, cudaStream_t s) {
  auto k = cross_kernel<T, D>;
  cudaError_t e = set_smem_limit(reinterpret_cast<const void*>(k), Cfg<D>::SMEM);
  if (e != cudaSuccess) return e;
  k<<<unsigned(items), THREADS, Cfg<D>::SMEM, s>>>(maps[0], maps[1], maps[2], maps[3], p);
  if (p.parts <= 1) return cudaGetLastError();
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned((int64_t(p.Tq) * p.Hkv * p.G + 3) / 4));
  cfg.blockDim = dim3(128);
  cfg.stream = s;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, combine_kernel<T, D>, p);
}

// The map of q or out [T, Hq, D] with boxes of G heads x tpt tokens x 64 columns (or 32), the nearer of
// heads and tokens in memory listed first.
static bool make_row_map(CUtensorMap* m, const void* base, int64_t T, int64_t Hq, int64_t D, int64_t st, int64_t sh, int G,
                         int tpt, int cols, int* th) {
  auto fn = encode_fn();
  if (!fn) return false;
  if (T <= 1) st = Hq <= 1 ? D : (sh > 0 ? sh * Hq : D);
  if (Hq <= 1) sh = st * T;
  *th = st < sh ? 1 : 0;
  const cuuint64_t dims[3] = {uint64_t(D), uint64_t(*th ? T : Hq), uint64_t(*th ? Hq : T)};
  const cuuint64_t strides[2] = {uint64_t(*th ? st : sh) * 2, uint64_t(*th ? sh : st) * 2};
  const cuuint32_t box[3] = {uint32_t(cols), uint32_t(*th ? tpt : G), uint32_t(*th ? G : tpt)};
  const cuuint32_t es[3] = {1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, es,
            CU_TENSOR_MAP_INTERLEAVE_NONE, cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace cross
}  // namespace l3d

using namespace l3d;

extern "C" size_t l3d_cross_attention_workspace_size(int64_t b, int64_t tq, int64_t tk, int64_t hq, int64_t hkv,
                                                     int64_t d, int ragged) {
  if (b <= 0 || tq <= 0 || tk < 0 || hq <= 0 || hkv <= 0 || hq % hkv || hq / hkv > l3d::cross::BQ || d <= 0) return 0;
  const int64_t G = hq / hkv, N = ragged || tq % b ? 0 : tq / b;
  if (l3d::cross::few_rows(b, N, G, tk)) return l3d::decode::workspace_size(b, N, G, hkv, tk, d);
  const int parts = l3d::cross::parts_for(b, tq, tk, G, hkv);
  if (parts <= 1) return 0;
  return (size_t(parts) * size_t(tq * hq) * 4 + 255) / 256 * 256 + size_t(parts) * size_t(tq * hq) * size_t(d) * 4;
}

extern "C" int l3d_cross_attention(const l3d_tensor* q, const l3d_tensor* k, const l3d_tensor* v,
                                   const l3d_tensor* k_offsets, const l3d_tensor* q_offsets, float scale,
                                   const l3d_tensor* out, void* workspace, size_t workspace_bytes,
                                   l3d_stream stream) {
  using namespace l3d::cross;
  const char* op = "l3d_cross_attention";
  if (!q || !k || !v || !k_offsets || !out)
    return fail(L3D_E_NULL, "%s: q, k, v, k_offsets and out are required", op);
  const l3d_tensor* all[] = {q, out, k, v};
  for (const l3d_tensor* t : all) {
    if (t->dtype != q->dtype || (t->dtype != L3D_BF16 && t->dtype != L3D_F16))
      return fail(L3D_E_DTYPE, "%s: q, k, v and out all BF16 or all F16", op);
    if (t->ndim != 3) return fail(L3D_E_SHAPE, "%s: q, out [Tq, Hq, D], k, v [Tk, Hkv, D]", op);
    if (numel(t) > 0 && t->strides[2] != 1) return fail(L3D_E_ALIGN, "%s: the head dim must be contiguous", op);
  }
  const int64_t Tq = q->dims[0], Hq = q->dims[1], D = q->dims[2], Tk = k->dims[0], Hkv = k->dims[1];
  if (D != 64 && D != 128) return fail(L3D_E_UNSUPPORTED, "%s: head dim must be 64 or 128", op);
  for (int i = 0; i < 3; ++i) {
    if (out->dims[i] != q->dims[i]) return fail(L3D_E_SHAPE, "%s: out must have q's shape", op);
    if (v->dims[i] != k->dims[i] || (i == 2 && k->dims[i] != D))
      return fail(L3D_E_SHAPE, "%s: k and v [Tk, Hkv, D]", op);
  }
  if (Hq > 0 && (Hkv <= 0 || Hq % Hkv))
    return fail(L3D_E_SHAPE, "%s: query heads must be a multiple of the key heads", op);
  auto index_list = [](const l3d_tensor* t) {
    return (t->dtype == L3D_I32 || t->dtype == L3D_I64) && t->ndim == 1 && t->dims[0] >= 1 &&
           (t->dims[0] == 1 || t->strides[0] == 1);
  };
  if (!index_list(k_offsets)) return fail(L3D_E_SHAPE, "%s: k_offsets must be contiguous [B + 1] I32 or I64", op);
  const int64_t B = k_offsets->dims[0] - 1;
  if (q_offsets && (!index_list(q_offsets) || q_offsets->dims[0] != B + 1))
    return fail(L3D_E_SHAPE, "%s: q_offsets must be contiguous [B + 1] I32 or I64, as k_offsets", op);
  if (!q_offsets && (B > 0 ? Tq % B != 0 : Tq > 0))
    return fail(L3D_E_SHAPE, "%s: without q_offsets the rows must divide evenly among the sequences", op);
  const float scale_log2 = scale * 1.4426950408889634f;  // finite too
  if (!(scale > 0.f) || !(scale_log2 < INFINITY))
    return fail(L3D_E_UNSUPPORTED, "%s: scale must be positive and finite", op);
  const int64_t big = int64_t(1) << 30;
  if (Tq > big || Tk > big || B > MAX_BATCH || Hq > 65535 || Tq * Hq > big || Hkv * B > MAX_HEADS || Hkv * Tq > big)
    return fail(L3D_E_UNSUPPORTED, "%s: dimensions too large (at most 2^20 sequences, 2^26 times their key heads)", op);
  if (Hkv > 0 && Hq / Hkv > BQ) return fail(L3D_E_UNSUPPORTED, "%s: at most %d query heads per key head", op, BQ);
  if (Tq * Hq == 0 || B == 0) return L3D_OK;
  for (const l3d_tensor* t : {k, v})
    if (Tk > 1 && t->strides[0] == 0) return fail(L3D_E_ALIGN, "%s: the keys must not be expanded (stride 0)", op);
  for (const l3d_tensor* t : {q, out})
    if ((Tq > 1 && t->strides[0] == 0) || (Hq > 1 && t->strides[1] == 0))
      return fail(L3D_E_ALIGN, "%s: q and out must not be expanded (stride 0)", op);
  const size_t need = l3d_cross_attention_workspace_size(B, Tq, Tk, Hq, Hkv, D, q_offsets != nullptr);
  if (need && (!workspace || workspace_bytes < need))
    return fail(L3D_E_WORKSPACE, "%s: workspace of %zu bytes required", op, need);
  if (reinterpret_cast<uintptr_t>(workspace) % 256)
    return fail(L3D_E_ALIGN, "%s: workspace must be 256-byte aligned", op);
  for (const l3d_tensor* t : all) {
    if (no_data(t)) return fail(L3D_E_NULL, "%s: null data pointer", op);
    if (numel(t) == 0) continue;
    if (reinterpret_cast<uintptr_t>(elem_ptr(t)) % 16)
      return fail(L3D_E_ALIGN, "%s: tensors must be 16-byte aligned", op);
    for (int d = 0; d < 2; ++d)
      if (t->dims[d] > 1 && t->strides[d] % 8)
        return fail(L3D_E_ALIGN, "%s: strides must be multiples of 16 bytes", op);
  }
  if (no_data(k_offsets) || (q_offsets && no_data(q_offsets))) return fail(L3D_E_NULL, "%s: null data pointer", op);
  const int64_t G = Hq / Hkv, N = q_offsets ? 0 : Tq / B;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (few_rows(B, N, G, Tk)) {
    l3d::decode::Params p{};
    p.B = int(B); p.N = int(N); p.G = int(G); p.Hkv = int(Hkv);
    p.q = elem_ptr(q);
    p.out = const_cast<char*>(elem_ptr(out));
    p.qb = q->strides[0] * N; p.qn = q->strides[0]; p.qh = q->strides[1];
    p.ob = out->strides[0] * N; p.on = out->strides[0]; p.oh = out->strides[1];
    p.keys = int(Tk);
    p.lengths = elem_ptr(k_offsets);
    p.len64 = k_offsets->dtype == L3D_I64;
    p.scale_log2 = scale_log2;
    const l3d::decode::Keys kv{elem_ptr(k), elem_ptr(v), {0, k->strides[0], k->strides[1]},
                               {0, v->strides[0], v->strides[1]}, D};
    return l3d::decode::launch(op, p, kv, q->dtype == L3D_F16, Tk, workspace, s);
  }
  Params p{};
  p.B = int(B); p.G = int(G); p.Hkv = int(Hkv); p.Tq = int(Tq); p.Tk = int(Tk); p.N = int(N);
  p.tpt = BQ / p.G;
  p.q_offsets = q_offsets ? elem_ptr(q_offsets) : nullptr;
  p.q64 = q_offsets && q_offsets->dtype == L3D_I64;
  p.k_offsets = elem_ptr(k_offsets);
  p.k64 = k_offsets->dtype == L3D_I64;
  p.out = const_cast<char*>(elem_ptr(out));
  p.ot = out->strides[0]; p.oh = out->strides[1];
  p.scale_log2 = scale_log2;
  p.parts = parts_for(B, Tq, Tk, G, Hkv);
  p.part_l = static_cast<float*>(workspace);
  p.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + (size_t(p.parts) * size_t(Tq * Hq) * 4 + 255) / 256 * 256);
  p.wait_ns = l3d::tc::WAIT_LIMIT_NS;
  CUtensorMap maps[4];
  p.k_hm = Hkv > 1 && k->strides[1] == 0 ? 0 : 1;
  p.v_hm = Hkv > 1 && v->strides[1] == 0 ? 0 : 1;
  bool ok = make_row_map(&maps[0], elem_ptr(q), Tq, Hq, D, q->strides[0], q->strides[1], p.G, p.tpt, 64, &p.q_th);
  // A warp's 32 rows as a box of the output: whole tokens with their heads, listed as the rows are.
  maps[3] = maps[0];
  if (p.parts == 1 && 32 % p.G == 0 && (p.G == 1 || !p.q_th)) {
    ok = ok && make_row_map(&maps[3], elem_ptr(out), Tq, Hq, D, out->strides[0], out->strides[1], p.G, 32 / p.G,
                            D == 64 ? Cfg<64>::OUT_COLS : Cfg<128>::OUT_COLS, &p.o_th);
    p.o_tma = ok && (p.G == 1 || !p.o_th);
  }
  if (Tk > 0)
    ok = ok && make_map4(&maps[1], elem_ptr(k), 1, p.k_hm ? Hkv : 1, Tk, D, k->strides[0], k->strides[1], 0, BKV, &p.k_hn) &&
         make_map4(&maps[2], elem_ptr(v), 1, p.v_hm ? Hkv : 1, Tk, D, v->strides[0], v->strides[1], 0, BKV, &p.v_hn);
  else
    maps[1] = maps[2] = maps[0];  // never read
  if (!ok) return fail(L3D_E_CUDA, "%s: cuTensorMapEncodeTiled failed", op);
  const int64_t items = Hkv * (Tq / p.tpt + B) * p.parts;  // at most: a sequence's last tile may be cut short
  if (q->dtype == L3D_BF16)
    e = D == 64 ? launch<__nv_bfloat16, 64>(maps, p, items, s) : launch<__nv_bfloat16, 128>(maps, p, items, s);
  else
    e = D == 64 ? launch<__half, 64>(maps, p, items, s) : launch<__half, 128>(maps, p, items, s);
  return e == cudaSuccess ? L3D_OK : fail(L3D_E_CUDA, "%s: %s", op, cudaGetErrorString(e));
}
