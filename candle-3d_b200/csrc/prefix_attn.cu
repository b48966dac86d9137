// Attention for a batch whose elements share a prefix of keys, plus each
// element's own keys, on the 5th-generation tensor cores:
//   out[b, h, i] = sum_j softmax_j(scale q[b, h, i] . K[j]) V[j]
// over the prefix keys j < P (one copy for the whole batch) and the own keys
// j < lengths[b] of element b; with `causal`, row i sees the own keys up to
// its own place, j <= lengths[b] - N + i.  Query heads h share the key head
// h / G, G = Hq / Hkv.  The reference's attention core is exact_sdpa_heads
// (crate/runtime/attention_math.rs:199-259); a shared prefix would be copied
// into every batch element there.
//
// The query rows of one key head are numbered f = (b N + i) G + g: a tile of
// 128 rows holds the rows of several query heads, and, for the prefix, of
// several batch elements, so that the prefix keys are read once per tile of
// rows and not once per element.  A block takes one item:
//   packed   (row tiles over the whole batch) x (a chunk of prefix tiles), and
//            (row tiles of one element) x (a chunk of its own key tiles);
//   joint    (row tiles of one element) x (a chunk of prefix, then own tiles).
// An item that sees all the keys of its rows stores the output; otherwise it
// stores its part's O / l and log2 of its sum in f32, and combine_kernel
// weighs the parts of each row.  Parts have fixed places, so results do not
// depend on the order in which blocks run.
//
// Within an item a TMA warp fills rings of 64-key K and V tiles; one MMA warp
// per row tile issues S = Q K^T and O += P V (P read from tensor memory); four
// softmax warps per row tile, one row per thread, turn S into P, and also load
// Q (their rows have no common stride) and zero the V rows past an element's
// keys: a masked probability is 0, but 0 x NaN is not.  S has two buffers of 64
// columns per row tile, P going over the scores it comes from: S(j + 2) is
// issued right after P(j) V, while softmax(j + 1) runs, so that neither the
// tensor core nor the softmax warps wait for a whole round trip of the other.
// (With one 128-column buffer a row tile's softmax warps waited 1,500 of 3,830
// clocks per 128 keys at D = 128, and both pipes were about half busy.)
// P is rounded to the type of V, whose product takes both operands in 16 bits: the
// rounding of each probability is as large as that of the output, and the output is
// 1.33 to 1.43 times as far from the 64-bit one as one formed in f32 and rounded
// once (bf16 0.0023 against 0.0017).  The sum of the probabilities, in f32, takes
// them before that rounding.
// Long items are bound at D = 128 by the round trip between the products and the
// softmax (1234 TFLOP/s over 16384 keys, 75% of a plain product's rate; 1455 without
// the softmax), at D = 64 by the softmax itself (694 TFLOP/s); short ones by an item's
// set-up and the rounds over the device.
// Every mbarrier wait is bounded (%globaltimer, 2 s); on expiry the block
// records an error in the device's status word and stops.
#include <type_traits>

#include "attn.cuh"
#include "common.cuh"
#include "tc.cuh"

namespace l3d {
namespace pattn {

using namespace l3d::attn;

constexpr int BQ = 128, BKV = 64;
constexpr int ST_TIMEOUT = 5, ST_MISALIGNED = 6;
// As in attn.cu: the running max moves only when it grows past 2^8.
constexpr float RESCALE_LOG2 = 8.f;

__device__ int g_pattn_status;

// NT row tiles of 128 rows per block; NT = 1 blocks share an SM in pairs, for
// short items, whose set-up one block's work then hides for the other.
template <int D, int NT>
struct Cfg {
  static constexpr int DC = D / 64;
  static constexpr int CTAS = NT == 1 ? 2 : 1;        // per SM
  static constexpr int Q_BYTES = BQ * D * 2;
  static constexpr int KV_BYTES = BKV * D * 2;
  static constexpr int REST = 512;                    // barriers
  // K and V tiles in rings of their own, each released when its product has
  // read it.
  static constexpr int FIT = ((227 * 1024 - (CTAS - 1) * 1024) / CTAS - REST - NT * Q_BYTES) / KV_BYTES;
  static constexpr int BUFS = FIT < 16 ? FIT : 16;
  static constexpr int KST = BUFS / 2, VST = BUFS - KST;
  static constexpr int SMEM = NT * Q_BYTES + BUFS * KV_BYTES + REST;
  static constexpr uint32_t COL_S = 0, COL_O = NT * 2 * BKV;
  static constexpr uint32_t TMEM_COLS = COL_O + NT * D <= 256 ? 256 : 512;
  static constexpr int THREADS = (4 + 4 * NT) * 32;   // TMA and MMA warps, softmax warps
  // Of 8 pairs of P, those of ex2_poly2 (it takes twice ex2's time, on other units).
  // 0, 1, 2 of them: 37 heads x 1024 x 4096 at D 64 70, 66, 64 us; at D 128 1370
  // keys for 8 x 16 heads x 2049 rows 240 us without, 225 with one (and with two).
  static constexpr int POLY = D == 64 ? 2 : 1;
  static_assert(COL_O + NT * D <= TMEM_COLS && TMEM_COLS * CTAS <= 512, "TMEM budget");
  static_assert((2 * BUFS + 7 * NT) * 8 + 16 <= REST, "barrier area");
};

struct View {        // a K or V map: heads listed before rows; 0 for a broadcast dimension
  int hn, hm, bm;
};

struct Params {
  int B, N, G, Hkv;
  int RG, F;                 // rows of one element, of the batch (per key head)
  int P, S;                  // at most 2^30
  View pk, pv, k, v;
  const void* q;
  void* out;
  int64_t qb, qh, qn, ob, oh, on;  // element strides
  const void* lengths;       // [B] or null (= S)
  int len64, causal;
  float scale_log2;          // softmax scale * log2(e), > 0
  float *part_o, *part_l;    // [slots, Hkv, F, D], [slots, Hkv, F]; slots > 1
  int slots, slots_p;        // parts of a row; those of the prefix (packed)
  int joint;
  int prefix_items, tiles_p, tiles_o;  // row tiles (of NT x 128) of the batch, of one element
  int chunk_p, chunk_o;      // key tiles of an item
  uint64_t wait_ns;
};

__device__ __forceinline__ int own_length(const Params& p, int b) {
  if (!p.lengths) return p.S;
  const int64_t v = p.len64 ? static_cast<const int64_t*>(p.lengths)[b]
                            : static_cast<const int32_t*>(p.lengths)[b];
  return v < 0 ? 0 : v < p.S ? int(v) : p.S;
}
// Row f of a key head is query i of head h G + g of element b, f = (b N + i) G + g.
struct Row {
  int b, i, g;
};
__device__ __forceinline__ Row row_at(const Params& p, int f) {
  const int b = f / p.RG, i = (f - b * p.RG) / p.G;
  return {b, i, f - b * p.RG - i * p.G};
}

// 16 consecutive 32-bit TMEM columns of this thread's lane <- registers.
__device__ __forceinline__ void tmem_st16u(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

template <typename T> __device__ __forceinline__ uint32_t pack_pair(float a, float b);
template <> __device__ __forceinline__ uint32_t pack_pair<__nv_bfloat16>(float a, float b) {
  return pack_bf16x2(a, b);
}
template <> __device__ __forceinline__ uint32_t pack_pair<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// As make_idesc, for either 16-bit type.
template <typename T>
constexpr uint32_t idesc_of(int m, int n) {
  return make_idesc(m, n) & ~(sizeof(T) == 2 && std::is_same<T, __half>::value ? (1u << 7) | (1u << 10) : 0u);
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(Cfg<D, NT>::THREADS, Cfg<D, NT>::CTAS)
    prefix_kernel(const __grid_constant__ CUtensorMap map_pk,
                  const __grid_constant__ CUtensorMap map_pv,
                  const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const Params p) {
  using C = Cfg<D, NT>;
  constexpr uint32_t IDESC_S = idesc_of<T>(128, BKV);
  constexpr uint32_t IDESC_O = idesc_of<T>(128, D) | (1u << 16);  // B (V) MN-major
  int* const status = &g_pattn_status;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  if (smem_u32(smem_raw) & 1023u) {
    if (threadIdx.x == 0) atomicCAS(status, 0, ST_MISALIGNED);
    return;
  }
  uint8_t* sq = smem_raw;                            // [NT][DC][128 x 64]
  uint8_t* sk = sq + NT * C::Q_BYTES;                // [KST][DC][128 x 64]
  uint8_t* sv = sk + C::KST * C::KV_BYTES;           // [VST][DC][128 x 64]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sv + C::VST * C::KV_BYTES);
  uint64_t* k_full = bars;                           // [KST]
  uint64_t* k_empty = k_full + C::KST;               // [KST]
  uint64_t* v_full = k_empty + C::KST;               // [VST]
  uint64_t* v_empty = v_full + C::VST;               // [VST]
  uint64_t* s_full = v_empty + C::VST;               // [NT][2] (by S buffer)
  uint64_t* p_full = s_full + 2 * NT;                // [NT][2]
  uint64_t* pv_done = p_full + 2 * NT;               // [NT][2]
  uint64_t* mma_drain = pv_done + 2 * NT;            // [NT] abort teardown only
  volatile int* abort_flag = reinterpret_cast<volatile int*>(mma_drain + NT);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_drain + NT + 1);

  // (The shuffle tells the compiler that the role is the same in all lanes.)
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.launch_dependents;");
  // ---- this block's item: rows [f0, fend) of key head h, prefix tiles
  // [pa, pa + np), own tiles [sa, sa + nkv - np) of element b.
  int idx = blockIdx.x;
  int f0, fend, h, b = 0, pa, np, sa = 0, nkv, slot;
  int len = 0;
  if (idx < p.prefix_items) {
    const int qt = idx % p.tiles_p;
    idx /= p.tiles_p;
    h = idx % p.Hkv;
    slot = idx / p.Hkv;
    f0 = qt * (NT * BQ);
    fend = p.F;
    const int tiles = (p.P + BKV - 1) / BKV;
    pa = slot * p.chunk_p;
    np = max(min(p.chunk_p, tiles - pa), 0);
    nkv = np;
  } else {
    idx -= p.prefix_items;
    const int qt = idx % p.tiles_o;
    idx /= p.tiles_o;
    h = idx % p.Hkv;
    idx /= p.Hkv;
    b = idx % p.B;
    const int part = idx / p.B;
    f0 = b * p.RG + qt * (NT * BQ);
    fend = (b + 1) * p.RG;
    len = own_length(p, b);
    // Own keys that the last of the item's rows sees.
    int seen = len;
    if (p.causal) seen = max(min(len, len - p.N + row_at(p, min(f0 + NT * BQ, fend) - 1).i + 1), 0);
    const int own = (seen + BKV - 1) / BKV;
    const int pre = p.joint ? (p.P + BKV - 1) / BKV : 0;
    const int c0 = part * p.chunk_o;
    const int c1 = min(c0 + p.chunk_o, pre + own);
    pa = min(c0, pre);
    np = max(min(c1, pre) - pa, 0);
    sa = max(c0 - pre, 0);
    nkv = max(c1 - c0, 0);
    slot = (p.joint ? 0 : p.slots_p) + part;
  }
  const int ntv = min((fend - f0 + BQ - 1) / BQ, NT);  // row tiles that hold rows
  // Key tile j of K or V into its ring (thread 0).
  int loaded_k = 0, loaded_v = 0;
  auto load = [&](uint8_t* dst, uint64_t* bar, int j, const CUtensorMap* mp, const CUtensorMap* mo,
                  const View& wp, const View& wo) {
    mbar_expect_tx(bar, C::KV_BYTES);
    const bool pre = j < np;
    const int row = (pre ? pa + j : sa + j - np) * BKV;
    const View& w = pre ? wp : wo;
    const int hh = h * w.hm, bb = pre ? 0 : b * w.bm;
    for (int dc = 0; dc < C::DC; ++dc)
      tma_load_4d(dst + dc * (BKV * 128), pre ? mp : mo, bar, dc * 64, w.hn ? hh : row, w.hn ? row : hh, bb);
  };
  auto load_k = [&] {
    const int s = loaded_k % C::KST;
    load(sk + s * C::KV_BYTES, &k_full[s], loaded_k++, &map_pk, &map_k, p.pk, p.k);
  };
  auto load_v = [&] {
    const int s = loaded_v % C::VST;
    load(sv + s * C::KV_BYTES, &v_full[s], loaded_v++, &map_pv, &map_v, p.pv, p.v);
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::KST; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], ntv);  // one commit per MMA warp with rows
    }
    for (int s = 0; s < C::VST; ++s) {
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], ntv);
    }
    for (int i = 0; i < 2 * NT; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&pv_done[i], 1);
    }
    for (int t = 0; t < NT; ++t) mbar_init(&mma_drain[t], 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    for (int j = 0; j < nkv && j < C::VST; ++j) {
      if (j < C::KST) load_k();
      load_v();
    }
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(C::TMEM_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  // The softmax threads' row: row tile st, TMEM lane quarter warp % 4.
  const int st = (warp - 4) >> 2;
  const int r = (warp & 3) * 32 + lane;
  const int f = f0 + st * BQ + r;                // flattened row
  const bool valid = f < fend;
  if (warp >= 4 && st < ntv) {
    const Row w = row_at(p, valid ? f : fend - 1);
    const T* qr = static_cast<const T*>(p.q) + w.b * p.qb + int64_t(h * p.G + w.g) * p.qh + w.i * p.qn;
    uint8_t* qt = sq + st * C::Q_BYTES + r * 128;
    uint4 u[D / 8];
#pragma unroll
    for (int c = 0; c < D / 8; ++c)
      u[c] = valid ? __ldg(reinterpret_cast<const uint4*>(qr) + c) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int c = 0; c < D / 8; ++c)
      *reinterpret_cast<uint4*>(qt + (c >> 3) * (BQ * 128) + (((c & 7) ^ (r & 7)) << 4)) = u[c];
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
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

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      while ((loaded_k < nkv || loaded_v < nkv) && !*abort_flag) {
        if (loaded_k < nkv) {
          if (!wait(&k_empty[loaded_k % C::KST], (loaded_k / C::KST - 1) & 1)) break;
          load_k();
        }
        if (loaded_v < nkv) {
          if (!wait(&v_empty[loaded_v % C::VST], (loaded_v / C::VST - 1) & 1)) break;
          load_v();
        }
      }
    }
  } else if (warp <= ntv) {
    // ------------------------------------------------------------------ MMA
    // One warp per row tile.  The whole warp keeps step and one elected lane
    // issues, so that loop state and descriptors stay in uniform registers
    // (issuing from a divergent branch took 27% longer per key tile).
    const int t = warp - 1;
    const bool leader = elect_one();
    auto commit = [&](uint64_t* bar) {
      if (leader) umma_commit(bar);
    };
    const uint32_t t_s = tmem_base + C::COL_S + t * (2 * BKV), t_o = tmem_base + C::COL_O + t * D;
    auto issue_s = [&](int j) {
      const uint64_t da = smem_desc_sw128(sq + t * C::Q_BYTES);
      const uint64_t db = smem_desc_sw128(sk + (j % C::KST) * C::KV_BYTES);
      if (leader) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          umma_f16<IDESC_S>(t_s + (j & 1) * BKV, da + uint64_t((k >> 2) * (BQ * 128 >> 4) + 2 * (k & 3)),
                            db + uint64_t((k >> 2) * (BKV * 128 >> 4) + 2 * (k & 3)), k ? 1u : 0u);
      }
      commit(&s_full[2 * t + (j & 1)]);
      commit(&k_empty[j % C::KST]);
    };
    auto issue_pv = [&](int j) {
      const uint64_t db = smem_desc_sw128_mn(sv + (j % C::VST) * C::KV_BYTES, BKV * 128);
      if (leader) {
#pragma unroll
        for (int ks = 0; ks < BKV / 16; ++ks)
          umma_f16_ts<IDESC_O>(t_o, t_s + (j & 1) * BKV + uint32_t(ks * 8),
                               db + uint64_t(ks * (16 * 128 >> 4)), (j | ks) ? 1u : 0u);
      }
      commit(&v_empty[j % C::VST]);
      commit(&pv_done[2 * t + (j & 1)]);  // the last commit of an item: the block waits for it
    };
    bool ok = true;
    for (int j = 0; ok && j < 2 && j < nkv; ++j) {
      ok = wait_warp(&k_full[j % C::KST], (j / C::KST) & 1);
      if (!ok) break;
      tc_fence_after();
      issue_s(j);
    }
    for (int j = 0; ok && j < nkv; ++j) {
      ok = wait_warp(&p_full[2 * t + (j & 1)], (j >> 1) & 1) &&
           wait_warp(&v_full[j % C::VST], (j / C::VST) & 1);
      if (!ok) break;
      tc_fence_after();
      issue_pv(j);
      if (j + 2 < nkv) {
        ok = wait_warp(&k_full[(j + 2) % C::KST], ((j + 2) / C::KST) & 1);
        if (!ok) break;
        tc_fence_after();
        issue_s(j + 2);  // over P(j), which the product before it has read
      }
    }
  } else if (warp >= 4 && st < ntv) {
    // ------------------------------------------------------ softmax / epilogue
    const int t = st, quarter = warp & 3;
    const bool active = f - lane < fend;  // the warp holds rows
    // Own keys that this row sees.
    const int lim = p.causal ? min(len, len - p.N + row_at(p, valid ? f : fend - 1).i + 1) : len;
    const uint32_t lane_off = uint32_t(quarter * 32) << 16;
    const uint32_t t_s = tmem_base + C::COL_S + t * (2 * BKV) + lane_off;
    const uint32_t t_o = tmem_base + C::COL_O + t * D + lane_off;
    const float2 sc2 = f2(p.scale_log2);
    float m = -INFINITY;                         // running max, log2 units
    float2 l2 = f2(0.f);                         // running row sum (two parts)
    bool ok = true;
    for (int j = 0; j < nkv; ++j) {
      ok = wait_warp(&s_full[2 * t + (j & 1)], (j >> 1) & 1);
      if (!ok) break;
      tc_fence_after();
      const bool pre = j < np;
      const int key0 = (pre ? pa + j : sa + j - np) * BKV;
      // V rows past the element's keys may hold anything: zero them, once the
      // tile has landed (two threads per row).
      const int held = pre ? BKV : min(len - key0, BKV);
      if (held < BKV) {
        ok = wait_warp(&v_full[j % C::VST], (j / C::VST) & 1);
        if (!ok) break;
        const int vrow = r & (BKV - 1);
        if (vrow >= held) {
          uint8_t* vr = sv + (j % C::VST) * C::KV_BYTES + vrow * 128;
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            const int c = (r / BKV) * (D / 16) + i;
            *reinterpret_cast<uint4*>(vr + (c >> 3) * (BKV * 128) + ((c & 7) << 4)) = make_uint4(0, 0, 0, 0);
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
      }
      if (!active) {  // no rows: keep the other warps' pace
        if (lane == 0) mbar_arrive(&p_full[2 * t + (j & 1)]);
        continue;
      }
      const uint32_t t_sj = t_s + (j & 1) * BKV;
      float s[BKV];
      tmem_ld64(t_sj, s);
      const int kvalid = (pre ? p.P : lim) - key0;  // keys of this tile that the row sees
      if (kvalid < BKV) {
#pragma unroll
        for (int e = 0; e < BKV; ++e)
          if (e >= kvalid) s[e] = -INFINITY;
      }
      __syncwarp();
      float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int e = 4; e < BKV; e += 2) mx[(e >> 1) & 3] = max_nan(mx[(e >> 1) & 3], s[e], s[e + 1]);
      const float mxs = max_nan(max_nan(mx[0], mx[1], mx[2]), mx[3]) * p.scale_log2;  // scale > 0
      const bool grow = !(mxs <= m + RESCALE_LOG2);       // always on the first key a row sees
      const float m_new = grow ? mxs : m;
      const float alpha = grow ? ex2f(m - m_new) : 1.f;   // 0 on the first
      if (j > 0 && __any_sync(0xffffffffu, grow)) {
        ok = wait_warp(&pv_done[2 * t + ((j - 1) & 1)], ((j - 1) >> 1) & 1);  // O_t is stable
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
      // P = exp2(s * scale * log2 e - m); a row that has seen no key yet has
      // m = -inf and all its scores masked: subtract 0, so that P = 0.
      const float2 nm2 = f2(m_new == -INFINITY ? 0.f : minus_max(m_new));
      l2 = mul2(l2, f2(alpha));
      // In pieces of 32 scores, stored to TMEM as they are formed (one store of
      // all 64 measured 7% slower over short key ranges).
#pragma unroll
      for (int c = 0; c < BKV; c += 32) {
        uint32_t u[16];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float2 x = fma2(make_float2(s[c + e], s[c + e + 1]), sc2, nm2);
          const float2 pr = ((e >> 1) & 7) < C::POLY ? ex2_poly2(x)
                                                     : make_float2(ex2f(x.x), ex2f(x.y));
          l2 = add2(l2, pr);
          u[e >> 1] = pack_pair<T>(pr.x, pr.y);
        }
        tmem_st16u(t_sj + uint32_t(c / 2), u);
      }
      m = m_new;
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[2 * t + (j & 1)]);
    }
    // Epilogue, after the last P V: the output, or this part's O / l and log2 sum.
    // (A barrier per S buffer: of one barrier for all products, two phases could
    // pass before this thread looks.  S(j) complete says that P(j - 2) V is done.)
    if (ok && nkv > 0) ok = wait_warp(&pv_done[2 * t + ((nkv - 1) & 1)], ((nkv - 1) >> 1) & 1);
    tc_fence_after();
    if (ok && active) {
      // (A row that has seen no key: ex2_poly2 gives 1e-42 for -inf, not 0.)
      float l = l2.x + l2.y;
      if (m == -INFINITY && l == l) l = 0.f;
      const float inv = l > 0.f ? 1.f / l : l == l ? 0.f : l;  // no keys: zeros; NaN stays
      const int64_t pr = (int64_t(slot) * p.Hkv + h) * p.F + f;
      if (p.slots > 1 && valid) p.part_l[pr] = l > 0.f ? m + log2f(l) : l == l ? -INFINITY : l;
      const Row w = row_at(p, valid ? f : fend - 1);
      T* orow = static_cast<T*>(p.out) + w.b * p.ob + int64_t(h * p.G + w.g) * p.oh + w.i * p.on;
      __syncwarp();  // the loads from tensor memory are the whole warp's
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        float o[32];
        if (nkv > 0) {
          tmem_ld32(t_o + uint32_t(c), o);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0.f;
        }
        if (valid) {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] *= inv;
          if (p.slots > 1) {
            float4* dst = reinterpret_cast<float4*>(p.part_o + pr * D + c);
#pragma unroll
            for (int e = 0; e < 8; ++e) dst[e] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              float v[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] = o[8 * q + e];
              *reinterpret_cast<uint4*>(orow + c + 8 * q) = pack(v, T());
            }
          }
        }
        __syncwarp();
      }
    }
  }

  // Teardown, as in attn.cu: after an abort nothing the block started may
  // still be running when it frees TMEM and exits.
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    if (warp >= 1 && warp <= NT && elect_one()) {  // the lane that issued
      umma_commit(&mma_drain[warp - 1]);
      mbar_drain(&mma_drain[warp - 1], 0, p.wait_ns);
    }
    if (threadIdx.x == 0) {
      // The newest load of each ring buffer.
      for (int i = max(loaded_k - C::KST, 0); i < loaded_k; ++i)
        mbar_drain(&k_full[i % C::KST], uint32_t(i / C::KST) & 1u, p.wait_ns);
      for (int i = max(loaded_v - C::VST, 0); i < loaded_v; ++i)
        mbar_drain(&v_full[i % C::VST], uint32_t(i / C::VST) & 1u, p.wait_ns);
    }
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base),
                 "r"(C::TMEM_COLS));
  }
}

// Bound by the parts' bytes.  The parts of each row weighed by 2^(their log2 sum - the largest): a block of
// four warps per row, each with every fourth part, D / 32 elements per lane;
// added up in a fixed order.
constexpr int MAX_SLOTS = 64;
template <typename T, int D>
__global__ void __launch_bounds__(128) combine_kernel(const Params p) {
  constexpr int E = D / 32, W = 4, PER = MAX_SLOTS / W;
  using Vec = typename std::conditional<E == 4, float4, float2>::type;
  __shared__ Vec red[W - 1][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = blockIdx.x;  // h F + f
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t stride = int64_t(p.Hkv) * p.F;
  float w[2], mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int s = lane + 32 * i;
    w[i] = s < p.slots ? p.part_l[s * stride + row] : -INFINITY;
    mx = fmaxf(mx, w[i]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    w[i] = w[i] == -INFINITY ? 0.f : exp2f(w[i] - mx);
    sum += w[i];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  alignas(16) float acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  const Vec* src = reinterpret_cast<const Vec*>(p.part_o + row * D) + lane;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int s = i * W + warp;
    if (s >= p.slots) break;
    const float ws = __shfl_sync(0xffffffffu, i * W < 32 ? w[0] : w[1], s & 31);
    if (ws == 0.f) continue;  // a part without keys: nothing is stored there
    const Vec v = src[s * stride * (D / E)];
    acc[0] = fmaf(ws, v.x, acc[0]);
    acc[1] = fmaf(ws, v.y, acc[1]);
    if constexpr (E == 4) {
      acc[2] = fmaf(ws, v.z, acc[2]);
      acc[3] = fmaf(ws, v.w, acc[3]);
    }
  }
  if (warp > 0) red[warp - 1][lane] = *reinterpret_cast<const Vec*>(acc);
  __syncthreads();
  if (warp > 0) return;
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
  const int h = int(row / p.F);
  const Row at = row_at(p, int(row % p.F));
  T* orow = static_cast<T*>(p.out) + at.b * p.ob + int64_t(h * p.G + at.g) * p.oh + at.i * p.on + lane * E;
  alignas(8) T o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    float t = acc[e];
#pragma unroll
    for (int i = 0; i < W - 1; ++i) t += reinterpret_cast<const float*>(&red[i][lane])[e];
    o[e] = from_f<T>(t * inv);
  }
  if constexpr (E == 4) *reinterpret_cast<uint2*>(orow) = *reinterpret_cast<const uint2*>(o);
  else *reinterpret_cast<uint32_t*>(orow) = *reinterpret_cast<const uint32_t*>(o);
}

// How the rows and keys are divided into items (host).
struct Plan {
  int nt, joint, tiles_p, tiles_o, chunk_p, chunk_o, slots_p, slots, items;
};

// The plan with the least estimated time: one or two row tiles per block, the
// prefix for the rows of the whole batch (packed) or of each element (joint),
// and some lengths of an item.  An item of `len` key tiles takes about
//   D = 128: 5.5 + 1.00 len us (one row tile, two blocks per SM), 7.5 + 0.96 len (two),
//   D = 64:  2.0 + 0.89 len us,                                   2.5 + 0.87 len,
// fitted to 37 heads x 1024 rows x 256 .. 16384 keys; a call takes 5 us besides, and
// parts 3 us and their bytes.  Measured, with the estimate behind it:
//   8 x 16 heads x 2049 rows, 1370 keys, D 128: one tile 194 us (197), two 225 (234);
//   8 x 16 heads x 300 rows, 1370 + 300 keys, D 128: joint 66 us (70), packed 86 (84);
//   64 x 4 key heads x 4 rows, 32768 + 512 keys: packed 41 us, joint 428.
static Plan make_plan(int64_t B, int64_t Hq, int64_t Hkv, int64_t N, int64_t P, int64_t S, int64_t D) {
  auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  const int64_t RG = N * (Hq / Hkv), F = B * RG, kp = up(P, BKV), ko = up(S, BKV), half = MAX_SLOTS / 2;
  Plan best{};
  double least = 1e300;
  for (int nt = 1; nt <= 2; ++nt) {
    const double fixed = D == 64 ? (nt == 1 ? 2.0 : 2.5) : nt == 1 ? 5.5 : 7.5;
    const double tile = D == 64 ? (nt == 1 ? 0.89 : 0.87) : nt == 1 ? 1.0 : 0.96;
    const double cap = double(sm_count()) * (nt == 1 ? 2 : 1);
    const int64_t tp = up(F, nt * BQ), to = up(RG, nt * BQ);
    if (nt == 2 && F <= BQ) break;  // the second tile would be empty
    for (int joint = 0; joint <= (S > 0 ? 1 : 0); ++joint) {
      const int64_t kmax = joint ? kp + ko : kp > ko ? kp : ko;
      const double work = double(Hkv) * (joint ? double(B * to) * double(kp + ko) : double(tp) * double(kp) + double(B * to) * double(ko));
      const int64_t even = int64_t(work / cap) + 1;
      for (const int64_t want : {kmax, even, even + even / 4 + 1}) {  // whole, or a device's worth
        int64_t chunk = want < 2 ? 2 : want;
        if (chunk * half < kmax) chunk = up(kmax, half);
        Plan pl{nt, joint, int(tp), int(to), joint ? 0 : int(chunk), int(chunk), 0, 0, 0};
        double time, items, longest;
        if (joint) {
          pl.slots = kmax > 0 ? int(up(kmax, chunk)) : 1;
          items = double(Hkv * B * to) * pl.slots;
          longest = fixed + tile * double(chunk < kmax ? chunk : kmax);
          time = ceil(items / cap) * longest;
        } else {
          const int so = int(up(ko, chunk));
          pl.slots_p = kp > 0 || so == 0 ? int(kp > 0 ? up(kp, chunk) : 1) : 0;
          pl.slots = pl.slots_p + so;
          const double np = double(Hkv * tp) * pl.slots_p, no = double(Hkv * B * to) * so;
          const double lp = fixed + tile * double(chunk < kp ? chunk : kp), lo = fixed + tile * double(chunk < ko ? chunk : ko);
          items = np + no;
          longest = np > 0 && (no == 0 || lp > lo) ? lp : lo;
          time = np == 0 || no == 0 ? ceil(items / cap) * longest : (np * lp + no * lo) / cap + 0.5 * longest;
          if (time < longest) time = longest;
        }
        if (pl.slots > 1) time += 3.0 + double(pl.slots) * double(Hkv * F) * double(D) * 8.0 / 8e6;
        if (time < least * 0.999 && items < 2147483648.0) {
          least = time;
          best = pl;
          best.items = int(items);
        }
      }
    }
  }
  return best;
}

template <typename T, int D, int NT>
static cudaError_t launch(const CUtensorMap (&maps)[4], const Params& p, int items, cudaStream_t s) {
  auto k = prefix_kernel<T, D, NT>;
  const cudaError_t e = set_smem_limit(reinterpret_cast<const void*>(k), Cfg<D, NT>::SMEM);
  if (e != cudaSuccess) return e;
  k<<<unsigned(items), Cfg<D, NT>::THREADS, Cfg<D, NT>::SMEM, s>>>(maps[0], maps[1], maps[2], maps[3], p);
  if (p.slots <= 1) return cudaGetLastError();
  // The combination may be scheduled while the items finish; it waits for them.
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(p.Hkv) * unsigned(p.F));
  cfg.blockDim = dim3(128);
  cfg.stream = s;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, combine_kernel<T, D>, p);
}

template <typename T>
static cudaError_t launch_d(int D, int nt, const CUtensorMap (&maps)[4], const Params& p, int items,
                            cudaStream_t s) {
  if (D == 64) return nt == 1 ? launch<T, 64, 1>(maps, p, items, s) : launch<T, 64, 2>(maps, p, items, s);
  return nt == 1 ? launch<T, 128, 1>(maps, p, items, s) : launch<T, 128, 2>(maps, p, items, s);
}

// The map of a K or V view [B, H, rows, D]; a broadcast dimension (stride 0)
// is described once.
static bool make_view(CUtensorMap* m, View* w, const void* base, int64_t B, int64_t H, int64_t rows,
                      int64_t D, int64_t sb, int64_t sh, int64_t sn) {
  w->bm = B > 1 && sb == 0 ? 0 : 1;
  w->hm = H > 1 && sh == 0 ? 0 : 1;
  return make_map4(m, base, w->bm ? B : 1, w->hm ? H : 1, rows, D, sn, sh, sb, BKV, &w->hn);
}

cudaError_t status_read(int* status, int reset) {
  cudaError_t e = cudaMemcpyFromSymbol(status, g_pattn_status, sizeof(int));
  if (e == cudaSuccess && reset) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_pattn_status, &zero, sizeof(int));
  }
  return e;
}

}  // namespace pattn
}  // namespace l3d

using namespace l3d;

extern "C" size_t l3d_shared_prefix_attention_workspace_size(int64_t b, int64_t hq, int64_t hkv,
                                                             int64_t n, int64_t p, int64_t s,
                                                             int64_t d) {
  if (b <= 0 || hq <= 0 || hkv <= 0 || n <= 0 || p < 0 || s < 0 || d <= 0 || hq % hkv) return 0;
  const l3d::pattn::Plan pl = l3d::pattn::make_plan(b, hq, hkv, n, p, s, d);
  // O and the log2 sums of each row's parts, in f32.
  return pl.slots > 1 ? size_t(pl.slots) * size_t(b) * size_t(hq) * size_t(n) * (size_t(d) + 1) * 4 : 0;
}

extern "C" int l3d_shared_prefix_attention(const l3d_tensor* q, const l3d_tensor* prefix_k,
                                           const l3d_tensor* prefix_v, const l3d_tensor* k,
                                           const l3d_tensor* v, const l3d_tensor* lengths,
                                           int causal, float scale, const l3d_tensor* out,
                                           void* workspace, size_t workspace_bytes,
                                           l3d_stream stream) {
  using namespace l3d::pattn;
  const char* op = "l3d_shared_prefix_attention";
  if (!q || !prefix_k || !prefix_v || !out)
    return fail(L3D_E_NULL, "%s: q, prefix_k, prefix_v and out are required", op);
  if (!k != !v) return fail(L3D_E_NULL, "%s: k and v come together", op);
  if (!k && (lengths || causal))
    return fail(L3D_E_SHAPE, "%s: lengths and causal need own keys", op);
  const l3d_tensor* all[] = {q, out, prefix_k, prefix_v, k, v};
  for (int i = 0; i < 6; ++i) {
    const l3d_tensor* t = all[i];
    if (!t) continue;
    const int nd = i == 2 || i == 3 ? 3 : 4;
    if (t->dtype != q->dtype || (t->dtype != L3D_BF16 && t->dtype != L3D_F16))
      return fail(L3D_E_DTYPE, "%s: all tensors BF16 or all F16", op);
    if (t->ndim != nd)
      return fail(L3D_E_SHAPE, "%s: q, k, v, out [B, H, N, D], prefix_k, prefix_v [H, P, D]", op);
    if (numel(t) > 0 && t->strides[nd - 1] != 1)
      return fail(L3D_E_ALIGN, "%s: the head dim must be contiguous", op);
  }
  const int64_t B = q->dims[0], Hq = q->dims[1], N = q->dims[2], D = q->dims[3];
  const int64_t Hkv = prefix_k->dims[0], P = prefix_k->dims[1], S = k ? k->dims[2] : 0;
  if (D != 64 && D != 128) return fail(L3D_E_UNSUPPORTED, "%s: head dim must be 64 or 128", op);
  for (int i = 0; i < 4; ++i)
    if (out->dims[i] != q->dims[i]) return fail(L3D_E_SHAPE, "%s: out must have q's shape", op);
  if (prefix_k->dims[2] != D || prefix_v->dims[0] != Hkv || prefix_v->dims[1] != P || prefix_v->dims[2] != D)
    return fail(L3D_E_SHAPE, "%s: prefix_k and prefix_v [Hkv, P, D]", op);
  if (k && (k->dims[0] != B || k->dims[1] != Hkv || k->dims[3] != D || v->dims[0] != B ||
            v->dims[1] != Hkv || v->dims[2] != S || v->dims[3] != D))
    return fail(L3D_E_SHAPE, "%s: k and v [B, Hkv, S, D]", op);
  if (Hq > 0 && (Hkv <= 0 || Hq % Hkv))
    return fail(L3D_E_SHAPE, "%s: query heads must be a multiple of the key heads", op);
  if (lengths) {
    if (lengths->dtype != L3D_I32 && lengths->dtype != L3D_I64)
      return fail(L3D_E_DTYPE, "%s: lengths must be I32 or I64", op);
    if (lengths->ndim != 1 || lengths->dims[0] != B || (B > 1 && lengths->strides[0] != 1))
      return fail(L3D_E_SHAPE, "%s: lengths must be contiguous [B]", op);
    if (no_data(lengths)) return fail(L3D_E_NULL, "%s: null data pointer", op);
  }
  const float scale_log2 = scale * 1.4426950408889634f;  // finite too
  if (!(scale > 0.f) || !(scale_log2 < INFINITY))
    return fail(L3D_E_UNSUPPORTED, "%s: scale must be positive and finite", op);
  const int64_t big = int64_t(1) << 30;  // also keeps key and row arithmetic in 32 bits
  if (B > 65535 || Hq > 65535 || N > big || P > big || S > big || B * Hq * N > big)
    return fail(L3D_E_UNSUPPORTED, "%s: dimensions too large", op);
  const l3d_tensor* kvs[] = {prefix_k, prefix_v, k, v};
  for (const l3d_tensor* t : kvs)
    if (t && t->dims[t->ndim - 2] > 1 && t->strides[t->ndim - 2] == 0)
      return fail(L3D_E_ALIGN, "%s: the keys must not be expanded (stride 0)", op);
  const size_t need = l3d_shared_prefix_attention_workspace_size(B, Hq, Hkv, N, P, S, D);
  if (need && (!workspace || workspace_bytes < need))
    return fail(L3D_E_WORKSPACE, "%s: workspace of %zu bytes required", op, need);
  if (reinterpret_cast<uintptr_t>(workspace) % 256)
    return fail(L3D_E_ALIGN, "%s: workspace must be 256-byte aligned", op);
  if (B * Hq * N == 0) return L3D_OK;
  for (int i = 0; i < 6; ++i) {
    const l3d_tensor* t = all[i];
    if (!t) continue;
    if (no_data(t)) return fail(L3D_E_NULL, "%s: null data pointer", op);
    if (numel(t) == 0) continue;
    if (reinterpret_cast<uintptr_t>(elem_ptr(t)) % 16)
      return fail(L3D_E_ALIGN, "%s: tensors must be 16-byte aligned", op);
    for (int d = 0; d < t->ndim - 1; ++d)
      if (t->dims[d] > 1 && t->strides[d] % 8)
        return fail(L3D_E_ALIGN, "%s: strides must be multiples of 16 bytes", op);
  }
  const Plan pl = make_plan(B, Hq, Hkv, N, P, S, D);
  Params p{};
  p.B = int(B); p.N = int(N); p.G = int(Hq / Hkv); p.Hkv = int(Hkv);
  p.RG = int(N * p.G); p.F = int(B) * p.RG;
  p.P = int(P); p.S = int(S);
  p.q = elem_ptr(q);
  p.out = const_cast<char*>(elem_ptr(out));
  p.qb = q->strides[0]; p.qh = q->strides[1]; p.qn = q->strides[2];
  p.ob = out->strides[0]; p.oh = out->strides[1]; p.on = out->strides[2];
  p.lengths = lengths ? elem_ptr(lengths) : nullptr;
  p.len64 = lengths && lengths->dtype == L3D_I64;
  p.causal = causal != 0;
  p.scale_log2 = scale_log2;
  p.slots = pl.slots; p.slots_p = pl.slots_p; p.joint = pl.joint;
  p.tiles_p = pl.tiles_p; p.tiles_o = pl.tiles_o;
  p.chunk_p = pl.chunk_p; p.chunk_o = pl.chunk_o;
  p.prefix_items = pl.joint ? 0 : int(Hkv) * pl.tiles_p * pl.slots_p;
  p.part_o = static_cast<float*>(workspace);
  p.part_l = p.part_o + size_t(pl.slots) * Hkv * p.F * D;
  p.wait_ns = l3d::tc::WAIT_LIMIT_NS;
  // Views without elements are never read; any valid map stands in for theirs.
  CUtensorMap maps[4];
  bool ok = true;
  if (P > 0)
    ok = make_view(&maps[0], &p.pk, elem_ptr(prefix_k), 1, Hkv, P, D, 0, prefix_k->strides[0], prefix_k->strides[1]) &&
         make_view(&maps[1], &p.pv, elem_ptr(prefix_v), 1, Hkv, P, D, 0, prefix_v->strides[0], prefix_v->strides[1]);
  if (ok && S > 0)
    ok = make_view(&maps[2], &p.k, elem_ptr(k), B, Hkv, S, D, k->strides[0], k->strides[1], k->strides[2]) &&
         make_view(&maps[3], &p.v, elem_ptr(v), B, Hkv, S, D, v->strides[0], v->strides[1], v->strides[2]);
  if (!ok) return fail(L3D_E_CUDA, "%s: cuTensorMapEncodeTiled failed", op);
  if (P == 0 && S > 0) { maps[0] = maps[2]; maps[1] = maps[3]; }
  if (S == 0 && P > 0) { maps[2] = maps[0]; maps[3] = maps[1]; }
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const cudaError_t e = q->dtype == L3D_BF16 ? launch_d<__nv_bfloat16>(int(D), pl.nt, maps, p, pl.items, s)
                                             : launch_d<__half>(int(D), pl.nt, maps, p, pl.items, s);
  if (e != cudaSuccess) return fail(L3D_E_CUDA, "%s: %s", op, cudaGetErrorString(e));
  return L3D_OK;
}
