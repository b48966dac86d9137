// Attention of the newest token (or a few) of each request over its cached keys:
//   out[b, i, h] = sum_j softmax_j(scale q[b, i, h] . K[j]) V[j]
// over the keys j < lengths[b] - N + 1 + i, which lie in pages: key j of request b in slot j % size of page
// table[b, j / size]; or, for single rows of cross attention, over a packed stretch of an encoder's states.
// The reference's attention core is exact_sdpa_heads (crate/runtime/attention_math.rs:199-259); it has no cache.
//
// Bound by the bytes of K and V, each read once: a key head's rows (i, g), N G of them, in tiles of 8 or 16.
// The products are taken the other way round, S^T = K Q^T and O^T = V^T P^T, so that keys and head dim fill the 16
// rows of mma.m16n8k16 and the query rows its 8 columns: up to 8 rows cost half of what they would as the 16 rows
// of S = Q K^T (in instructions, products and registers).  The 5th-generation tensor core takes tiles of 128
// rows, and a round trip through its memory for each.
//
// Work is divided by keys alone: all (request, key head, row tile) have their keys in tiles of 16 (32 at
// D = 64: 8 KB of K and V either way), the tiles of all of them in one line, and every warp of the device takes an
// equal stretch of the line, whatever the lengths are; the lengths are read on the device, and each block sums them
// up for itself.  A warp works
// alone: its own ring of tiles in shared memory, filled by TMA boxes that lie in one page each and run on across
// the ends of requests, its own running maximum and sum, no barrier with another warp.  Where a stretch holds all
// the keys of a request's head, the warp stores the output; otherwise O / l and the log2 of the sum in f32, and
// combine_kernel weighs the parts of each row.  A part's place follows from the lengths, so results do not
// depend on the order in which warps run.
// Short caches of a few requests need neither line nor second kernel: a block takes all the keys of a head and row
// tile, a stretch of them per warp, and joins the parts in shared memory (ALONE).  What a table has room for decides, for
// lengths are not on the host: 300 keys in a table for 16384 take 3.6 us more than in one for 304.
//
// Scores with f32 accumulators, P in two 16-bit parts whose sum keeps 16 bits of each probability, or in f16 2^-31 of
// the row's largest where that is more (the products are not what bounds the kernel).
// A table entry outside the cache makes the key's score NaN, and so its row; a length past the table the same.
// Every wait for a load is bounded (%globaltimer, 2 s); on expiry the warp records an error in the device's
// status word and stops.
// Measured, D = 128: 8 x 65536 keys x 4 heads 172 us (6.25 TB/s, 95% of a plain copy); 64 x up to 4096 keys x 4 heads
// 50 us (4.82 TB/s): 3.7 us until the first loads go out, 2 for the second kernel.  One request of 300 keys x 2 heads of
// 64: 5.7 us.  The 64 requests with pages of 17 tokens, or of one, whose loads bring one row each: 73 us (D = 64: 47
// for 34.5).
#include <type_traits>

#include "attn.cuh"
#include "decode_attn.cuh"
#include "tc.cuh"

namespace l3d {
namespace decode {

using namespace l3d::attn;

constexpr int WARPS = 12;               // of a block (one per SM)
constexpr int MIN_TILES = 1;            // of a warp
constexpr float RESCALE_LOG2 = 8.f;     // the running maximum moves only when it grows past 2^8
// log2 of a row's largest probability: f16 goes down to 2^-24 only, and up to 2^15 there is room.  (At 2^0 the
// weight of 255 keys of 2^-18 each beside one of 1 was off by up to 1%.)
template <typename T>
constexpr float HELD_LOG2 = std::is_same<T, __half>::value ? 7.f : 0.f;
constexpr int ST_TIMEOUT = 5, ST_MISALIGNED = 6;

__device__ int g_decode_status;

// Keys of a tile.
__host__ __device__ constexpr int tile_keys(int D) { return D == 64 ? 32 : 16; }

template <int D>
struct Cfg {
  static constexpr int KT = tile_keys(D), MK = KT / 16;
  static constexpr int DC = D / 64, HALF = KT * 128;       // a tile lies as DC pieces of KT rows x 128 bytes
  static constexpr int TILE = DC * HALF;                   // bytes of K, or of V
  static constexpr int STAGES = 2;
  static constexpr int RING = STAGES * 2 * TILE;           // of one warp
  static constexpr int BARS = 512;                         // barriers of all warps
  static_assert(WARPS * STAGES * 8 + 8 <= BARS, "barrier area");
  static_assert(WARPS * RING + BARS + (MAX_BATCH + 1) * 4 <= 226 * 1024, "shared memory");
};

__device__ __forceinline__ int64_t value_at(const void* p, int is64, int64_t i) {
  return is64 ? static_cast<const int64_t*>(p)[i] : int64_t(static_cast<const int32_t*>(p)[i]);
}
// First packed row of sequence b (the end of b - 1).
__device__ __forceinline__ int packed_start(const Params& p, int b) {
  const int64_t v = value_at(p.lengths, p.len64, b);
  return v < 0 ? 0 : v < p.keys ? int(v) : p.keys;
}
// Keys of sequence b that can be read, and whether its length does not fit its table.
__device__ __forceinline__ int length_of(const Params& p, int b, bool* bad) {
  *bad = false;
  if (p.size == 0) return max(packed_start(p, b + 1) - packed_start(p, b), 0);
  const int64_t v = value_at(p.lengths, p.len64, b), room = int64_t(p.width) * p.size;
  *bad = v > room;
  return v < 0 ? 0 : int(v < room ? v : room);
}

// a / b of values that are seldom past 32 bits (a 64-bit division takes some 150 clocks more).
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  return ((a | b) >> 32) == 0 ? int64_t(uint32_t(a) / uint32_t(b)) : a / b;
}

// The line of tiles: sequence b's begin at starts[b] * heads, heads = Hkv * row tiles.
struct Line {
  int64_t total, per;   // tiles, tiles of a warp
};
__device__ __forceinline__ Line line_of(const Params& p, int tiles) {
  const int64_t total = int64_t(tiles) * p.Hkv * p.tiles;
  const int64_t even = quotient(total + p.total_warps - 1, p.total_warps);
  return {total, even > MIN_TILES ? even : MIN_TILES};
}

// The second part of a probability, at least the type's smallest number where the first is not 0: it meets an infinite
// V too, and 0 times that (or an infinity less another, were the first rounded up) is no number.  Values without a sign
// are ordered as their bits.
__device__ __forceinline__ uint32_t not_zero(uint32_t second, uint32_t first) {
  return __vmaxu2(second, __vminu2(first, 0x00010001u));
}

template <typename T> struct Mma;
template <> struct Mma<__nv_bfloat16> {
  static __device__ __forceinline__ void run(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  // a, b >= 0 cut off to a pair of the type, and what that leaves of them, rounded.
  static __device__ __forceinline__ uint32_t split(float a, float b, uint32_t& rest) {
    const uint32_t x = __float_as_uint(a), y = __float_as_uint(b), hi = __byte_perm(x, y, 0x7632);
    const __nv_bfloat162 l = __floats2bfloat162_rn(a - __uint_as_float(x & 0xffff0000u), b - __uint_as_float(y & 0xffff0000u));
    rest = not_zero(*reinterpret_cast<const uint32_t*>(&l), hi);
    return hi;
  }
};
template <> struct Mma<__half> {
  static __device__ __forceinline__ void run(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t split(float a, float b, uint32_t& rest) {
    uint32_t hi;
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(b), "f"(a));
    const __half2 h = *reinterpret_cast<const __half2*>(&hi);
    const __half2 l = __floats2half2_rn(a - __low2float(h), b - __high2float(h));
    rest = not_zero(*reinterpret_cast<const uint32_t*>(&l), hi);
    return hi;
  }
};
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// An 8 x 8 matrix of 16-bit values across the warp, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
// (Keys and values are the first to leave L2: the parts written meanwhile are read again.)
__device__ __forceinline__ uint64_t first_to_leave() {
  uint64_t policy;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
  return policy;
}
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, uint32_t bar, uint64_t policy, int c0, int c1,
                                        int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4, %5, %6}], [%2], %7;" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "l"(policy)
      : "memory");
}
__device__ __forceinline__ void store16(uint32_t dst, uint32_t v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst), "r"(v) : "memory");
}

// The exponent of infinities and NaN.
template <typename T>
constexpr uint32_t INF_BITS = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
// Whether one of the 8 values at a shared address is not finite.
template <typename T>
__device__ __forceinline__ bool not_finite(uint32_t at) {
  uint32_t r[4];
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
  bool any = false;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    any |= (r[i] & INF_BITS<T>) == INF_BITS<T> || (r[i] >> 16 & INF_BITS<T>) == INF_BITS<T>;
  return any;
}

// A place in the line of tiles: sequence b, head and row tile hr, key tile t of `tiles`.
struct Cursor {
  int b, hr, t, tiles;
  __device__ __forceinline__ void seek(const int* starts, int B, int heads, int64_t x) {
    const int64_t y = quotient(x, heads);
    int lo = 0, hi = B;  // the last b with starts[b] <= y
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (starts[mid] <= y) lo = mid;
      else hi = mid;
    }
    b = lo;
    tiles = starts[b + 1] - starts[b];
    const int64_t rem = x - int64_t(starts[b]) * heads;
    hr = int(quotient(rem, tiles));
    t = int(rem - int64_t(hr) * tiles);
  }
  // To the next tile (not past the line's last one); whether its head or row tile is another one.
  __device__ __forceinline__ bool next(const int* starts, int heads) {
    if (++t < tiles) return false;
    t = 0;
    if (++hr < heads) return true;
    hr = 0;
    do {
      ++b;
      tiles = starts[b + 1] - starts[b];
    } while (tiles == 0);
    return true;
  }
};

// NB: columns of 8 rows in a row tile.
template <typename T, int D, int NB, bool ALONE>
__global__ void __launch_bounds__(WARPS * 32, 1)
    decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Params p) {
  using C = Cfg<D>;
  constexpr int KT = C::KT, MK = C::MK, NT = D / 16;   // 16-key tiles of S^T, 16-wide tiles of O^T
  int* const status = &g_decode_status;
  extern __shared__ __align__(1024) uint8_t smem[];
  const bool aligned = (smem_u32(smem) & 1023u) == 0;  // (else no tile is loaded, but what is joined is still told)
  if (!aligned && threadIdx.x == 0) atomicCAS(status, 0, ST_MISALIGNED);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + WARPS * C::RING);  // [WARPS][STAGES]
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + WARPS * C::STAGES);
  int* starts = reinterpret_cast<int*>(smem + WARPS * C::RING + C::BARS);  // [B + 1]
  __shared__ int s_warp[WARPS];
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.launch_dependents;");

  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
  }
  if (threadIdx.x < WARPS * C::STAGES) mbar_init(&bars[threadIdx.x], 1);
  if (threadIdx.x == 0) *abort_flag = 0;
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");  // for the kernel before: nothing global is touched earlier
  const int heads = p.Hkv * p.tiles;
  const int me = warp * gridDim.x + blockIdx.x;  // a short line spreads over the device first
  int64_t x0 = 0;
  int count = 0;
  // ---- key tiles before each sequence: a sum over the batch, a stretch of it per thread
  if constexpr (!ALONE) {
    const int per = (p.B + WARPS * 32 - 1) / (WARPS * 32), b0 = min(int(threadIdx.x) * per, p.B), b1 = min(b0 + per, p.B);
    int sum = 0;
    for (int b = b0; b < b1; ++b) {
      bool bad;
      const int n = (length_of(p, b, &bad) + KT - 1) / KT;
      starts[b] = n;
      sum += n;
    }
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    if (lane == 31) s_warp[warp] = incl;
    __syncthreads();
    int at = incl - sum;
    for (int w = 0; w < warp; ++w) at += s_warp[w];
    for (int b = b0; b < b1; ++b) {
      const int n = starts[b];
      starts[b] = at;
      at += n;
    }
    if (threadIdx.x == WARPS * 32 - 1) starts[p.B] = at;  // (its stretch is the last, or empty)
    __syncthreads();
    if (p.edges) {  // rows without keys, which no warp comes to
      for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
        if (starts[b + 1] != starts[b]) continue;
        bool bad;
        length_of(p, b, &bad);
        const int Hq = p.Hkv * p.G;
        for (int64_t x = threadIdx.x; x < int64_t(p.N) * Hq * D; x += WARPS * 32) {
          const int row = int(x / D), i = row / Hq;
          reinterpret_cast<T*>(p.out)[b * p.ob + i * p.on + (row - i * Hq) * p.oh + x % D] =
              from_f<T>(bad ? __int_as_float(0x7fffffff) : 0.f);
        }
      }
    } else if (blockIdx.x == 0) {
      for (int b = threadIdx.x; b <= p.B; b += WARPS * 32) p.starts[b] = starts[b];
    }
  }
  int64_t per = 0;  // tiles of a warp
  if constexpr (!ALONE) {
    const Line line = line_of(p, starts[p.B]);
    per = line.per;
    x0 = int64_t(me) * per;
    // (Nothing to join, until the stretch is done: also where a wait runs out, for the joining kernel follows either way.)
    if (p.edges && lane == 0) p.edges[me] = make_int4(0, 0, 0, 0);
    if (x0 >= line.total || !aligned) return;
    count = int(min(per, line.total - x0));
  } else {
    __syncthreads();  // (the barriers are there)
  }
  // Where this warp begins.
  auto seek = [&](Cursor& c) {
    if constexpr (ALONE) {
      c.b = blockIdx.x / heads;
      c.hr = blockIdx.x - c.b * heads;
      bool bad;
      c.tiles = (length_of(p, c.b, &bad) + KT - 1) / KT;
      const int per = (c.tiles + WARPS - 1) / WARPS;
      c.t = warp * per;
      count = aligned ? max(min(c.tiles - c.t, per), 0) : 0;
    } else {
      c.seek(starts, p.B, heads, x0);
    }
  };

  // ---- loads, STAGES tiles ahead of the work: lane i takes box i of a tile.  A tile's table entries are looked
  // up one tile early, so that their latency is not waited for.
  const uint32_t ring = smem_u32(smem) + warp * C::RING;
  uint64_t* full = bars + warp * C::STAGES;
  Cursor ld;
  seek(ld);
  int ld_page = 0, ld_slot = 0, ld_h = 0, ld_len = 0, ld_first = 0;
  bool ld_ok = false, ld_new = true;
  auto look_up = [&] {
    if (ld_new) {
      bool bad;
      ld_len = length_of(p, ld.b, &bad);
      ld_first = p.size ? 0 : packed_start(p, ld.b);
      ld_h = ld.hr / p.tiles;
    }
    const int j = ld.t * KT + lane * p.box;
    ld_ok = lane * p.box < KT && j < ld_len;
    ld_page = 0;
    ld_slot = ld_first + j;
    if (p.size) {
      const int page = p.size == 1 ? j : int(__umulhi(uint32_t(j), p.mul) >> p.shift);
      ld_slot = j - page * p.size;
      if (ld_ok) ld_page = p.table[ld.b * p.table_stride + page];
    }
  };
  if (count > 0) look_up();
  int issued = 0, ld_stage = 0;
  const uint64_t policy = first_to_leave();
  auto issue = [&] {
    if (issued >= count) return;
    // (Only now is the table's entry needed.)
    const bool in = ld_ok && (p.size == 0 || (ld_page >= 0 && ld_page < p.keys));
    const uint32_t kd = ring + ld_stage * (2 * C::TILE), vd = kd + C::TILE;
    const int boxes = __popc(__ballot_sync(0xffffffffu, in));
    if (lane == 0) mbar_expect_tx(&full[ld_stage], boxes * p.box_bytes);
    __syncwarp();
    if (in) {
      const uint32_t at = lane * p.box * 128, bar = smem_u32(&full[ld_stage]);
#pragma unroll
      for (int dc = 0; dc < C::DC; ++dc) {
        tma_box(kd + dc * C::HALF + at, &map_k, bar, policy, dc * 64, p.kw.hn ? ld_h * p.kw.hm : ld_slot,
                p.kw.hn ? ld_slot : ld_h * p.kw.hm, ld_page);
        tma_box(vd + dc * C::HALF + at, &map_v, bar, policy, dc * 64, p.vw.hn ? ld_h * p.vw.hm : ld_slot,
                p.vw.hn ? ld_slot : ld_h * p.vw.hm, ld_page);
      }
    } else if (ld_ok) {  // a page that is none of the cache: K of NaN
      for (int r = lane * p.box; r < (lane + 1) * p.box; ++r)
        for (int c = 0; c < 8 * C::DC; ++c) store16(kd + (c >> 3) * C::HALF + r * 128 + (c & 7) * 16, 0xffffffffu);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (++ld_stage == C::STAGES) ld_stage = 0;
    if (++issued < count) {
      ld_new = ld.next(starts, heads);
      look_up();
    }
  };
  for (int s = 0; s < C::STAGES; ++s) issue();

  // ---- work
  Cursor cu;
  seek(cu);
  // This thread's keys (or head dims) g and g + 8 of 16, its rows q2 and q2 + 1 of 8; Q is loaded for row g.
  const int g8 = lane >> 2, q2 = (lane & 3) * 2;
  const int R = p.N * p.G;
  // Addresses of this lane's rows for ldmatrix, within a piece: 16-byte chunk c of row r at (c ^ r % 8) * 16.
  const int r8 = lane & 7, mi = lane >> 3;
  const uint32_t k_row = (r8 + (mi & 1) * 8) * 128, v_row = C::TILE + (r8 + (mi >> 1) * 8) * 128;
  uint32_t k_at[4], v_at[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    k_at[i] = k_row + (((2 * i + (mi >> 1)) ^ r8) << 4);
    v_at[i] = v_row + (((2 * i + (mi & 1)) ^ r8) << 4);
  }
  // ALONE: this warp's part, over its ring.
  float* const alone_o = reinterpret_cast<float*>(smem + warp * C::RING);
  float* const alone_l = alone_o + 8 * NB * D;
  if (ALONE && count == 0 && lane < 8 * NB) alone_l[lane] = -INFINITY;
  uint32_t qf[D / 16][NB][2];
  float o[NT][NB][4];
  float m[NB][2], l[NB][2];
  int lim[NB][2], len = 0, t_first = 0, least = 0, stage = 0, turn = 0;
  bool fresh = true, ok = true;
#pragma unroll 1
  for (int n = 0; n < count; ++n) {
    if (fresh) {  // the first tile of a part
      fresh = false;
      t_first = cu.t;
      bool bad;
      len = length_of(p, cu.b, &bad);
      least = p.causal ? len - p.N + 1 : len;
      const int h = cu.hr / p.tiles, f0 = (cu.hr - h * p.tiles) * (8 * NB);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int f = f0 + nb * 8 + q2 + e;
          lim[nb][e] = f >= R ? 0 : p.causal ? len - p.N + 1 + f / p.G : len;
          m[nb][e] = -INFINITY;
          l[nb][e] = bad ? __int_as_float(0x7fffffff) : 0.f;
        }
        const int f = f0 + nb * 8 + g8, i = f / p.G, g = f - i * p.G;
        const T* qr = reinterpret_cast<const T*>(p.q) + cu.b * p.qb + i * p.qn + (h * p.G + g) * p.qh + q2;
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
          for (int x = 0; x < 2; ++x)
            qf[k][nb][x] = f < R ? *reinterpret_cast<const uint32_t*>(qr + k * 16 + x * 8) : 0u;
#pragma unroll
        for (int i2 = 0; i2 < NT; ++i2)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i2][nb][e] = 0.f;
      }
    }
    ok = __all_sync(0xffffffffu, mbar_wait(&full[stage], turn & 1, abort_flag, status, ST_TIMEOUT, p.wait_ns));
    if (!ok) break;
    __syncwarp();
    const uint32_t tile = ring + stage * (2 * C::TILE);
    // S^T = K Q^T; even and odd steps of 16 head dims summed apart (two chains of products)
    float sc[MK][NB][4], sd[MK][NB][4];
#pragma unroll
    for (int i = 0; i < MK * NB * 4; ++i) (&sc[0][0][0])[i] = (&sd[0][0][0])[i] = 0.f;
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
#pragma unroll
      for (int mk = 0; mk < MK; ++mk) {
        uint32_t a[4];
        ldsm4(a, tile + (k >> 2) * C::HALF + mk * (16 * 128) + k_at[k & 3]);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) Mma<T>::run(k & 1 ? sd[mk][nb] : sc[mk][nb], a, qf[k][nb][0], qf[k][nb][1]);
      }
#pragma unroll
    for (int i = 0; i < MK * NB * 4; ++i) (&sc[0][0][0])[i] += (&sd[0][0][0])[i];
    const int key0 = cu.t * KT;
    bool mixed = false;
    if (key0 + KT > least) {  // some row does not see some key
#pragma unroll
      for (int mk = 0; mk < MK; ++mk)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (key0 + mk * 16 + g8 + (e >> 1) * 8 >= lim[nb][e & 1]) sc[mk][nb][e] = -INFINITY;
      // V rows past the keys may hold anything: zero them, for 0 x NaN is not 0.
      bool wild = false;  // a V that is not finite, of a key that only the later rows see
      for (int c = lane; c < C::TILE / 16; c += 32) {
        const int r = (c >> 3) % KT;
        const uint32_t at = tile + C::TILE + c * 16;
        if (key0 + r >= len) store16(at, 0u);
        else if (key0 + r >= least) wild |= not_finite<T>(at);
      }
      mixed = __any_sync(0xffffffffu, wild);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
    }
    // The running maximum (less HELD_LOG2) and sum of this thread's two rows (the maximum over all its warp's keys,
    // the sum over its own ones).
    bool grown = false;
    float al[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mx = max_nan(sc[0][nb][e], sc[0][nb][e + 2]);
#pragma unroll
        for (int mk = 1; mk < MK; ++mk) mx = max_nan(mx, sc[mk][nb][e], sc[mk][nb][e + 2]);
        mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 16)) * p.scale_log2;
        const bool grow = !(mx <= m[nb][e] + (RESCALE_LOG2 + HELD_LOG2<T>));
        mx -= HELD_LOG2<T>;
        al[nb][e] = grow ? ex2f(m[nb][e] - mx) : 1.f;  // 0 on the first key a row sees
        if (grow) m[nb][e] = mx;
        grown |= grow;
      }
    if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int e = 0; e < 2; ++e) l[nb][e] *= al[nb][e];
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][nb][e] *= al[nb][e & 1];
      }
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float nm = m[nb][e] == -INFINITY ? 0.f : minus_max(m[nb][e]);
#pragma unroll
        for (int mk = 0; mk < MK; ++mk)
#pragma unroll
          for (int x = 0; x < 4; x += 2) {
            sc[mk][nb][e + x] = ex2f(fmaf(sc[mk][nb][e + x], p.scale_log2, nm));
            l[nb][e] += sc[mk][nb][e + x];
          }
      }
    if (mixed) {
      // What a row does not see, it does not meet times zero either: such elements go to the rows that see them
      // one by one, and out of the tile.
#pragma unroll
      for (int mk = 0; mk < MK; ++mk)
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll 1
          for (int x = 0; x < 8; ++x) {
            const int key = mk * 16 + half * 8 + x, src = x * 4 + (lane & 3);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float pv = __shfl_sync(0xffffffffu, sc[mk][nb][half * 2 + e], src);
                if (key0 + key < lim[nb][e]) {
#pragma unroll
                  for (int i = 0; i < 2 * NT; ++i) {
                    const uint32_t at = tile + C::TILE + (i >> 3) * C::HALF + key * 128 + (((i & 7) ^ (key & 7)) << 4) + g8 * 2;
                    uint16_t bits;
                    asm volatile("ld.shared.b16 %0, [%1];" : "=h"(bits) : "r"(at) : "memory");
                    if ((bits & INF_BITS<T>) == INF_BITS<T>) {
                      float& acc = o[i >> 1][nb][(i & 1) * 2 + e];
                      acc = fmaf(pv, to_f(*reinterpret_cast<const T*>(&bits)), acc);
                    }
                  }
                }
              }
          }
      __syncwarp();
      for (int c = lane; c < C::TILE / 4; c += 32) {
        if (key0 + (c >> 5) % KT < least) continue;
        const uint32_t at = tile + C::TILE + c * 4;
        uint32_t raw;
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(raw) : "r"(at) : "memory");
        if ((raw & INF_BITS<T>) == INF_BITS<T>) raw &= 0xffff0000u;
        if ((raw >> 16 & INF_BITS<T>) == INF_BITS<T>) raw &= 0xffffu;
        asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(raw) : "memory");
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
    }
    // O^T += V^T P^T
#pragma unroll
    for (int mk = 0; mk < MK; ++mk) {
      uint32_t hi[NB][2], lo[NB][2];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          uint32_t rest;
          hi[nb][x] = transposed(Mma<T>::split(sc[mk][nb][2 * x], sc[mk][nb][2 * x + 1], rest));
          lo[nb][x] = transposed(rest);
        }
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        uint32_t a[4];
        ldsm4t(a, tile + (i >> 2) * C::HALF + mk * (16 * 128) + v_at[i & 3]);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          Mma<T>::run(o[i][nb], a, hi[nb][0], hi[nb][1]);
          Mma<T>::run(o[i][nb], a, lo[nb][0], lo[nb][1]);
        }
      }
    }
    __syncwarp();
    issue();
    if (++stage == C::STAGES) {
      stage = 0;
      ++turn;
    }
    if (cu.t + 1 == cu.tiles || n + 1 == count) {
      // The end of a part: the output, or O / l and the log2 sum.
      fresh = true;
      const bool whole = t_first == 0 && cu.t + 1 == cu.tiles;
      if constexpr (ALONE) __syncwarp();  // (the tiles are read: the part goes over them)
      const int h = cu.hr / p.tiles, f0 = (cu.hr - h * p.tiles) * (8 * NB);
      const int64_t part = (2 * int64_t(me) + (t_first == 0 ? 1 : 0)) * p.rows;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float inv[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float sum = l[nb][e];
          sum += __shfl_xor_sync(0xffffffffu, sum, 4);
          sum += __shfl_xor_sync(0xffffffffu, sum, 8);
          sum += __shfl_xor_sync(0xffffffffu, sum, 16);
          inv[e] = sum > 0.f ? 1.f / sum : sum == sum ? 0.f : sum;
          const int r = nb * 8 + q2 + e;
          if (ALONE ? g8 == 0 : !whole && g8 == 0 && f0 + r < R)
            (ALONE ? alone_l + r : p.part_l + part + r)[0] = sum > 0.f ? m[nb][e] + log2f(sum) : sum == sum ? -INFINITY : sum;
        }
        if constexpr (ALONE) {
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int c = 0; c < 2 * NT; ++c)
              alone_o[(nb * 8 + q2 + e) * D + c * 8 + g8] = o[c >> 1][nb][(c & 1) * 2 + e] * inv[e];
        } else if (whole) {
          const int f = f0 + nb * 8 + g8, i = f / p.G, g = f - i * p.G;
          T* orow = reinterpret_cast<T*>(p.out) + cu.b * p.ob + i * p.on + (h * p.G + g) * p.oh + q2;
#pragma unroll
          for (int c = 0; c < 2 * NT; ++c) {
            const float* v = &o[c >> 1][nb][(c & 1) * 2];
            const uint32_t pair = transposed(pack_pair<T>(v[0] * inv[0], v[1] * inv[1]));
            if (f < R) *reinterpret_cast<uint32_t*>(orow + c * 8) = pair;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = nb * 8 + q2 + e;
            if (f0 + r >= R) continue;
            float* orow = p.part_o + (part + r) * D + g8;
#pragma unroll
            for (int c = 0; c < 2 * NT; ++c) orow[c * 8] = o[c >> 1][nb][(c & 1) * 2 + e] * inv[e];
          }
        }
      }
    }
    if (n + 1 < count) cu.next(starts, heads);
    else if (!ALONE && p.edges && lane == 0) {  // the item that begins in this stretch and goes on behind it, if any
      const int rest = cu.tiles - (cu.t + 1);
      p.edges[me] = make_int4(cu.b, cu.hr, t_first == 0 && rest > 0 ? 1 + int((rest + per - 1) / per) : 0, 0);
    }
  }
  if (!ok && lane == 0) {  // the newest load of each stage: no copy may be in flight when the block exits
    for (int i = max(issued - C::STAGES, 0); i < issued; ++i)
      mbar_drain(&full[i % C::STAGES], uint32_t(i / C::STAGES) & 1u, p.wait_ns);
  }
  if constexpr (ALONE) {
    // The warps' parts of each row weighed by 2^(their log2 sum - the largest), in the warps' order.
    __syncthreads();
    if (*abort_flag) return;
    constexpr int E = D / 32;
    bool bad;
    length_of(p, cu.b, &bad);
    const int h = cu.hr / p.tiles, f0 = (cu.hr - h * p.tiles) * (8 * NB);
    for (int r = warp; r < 8 * NB && f0 + r < R; r += WARPS) {
      auto part_l = [&](int w) { return reinterpret_cast<const float*>(smem + w * C::RING)[8 * NB * D + r]; };
      float wgt = lane < WARPS ? part_l(lane) : -INFINITY, mx = wgt;
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, x));
      wgt = wgt == -INFINITY ? 0.f : exp2f(wgt - mx);
      float sum = wgt;
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      float acc[E] = {};
      for (int w = 0; w < WARPS; ++w) {
        const float ww = __shfl_sync(0xffffffffu, wgt, w);
        if (ww == 0.f) continue;  // a part without keys: nothing is stored there
        const float* src = reinterpret_cast<const float*>(smem + w * C::RING) + r * D + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(ww, src[e], acc[e]);
      }
      const float inv = bad ? __int_as_float(0x7fffffff) : sum != 0.f ? 1.f / sum : 0.f;
      const int i = (f0 + r) / p.G;
      T* orow = reinterpret_cast<T*>(p.out) + cu.b * p.ob + i * p.on + (h * p.G + f0 + r - i * p.G) * p.oh + lane * E;
      alignas(8) T v[E];
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = from_f<T>(acc[e] * inv);
      if constexpr (E == 4) *reinterpret_cast<uint2*>(orow) = *reinterpret_cast<const uint2*>(v);
      else *reinterpret_cast<uint32_t*>(orow) = *reinterpret_cast<const uint32_t*>(v);
    }
  }
}

// A running sum of parts, each weighed by 2^(its log2 sum - the largest): D / 32 elements per lane.
template <int D>
struct Joined {
  static constexpr int E = D / 32;
  using Vec = typename std::conditional<E == 4, float4, float2>::type;
  float m = -INFINITY, l = 0.f;
  alignas(16) float acc[E] = {};
  // Parts k0, k0 + step, .. up to `parts`, U of them at a time.  The first part lies in its warp's second place: it
  // holds the row's first key.
  template <int U>
  __device__ __forceinline__ void add(const Params& p, int w0, int parts, int r, int k0, int step) {
    const int lane = threadIdx.x & 31;
    auto row_at = [&](int k) { return (2 * int64_t(w0 + k) + (k == 0 ? 1 : 0)) * p.rows + r; };
    for (; k0 < parts; k0 += step * U) {
      float pl[U];
      Vec v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = k0 + u * step;
        pl[u] = k < parts ? p.part_l[row_at(k)] : -INFINITY;
        v[u] = reinterpret_cast<const Vec*>(p.part_o + row_at(k < parts ? k : k0) * D)[lane];
      }
      float mx = m;
#pragma unroll
      for (int u = 0; u < U; ++u) mx = max_nan(mx, pl[u]);
      if (mx == -INFINITY) continue;
      const float a = exp2f(m - mx);
      l *= a;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] *= a;
      m = mx;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (pl[u] == -INFINITY) continue;
        const float wgt = exp2f(pl[u] - m);
        l += wgt;
        const float* vv = reinterpret_cast<const float*>(&v[u]);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(wgt, vv[e], acc[e]);
      }
    }
  }
  template <typename T>
  __device__ __forceinline__ void store(T* orow) const {
    const float inv = l > 0.f ? 1.f / l : l == l ? 0.f : l;
    alignas(8) T o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = from_f<T>(acc[e] * inv);
    orow += (threadIdx.x & 31) * E;
    if constexpr (E == 4) *reinterpret_cast<uint2*>(orow) = *reinterpret_cast<const uint2*>(o);
    else *reinterpret_cast<uint32_t*>(orow) = *reinterpret_cast<const uint32_t*>(o);
  }
};

// The parts of each row joined, in a fixed order: W warps for a row, with every W-th part each; a block of 4 rows
// where one warp does.  Rows without keys are zeroed here, and no others touched that one warp has finished.
template <typename T, int D, int W>
__global__ void __launch_bounds__(W == 1 ? 128 : W * 32) combine_kernel(const Params p) {
  constexpr int E = D / 32;
  using Vec = typename Joined<D>::Vec;
  __shared__ alignas(16) float red[W][D];
  __shared__ float red_m[W], red_l[W];
  const int lane = threadIdx.x & 31, warp = W == 1 ? 0 : threadIdx.x >> 5;
  const int R = p.N * p.G;
  const uint32_t row = W == 1 ? blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;  // at most 2^30 of them
  if (W == 1 && row >= uint32_t(p.B) * p.Hkv * R) return;
  const int head = int(row / uint32_t(R)), f = int(row) - head * R, b = head / p.Hkv, h = head - b * p.Hkv;
  const int i = f / p.G, rt = f / p.height, hr = h * p.tiles + rt, heads = p.Hkv * p.tiles;
  T* orow = reinterpret_cast<T*>(p.out) + b * p.ob + i * p.on + (h * p.G + f - i * p.G) * p.oh;
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int before = p.starts[b], tiles = p.starts[b + 1] - before;
  if (tiles == 0) {
    bool bad;
    length_of(p, b, &bad);
    if (warp == 0) {
#pragma unroll
      for (int e = 0; e < E; ++e) orow[lane * E + e] = from_f<T>(bad ? __int_as_float(0x7fffffff) : 0.f);
    }
    return;
  }
  const Line line = line_of(p, p.starts[p.B]);
  const int64_t first = int64_t(before) * heads + int64_t(hr) * tiles, last = first + tiles - 1;
  const int w0 = int(quotient(first, line.per)), parts = int(quotient(last, line.per)) - w0 + 1;
  if (parts == 1) return;
  Joined<D> sum;
  sum.template add<W == 1 || W == 32 ? 8 : 4>(p, w0, parts, f - rt * p.height, warp, W);
  if constexpr (W == 1) {
    sum.store(orow);
    return;
  }
  *reinterpret_cast<Vec*>(&red[warp][lane * E]) = *reinterpret_cast<const Vec*>(sum.acc);
  if (lane == 0) {
    red_m[warp] = sum.m;
    red_l[warp] = sum.l;
  }
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += W * 32) {
    float mx = -INFINITY, all = 0.f, val = 0.f;
    for (int w = 0; w < W; ++w) mx = max_nan(mx, red_m[w]);
    if (mx != -INFINITY)
      for (int w = 0; w < W; ++w) {
        if (red_m[w] == -INFINITY) continue;
        const float wgt = exp2f(red_m[w] - mx);
        all = fmaf(wgt, red_l[w], all);
        val = fmaf(wgt, red[w][d], val);
      }
    orow[d] = from_f<T>(all > 0.f ? val / all : all == all ? 0.f : all);
  }
}

// The same where there are more heads and row tiles than warps: few of them are divided at all, at most one per
// end of a warp's stretch, and those are listed there.  A block per end, a row per warp.  (Looking at every row took
// 90 of 119 us for 237 requests x 16 heads x 64 rows of 3 keys.)
template <typename T, int D>
__global__ void __launch_bounds__(128) combine_edges_kernel(const Params p) {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 edge = p.edges[blockIdx.x];  // request, head and row tile, parts
  if (edge.z == 0) return;
  const int h = edge.y / p.tiles, f0 = (edge.y - h * p.tiles) * p.height;
  for (int r = threadIdx.x >> 5; r < p.rows && f0 + r < p.N * p.G; r += 4) {
    const int i = (f0 + r) / p.G;
    Joined<D> sum;
    sum.template add<8>(p, blockIdx.x, edge.z, r, 0, 1);
    sum.store(reinterpret_cast<T*>(p.out) + edge.x * p.ob + i * p.on + (h * p.G + f0 + r - i * p.G) * p.oh);
  }
}

// Rows of a row tile: 8 hold all of a key head's, or 16.
static int height_for(int64_t R) { return R <= 8 ? 8 : 16; }

static int blocks_for(int64_t B, int64_t N, int64_t G, int64_t Hkv, int64_t longest, int64_t D) {
  // (Warps past the line's end only cost their start.)
  const int64_t h = height_for(N * G), most = B * Hkv * ((N * G + h - 1) / h) * ((longest + tile_keys(int(D)) - 1) / tile_keys(int(D)));
  const int64_t want = (most + MIN_TILES - 1) / MIN_TILES;
  return int(want < 1 ? 1 : want < sm_count() ? want : sm_count());
}

// A block for each head and row tile: as many as run at once, with few tiles for each warp, more the nearer the
// blocks come to filling the device.  t tiles a warp, D = 128, us: 8 blocks, t = 2 7.7 alone, 9.8 divided over the device;
// 8, 4 9.8, 10.0; 32, 4 10.1, 10.6; 32, 6 12.1, 11.9; 64, 4 9.9, 11.6; 64, 6 12.1, 13.7; 128, 8 15.0, 20.5; 128, 16 24.2,
// 30.9; but 16, 16 22.4, 14.0, and alone the longest cache decides, so that t stays small.
static bool alone(int64_t B, int64_t N, int64_t G, int64_t Hkv, int64_t longest, int64_t D) {
  const int64_t h = height_for(N * G);
  const int64_t blocks = B * Hkv * ((N * G + h - 1) / h), stretch = WARPS * tile_keys(int(D));
  return blocks <= sm_count() && longest <= (4 + blocks / 24) * stretch;
}

size_t workspace_size(int64_t B, int64_t N, int64_t G, int64_t Hkv, int64_t longest, int64_t D) {
  if (B <= 0 || N <= 0 || G <= 0 || Hkv <= 0 || longest < 0 || D <= 0 || alone(B, N, G, Hkv, longest, D)) return 0;
  const int64_t h = height_for(N * G), rows = N * G < h ? N * G : h;
  const int64_t parts = 2 * int64_t(blocks_for(B, N, G, Hkv, longest, D)) * WARPS;
  return (size_t(B + 1) * 4 + 255) / 256 * 256 + size_t(parts) * 8 + (size_t(parts * rows) * 4 + 255) / 256 * 256 + size_t(parts * rows * D) * 4;
}

template <typename T, int D>
static cudaError_t launch_t(const CUtensorMap (&maps)[2], const Params& p, int blocks, int64_t longest, cudaStream_t s) {
  const bool one = p.total_warps == 0;
  auto k = p.height == 8 ? (one ? decode_kernel<T, D, 1, true> : decode_kernel<T, D, 1, false>)
                         : (one ? decode_kernel<T, D, 2, true> : decode_kernel<T, D, 2, false>);
  constexpr int fixed = WARPS * Cfg<D>::RING + Cfg<D>::BARS;
  cudaError_t e = set_smem_limit(reinterpret_cast<const void*>(k), fixed + (MAX_BATCH + 1) * 4);
  if (e != cudaSuccess) return e;
  // Both may be scheduled while the kernel before them runs, and wait for it.
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  cfg.stream = s;
  cfg.gridDim = dim3(unsigned(blocks));
  cfg.blockDim = dim3(WARPS * 32);
  cfg.dynamicSmemBytes = fixed + (one ? 0 : (p.B + 1) * 4);
  e = cudaLaunchKernelEx(&cfg, k, maps[0], maps[1], p);
  if (e != cudaSuccess || one) return e;
  if (p.edges) {
    cfg.gridDim = dim3(unsigned(p.total_warps));
    cfg.blockDim = dim3(128);
    cfg.dynamicSmemBytes = 0;
    return cudaLaunchKernelEx(&cfg, combine_edges_kernel<T, D>, p);
  }
  // Warps for a row by the parts that it has where the caches are full: one takes eight in a round, sixteen 64,
  // thirty-two 256.  (64 requests, 7 parts: 53.8 us with one, 54.6 with eight; 12 requests x 12 heads, 13 parts, up to 29:
  // 576 rows 47.2 with one, 41.3 with eight, 144 rows 37.5 with eight, 34.9 with sixteen; one request x 8 heads, 125
  // parts: 12.8 with sixteen, 13.3 with thirty-two; 2 x 2 heads, 417 parts: 22.8 and 18.1.)
  const int64_t rows = int64_t(p.B) * p.Hkv * p.N * p.G, items = int64_t(p.B) * p.Hkv * p.tiles;
  const int64_t tiles = (longest + tile_keys(D) - 1) / tile_keys(D), per = (items * tiles + p.total_warps - 1) / p.total_warps;
  const int64_t parts = tiles / (per > MIN_TILES ? per : MIN_TILES);
  const int warps = parts <= 8 ? 1 : rows > 2 * sm_count() ? 8 : parts <= 160 ? 16 : 32;
  cfg.gridDim = dim3(unsigned(warps > 1 ? rows : (rows + 3) / 4));
  cfg.blockDim = dim3(warps > 1 ? warps * 32 : 128);
  cfg.dynamicSmemBytes = 0;
  auto join = warps == 1 ? combine_kernel<T, D, 1> : warps == 8 ? combine_kernel<T, D, 8>
              : warps == 16 ? combine_kernel<T, D, 16> : combine_kernel<T, D, 32>;
  return cudaLaunchKernelEx(&cfg, join, p);
}

int launch(const char* op, Params p, const Keys& kv, bool f16, int64_t longest, void* workspace, cudaStream_t s,
           uint64_t timeout_ns) {
  const int R = p.N * p.G;
  const bool one = alone(p.B, p.N, p.G, p.Hkv, longest, kv.D);
  p.height = height_for(R);
  p.tiles = (R + p.height - 1) / p.height;
  p.rows = R < p.height ? R : p.height;
  const int blocks = one ? p.B * p.Hkv * p.tiles : blocks_for(p.B, p.N, p.G, p.Hkv, longest, kv.D);
  p.total_warps = one ? 0 : blocks * WARPS;
  p.wait_ns = timeout_ns ? timeout_ns : tc::WAIT_LIMIT_NS;
  char* w = static_cast<char*>(workspace);
  p.starts = reinterpret_cast<int*>(w);
  w += (size_t(p.B + 1) * 4 + 255) / 256 * 256;
  p.edges = int64_t(p.B) * p.Hkv * p.tiles > p.total_warps ? reinterpret_cast<int4*>(w) : nullptr;
  w += size_t(p.total_warps) * 16;
  p.part_l = reinterpret_cast<float*>(w);
  w += (size_t(2) * p.total_warps * p.rows * 4 + 255) / 256 * 256;
  p.part_o = reinterpret_cast<float*>(w);
  p.box = tile_keys(int(kv.D));
  if (p.size) {
    while (p.size % p.box) p.box /= 2;
    // shift = floor(log2(size - 1)): mul exceeds 2^(32 + shift) / size by at most 1, so that the product is
    // over by less than j / 2^(32 + shift) < 1 / size for j < 2^30.
    while (p.size > 1 && (int64_t(2) << p.shift) <= p.size - 1) ++p.shift;
    if (p.size > 1) p.mul = uint32_t((uint64_t(1) << (32 + p.shift)) / uint64_t(p.size) + 1);
  }
  p.box_bytes = p.box * 2 * int(kv.D) * 2 + (timeout_ns ? 16 : 0);
  CUtensorMap maps[2] = {};
  if (p.keys > 0) {  // (without keys nothing is loaded)
    const int64_t pages = p.size ? p.keys : 1, slots = p.size ? p.size : p.keys;
    const void* base[] = {kv.k, kv.v};
    const int64_t* st[] = {kv.ks, kv.vs};
    View* view[] = {&p.kw, &p.vw};
    for (int i = 0; i < 2; ++i) {
      view[i]->hm = p.Hkv > 1 && st[i][2] == 0 ? 0 : 1;
      if (!make_map4(&maps[i], base[i], pages, view[i]->hm ? p.Hkv : 1, slots, kv.D, st[i][1], st[i][2], st[i][0],
                     uint32_t(p.box), &view[i]->hn))
        return fail(L3D_E_CUDA, "%s: cuTensorMapEncodeTiled failed", op);
    }
  }
  const cudaError_t e = f16 ? (kv.D == 64 ? launch_t<__half, 64>(maps, p, blocks, longest, s) : launch_t<__half, 128>(maps, p, blocks, longest, s))
                            : (kv.D == 64 ? launch_t<__nv_bfloat16, 64>(maps, p, blocks, longest, s)
                                          : launch_t<__nv_bfloat16, 128>(maps, p, blocks, longest, s));
  return e == cudaSuccess ? L3D_OK : fail(L3D_E_CUDA, "%s: %s", op, cudaGetErrorString(e));
}

cudaError_t status_read(int* status, int reset) {
  cudaError_t e = cudaMemcpyFromSymbol(status, g_decode_status, sizeof(int));
  if (e == cudaSuccess && reset) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_decode_status, &zero, sizeof(int));
  }
  return e;
}

}  // namespace decode
}  // namespace l3d

using namespace l3d;

extern "C" size_t l3d_paged_attention_workspace_size(int64_t b, int64_t hq, int64_t hkv, int64_t n, int64_t capacity,
                                                     int64_t d) {
  if (hkv <= 0 || hq <= 0 || hq % hkv) return 0;
  return l3d::decode::workspace_size(b, n, hq / hkv, hkv, capacity, d);
}

static int run_paged_attention(const l3d_tensor* q, const l3d_tensor* k_pages, const l3d_tensor* v_pages,
                               const l3d_tensor* table, const l3d_tensor* lengths, float scale, const l3d_tensor* out,
                               void* workspace, size_t workspace_bytes, l3d_stream stream, uint64_t timeout_ns,
                               const char* op) {
  if (!q || !k_pages || !v_pages || !table || !lengths || !out)
    return fail(L3D_E_NULL, "%s: q, k_pages, v_pages, table, lengths and out are required", op);
  const l3d_tensor* all[] = {q, out, k_pages, v_pages};
  for (const l3d_tensor* t : all) {
    if (t->dtype != q->dtype || (t->dtype != L3D_BF16 && t->dtype != L3D_F16))
      return fail(L3D_E_DTYPE, "%s: q, the pages and out all BF16 or all F16", op);
    if (t->ndim != 4) return fail(L3D_E_SHAPE, "%s: q and out [B, N, H, D], pages [pages, size, Hkv, D]", op);
    if (numel(t) > 0 && t->strides[3] != 1) return fail(L3D_E_ALIGN, "%s: the head dim must be contiguous", op);
  }
  const int64_t B = q->dims[0], N = q->dims[1], Hq = q->dims[2], D = q->dims[3];
  const int64_t pages = k_pages->dims[0], size = k_pages->dims[1], Hkv = k_pages->dims[2];
  if (D != 64 && D != 128) return fail(L3D_E_UNSUPPORTED, "%s: head dim must be 64 or 128", op);
  for (int i = 0; i < 4; ++i) {
    if (out->dims[i] != q->dims[i]) return fail(L3D_E_SHAPE, "%s: out must have q's shape", op);
    if (v_pages->dims[i] != k_pages->dims[i] || (i == 3 && k_pages->dims[i] != D))
      return fail(L3D_E_SHAPE, "%s: k_pages and v_pages [pages, size, Hkv, D]", op);
  }
  if (Hq > 0 && (Hkv <= 0 || Hq % Hkv))
    return fail(L3D_E_SHAPE, "%s: query heads must be a multiple of the key heads", op);
  if (table->dtype != L3D_I32) return fail(L3D_E_DTYPE, "%s: table must be I32", op);
  if (table->ndim != 2 || table->dims[0] != B || (table->dims[1] > 1 && table->strides[1] != 1))
    return fail(L3D_E_SHAPE, "%s: table must be [B, pages of a request] with contiguous rows", op);
  if (lengths->dtype != L3D_I32 && lengths->dtype != L3D_I64)
    return fail(L3D_E_DTYPE, "%s: lengths must be I32 or I64", op);
  if (lengths->ndim != 1 || lengths->dims[0] != B || (B > 1 && lengths->strides[0] != 1))
    return fail(L3D_E_SHAPE, "%s: lengths must be contiguous [B]", op);
  const float scale_log2 = scale * 1.4426950408889634f;  // finite too
  if (!(scale > 0.f) || !(scale_log2 < INFINITY))
    return fail(L3D_E_UNSUPPORTED, "%s: scale must be positive and finite", op);
  const int64_t big = int64_t(1) << 30, width = table->dims[1];
  if (size <= 0 || pages > big || size > big || width > big || width * size > big || B > l3d::decode::MAX_BATCH ||
      N > 65535 || Hq > 65535 || B * N * Hq > big || B * (width * size / 16 + 1) > big)
    return fail(L3D_E_UNSUPPORTED, "%s: dimensions too large (at most %d requests), or pages of no tokens", op,
                l3d::decode::MAX_BATCH);
  if (B * N * Hq == 0) return L3D_OK;
  const size_t need = l3d::decode::workspace_size(B, N, Hq / Hkv, Hkv, width * size, D);
  if (need && (!workspace || workspace_bytes < need))
    return fail(L3D_E_WORKSPACE, "%s: workspace of %zu bytes required", op, need);
  if (reinterpret_cast<uintptr_t>(workspace) % 256)
    return fail(L3D_E_ALIGN, "%s: workspace must be 256-byte aligned", op);
  for (const l3d_tensor* t : all) {
    if (no_data(t)) return fail(L3D_E_NULL, "%s: null data pointer", op);
    if (numel(t) == 0) continue;
    if (reinterpret_cast<uintptr_t>(elem_ptr(t)) % 16)
      return fail(L3D_E_ALIGN, "%s: tensors must be 16-byte aligned", op);
    for (int d = 0; d < 3; ++d)
      if (t->dims[d] > 1 && t->strides[d] % 8)
        return fail(L3D_E_ALIGN, "%s: strides must be multiples of 16 bytes", op);
  }
  for (const l3d_tensor* t : {k_pages, v_pages})
    if ((pages > 1 && t->strides[0] == 0) || (size > 1 && t->strides[1] == 0))
      return fail(L3D_E_ALIGN, "%s: the pages must not be expanded (stride 0)", op);
  for (int d = 0; d < 3; ++d)
    if (out->dims[d] > 1 && out->strides[d] == 0) return fail(L3D_E_ALIGN, "%s: out must not be expanded (stride 0)", op);
  if (no_data(table) || no_data(lengths)) return fail(L3D_E_NULL, "%s: null data pointer", op);
  l3d::decode::Params p{};
  p.B = int(B); p.N = int(N); p.G = int(Hq / Hkv); p.Hkv = int(Hkv);
  p.q = elem_ptr(q);
  p.out = const_cast<char*>(elem_ptr(out));
  p.qb = q->strides[0]; p.qn = q->strides[1]; p.qh = q->strides[2];
  p.ob = out->strides[0]; p.on = out->strides[1]; p.oh = out->strides[2];
  l3d::decode::Keys kv{elem_ptr(k_pages), elem_ptr(v_pages), {}, {}, D};
  for (int i = 0; i < 3; ++i) {
    kv.ks[i] = k_pages->strides[i];
    kv.vs[i] = v_pages->strides[i];
  }
  p.keys = int(pages); p.size = int(size); p.width = int(width);
  p.table = reinterpret_cast<const int32_t*>(elem_ptr(table));
  p.table_stride = table->strides[0];
  p.lengths = elem_ptr(lengths);
  p.len64 = lengths->dtype == L3D_I64;
  p.causal = 1;
  p.scale_log2 = scale_log2;
  return l3d::decode::launch(op, p, kv, q->dtype == L3D_F16, width * size, workspace, reinterpret_cast<cudaStream_t>(stream),
                             timeout_ns);
}

extern "C" int l3d_paged_attention(const l3d_tensor* q, const l3d_tensor* k_pages, const l3d_tensor* v_pages,
                                   const l3d_tensor* table, const l3d_tensor* lengths, float scale,
                                   const l3d_tensor* out, void* workspace, size_t workspace_bytes,
                                   l3d_stream stream) {
  return run_paged_attention(q, k_pages, v_pages, table, lengths, scale, out, workspace, workspace_bytes, stream, 0,
                             "l3d_paged_attention");
}

extern "C" int l3d_paged_attention_selftest_timeout(const l3d_tensor* q, const l3d_tensor* k_pages,
                                                    const l3d_tensor* v_pages, const l3d_tensor* table,
                                                    const l3d_tensor* lengths, float scale, const l3d_tensor* out,
                                                    void* workspace, size_t workspace_bytes, uint32_t wait_limit_ms,
                                                    l3d_stream stream) {
  const char* op = "l3d_paged_attention_selftest_timeout";
  if (wait_limit_ms == 0 || wait_limit_ms > 2000)
    return fail(L3D_E_UNSUPPORTED, "%s: wait_limit_ms must be in [1, 2000]", op);
  return run_paged_attention(q, k_pages, v_pages, table, lengths, scale, out, workspace, workspace_bytes, stream,
                             uint64_t(wait_limit_ms) * 1000000ull, op);
}
