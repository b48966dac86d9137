// The step between a block's projection and its attention over a paged cache, in one pass: for the newest
// tokens of a batch of requests, the queries and keys normed per head and rotated by the tokens' positions,
// and the keys and values put into the cache's pages.
//   n = x / sqrt(mean(x^2) + eps) * w                    per head (where weights are given)
//   (n_lo, n_hi) -> (n_lo cos t - n_hi sin t, n_hi cos t + n_lo sin t),   t = position[axis(i)] * freq(i)
// for the pairs i of a head; elements in no pair stay as they are.  The reference norms and rotates q and k
// for two fixed models (crate/runtime/attention_math.rs:104-146, crate/runtime/trellis2_blocks.rs:85-161,
// :306-319) and keeps no cache.
//
// Bound by bytes: q, k and v are read once, q and the new cache rows written once.  Eight elements per thread, a
// head's D / 8 threads side by side in a warp: four pairs, both of whose elements a thread holds (two loads of 8 bytes
// where they lie apart), so that only the norm's sum is shuffled.  (With 16 bytes in a row per thread and the other
// half of a pair by shuffles the kernel was bound by issue: 36 us for 10992 tokens x 48 heads x 64.)  A block takes a few tokens and forms their angles once for all heads, in 64 bits:
// at position 100,000 a product in 32 bits is off by up to 4e-3 radians, as much as bf16's rounding.  What is
// left after whole turns are taken off is at most half a turn, and goes on in 32 bits.
// Measured: 49152 tokens x 24 heads x 128, bf16: 109 us (5.55 TB/s, 84% of a plain copy; call after call 112); 10992 x
// 48 x 64, f16: 31 us (4.38 TB/s; each block looks its places and angles up before its first row); one token 4.5 us.
#include "common.cuh"

namespace l3d {
namespace paged {

constexpr int THREADS = 256;
constexpr int MAX_TOKENS = 32;  // of one block
constexpr int TPU = 4;          // tokens of a thread's unit

struct Rows {                   // a [T, H, D] view
  char* p;
  int64_t st, sh;               // element strides
};

struct Params {
  int T, B, Hq, Hkv;
  int tokens;                   // of one block
  Rows q, k, v, qo;
  char *kp, *vp;                // pages [pages, size, Hkv, D]
  int64_t ks[3], vs[3];         // strides of page, slot, head
  int pages, size, width;
  const int32_t* table;
  int64_t table_stride;
  const void *held, *offsets, *positions;
  int held64, offsets64, positions64, axes;
  int64_t position_stride, position_axis;
  ChanVec qw, kw;
  float eps;
  const float2* freqs;          // high and low part of each pair's frequency
  const int32_t* axis;
  int pairs, half;              // half 0: neighbours; else pairs lie `half` apart in blocks of 2 half
};

__device__ __forceinline__ int64_t index_at(const void* p, int is64, int64_t i) {
  return is64 ? static_cast<const int64_t*>(p)[i] : int64_t(static_cast<const int32_t*>(p)[i]);
}

// The last place of the offsets with a value up to t, -1: none.  A warp looks, 32 places at a time.
__device__ __forceinline__ int request_of(const Params& p, int t, int lane) {
  if (!p.offsets) return 0;
  int lo = -1, hi = p.B + 1;  // offsets[lo] <= t < offsets[hi], as far as there are such
  while (hi - lo > 1) {
    const int step = (hi - lo - 1 + 31) / 32, at = lo + (lane + 1) * step;
    const bool below = at < hi && index_at(p.offsets, p.offsets64, at) <= t;
    const int n = __popc(__ballot_sync(0xffffffffu, below));
    hi = min(hi, lo + (n + 1) * step);
    lo += n * step;
  }
  return lo;
}

// Four values of a 16-bit type as two pairs of f32, and back.
__device__ __forceinline__ void unpack4(uint2 u, float2 (&f)[2], __nv_bfloat16) {
  f[0] = make_float2(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u));
  f[1] = make_float2(__uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
}
__device__ __forceinline__ void unpack4(uint2 u, float2 (&f)[2], __half) {
  f[0] = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
  f[1] = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
}
__device__ __forceinline__ uint2 pack4(const float2 (&f)[2], __nv_bfloat16) {
  const __nv_bfloat162 a = __float22bfloat162_rn(f[0]), b = __float22bfloat162_rn(f[1]);
  return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}
__device__ __forceinline__ uint2 pack4(const float2 (&f)[2], __half) {
  const __half2 a = __float22half2_rn(f[0]), b = __float22half2_rn(f[1]);
  return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// APART: the elements of a pair do not lie side by side.
template <typename T, int D, bool APART>
__global__ void __launch_bounds__(THREADS) append_kernel(const Params p) {
  constexpr int LANES = D / 8;                  // threads of a row
  constexpr int SLOTS = THREADS / LANES;        // rows of a block at a time
  __shared__ alignas(16) float s_cos[MAX_TOKENS][D / 2], s_sin[MAX_TOKENS][D / 2];
  __shared__ int64_t s_at[MAX_TOKENS];          // place in the request's sequence
  __shared__ int64_t s_k[MAX_TOKENS], s_v[MAX_TOKENS];  // where its key and value go; -1: no room
  __shared__ int s_out[MAX_TOKENS];             // -1: a token of no request
  __shared__ int s_ends[2];
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");  // for the kernel before: nothing global is touched earlier
  const int t0 = blockIdx.x * p.tokens, n = min(p.tokens, p.T - t0);
  const int lane = threadIdx.x % LANES, slot = threadIdx.x / LANES, groups = (n + TPU - 1) / TPU;
  // This thread's elements: lo .. lo + 3 and hi .. hi + 3, the pairs pair0 .. pair0 + 3; or neighbours, the pairs
  // pair0 .. of lo .. lo + 7.
  const int pair0 = 4 * lane;
  int lo = 8 * lane, hi = lo + 4;
  if (APART && pair0 < p.pairs) {
    const int block = pair0 / p.half;
    lo = block * 2 * p.half + (pair0 - block * p.half);
    hi = lo + p.half;
  }
  // The tokens' places: the requests of the first and of the last by a warp each, of the others between them.
  if (threadIdx.x < 64) {
    const int end = threadIdx.x / 32, b = request_of(p, end ? t0 + n - 1 : t0, threadIdx.x % 32);
    if (threadIdx.x % 32 == 0) s_ends[end] = b;
  }
  __syncthreads();
  if (threadIdx.x < n) {
    const int t = t0 + threadIdx.x;
    int b = s_ends[0], hi = s_ends[1] + 1;
    int64_t first = 0, place = 0;
    int page = -1;
    if (p.offsets) {
      while (hi - b > 1) {
        const int mid = (b + hi) >> 1;
        if (index_at(p.offsets, p.offsets64, mid) <= t) b = mid;
        else hi = mid;
      }
      if (b >= p.B) b = -1;
    } else {
      b = t / (p.T / p.B);
    }
    if (b >= 0) {
      first = p.offsets ? index_at(p.offsets, p.offsets64, b) : int64_t(b) * (p.T / p.B);
      place = index_at(p.held, p.held64, b) + (t - first);
      if (place >= 0 && place < int64_t(p.width) * p.size) page = p.table[b * p.table_stride + place / p.size];
    }
    const bool room = page >= 0 && page < p.pages;
    s_out[threadIdx.x] = b;
    s_at[threadIdx.x] = place;
    s_k[threadIdx.x] = room ? page * p.ks[0] + place % p.size * p.ks[1] : -1;
    s_v[threadIdx.x] = room ? page * p.vs[0] + place % p.size * p.vs[1] : -1;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n * p.pairs; i += THREADS) {
    const int t = i / p.pairs, pair = i - t * p.pairs;
    int64_t at = s_at[t];
    if (p.positions)
      at = index_at(p.positions, p.positions64,
                    (t0 + t) * p.position_stride + min(max(p.axis[pair], 0), p.axes - 1) * p.position_axis);
    const float2 f = p.freqs[pair];
    const double turns = double(at) * (double(f.x) + double(f.y)) * 0.15915494309189533577;  // 1 / 2 pi
    sincospif(2.f * float(turns - rint(turns)), &s_sin[t][pair], &s_cos[t][pair]);
  }
  __syncthreads();

  // ---- queries and keys.  A thread's unit is one head of TPU tokens of the block, whose loads it issues together; the
  // head's address and weights are worked out once for them.  (All threads of a warp take every turn: they meet in
  // its shuffles.)
  const int heads = p.Hq + p.Hkv, units = heads * groups;
  for (int u0 = 0; u0 < units; u0 += SLOTS) {
    const int u = min(u0 + slot, units - 1), grp = u / heads, hh = u - grp * heads;
    const bool isq = hh < p.Hq;
    const int h = isq ? hh : hh - p.Hq, ta = grp * TPU, tn = u0 + slot < units ? min(n - ta, TPU) : 0;
    const int64_t step = isq ? p.q.st : p.k.st;
    const T* src = reinterpret_cast<const T*>(isq ? p.q.p : p.k.p) + (t0 + ta) * step + h * (isq ? p.q.sh : p.k.sh);
    uint2 raw[TPU][2];
#pragma unroll
    for (int i = 0; i < TPU; ++i) {
      if constexpr (APART) {
        raw[i][0] = i < tn ? *reinterpret_cast<const uint2*>(src + i * step + lo) : make_uint2(0, 0);
        raw[i][1] = i < tn ? *reinterpret_cast<const uint2*>(src + i * step + hi) : make_uint2(0, 0);
      } else {
        const uint4 v = i < tn ? *reinterpret_cast<const uint4*>(src + i * step + lo) : make_uint4(0, 0, 0, 0);
        raw[i][0] = make_uint2(v.x, v.y);
        raw[i][1] = make_uint2(v.z, v.w);
      }
    }
    float2 w[2][2];
    if (p.qw.ptr) {
      load_chan<4>(isq ? p.qw : p.kw, h, lo, *reinterpret_cast<float(*)[4]>(w[0]));
      load_chan<4>(isq ? p.qw : p.kw, h, hi, *reinterpret_cast<float(*)[4]>(w[1]));
    }
#pragma unroll
    for (int i = 0; i < TPU; ++i) {
      if (i >= n) break;  // (as many tokens in the block: the same for all threads)
      const int t = min(ta + i, n - 1);
      float2 x[2][2];
      unpack4(raw[i][0], x[0], T());
      unpack4(raw[i][1], x[1], T());
      if (p.qw.ptr) {
        float2 sq = mul2(x[0][0], x[0][0]);
        sq = fma2(x[0][1], x[0][1], sq);
        sq = fma2(x[1][0], x[1][0], sq);
        sq = fma2(x[1][1], x[1][1], sq);
        float sum = sq.x + sq.y;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const float2 inv = f2(rsqrtf(sum * (1.f / D) + p.eps));  // to 2 ulp; what it goes into is rounded to 16 bits
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int e = 0; e < 2; ++e) x[a][e] = mul2(x[a][e], mul2(inv, w[a][e]));
      }
      if (pair0 < p.pairs) {
        const float4 c4 = *reinterpret_cast<const float4*>(&s_cos[t][pair0]), s4 = *reinterpret_cast<const float4*>(&s_sin[t][pair0]);
        if constexpr (APART) {
          const float2 c[2] = {make_float2(c4.x, c4.y), make_float2(c4.z, c4.w)};
          const float2 s[2] = {make_float2(s4.x, s4.y), make_float2(s4.z, s4.w)};
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 a = x[0][e], b = x[1][e], bs = mul2(b, s[e]);
            x[0][e] = fma2(a, c[e], make_float2(-bs.x, -bs.y));
            x[1][e] = fma2(b, c[e], mul2(a, s[e]));
          }
        } else {
          const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (pair0 + e >= p.pairs) continue;  // (of a place behind the last pair, which may hold anything)
            float2& z = x[e >> 1][e & 1];
            z = make_float2(z.x * c[e] - z.y * s[e], z.y * c[e] + z.x * s[e]);
          }
        }
      }
      if (i >= tn || s_out[t] < 0 || (!isq && s_k[t] < 0)) continue;  // (the shuffles are behind us)
      uint2 y[2] = {pack4(x[0], T()), pack4(x[1], T())};
      if (isq && s_k[t] < 0)  // no room: nothing is stored, and the request's attention is not finite
        y[0] = y[1] = make_uint2(0x7fff7fffu, 0x7fff7fffu);
      T* dst = isq ? reinterpret_cast<T*>(p.qo.p) + (t0 + t) * p.qo.st + h * p.qo.sh
                   : reinterpret_cast<T*>(p.kp) + s_k[t] + h * p.ks[2];
      if constexpr (APART) {
        *reinterpret_cast<uint2*>(dst + lo) = y[0];
        *reinterpret_cast<uint2*>(dst + hi) = y[1];
      } else {
        *reinterpret_cast<uint4*>(dst + lo) = make_uint4(y[0].x, y[0].y, y[1].x, y[1].y);
      }
    }
  }
  // ---- values
  for (int u = slot; u < p.Hkv * groups; u += SLOTS) {
    const int grp = u / p.Hkv, h = u - grp * p.Hkv, ta = grp * TPU, tn = min(n - ta, TPU);
    const T* src = reinterpret_cast<const T*>(p.v.p) + (t0 + ta) * p.v.st + h * p.v.sh + 8 * lane;
    uint4 raw[TPU];
#pragma unroll
    for (int i = 0; i < TPU; ++i)
      if (i < tn) raw[i] = *reinterpret_cast<const uint4*>(src + i * p.v.st);
#pragma unroll
    for (int i = 0; i < TPU; ++i)
      if (i < tn && s_k[ta + i] >= 0)
        *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.vp) + s_v[ta + i] + h * p.vs[2] + 8 * lane) = raw[i];
  }
}

template <typename T, int D>
static cudaError_t launch(const Params& p, unsigned grid, cudaStream_t s) {
  // The kernel may be scheduled while the one before it runs, and waits for it.
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(THREADS);
  cfg.stream = s;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, p.half ? append_kernel<T, D, true> : append_kernel<T, D, false>, p);
}

}  // namespace paged
}  // namespace l3d

using namespace l3d;

extern "C" int l3d_paged_append(const l3d_tensor* q, const l3d_tensor* k, const l3d_tensor* v,
                                const l3d_tensor* q_weight, const l3d_tensor* k_weight, float eps,
                                const l3d_tensor* freqs, const l3d_tensor* axes, int half,
                                const l3d_tensor* positions, const l3d_tensor* table,
                                const l3d_tensor* held, const l3d_tensor* offsets,
                                const l3d_tensor* q_out, const l3d_tensor* k_pages,
                                const l3d_tensor* v_pages, l3d_stream stream) {
  using namespace l3d::paged;
  const char* op = "l3d_paged_append";
  if (!q || !k || !v || !table || !held || !q_out || !k_pages || !v_pages)
    return fail(L3D_E_NULL, "%s: q, k, v, table, held, q_out, k_pages and v_pages are required", op);
  if (!q_weight != !k_weight) return fail(L3D_E_NULL, "%s: q_weight and k_weight come together", op);
  if (!freqs != !axes) return fail(L3D_E_NULL, "%s: freqs and axes come together", op);
  if (positions && !freqs) return fail(L3D_E_SHAPE, "%s: positions need freqs", op);
  const l3d_tensor* all[] = {q, k, v, q_out, k_pages, v_pages};
  for (int i = 0; i < 6; ++i) {
    const l3d_tensor* t = all[i];
    const int nd = i < 4 ? 3 : 4;
    if (t->dtype != q->dtype || (t->dtype != L3D_BF16 && t->dtype != L3D_F16))
      return fail(L3D_E_DTYPE, "%s: q, k, v, q_out and the pages all BF16 or all F16", op);
    if (t->ndim != nd)
      return fail(L3D_E_SHAPE, "%s: q, k, v, q_out [T, H, D], pages [pages, size, H, D]", op);
    if (numel(t) > 0 && t->strides[nd - 1] != 1)
      return fail(L3D_E_ALIGN, "%s: the head dim must be contiguous", op);
  }
  const int64_t T = q->dims[0], Hq = q->dims[1], D = q->dims[2], Hkv = k->dims[1];
  const int64_t pages = k_pages->dims[0], size = k_pages->dims[1], B = table->ndim == 2 ? table->dims[0] : 0;
  if (D != 64 && D != 128) return fail(L3D_E_UNSUPPORTED, "%s: head dim must be 64 or 128", op);
  for (int i = 0; i < 3; ++i) {
    if (q_out->dims[i] != q->dims[i]) return fail(L3D_E_SHAPE, "%s: q_out must have q's shape", op);
    if (v->dims[i] != k->dims[i]) return fail(L3D_E_SHAPE, "%s: k and v [T, Hkv, D]", op);
  }
  if (k->dims[0] != T || k->dims[2] != D) return fail(L3D_E_SHAPE, "%s: k and v [T, Hkv, D]", op);
  for (int i = 0; i < 4; ++i)
    if (v_pages->dims[i] != k_pages->dims[i] || (i == 2 && k_pages->dims[i] != Hkv) || (i == 3 && k_pages->dims[i] != D))
      return fail(L3D_E_SHAPE, "%s: k_pages and v_pages [pages, size, Hkv, D]", op);
  if (table->ndim != 2 || table->dtype != L3D_I32 || (table->dims[1] > 1 && table->strides[1] != 1))
    return fail(table->ndim == 2 && table->dtype != L3D_I32 ? L3D_E_DTYPE : L3D_E_SHAPE,
                "%s: table must be [B, pages of a request] I32 with contiguous rows", op);
  auto index_list = [&](const l3d_tensor* t, int64_t n) {
    return (t->dtype == L3D_I32 || t->dtype == L3D_I64) && t->ndim == 1 && t->dims[0] == n && (n <= 1 || t->strides[0] == 1);
  };
  if (!index_list(held, B)) return fail(L3D_E_SHAPE, "%s: held must be contiguous [B] I32 or I64", op);
  if (offsets && !index_list(offsets, B + 1))
    return fail(L3D_E_SHAPE, "%s: offsets must be contiguous [B + 1] I32 or I64", op);
  if (!offsets && (B > 0 ? T % B != 0 : T > 0))
    return fail(L3D_E_SHAPE, "%s: without offsets the tokens must divide evenly among the requests", op);
  const int64_t big = int64_t(1) << 30;
  if (T > big || B > big || pages > big || size > big || table->dims[1] > big || Hq + 2 * Hkv > 65535 || size <= 0)
    return fail(L3D_E_UNSUPPORTED, "%s: dimensions too large, or pages of no tokens", op);
  if (!(eps >= 0.f) || !(eps < INFINITY)) return fail(L3D_E_UNSUPPORTED, "%s: eps must be finite and >= 0", op);
  int64_t pairs = 0;
  if (freqs) {
    pairs = freqs->dims[0];
    if (freqs->dtype != L3D_F32 || axes->dtype != L3D_I32) return fail(L3D_E_DTYPE, "%s: freqs F32, axes I32", op);
    if (freqs->ndim != 2 || freqs->dims[1] != 2 || axes->ndim != 1 || axes->dims[0] != pairs || pairs < 1 ||
        2 * pairs > D || freqs->strides[1] != 1 || (pairs > 1 && (freqs->strides[0] != 2 || axes->strides[0] != 1)))
      return fail(L3D_E_SHAPE, "%s: freqs [pairs, 2] and axes [pairs], contiguous, at most D / 2 pairs", op);
    if (half < 0 || half % 8 || (half && pairs % half))
      return fail(L3D_E_UNSUPPORTED, "%s: half must be 0 or a multiple of 8 that divides the pairs", op);
    if (no_data(freqs) || no_data(axes) || reinterpret_cast<uintptr_t>(elem_ptr(freqs)) % 8)
      return fail(L3D_E_ALIGN, "%s: freqs must be 8-byte aligned", op);
  }
  if (positions) {
    if (positions->dtype != L3D_I32 && positions->dtype != L3D_I64)
      return fail(L3D_E_DTYPE, "%s: positions must be I32 or I64", op);
    if (positions->ndim != 2 || positions->dims[0] != T || positions->dims[1] < 1)
      return fail(L3D_E_SHAPE, "%s: positions must be [T, axes]", op);
  }
  Params p{};
  if (q_weight) {
    bool aligned = true;
    const l3d_tensor* w[] = {q_weight, k_weight};
    const char* names[] = {"q_weight", "k_weight"};
    for (int i = 0; i < 2; ++i) {
      if (int e = make_chanvec(w[i], names[i], D, i ? Hkv : Hq, i ? &p.kw : &p.qw, &aligned)) return e;
      if (!aligned) return fail(L3D_E_ALIGN, "%s: %s must be 16-byte aligned", op, names[i]);
    }
  }
  if (T == 0) return L3D_OK;
  for (const l3d_tensor* t : all) {
    if (no_data(t)) return fail(L3D_E_NULL, "%s: null data pointer", op);
    if (numel(t) == 0) continue;
    if (reinterpret_cast<uintptr_t>(elem_ptr(t)) % 16)
      return fail(L3D_E_ALIGN, "%s: tensors must be 16-byte aligned", op);
    for (int d = 0; d < t->ndim - 1; ++d)
      if (t->dims[d] > 1 && t->strides[d] % 8)
        return fail(L3D_E_ALIGN, "%s: strides must be multiples of 16 bytes", op);
  }
  const l3d_tensor* written[] = {q_out, k_pages, v_pages};
  for (const l3d_tensor* t : written)
    for (int d = 0; d < t->ndim - 1; ++d)
      if (t->dims[d] > 1 && t->strides[d] == 0)
        return fail(L3D_E_ALIGN, "%s: q_out and the pages must not be expanded (stride 0)", op);
  const l3d_tensor* lists[] = {table, held, offsets, positions};
  for (const l3d_tensor* t : lists)
    if (t && no_data(t)) return fail(L3D_E_NULL, "%s: null data pointer", op);
  auto rows = [](const l3d_tensor* t) {
    return Rows{const_cast<char*>(elem_ptr(t)), t->strides[0], t->strides[1]};
  };
  p.T = int(T); p.B = int(B); p.Hq = int(Hq); p.Hkv = int(Hkv);
  p.q = rows(q); p.k = rows(k); p.v = rows(v); p.qo = rows(q_out);
  p.kp = const_cast<char*>(elem_ptr(k_pages));
  p.vp = const_cast<char*>(elem_ptr(v_pages));
  for (int i = 0; i < 3; ++i) {
    p.ks[i] = k_pages->strides[i];
    p.vs[i] = v_pages->strides[i];
  }
  p.pages = int(pages); p.size = int(size); p.width = int(table->dims[1]);
  p.table = reinterpret_cast<const int32_t*>(elem_ptr(table));
  p.table_stride = table->strides[0];
  p.held = elem_ptr(held);
  p.held64 = held->dtype == L3D_I64;
  p.offsets = offsets ? elem_ptr(offsets) : nullptr;
  p.offsets64 = offsets && offsets->dtype == L3D_I64;
  if (positions) {
    p.positions = elem_ptr(positions);
    p.positions64 = positions->dtype == L3D_I64;
    p.axes = int(positions->dims[1]);
    p.position_stride = positions->strides[0];
    p.position_axis = positions->strides[1];
  }
  p.eps = eps;
  p.freqs = freqs ? reinterpret_cast<const float2*>(elem_ptr(freqs)) : nullptr;
  p.axis = axes ? reinterpret_cast<const int32_t*>(elem_ptr(axes)) : nullptr;
  p.pairs = int(pairs);
  p.half = freqs ? half : 0;
  // One token per block as long as the device (four blocks an SM) is not full, so that a few tokens spread over it;
  // then as many as fill it once, for a block's tokens are looked up together.
  const int64_t per = (T + 4 * int64_t(sm_count()) - 1) / (4 * int64_t(sm_count()));
  p.tokens = per > MAX_TOKENS ? MAX_TOKENS : int(per);
  const unsigned grid = unsigned((T + p.tokens - 1) / p.tokens);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (q->dtype == L3D_BF16) e = D == 64 ? launch<__nv_bfloat16, 64>(p, grid, s) : launch<__nv_bfloat16, 128>(p, grid, s);
  else e = D == 64 ? launch<__half, 64>(p, grid, s) : launch<__half, 128>(p, grid, s);
  return e == cudaSuccess ? L3D_OK : fail(L3D_E_CUDA, "%s: %s", op, cudaGetErrorString(e));
}
