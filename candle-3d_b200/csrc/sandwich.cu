// Block seam with a norm on either side of the residual (a "sandwich" norm):
//   n = Norm(h) [* post_weight] [+ post_bias]
//   r = res_scale * x + [gate *] n
//   y = Norm(r) [* weight] [+ bias] [* (1 + scale) + shift]
// Norm: RMS, v / sqrt(mean(v^2) + eps), or Layer, (v - mean) / sqrt(var + eps).
// The reference composes such seams from its norms and residual adds
// (crate/runtime/trellis2_blocks.rs:280-286,627-645, crate/runtime/vggt.rs:104-123);
// here x and h are read once and r and y written once.
#include <type_traits>

#include "common.cuh"
#include "ring.cuh"

namespace l3d {
namespace sandwich {

enum { NORM_LAYER = 1, NORM_RMS = 2 };

struct Params {
  int64_t rows, C, rows_per_batch;
  RowMap xm, hm, rm, ym;
  const void *x, *h;
  void *r, *y;                 // y null: no next norm
  ChanVec pw, pb, gate;        // after the block
  ChanVec w, b, scale, shift;  // before the next one
  float res_scale, post_eps, eps;
  int norm;
};

constexpr int kRowBlock = 1024, kBlock = 256;

__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) red[warp] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kRowBlock / 32; ++i) s += red[i];
  __syncthreads();
  return s;
}

__device__ __forceinline__ float chan_or(const ChanVec& v, int64_t b, int64_t c, float none) {
  if (!v.ptr) return none;
  float f[1];
  load_chan<1>(v, b, c, f);
  return f[0];
}

// Mean (0 for RMS) and 1 / sqrt(.. + eps) of the C values at s, by the whole block.
__device__ __forceinline__ void block_stats(int norm, const float* s, int64_t C, float eps, float* red,
                                            float& mean, float& inv) {
  mean = 0.f;
  if (norm == NORM_LAYER) {
    float a = 0.f;
    for (int64_t c = threadIdx.x; c < C; c += kRowBlock) a += s[c];
    mean = block_sum(a, red) / float(C);
  }
  float q = 0.f;
  for (int64_t c = threadIdx.x; c < C; c += kRowBlock) {
    const float d = s[c] - mean;
    q = fmaf(d, d, q);
  }
  inv = 1.f / sqrtf(block_sum(q, red) / float(C) + eps);
}

// One row per block at a time, the row held in shared memory as f32; any
// row length, alignment and strides.  Bound by its element-wise accesses and the
// waits between its passes: 4096 x 16384 bf16 501 us (1.1 TB/s; 256 threads 1145).
template <typename T>
__global__ void __launch_bounds__(kRowBlock, 2) row_kernel(const Params p) {
  extern __shared__ float s[];
  __shared__ float red[kRowBlock / 32];
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const int64_t b = row / p.rows_per_batch;
    const T* xr = static_cast<const T*>(p.x) + row_offset(p.xm, row);
    const T* hr = static_cast<const T*>(p.h) + row_offset(p.hm, row);
    for (int64_t c = threadIdx.x; c < p.C; c += kRowBlock) s[c] = to_f(hr[c]);
    __syncthreads();
    float mean, inv;
    block_stats(p.norm, s, p.C, p.post_eps, red, mean, inv);
    T* rr = static_cast<T*>(p.r) + row_offset(p.rm, row);
    for (int64_t c = threadIdx.x; c < p.C; c += kRowBlock) {
      const float n = (s[c] - mean) * inv * chan_or(p.pw, 0, c, 1.f) + chan_or(p.pb, 0, c, 0.f);
      const float r = fmaf(chan_or(p.gate, b, c, 1.f), n, p.res_scale * to_f(xr[c]));
      rr[c] = from_f<T>(r);
      s[c] = r;
    }
    __syncthreads();
    if (p.y) {
      block_stats(p.norm, s, p.C, p.eps, red, mean, inv);
      T* yr = static_cast<T*>(p.y) + row_offset(p.ym, row);
      for (int64_t c = threadIdx.x; c < p.C; c += kRowBlock) {
        const float n = (s[c] - mean) * inv * chan_or(p.w, 0, c, 1.f) + chan_or(p.b, 0, c, 0.f);
        yr[c] = from_f<T>(fmaf(n, 1.f + chan_or(p.scale, b, c, 0.f), chan_or(p.shift, b, c, 0.f)));
      }
      __syncthreads();
    }
  }
}

// The per-channel vectors are folded into f32 coefficients in shared memory,
//   r = res_scale x + A1 (h - mean) inv + B1,  A1 = gate post_weight, B1 = gate post_bias
//   y = A2 (r - mean) inv + B2,  A2 = weight (1 + scale), B2 = bias (1 + scale) + shift
// B1 and B2 only where one of their vectors is given.
struct Coefs {
  int has_b1, has_b2;
  int ld;                  // floats of a coefficient row (a multiple of 4)
  int chan_vec;            // the vectors are 16-byte aligned
  int same;                // and of the activations' type
};

// Place of channel c in a coefficient row read in vectors of VEC: in planes of
// four floats, so that consecutive vectors lie 16 bytes apart and their loads
// meet no bank twice.
template <int VEC>
__device__ __forceinline__ int coef_at(int c, int ld) {
  if constexpr (VEC == 8) return ((c >> 2) & 1) * (ld / 2) + (c >> 3) * 4 + (c & 3);
  else return c;
}

// One channel, or VEC consecutive ones, of batch element b folded into `coef`.
template <typename T, int VEC>
__device__ __forceinline__ void fold(const Params& p, const Coefs& k, float* coef, int64_t b) {
  const int C = int(p.C);
  float* row = coef;
  float *a1 = row, *a2 = row + k.ld, *b1 = row + 2 * k.ld, *b2 = row + (2 + k.has_b1) * k.ld;
  if constexpr (VEC > 1) {
    if (k.chan_vec && k.same) {
      // All vectors' loads at once (without branches between them): this is what
      // a call on a few rows waits for.
      for (int c = int(threadIdx.x) * VEC; c < C; c += int(blockDim.x) * VEC) {
        const ChanVec* const vecs[7] = {&p.gate, &p.pw, &p.pb, &p.scale, &p.w, &p.b, &p.shift};
        uint4 raw[7];
#pragma unroll
        for (int i = 0; i < 7; ++i)
          raw[i] = vecs[i]->ptr ? __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(vecs[i]->ptr) +
                                                                       b * vecs[i]->bstride + c))
                                : make_uint4(0, 0, 0, 0);
        float f[7][VEC];
#pragma unroll
        for (int i = 0; i < 7; ++i) unpack(raw[i], f[i], T());
        float o[4][VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float g = p.gate.ptr ? f[0][e] : 1.f, t = 1.f + f[3][e];
          o[0][e] = g * (p.pw.ptr ? f[1][e] : 1.f);
          o[1][e] = t * (p.w.ptr ? f[4][e] : 1.f);
          o[2][e] = g * f[2][e];
          o[3][e] = fmaf(t, f[5][e], f[6][e]);
        }
#pragma unroll
        for (int e = 0; e < VEC; e += 4) {
          const int at = coef_at<VEC>(c + e, k.ld);
          auto four = [&](int i) { return make_float4(o[i][e], o[i][e + 1], o[i][e + 2], o[i][e + 3]); };
          *reinterpret_cast<float4*>(a1 + at) = four(0);
          *reinterpret_cast<float4*>(a2 + at) = four(1);
          if (k.has_b1) *reinterpret_cast<float4*>(b1 + at) = four(2);
          if (k.has_b2) *reinterpret_cast<float4*>(b2 + at) = four(3);
        }
      }
      return;
    }
  }
  if constexpr (VEC == 1) {
    if (k.same) {  // as above, four channels at once
      constexpr int U = 4;
      for (int c0 = threadIdx.x; c0 < C; c0 += U * int(blockDim.x)) {
        const ChanVec* const vecs[7] = {&p.gate, &p.pw, &p.pb, &p.scale, &p.w, &p.b, &p.shift};
        T raw[7][U];
#pragma unroll
        for (int i = 0; i < 7; ++i)
#pragma unroll
          for (int u = 0; u < U; ++u)
            raw[i][u] = vecs[i]->ptr ? __ldg(static_cast<const T*>(vecs[i]->ptr) + b * vecs[i]->bstride +
                                             min(c0 + u * int(blockDim.x), C - 1))
                                     : from_f<T>(0.f);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int c = c0 + u * int(blockDim.x);
          if (c >= C) break;
          const float g = p.gate.ptr ? to_f(raw[0][u]) : 1.f, t = 1.f + to_f(raw[3][u]);
          a1[c] = g * (p.pw.ptr ? to_f(raw[1][u]) : 1.f);
          a2[c] = t * (p.w.ptr ? to_f(raw[4][u]) : 1.f);
          if (k.has_b1) b1[c] = g * to_f(raw[2][u]);
          if (k.has_b2) b2[c] = fmaf(t, to_f(raw[5][u]), to_f(raw[6][u]));
        }
      }
      return;
    }
  }
  if (VEC > 1 && k.chan_vec) {
    for (int c = int(threadIdx.x) * VEC; c < C; c += int(blockDim.x) * VEC) {
      float g[VEC], w[VEC], t[VEC];
      auto get = [&](const ChanVec& v, int64_t bb, float none, float (&o)[VEC]) {
        if (v.ptr) {
          load_chan<VEC>(v, bb, c, o);
        } else {
#pragma unroll
          for (int e = 0; e < VEC; ++e) o[e] = none;
        }
      };
      auto put = [&](float* dst, const float (&o)[VEC]) {
#pragma unroll
        for (int e = 0; e < VEC; e += 4)
          *reinterpret_cast<float4*>(dst + coef_at<VEC>(c + e, k.ld)) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
      };
      get(p.gate, b, 1.f, g);
      get(p.pw, 0, 1.f, w);
      get(p.scale, b, 0.f, t);
#pragma unroll
      for (int e = 0; e < VEC; ++e) { w[e] *= g[e]; t[e] += 1.f; }
      put(a1, w);
      if (k.has_b1) {
        get(p.pb, 0, 0.f, w);
#pragma unroll
        for (int e = 0; e < VEC; ++e) w[e] *= g[e];
        put(b1, w);
      }
      get(p.w, 0, 1.f, w);
#pragma unroll
      for (int e = 0; e < VEC; ++e) w[e] *= t[e];
      put(a2, w);
      if (k.has_b2) {
        get(p.b, 0, 0.f, w);
        get(p.shift, b, 0.f, g);
#pragma unroll
        for (int e = 0; e < VEC; ++e) w[e] = fmaf(w[e], t[e], g[e]);
        put(b2, w);
      }
    }
  } else {
    for (int c = threadIdx.x; c < C; c += blockDim.x) {
      const int at = coef_at<VEC>(c, k.ld);
      const float g = chan_or(p.gate, b, c, 1.f), t = 1.f + chan_or(p.scale, b, c, 0.f);
      a1[at] = g * chan_or(p.pw, 0, c, 1.f);
      if (k.has_b1) b1[at] = g * chan_or(p.pb, 0, c, 0.f);
      a2[at] = t * chan_or(p.w, 0, c, 1.f);
      if (k.has_b2) b2[at] = fmaf(t, chan_or(p.b, 0, c, 0.f), chan_or(p.shift, b, c, 0.f));
    }
  }
}

// row_offset for fewer than 2^32 rows: a 64-bit division is a call, around which
// a row held in registers would be spilled.
__device__ __forceinline__ int64_t row_offset32(const RowMap& m, uint32_t r) {
  int64_t off = m.base;
#pragma unroll
  for (int i = 4; i >= 1; --i) {
    if (i < m.nd) {
      const uint32_t d = uint32_t(m.dims[i]), q = r / d;
      off += int64_t(r - q * d) * m.strides[i];
      r = q;
    }
  }
  return off + int64_t(r) * m.strides[0];
}

// Sum over the G threads of a row, the same value in each of them.  `red`: two
// buffers in turn, since a warp can be one sum ahead of another, not two.
template <int G>
__device__ __forceinline__ float group_sum(float v, float* red, int& turn) {
#pragma unroll
  for (int o = (G < 32 ? G : 32) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (G > 32) {
    constexpr int W = G / 32;
    const int grp = threadIdx.x / G;
    float* r = red + turn * 20 + grp * W;
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) r[(threadIdx.x % G) >> 5] = v;
    asm volatile("bar.sync %0, %1;" ::"r"(1 + grp), "n"(G) : "memory");
    v = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) v += r[i];
  }
  return v;
}
// Whether `ok` holds in all threads of the unit.
template <int G>
__device__ __forceinline__ bool unit_all(bool ok) {
  if constexpr (G <= 32) {
    return __all_sync(0xffffffffu, ok);
  } else {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
        "bar.red.and.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"(uint32_t(ok)), "r"(1 + int(threadIdx.x / G)), "n"(G)
        : "memory");
    return r != 0;
  }
}

// The ring kernel (16-byte aligned rows): one block per SM (fewer for few rows),
// a contiguous range of rows each, worked through by units of max(G, 32)
// threads.  G threads hold a row's h in registers as f32 (64 elements a thread,
// 32 of f32 rows), and r in its place; G = 8 puts four rows in a warp.  Each
// unit keeps two packs of rows (x and h) in shared memory that bulk copies
// fill ahead of it, so that the loads in flight do not occupy registers; its
// first thread issues the next copy once the unit has read a slot.
// Both norms' sums are taken in two passes over the registers (mean, then
// centred squares: one pass of shifted moments loses digits where one channel
// lies far out).
// Bound by memory: 131072 x 2048 bf16 takes 376 us (5.7 TB/s, 87% of a plain copy).
// G and NV by the row's length, bf16: 65536 x 256 takes 34 us with 8 threads a row
// and 4 vectors a thread, 41 with 8 and 8, 56 with 32 and 4; 65536 x 1024 102 us with
// 32 and 4, 120 with 32 and 8; 8192 x 8192 117 us with 128 and 8, 169 with 256 and 4.
// Threads of a block: 12 warps of 168 registers for 8 vectors a thread, 20 of 96
// for rows of half that length.
constexpr int threads_of(int nv) { return nv == 8 ? 384 : 640; }

struct Ring {
  int64_t rows_per_batch;  // rows that share per-batch vectors (all, without such vectors)
  int units;               // per block
  int slots;               // of a unit: 2, or 1
  uint32_t row_bytes;
  uint64_t wait_ns;
};

__device__ int g_sandwich_status;

template <typename T, int G, int NV, int NORM>
__global__ void __launch_bounds__(threads_of(NV), 1)
    ring_kernel(const Params p, const Coefs kc, const Ring sp) {
  constexpr int VEC = Vec16<T>::N, P = VEC / 2;          // pairs of a vector (NV of them a thread)
  constexpr int U = G < 32 ? 32 : G, RPU = U / G;        // threads and rows of a unit
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float red[40];
  float* coef = reinterpret_cast<float*>(smem);
  uint8_t* slots = smem + size_t(2 + kc.has_b1 + kc.has_b2) * kc.ld * 4;
  const uint32_t slot_bytes = 2 * RPU * sp.row_bytes;    // the pack's h rows, then its x rows
  uint64_t* full = reinterpret_cast<uint64_t*>(slots + size_t(sp.units) * sp.slots * slot_bytes);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(full + sp.units * sp.slots);
  const int unit = threadIdx.x / U, tu = threadIdx.x % U;
  const int t = threadIdx.x % G, sub = tu / G;           // thread of the row, row of the pack
  const int nvec = int(p.C) / VEC;
  const int64_t lo = p.rows * blockIdx.x / gridDim.x, hi = p.rows * (blockIdx.x + 1) / gridDim.x;
  const int64_t packs = (hi - lo + RPU - 1) / RPU;       // pack k: rows lo + k RPU ..
  if (threadIdx.x == 0) {
    for (int i = 0; i < sp.units * sp.slots; ++i) ring_bar_init(&full[i], 2 * RPU);
    *abort_flag = 0;
    ring_init_fence();
  }
  __syncthreads();
  const bool works = unit < sp.units;                    // the other threads only fold
  uint8_t* my_slots = slots + size_t(works ? unit : 0) * sp.slots * slot_bytes;
  uint64_t* my_full = full + (works ? unit : 0) * sp.slots;
  // The unit's n-th pack (pack n units + unit) into slot n mod slots.
  auto issue = [&](int64_t n) {
    const int64_t k = n * sp.units + unit;
    if (k >= packs) return;
    uint8_t* slot = my_slots + (n & (sp.slots - 1)) * slot_bytes;
    uint64_t* bar = &my_full[n & (sp.slots - 1)];
    for (int i = 0; i < RPU; ++i) {
      const int64_t row = lo + k * RPU + i;
      if (row < hi) {
        ring_load(slot + i * sp.row_bytes, static_cast<const T*>(p.h) + row_offset32(p.hm, uint32_t(row)),
                  sp.row_bytes, bar);
        ring_load(slot + (RPU + i) * sp.row_bytes,
                  static_cast<const T*>(p.x) + row_offset32(p.xm, uint32_t(row)), sp.row_bytes, bar);
      } else {
        ring_arrive(bar);
        ring_arrive(bar);
      }
    }
  };
  if (works && tu == 0)
    for (int n = 0; n < sp.slots; ++n) issue(n);
  const float inv_c = 1.f / float(p.C);
  const float2 rs = f2(p.res_scale);
  int turn = 0;
  bool dead = false;
  int64_t n = 0;  // the unit's next pack
  for (int64_t s0 = lo; s0 < hi;) {
    // Rows [s0, s1): one batch element's.
    const int64_t b = s0 / sp.rows_per_batch;
    const int64_t s1 = min((b + 1) * sp.rows_per_batch, hi);
    if (s0 != lo) __syncthreads();
    fold<T, VEC>(p, kc, coef, b);
    __syncthreads();
    // Vector i of this thread of coefficient row k.
    auto coefs = [&](int k, int i, float2 (&o)[P]) {
      const float* c = coef + k * kc.ld + (t + i * G) * 4;
#pragma unroll
      for (int e = 0; e < P; e += 2) {
        const float4 v = *reinterpret_cast<const float4*>(c + (e / 2) * (kc.ld / 2));
        o[e] = make_float2(v.x, v.y);
        o[e + 1] = make_float2(v.z, v.w);
      }
    };
    for (; works && !dead; ++n) {
      const int64_t row0 = lo + (n * sp.units + unit) * RPU;  // first row of the pack
      if (row0 >= s1) break;
      const int slot = int(n & (sp.slots - 1));
      if (!unit_all<G>(ring_wait(&my_full[slot], uint32_t(n >> (sp.slots - 1)) & 1u, abort_flag, sp.wait_ns, false,
                                 &g_sandwich_status))) {
        dead = true;
        break;
      }
      const int64_t row = row0 + sub;
      const bool valid = row >= s0 && row < s1;
      const uint32_t at = uint32_t(valid ? row : s0);
      const uint4* hs = reinterpret_cast<const uint4*>(my_slots + slot * slot_bytes + sub * sp.row_bytes) + t;
      const uint4* xs = reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(hs) + RPU * sp.row_bytes);
      float2 f[NV][P];
#pragma unroll
      for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int e = 0; e < P; ++e) f[i][e] = f2(0.f);
        if (t + i * G < nvec) unpack2(hs[i * G], f[i], T());
      }
      // Mean and 1 / sqrt(mean square + eps) of the row in f (zero past its end).
      float2 nm = f2(0.f);
      auto stats = [&](float eps) {
        if constexpr (NORM == NORM_LAYER) {
          float2 s = f[0][0];
#pragma unroll
          for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < P; ++e)
              if (i + e > 0) s = add2(s, f[i][e]);
          nm = f2(-group_sum<G>(s.x + s.y, red, turn) * inv_c);
        }
        float2 q = f2(0.f);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          if (NORM == NORM_LAYER && t + i * G >= nvec) continue;
#pragma unroll
          for (int e = 0; e < P; ++e) {
            const float2 d = NORM == NORM_LAYER ? add2(f[i][e], nm) : f[i][e];
            q = fma2(d, d, q);
          }
        }
        return f2(1.f / sqrtf(fmaf(group_sum<G>(q.x + q.y, red, turn), inv_c, eps)));
      };
      float2 iv = stats(p.post_eps);
      {
        uint4* rd = reinterpret_cast<uint4*>(static_cast<T*>(p.r) + row_offset32(p.rm, at)) + t;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          if (t + i * G >= nvec) continue;
          float2 a[P], c[P], x[P];
          coefs(0, i, a);
          if (kc.has_b1) coefs(2, i, c);
          unpack2(xs[i * G], x, T());
#pragma unroll
          for (int e = 0; e < P; ++e) {
            const float2 d = mul2(NORM == NORM_LAYER ? add2(f[i][e], nm) : f[i][e], iv);
            const float2 base = kc.has_b1 ? fma2(rs, x[e], c[e]) : mul2(rs, x[e]);
            f[i][e] = fma2(a[e], d, base);
          }
          if (valid) st_act_raw(rd + i * G, pack2(f[i], T()));
        }
      }
      // The slot has been read; a pack that reaches into the next batch
      // element is taken up again there.
      const bool whole = RPU == 1 || row0 + RPU <= s1 || s1 == hi;
      if (whole) {
        if constexpr (G <= 32) __syncwarp();
        else unit_all<G>(true);
        if (tu == 0) issue(n + sp.slots);
      }
      if (p.y) {
        iv = stats(p.eps);
        uint4* yd = reinterpret_cast<uint4*>(static_cast<T*>(p.y) + row_offset32(p.ym, at)) + t;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          if (t + i * G >= nvec) continue;
          float2 a[P], c[P];
          coefs(1, i, a);
          if (kc.has_b2) coefs(2 + kc.has_b1, i, c);
#pragma unroll
          for (int e = 0; e < P; ++e) {
            const float2 d = mul2(NORM == NORM_LAYER ? add2(f[i][e], nm) : f[i][e], iv);
            f[i][e] = kc.has_b2 ? fma2(a[e], d, c[e]) : mul2(a[e], d);
          }
          if (valid) st_act_raw(yd + i * G, pack2(f[i], T()));
        }
      }
      if (!whole) break;
    }
    s0 = s1;
  }
  // After an abort no copy may still be in flight when the block exits.
  if (dead && tu == 0)
    for (int64_t k = n; k < n + sp.slots; ++k)
      if (k * sp.units + unit < packs)
        ring_wait(&my_full[k & (sp.slots - 1)], uint32_t(k >> (sp.slots - 1)) & 1u, abort_flag, sp.wait_ns, true, &g_sandwich_status);
}

// The element kernel (any alignment): G threads per row, NE elements a thread,
// blocks that keep to one batch element.  Bound by the number of its accesses,
// an element each: 65536 x 1023 bf16 takes 237 us (2.3 TB/s), where the ring
// takes 102 for rows of 1024; a few rows by the folding (572 x 5252 18 us, 36 with
// a channel at a time and a second wave of blocks that folds again).  NE and G by
// the row's length: 262144 x 63 takes 121 us with 8 elements a thread, 407 with 32;
// 32768 x 2047 243 us with 64 threads a row, 577 with 256.
struct Blocks {
  int64_t rows, rows_per_block;  // of a batch element
  int per_batch;
};
constexpr int elem_blocks(int ne) { return ne == 8 ? 6 : 2; }  // per SM
template <typename T, int G, int NE, int NORM>
__global__ void __launch_bounds__(kBlock, elem_blocks(NE))
    elem_kernel(const Params p, const Coefs kc, const Blocks sp) {
  constexpr int RPB = kBlock / G;
  extern __shared__ __align__(16) float coef[];
  __shared__ float red[40];
  const int t = threadIdx.x % G, C = int(p.C);
  const int64_t b = blockIdx.x / sp.per_batch;
  const int64_t first = int64_t(blockIdx.x % sp.per_batch) * sp.rows_per_block;
  const int64_t last = min(first + sp.rows_per_block, sp.rows);
  fold<T, 1>(p, kc, coef, b);
  __syncthreads();
  const float *a1 = coef, *a2 = coef + kc.ld, *b1 = coef + 2 * kc.ld, *b2 = coef + (2 + kc.has_b1) * kc.ld;
  const float inv_c = 1.f / float(C);
  int turn = 0;
  for (int64_t row = first + threadIdx.x / G; row < last; row += RPB) {
    const uint32_t at = uint32_t(b * sp.rows + row);
    const T* hs = static_cast<const T*>(p.h) + row_offset32(p.hm, at);
    const T* xs = static_cast<const T*>(p.x) + row_offset32(p.xm, at);
    T* rd = static_cast<T*>(p.r) + row_offset32(p.rm, at);
    T* yd = p.y ? static_cast<T*>(p.y) + row_offset32(p.ym, at) : nullptr;
    // Both rows' loads at once (a load of x in the loop below would wait for the
    // stores before it: 65536 x 1024 bf16 took 476 us that way).
    float f[NE], x[NE];
#pragma unroll
    for (int i = 0; i < NE; ++i) f[i] = t + i * G < C ? to_f(hs[t + i * G]) : 0.f;
#pragma unroll
    for (int i = 0; i < NE; ++i) x[i] = t + i * G < C ? to_f(xs[t + i * G]) : 0.f;
    float nm = 0.f;
    auto stats = [&](float eps) {
      if constexpr (NORM == NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NE; ++i) s += f[i];
        nm = -group_sum<G>(s, red, turn) * inv_c;
      }
      float q = 0.f;
#pragma unroll
      for (int i = 0; i < NE; ++i) {
        const float d = NORM == NORM_LAYER ? (t + i * G < C ? f[i] + nm : 0.f) : f[i];
        q = fmaf(d, d, q);
      }
      return 1.f / sqrtf(fmaf(group_sum<G>(q, red, turn), inv_c, eps));
    };
    float iv = stats(p.post_eps);
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const int c = t + i * G;
      if (c >= C) continue;
      const float base = fmaf(p.res_scale, x[i], kc.has_b1 ? b1[c] : 0.f);
      f[i] = fmaf(a1[c], (f[i] + nm) * iv, base);
      rd[c] = from_f<T>(f[i]);
    }
    if (!p.y) continue;
    iv = stats(p.eps);
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const int c = t + i * G;
      if (c < C) yd[c] = from_f<T>(fmaf(a2[c], (f[i] + nm) * iv, kc.has_b2 ? b2[c] : 0.f));
    }
  }
}

constexpr int64_t kMaxC = 24 * 1024;  // the row in shared memory: 96 KB

static int check_like(const l3d_tensor* t, const l3d_tensor* x, const char* op, const char* name) {
  if (no_data(t)) return fail(L3D_E_NULL, "%s: %s has a null data pointer", op, name);
  if (t->dtype != x->dtype)
    return fail(L3D_E_DTYPE, "%s: %s dtype %s != x dtype %s", op, name, dtype_name(t->dtype),
                dtype_name(x->dtype));
  bool same = t->ndim == x->ndim;
  for (int i = 0; same && i < x->ndim; ++i) same = t->dims[i] == x->dims[i];
  if (!same) return fail(L3D_E_SHAPE, "%s: %s shape differs from x", op, name);
  if (t->dims[t->ndim - 1] > 1 && t->strides[t->ndim - 1] != 1)
    return fail(L3D_E_ALIGN, "%s: %s last dim must be contiguous", op, name);
  return L3D_OK;
}

constexpr int kSmem = 227 * 1024 - 1024;
constexpr const char* kNoSmem = "l3d_sandwich_residual_norm: cannot reserve shared memory";

// Returns 1 when launched, 0 when the row does not fit this kernel, or fails.
template <typename T, int G, int NV, int NORM>
static int launch_ring(const Params& p, const Coefs& kc, Ring sp, size_t coef, cudaStream_t s) {
  constexpr int U = G < 32 ? 32 : G, RPU = U / G;
  // One slot, not filled ahead, where two do not fit: 8192 x 8192 f32 with
  // all vectors takes 205 us so, 1170 with a block per row.
  size_t slot = 2 * (size_t(2) * RPU * sp.row_bytes + 8);
  sp.slots = coef + slot + 16 > size_t(kSmem) ? 1 : 2;
  if (sp.slots == 1) slot /= 2;
  if (coef + slot + 16 > size_t(kSmem)) return 0;
  auto k = ring_kernel<T, G, NV, NORM>;
  if (set_smem_limit(reinterpret_cast<const void*>(k), kSmem) != cudaSuccess) return -fail(L3D_E_CUDA, "%s", kNoSmem);
  const int64_t packs = (p.rows + RPU - 1) / RPU;
  const int64_t blocks = packs < sm_count() ? packs : sm_count();
  const int64_t per_block = ((p.rows + blocks - 1) / blocks + RPU - 1) / RPU;
  int64_t units = threads_of(NV) / U;
  if (units > per_block) units = per_block;
  const int64_t room = int64_t((size_t(kSmem) - coef - 16) / slot);
  sp.units = int(units < room ? units : room);
  k<<<unsigned(blocks), threads_of(NV), coef + size_t(sp.units) * slot + 16, s>>>(p, kc, sp);
  return 1;
}

template <typename T, int G, int NE, int NORM>
static int launch_elem(const Params& p, const Coefs& kc, int64_t batches, size_t coef, cudaStream_t s) {
  constexpr int RPB = kBlock / G;
  if (coef > 100 * 1024) return 0;
  auto k = elem_kernel<T, G, NE, NORM>;
  if (set_smem_limit(reinterpret_cast<const void*>(k), 100 * 1024) != cudaSuccess) return -fail(L3D_E_CUDA, "%s", kNoSmem);
  Blocks sp{};
  sp.rows = p.rows / batches;
  // One wave of blocks, shared out between the batch elements.
  const int64_t most = (sp.rows + RPB - 1) / RPB;
  int64_t per = int64_t(sm_count()) * elem_blocks(NE) / batches;
  per = per < 1 ? 1 : per > most ? most : per;
  sp.rows_per_block = ((sp.rows + per - 1) / per + RPB - 1) / RPB * RPB;
  sp.per_batch = int((sp.rows + sp.rows_per_block - 1) / sp.rows_per_block);
  k<<<unsigned(sp.per_batch) * unsigned(batches), kBlock, coef, s>>>(p, kc, sp);
  return 1;
}

template <typename T, int NORM>
static int try_fast(const Params& p, bool vec_ok, bool chan_vec, int64_t batches, cudaStream_t s) {
  if (p.rows >= (int64_t(1) << 31)) return 0;
  Coefs kc{};
  kc.has_b1 = p.pb.ptr != nullptr;
  kc.has_b2 = p.b.ptr || p.shift.ptr;
  kc.ld = int((p.C + 7) & ~int64_t(7));
  kc.chan_vec = chan_vec;
  const int dt = std::is_same<T, float>::value ? L3D_F32 : std::is_same<T, __half>::value ? L3D_F16 : L3D_BF16;
  kc.same = 1;
  for (const ChanVec* v : {&p.gate, &p.pw, &p.pb, &p.scale, &p.w, &p.b, &p.shift})
    if (v->ptr && v->dtype != dt) kc.same = 0;
  const size_t coef = size_t(2 + kc.has_b1 + kc.has_b2) * kc.ld * 4;
  if (vec_ok) {
    Ring sp{};
    sp.rows_per_batch = p.rows / batches;
    sp.row_bytes = uint32_t(p.C * sizeof(T));
    sp.wait_ns = 2000000000ull;
    constexpr int E = 8 * Vec16<T>::N;  // elements of a thread
    const int rc = p.C <= 4 * E ? launch_ring<T, 8, 4, NORM>(p, kc, sp, coef, s)
                   : p.C <= 8 * E ? launch_ring<T, 8, 8, NORM>(p, kc, sp, coef, s)
                   : p.C <= 16 * E ? launch_ring<T, 32, 4, NORM>(p, kc, sp, coef, s)
                   : p.C <= 32 * E ? launch_ring<T, 32, 8, NORM>(p, kc, sp, coef, s)
                   : p.C <= 64 * E ? launch_ring<T, 64, 8, NORM>(p, kc, sp, coef, s)
                   : p.C <= 128 * E ? launch_ring<T, 128, 8, NORM>(p, kc, sp, coef, s)
                   : p.C <= 256 * E ? launch_ring<T, 256, 8, NORM>(p, kc, sp, coef, s) : 0;
    if (rc) return rc;
  }
  return p.C <= 32 * 8 ? launch_elem<T, 32, 8, NORM>(p, kc, batches, coef, s)
         : p.C <= 32 * 32 ? launch_elem<T, 32, 32, NORM>(p, kc, batches, coef, s)
         : p.C <= 64 * 32 ? launch_elem<T, 64, 32, NORM>(p, kc, batches, coef, s)
         : p.C <= 128 * 32 ? launch_elem<T, 128, 32, NORM>(p, kc, batches, coef, s)
         : p.C <= 256 * 32 ? launch_elem<T, 256, 32, NORM>(p, kc, batches, coef, s) : 0;
}

template <typename T>
static int launch(const Params& p, bool vec_ok, bool chan_vec, int64_t batches, cudaStream_t s) {
  const int rc = p.norm == NORM_LAYER ? try_fast<T, NORM_LAYER>(p, vec_ok, chan_vec, batches, s)
                                      : try_fast<T, NORM_RMS>(p, vec_ok, chan_vec, batches, s);
  if (rc) return rc < 0 ? -rc : L3D_OK;
  // Rows too long for either (or 2^31 of them): a block per row.
  auto k = row_kernel<T>;
  if (set_smem_limit(reinterpret_cast<const void*>(k), int(kMaxC * 4)) != cudaSuccess)
    return fail(L3D_E_CUDA, "l3d_sandwich_residual_norm: cannot reserve shared memory");
  const int64_t cap = int64_t(sm_count()) * 8;
  k<<<unsigned(p.rows < cap ? p.rows : cap), kRowBlock, size_t(p.C) * 4, s>>>(p);
  return L3D_OK;
}

cudaError_t status_read(int* status, int reset) {
  cudaError_t e = cudaMemcpyFromSymbol(status, g_sandwich_status, sizeof(int));
  if (e == cudaSuccess && reset) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_sandwich_status, &zero, sizeof(int));
  }
  return e;
}

}  // namespace sandwich
}  // namespace l3d

using namespace l3d;

extern "C" int l3d_sandwich_residual_norm(const l3d_tensor* x, const l3d_tensor* h, int norm,
                                          const l3d_tensor* post_weight,
                                          const l3d_tensor* post_bias, const l3d_tensor* gate,
                                          float res_scale, const l3d_tensor* weight,
                                          const l3d_tensor* bias, const l3d_tensor* shift,
                                          const l3d_tensor* scale, float post_eps, float eps,
                                          const l3d_tensor* r_out, const l3d_tensor* y,
                                          l3d_stream stream) {
  using namespace l3d::sandwich;
  const char* op = "l3d_sandwich_residual_norm";
  if (!x || !h || !r_out) return fail(L3D_E_NULL, "%s: x, h and r_out are required", op);
  if (no_data(x)) return fail(L3D_E_NULL, "%s: x has a null data pointer", op);
  if (!is_float_dtype(x->dtype)) return fail(L3D_E_DTYPE, "%s: x must be F32/F16/BF16", op);
  if (x->ndim < 1 || x->ndim > L3D_MAX_DIMS) return fail(L3D_E_SHAPE, "%s: bad rank", op);
  if (norm != NORM_LAYER && norm != NORM_RMS)
    return fail(L3D_E_UNSUPPORTED, "%s: norm must be 1 (layer) or 2 (RMS)", op);
  if (!y && (weight || bias || shift || scale))
    return fail(L3D_E_NULL, "%s: weight, bias, shift and scale need y", op);
  int rc;
  if ((rc = check_like(x, x, op, "x")) || (rc = check_like(h, x, op, "h")) ||
      (rc = check_like(r_out, x, op, "r_out")) || (y && (rc = check_like(y, x, op, "y"))))
    return rc;
  if (!(post_eps >= 0.f) || !(eps >= 0.f))
    return fail(L3D_E_UNSUPPORTED, "%s: eps must not be negative", op);
  Params p{};
  p.C = x->dims[x->ndim - 1];
  p.rows = 1;
  for (int i = 0; i < x->ndim - 1; ++i) p.rows *= x->dims[i];
  if (p.C <= 0) return fail(L3D_E_SHAPE, "%s: empty rows (C = 0)", op);
  if (p.C > kMaxC)
    return fail(L3D_E_UNSUPPORTED, "%s: row length %lld exceeds %lld", op, (long long)p.C,
                (long long)kMaxC);
  const int64_t B = x->ndim >= 3 ? x->dims[0] : 1;
  bool al = true;
  if ((rc = make_chanvec(post_weight, "post_weight", p.C, 1, &p.pw, &al)) ||
      (rc = make_chanvec(post_bias, "post_bias", p.C, 1, &p.pb, &al)) ||
      (rc = make_chanvec(gate, "gate", p.C, B, &p.gate, &al)) ||
      (rc = make_chanvec(weight, "weight", p.C, 1, &p.w, &al)) ||
      (rc = make_chanvec(bias, "bias", p.C, 1, &p.b, &al)) ||
      (rc = make_chanvec(shift, "shift", p.C, B, &p.shift, &al)) ||
      (rc = make_chanvec(scale, "scale", p.C, B, &p.scale, &al)))
    return rc;
  const int lead = x->ndim - 1;
  if (!make_rowmap(x, lead, &p.xm) || !make_rowmap(h, lead, &p.hm) ||
      !make_rowmap(r_out, lead, &p.rm) || (y && !make_rowmap(y, lead, &p.ym)))
    return fail(L3D_E_UNSUPPORTED, "%s: more than 5 non-collapsible leading dims", op);
  if (p.rows == 0) return L3D_OK;
  p.rows_per_batch = p.rows / B;
  p.x = x->data;
  p.h = h->data;
  p.r = r_out->data;
  p.y = y ? y->data : nullptr;
  p.res_scale = res_scale;
  p.post_eps = post_eps;
  p.eps = eps;
  p.norm = norm;
  // 16-byte vectors where every row of every activation is so aligned.
  const int vec = 16 / dtype_size(x->dtype);
  auto rows_ok = [&](const l3d_tensor* t, const RowMap& m) {
    return !t || (reinterpret_cast<uintptr_t>(t->data) % 16 == 0 && rowmap_aligned(m, vec));
  };
  const bool vec_ok = p.C % vec == 0 && rows_ok(x, p.xm) && rows_ok(h, p.hm) && rows_ok(r_out, p.rm) &&
                      rows_ok(y, p.ym);
  const bool per_batch = p.gate.bstride || p.shift.bstride || p.scale.bstride;
  const int64_t batches = per_batch ? B : 1;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  L3D_DISPATCH_FLOAT(x->dtype, T, {
    rc = launch<T>(p, vec_ok, al, batches, s);
  });
  return rc ? rc : check_launch(op);
}
