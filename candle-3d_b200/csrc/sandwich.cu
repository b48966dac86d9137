// Block seam with a norm on either side of the residual (a "sandwich" norm):
//   n = Norm(h) [* post_weight] [+ post_bias]
//   r = res_scale * x + [gate *] n
//   y = Norm(r) [* weight] [+ bias] [* (1 + scale) + shift]
// Norm: RMS, v / sqrt(mean(v^2) + eps), or Layer, (v - mean) / sqrt(var + eps).
// The reference composes such seams from its norms and residual adds
// (crate/runtime/trellis2_blocks.rs:280-286,627-645, crate/runtime/vggt.rs:104-123);
// here x and h are read once and r and y written once.
#include "common.cuh"

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
};

constexpr int kBlock = 256;

__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) red[warp] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kBlock / 32; ++i) s += red[i];
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
template <int NORM>
__device__ __forceinline__ void block_stats(const float* s, int64_t C, float eps, float* red,
                                            float& mean, float& inv) {
  mean = 0.f;
  if constexpr (NORM == NORM_LAYER) {
    float a = 0.f;
    for (int64_t c = threadIdx.x; c < C; c += kBlock) a += s[c];
    mean = block_sum(a, red) / float(C);
  }
  float q = 0.f;
  for (int64_t c = threadIdx.x; c < C; c += kBlock) {
    const float d = s[c] - mean;
    q = fmaf(d, d, q);
  }
  inv = 1.f / sqrtf(block_sum(q, red) / float(C) + eps);
}

// One row per block at a time, the row held in shared memory as f32; any
// row length, alignment and strides.
template <typename T, int NORM>
__global__ void __launch_bounds__(kBlock) row_kernel(const Params p) {
  extern __shared__ float s[];
  __shared__ float red[kBlock / 32];
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const int64_t b = row / p.rows_per_batch;
    const T* xr = static_cast<const T*>(p.x) + row_offset(p.xm, row);
    const T* hr = static_cast<const T*>(p.h) + row_offset(p.hm, row);
    for (int64_t c = threadIdx.x; c < p.C; c += kBlock) s[c] = to_f(hr[c]);
    __syncthreads();
    float mean, inv;
    block_stats<NORM>(s, p.C, p.post_eps, red, mean, inv);
    T* rr = static_cast<T*>(p.r) + row_offset(p.rm, row);
    for (int64_t c = threadIdx.x; c < p.C; c += kBlock) {
      const float n = (s[c] - mean) * inv * chan_or(p.pw, 0, c, 1.f) + chan_or(p.pb, 0, c, 0.f);
      const float r = fmaf(chan_or(p.gate, b, c, 1.f), n, p.res_scale * to_f(xr[c]));
      rr[c] = from_f<T>(r);
      s[c] = r;
    }
    __syncthreads();
    if (p.y) {
      block_stats<NORM>(s, p.C, p.eps, red, mean, inv);
      T* yr = static_cast<T*>(p.y) + row_offset(p.ym, row);
      for (int64_t c = threadIdx.x; c < p.C; c += kBlock) {
        const float n = (s[c] - mean) * inv * chan_or(p.w, 0, c, 1.f) + chan_or(p.b, 0, c, 0.f);
        yr[c] = from_f<T>(fmaf(n, 1.f + chan_or(p.scale, b, c, 0.f), chan_or(p.shift, b, c, 0.f)));
      }
      __syncthreads();
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

template <typename T, int NORM>
static int launch(const Params& p, cudaStream_t s) {
  auto k = row_kernel<T, NORM>;
  if (set_smem_limit(reinterpret_cast<const void*>(k), int(kMaxC * 4)) != cudaSuccess)
    return fail(L3D_E_CUDA, "l3d_sandwich_residual_norm: cannot reserve shared memory");
  const int64_t cap = int64_t(sm_count()) * 8;
  k<<<unsigned(p.rows < cap ? p.rows : cap), kBlock, size_t(p.C) * 4, s>>>(p);
  return L3D_OK;
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
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  L3D_DISPATCH_FLOAT(x->dtype, T, {
    rc = norm == NORM_LAYER ? launch<T, NORM_LAYER>(p, s) : launch<T, NORM_RMS>(p, s);
  });
  return rc ? rc : check_launch(op);
}
