// Shared projection with low-rank adapters of many requests:
//   y[m] = [residual +] [gate *] act( W x[m] + bias + scale_a B_a (A_a x[m]) ),  a = ids(m)
// (rows whose id is outside [0, adapters) take the projection alone).  The
// projection is the reference's Linear::forward / ops::mul_mat_add
// (crate/runtime/nn_blocks.rs:82,179-195) with the element-wise ops of its
// blocks; the adapters have no counterpart there.
#include "act.cuh"
#include "common.cuh"

namespace l3d {
namespace lora {

struct Params {
  int M, N, K, R, A;
  const __nv_bfloat16 *x, *w, *a, *b;
  int64_t x_ld, w_ld, y_ld, res_ld;
  const float* scale;     // [A]
  const int32_t* ranks;   // [A] or null (= R)
  const void* ids;        // row m has id ids[m / per]
  int ids64, per;
  const void* bias;
  int bias_dtype;
  const void* gate;
  int gate_dtype;
  const void* res;
  void* y;
  int y_dtype, act;
  float* t;               // [M, R] scale_a A_a x[m]
};

__device__ __forceinline__ int adapter_of(const Params& p, int m) {
  const int g = m / p.per;
  const int64_t id = p.ids64 ? static_cast<const int64_t*>(p.ids)[g] : static_cast<const int32_t*>(p.ids)[g];
  return id >= 0 && id < p.A ? int(id) : -1;
}
__device__ __forceinline__ float vec_at(const void* v, int dtype, int i) {
  return dtype == L3D_F32 ? static_cast<const float*>(v)[i]
                          : __bfloat162float(static_cast<const __nv_bfloat16*>(v)[i]);
}

// One row per block, one rank per warp at a time.
__global__ void __launch_bounds__(256) shrink_kernel(const Params p) {
  const int m = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int a = adapter_of(p, m);
  const int rank = a < 0 ? 0 : p.ranks ? min(max(p.ranks[a], 0), p.R) : p.R;
  const __nv_bfloat16* xr = p.x + int64_t(m) * p.x_ld;
  for (int r = warp; r < p.R; r += 8) {
    float acc = 0.f;
    if (r < rank) {
      const __nv_bfloat16* ar = p.a + (int64_t(a) * p.R + r) * p.K;
      for (int k = lane; k < p.K; k += 32) acc = fmaf(to_f(xr[k]), to_f(ar[k]), acc);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if (lane == 0) p.t[int64_t(m) * p.R + r] = r < rank ? acc * p.scale[a] : 0.f;
  }
}

// 16 rows x 16 columns per block.
__global__ void __launch_bounds__(256) expand_kernel(const Params p) {
  __shared__ float sx[16][17], sw[16][17];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int m = blockIdx.y * 16 + ty, n = blockIdx.x * 16 + tx, nl = blockIdx.x * 16 + ty;
  float acc = 0.f;
  for (int k0 = 0; k0 < p.K; k0 += 16) {
    const int k = k0 + tx;
    sx[ty][tx] = m < p.M && k < p.K ? to_f(p.x[int64_t(m) * p.x_ld + k]) : 0.f;
    sw[ty][tx] = nl < p.N && k < p.K ? to_f(p.w[int64_t(nl) * p.w_ld + k]) : 0.f;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; ++i) acc = fmaf(sx[ty][i], sw[tx][i], acc);
    __syncthreads();
  }
  if (m >= p.M || n >= p.N) return;
  const int a = adapter_of(p, m);
  if (a >= 0) {
    const __nv_bfloat16* br = p.b + (int64_t(a) * p.N + n) * p.R;
    for (int r = 0; r < p.R; ++r) acc = fmaf(p.t[int64_t(m) * p.R + r], to_f(br[r]), acc);
  }
  if (p.bias) acc += vec_at(p.bias, p.bias_dtype, n);
  acc = act_dyn(p.act, acc);
  if (p.res) acc = fmaf(p.gate ? vec_at(p.gate, p.gate_dtype, n) : 1.f, acc,
                        (p.y_dtype == L3D_F32
                            ? static_cast<const float*>(p.res)[int64_t(m) * p.res_ld + n]
                            : to_f(static_cast<const __nv_bfloat16*>(p.res)[int64_t(m) * p.res_ld + n])));
  if (p.y_dtype == L3D_F32) static_cast<float*>(p.y)[int64_t(m) * p.y_ld + n] = acc;
  else static_cast<__nv_bfloat16*>(p.y)[int64_t(m) * p.y_ld + n] = __float2bfloat16_rn(acc);
}

}  // namespace lora
}  // namespace l3d

using namespace l3d;

extern "C" size_t l3d_lora_linear_workspace_size(int64_t m, int64_t r) {
  if (m < 0 || r < 0) return 0;
  return size_t(m) * size_t(r) * 4 + 256;
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
  p.w = reinterpret_cast<const __nv_bfloat16*>(elem_ptr(weight));
  p.a = reinterpret_cast<const __nv_bfloat16*>(elem_ptr(lora_a));
  p.b = reinterpret_cast<const __nv_bfloat16*>(elem_ptr(lora_b));
  p.x_ld = x_ld; p.w_ld = w_ld; p.y_ld = y_ld; p.res_ld = res_ld;
  p.scale = reinterpret_cast<const float*>(elem_ptr(lora_scale));
  p.ranks = ranks ? reinterpret_cast<const int32_t*>(elem_ptr(ranks)) : nullptr;
  p.ids = elem_ptr(ids);
  p.ids64 = ids->dtype == L3D_I64;
  p.per = int(M / ids->dims[0]);
  p.bias = bias ? elem_ptr(bias) : nullptr;
  p.bias_dtype = bias ? bias->dtype : L3D_F32;
  p.gate = gate ? elem_ptr(gate) : nullptr;
  p.gate_dtype = gate ? gate->dtype : L3D_F32;
  p.res = residual ? elem_ptr(residual) : nullptr;
  p.y = const_cast<char*>(elem_ptr(y));
  p.y_dtype = y->dtype;
  p.act = act;
  p.t = static_cast<float*>(workspace);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  shrink_kernel<<<unsigned(M), 256, 0, s>>>(p);
  expand_kernel<<<dim3(unsigned((n + 15) / 16), unsigned((M + 15) / 16)), 256, 0, s>>>(p);
  return check_launch(op);
}
