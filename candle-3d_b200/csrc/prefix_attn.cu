// Attention for a batch whose elements share a prefix of keys, plus each
// element's own keys:
//   out[b, h, i] = sum_j softmax_j(scale q[b, h, i] . K[j]) V[j]
// over the prefix keys j < P (one copy for the whole batch) and the own keys
// j < lengths[b] of element b; with `causal`, row i sees the own keys up to
// its own place, j <= lengths[b] - N + i.  Query heads h share the key head
// h / (Hq / Hkv).  The reference's attention core is exact_sdpa_heads
// (crate/runtime/attention_math.rs:199-259); a shared prefix would be copied
// into every batch element there.
#include "common.cuh"

namespace l3d {
namespace pattn {

struct Params {
  int B, Hq, Hkv, N, D;
  int64_t P, S;
  const void *q, *pk, *pv, *k, *v;
  void* out;
  int64_t qb, qh, qn, pkh, pkn, pvh, pvn, kb, kh, kn, vb, vh, vn, ob, oh, on;  // element strides
  const void* lengths;  // [B] or null (= S)
  int len64, causal;
  float scale;
};

// One query row per warp, keys one at a time, the head dim over the lanes.
template <typename T>
__global__ void __launch_bounds__(128) row_kernel(const Params p) {
  const int lane = threadIdx.x & 31, E = p.D / 32;
  const int64_t row = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (row >= int64_t(p.B) * p.Hq * p.N) return;
  const int64_t i = row % p.N, h = row / p.N % p.Hq, b = row / p.N / p.Hq;
  const int64_t kvh = h / (p.Hq / p.Hkv);
  const T* qr = static_cast<const T*>(p.q) + b * p.qb + h * p.qh + i * p.qn;
  float q[4], o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int e = 0; e < E; ++e) q[e] = to_f(qr[lane + 32 * e]) * p.scale;
  float m = -INFINITY, l = 0.f;
  auto key = [&](const T* kr, const T* vr) {
    float s = 0.f;
    for (int e = 0; e < E; ++e) s = fmaf(q[e], to_f(kr[lane + 32 * e]), s);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    const float mn = fmaxf(m, s);
    const float alpha = mn == -INFINITY ? 1.f : expf(m - mn);
    const float pr = mn == -INFINITY ? 0.f : expf(s - mn);
    l = l * alpha + pr;
    for (int e = 0; e < E; ++e) o[e] = o[e] * alpha + pr * to_f(vr[lane + 32 * e]);
    m = mn;
  };
  for (int64_t j = 0; j < p.P; ++j)
    key(static_cast<const T*>(p.pk) + kvh * p.pkh + j * p.pkn,
        static_cast<const T*>(p.pv) + kvh * p.pvh + j * p.pvn);
  int64_t len = p.S;
  if (p.lengths) {
    const int64_t v = p.len64 ? static_cast<const int64_t*>(p.lengths)[b] : static_cast<const int32_t*>(p.lengths)[b];
    len = v < 0 ? 0 : v < p.S ? v : p.S;
  }
  if (p.causal && len - p.N + i + 1 < len) len = len - p.N + i + 1;
  for (int64_t j = 0; j < len; ++j)
    key(static_cast<const T*>(p.k) + b * p.kb + kvh * p.kh + j * p.kn,
        static_cast<const T*>(p.v) + b * p.vb + kvh * p.vh + j * p.vn);
  T* orow = static_cast<T*>(p.out) + b * p.ob + h * p.oh + i * p.on;
  for (int e = 0; e < E; ++e) orow[lane + 32 * e] = from_f<T>(l != 0.f ? o[e] / l : 0.f);
}

}  // namespace pattn
}  // namespace l3d

using namespace l3d;

extern "C" size_t l3d_shared_prefix_attention_workspace_size(int64_t b, int64_t hq, int64_t hkv,
                                                             int64_t n, int64_t p, int64_t s,
                                                             int64_t d) {
  (void)b; (void)hq; (void)hkv; (void)n; (void)p; (void)s; (void)d;
  return 0;
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
    if (t->strides[nd - 1] != 1) return fail(L3D_E_ALIGN, "%s: the head dim must be contiguous", op);
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
  if (!(scale > 0.f) || !(scale < 3.0e38f))
    return fail(L3D_E_UNSUPPORTED, "%s: scale must be positive and finite", op);
  const int64_t big = int64_t(1) << 30;
  if (B > 65535 || Hq > 65535 || N > big || P > big || S > big || B * Hq * N > big)
    return fail(L3D_E_UNSUPPORTED, "%s: dimensions too large", op);
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
  Params p{};
  p.B = int(B); p.Hq = int(Hq); p.Hkv = int(Hkv); p.N = int(N); p.D = int(D);
  p.P = P; p.S = S;
  p.q = elem_ptr(q); p.pk = elem_ptr(prefix_k); p.pv = elem_ptr(prefix_v);
  p.k = k ? elem_ptr(k) : nullptr; p.v = v ? elem_ptr(v) : nullptr;
  p.out = const_cast<char*>(elem_ptr(out));
  p.qb = q->strides[0]; p.qh = q->strides[1]; p.qn = q->strides[2];
  p.ob = out->strides[0]; p.oh = out->strides[1]; p.on = out->strides[2];
  p.pkh = prefix_k->strides[0]; p.pkn = prefix_k->strides[1];
  p.pvh = prefix_v->strides[0]; p.pvn = prefix_v->strides[1];
  if (k) {
    p.kb = k->strides[0]; p.kh = k->strides[1]; p.kn = k->strides[2];
    p.vb = v->strides[0]; p.vh = v->strides[1]; p.vn = v->strides[2];
  }
  p.lengths = lengths ? elem_ptr(lengths) : nullptr;
  p.len64 = lengths && lengths->dtype == L3D_I64;
  p.causal = causal != 0;
  p.scale = scale;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const unsigned grid = unsigned((B * Hq * N + 3) / 4);
  if (q->dtype == L3D_BF16) row_kernel<__nv_bfloat16><<<grid, 128, 0, s>>>(p);
  else row_kernel<__half><<<grid, 128, 0, s>>>(p);
  return check_launch(op);
}
