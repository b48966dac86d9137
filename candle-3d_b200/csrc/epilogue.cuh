// The fused epilogue of the GEMM kernels, y = res + gate * act(acc + bias), on
// accumulator columns held by one thread.  Params names M, N, bias, bias_dtype,
// bias_vec (16-byte aligned), act, y_dtype, res, res_ld, res_vec (16-byte
// aligned rows), gate and gate_dtype.
#pragma once
#include "act.cuh"
#include "common.cuh"

namespace l3d {
namespace gemm {

// The fused epilogue ops on NC consecutive columns [col0, col0 + NC) of one
// row, after the bias: the activation (the reduced-cost forms for 16-bit
// outputs), then the gated residual, 8 columns at a time.  Columns past N are
// left alone.
template <int A, bool FAST, int NC>
__device__ __forceinline__ void act_chunk(float (&v)[NC]) {
#pragma unroll
  for (int i = 0; i < NC; ++i) v[i] = act_t<A, FAST>(v[i]);
}
// One dispatch per chunk, so each variant's loop is contiguous code.  REL: the
// tanh GELU is accurate relative to its value (gelu_tanh_rel).
template <int NC, bool REL = false>
__device__ __forceinline__ void epi_act(int act, bool fast, float (&v)[NC]) {
  if (fast) {
    switch (act) {
      case ACT_SILU: act_chunk<ACT_SILU, true>(v); break;
      case ACT_GELU_ERF: act_chunk<ACT_GELU_ERF, true>(v); break;
      case ACT_GELU_TANH:
        if constexpr (REL) {
#pragma unroll
          for (int i = 0; i < NC; ++i) v[i] = gelu_tanh_rel(v[i]);
        } else {
          act_chunk<ACT_GELU_TANH, true>(v);
        }
        break;
      default: break;
    }
  } else {
    switch (act) {
      case ACT_SILU: act_chunk<ACT_SILU, false>(v); break;
      case ACT_GELU_ERF: act_chunk<ACT_GELU_ERF, false>(v); break;
      case ACT_GELU_TANH: act_chunk<ACT_GELU_TANH, false>(v); break;
      default: break;
    }
  }
}

template <int NC, typename Params>
__device__ __forceinline__ void epi_post(const Params& p, int row, int col0, float (&v)[NC]) {
  if (p.act) epi_act<NC>(p.act, p.y_dtype != L3D_F32, v);
  if (!p.res || row >= p.M) return;
  const bool bf = p.y_dtype == L3D_BF16;
  const char* rrow = static_cast<const char*>(p.res) + (int64_t(row) * p.res_ld + col0) * (bf ? 2 : 4);
#pragma unroll
  for (int q = 0; q < NC / 8; ++q) {
    const int c = col0 + 8 * q;
    if (c >= p.N) break;
    float r[8], g[8];
    if (c + 8 <= p.N && p.res_vec) {
      if (bf) {
        unpack(__ldg(reinterpret_cast<const uint4*>(rrow) + q), r, __nv_bfloat16());
      } else {
        const float4 a = __ldg(reinterpret_cast<const float4*>(rrow) + 2 * q);
        const float4 b = __ldg(reinterpret_cast<const float4*>(rrow) + 2 * q + 1);
        r[0] = a.x; r[1] = a.y; r[2] = a.z; r[3] = a.w; r[4] = b.x; r[5] = b.y; r[6] = b.z; r[7] = b.w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int i = c + e < p.N ? 8 * q + e : 8 * q;  // clamp to a valid column
        r[e] = bf ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(rrow)[i])
                  : __ldg(reinterpret_cast<const float*>(rrow) + i);
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int col = c + e < p.N ? c + e : p.N - 1;
      g[e] = !p.gate ? 1.f
             : p.gate_dtype == L3D_F32 ? __ldg(static_cast<const float*>(p.gate) + col)
                                       : __bfloat162float(static_cast<const __nv_bfloat16*>(p.gate)[col]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < p.N) v[8 * q + e] = fmaf(g[e], v[8 * q + e], r[e]);
  }
}

// v[i] += bias[col0 + i] for NC columns: 16-byte loads through the read-only
// path when the chunk lies inside N and the bias is 16-byte aligned (f32 or
// bf16), else one element at a time (columns past N are left alone).
template <int NC, typename Params>
__device__ __forceinline__ void add_bias(const Params& p, int col0, float (&v)[NC]) {
  if (col0 + NC <= p.N && p.bias_vec) {
    if (p.bias_dtype == L3D_F32) {
      const float4* b4 = reinterpret_cast<const float4*>(static_cast<const float*>(p.bias) + col0);
#pragma unroll
      for (int q = 0; q < NC / 4; ++q) {
        const float4 t = __ldg(b4 + q);
        v[4 * q] += t.x; v[4 * q + 1] += t.y; v[4 * q + 2] += t.z; v[4 * q + 3] += t.w;
      }
    } else {
      const uint4* b8 = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.bias) + col0);
#pragma unroll
      for (int q = 0; q < NC / 8; ++q) {
        const uint4 t = __ldg(b8 + q);
        const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[8 * q + 2 * e] += __uint_as_float(w[e] << 16);
          v[8 * q + 2 * e + 1] += __uint_as_float(w[e] & 0xffff0000u);
        }
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int col = col0 + i;
    if (col < p.N)
      v[i] += p.bias_dtype == L3D_F32
                  ? __ldg(static_cast<const float*>(p.bias) + col)
                  : __uint_as_float(uint32_t(__ldg(static_cast<const unsigned short*>(p.bias) + col)) << 16);
  }
}

// v[i] *= gate[col0 + i] for NC columns inside N: 16-byte loads where the gate
// is so aligned.
template <int NC, typename Params>
__device__ __forceinline__ void mul_gate(const Params& p, int col0, float (&v)[NC]) {
  const bool al = (reinterpret_cast<uintptr_t>(p.gate) & 15) == 0;
  if (p.gate_dtype == L3D_F32) {
    const float* g = static_cast<const float*>(p.gate) + col0;
#pragma unroll
    for (int q = 0; q < NC / 4; ++q) {
      const float4 t = al ? __ldg(reinterpret_cast<const float4*>(g) + q)
                          : make_float4(g[4 * q], g[4 * q + 1], g[4 * q + 2], g[4 * q + 3]);
      v[4 * q] *= t.x; v[4 * q + 1] *= t.y; v[4 * q + 2] *= t.z; v[4 * q + 3] *= t.w;
    }
  } else {
    const __nv_bfloat16* g = static_cast<const __nv_bfloat16*>(p.gate) + col0;
#pragma unroll
    for (int q = 0; q < NC / 8; ++q) {
      float t[8];
      if (al) {
        unpack(__ldg(reinterpret_cast<const uint4*>(g) + q), t, __nv_bfloat16());
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = __bfloat162float(g[8 * q + e]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) v[8 * q + e] *= t[e];
    }
  }
}

}  // namespace gemm
}  // namespace l3d
