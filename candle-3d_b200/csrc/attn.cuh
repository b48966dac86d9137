// Pieces shared by the attention kernels (attn.cu, prefix_attn.cu, cross_attn.cu, decode_attn.cu): 4-D TMA
// tile loads and maps, the MN-major V operand, P read from tensor memory, wide
// TMEM accesses and the exponentials.
#pragma once
#include <type_traits>

#include "common.cuh"
#include "tc.cuh"

namespace l3d {
namespace attn {

using namespace l3d::tc;

// exp2 on the FMA pipe, for part of the elements, so that the MUFU unit (16
// exp2 per clock per SM) is not the only one doing them: Cody-Waite style
// range reduction x = j + f with j = round(x) (the 1.5 * 2^23 shifter) and f
// in [-1/2, 1/2], 2^f by a degree-3 minimax polynomial (Remez fit made for
// this kernel, relative error 7.5e-5, far below the bf16 rounding of P), and
// 2^j added to the exponent field.  x is clamped just above -127, where q > 1 and
// the exponent field comes to 0: what is left, 1e-42, is 0 in either 16-bit type,
// as a masked key's probability has to be (2^-126 would add 4 to an output where
// its V is at the end of bf16's range).  The inputs here are <= 8 (the rescale
// threshold), or 15 where f16 probabilities are held higher.  A NaN is clamped
// too: the running maximum carries it past this function (max_nan).
constexpr float EX2_C0 = 0.99992806f, EX2_C1 = 0.69326097f, EX2_C2 = 0.24261113f,
                EX2_C3 = 0.05517167f, EX2_MIN = -127.f + 0x1p-12f;
__device__ __forceinline__ float2 ex2_poly2(float2 x) {
  x = make_float2(fmaxf(x.x, EX2_MIN), fmaxf(x.y, EX2_MIN));
  const float2 t = add2(x, f2(12582912.f));          // low mantissa bits = round(x)
  const float2 r = add2(t, f2(-12582912.f));
  const float2 f = add2(x, make_float2(-r.x, -r.y));
  float2 q = fma2(f, f2(EX2_C3), f2(EX2_C2));
  q = fma2(q, f, f2(EX2_C1));
  q = fma2(q, f, f2(EX2_C0));
  return make_float2(__int_as_float(__float_as_int(q.x) + (__float_as_int(t.x) << 23)),
                     __int_as_float(__float_as_int(q.y) + (__float_as_int(t.y) << 23)));
}

// A score that is NaN or +inf has no softmax: its row is NaN, wherever in a tile
// the score lies.  The running maximum m carries it: the largest of the scores, NaN
// where one is (fmaxf drops it), moves m where !(largest <= m + threshold), and the
// rescaling spoils all that was summed before.  An infinite m becomes NaN either
// in what is added to the scaled scores (minus_max, where m can be -inf for a row
// that has seen no key) or in the row's sum (m * 0, off the path to the exponentials:
// 16 heads x 10992 x 10992, D 64: 0.9% in attn.cu).
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ float minus_max(float m) { return fmaf(m, 0.f, -m); }

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar,
                                            int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2),
      "r"(c3)
      : "memory");
}

// MN-major, 128B-swizzled operand tile (B = V: N = D contiguous in rows of 128
// B, one row per K index): 8-row K groups 1024 B apart (SBO), 64-wide N blocks
// `lbo` bytes apart (LBO).
__device__ __forceinline__ uint64_t smem_desc_sw128_mn(const void* tile, uint32_t lbo) {
  const uint64_t addr = smem_u32(tile);
  uint64_t d = 0;
  d |= (addr >> 4) & 0x3fffull;
  d |= uint64_t((lbo >> 4) & 0x3fff) << 16;
  d |= uint64_t(1024 >> 4) << 32;
  d |= uint64_t(1) << 46;
  d |= uint64_t(2) << 61;
  return d;
}

// D[tmem] (+)= A[tmem] * B[smem]^T: A (M 128 x K 16, bf16 pairs packed in 32-bit
// columns, rows = TMEM lanes) from tensor memory, B from a shared-memory
// descriptor.
template <uint32_t IDESC_>
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t db,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(db), "r"(IDESC_), "r"(accumulate));
}

// 64 consecutive f32 TMEM columns of this thread's lane -> registers; the
// wait is inside the same statement, so no use can move above it.
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, float* v) {
  uint32_t r[64];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, "
      "%28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, "
      "%45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, "
      "%62, %63}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
        "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
        "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]),
        "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]),
        "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]),
        "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]),
        "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]),
        "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(r[i]);
}

// 32 consecutive 32-bit TMEM columns of this thread's lane <- registers.
__device__ __forceinline__ void tmem_st32u(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, "
      "%28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]),
      "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]),
      "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]),
      "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}

__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two floats -> packed bf16 pair (lo = a, the lower K index).
__device__ __forceinline__ uint32_t pack_bf16x2(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
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

// 4-D bf16 view [B, H, rows, cols] (cols contiguous) as a TMA map with a box
// of 64 columns x box_rows rows, 128B swizzle.  The map's dimensions are
// ordered by stride: (cols, rows, H, B), or (cols, H, rows, B) when heads are
// closer in memory than rows (*hn = 1; the kernel swaps those coordinates).
// Strides of size-1 dimensions are replaced by packed ones.
inline bool make_map4(CUtensorMap* m, const void* base, int64_t B, int64_t H, int64_t rows,
                      int64_t cols, int64_t s_row, int64_t s_h, int64_t s_b, uint32_t box_rows,
                      int* hn) {
  auto fn = encode_fn();
  if (!fn) return false;
  if (rows <= 1) s_row = cols;
  if (H <= 1) s_h = s_row * rows;
  if (B <= 1) s_b = (s_h > s_row ? s_h * H : s_row * rows);
  *hn = s_h < s_row ? 1 : 0;
  const cuuint64_t dims[4] = {uint64_t(cols), uint64_t(*hn ? H : rows), uint64_t(*hn ? rows : H),
                              uint64_t(B)};
  const cuuint64_t strides[3] = {uint64_t(*hn ? s_h : s_row) * 2, uint64_t(*hn ? s_row : s_h) * 2,
                                 uint64_t(s_b) * 2};
  const cuuint32_t box[4] = {64u, *hn ? 1u : box_rows, *hn ? box_rows : 1u, 1u};
  const cuuint32_t es[4] = {1, 1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box,
            es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace attn
}  // namespace l3d
