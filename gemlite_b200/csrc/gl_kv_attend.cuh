// What the two attention kernels over the quantised cache share: parameters, exact conversion of codes to fp16, output.
#pragma once
#include "gl_kv.cuh"

struct KvAttendParams {
  KvBatch kb;
  const uint8_t *k_codes, *v_codes, *k_zeros, *v_zeros;
  const float *k_scales, *v_scales;
  const void* q;
  void* out;
  const uint8_t* mask;
  float* part_o;               // [splits][n_tokens * hq][D], unnormalised
  float2* part_ml;             // [splits][n_tokens * hq]: maximum and sum (0: nothing seen)
  int64_t q_sn, q_sh, mask_stride;
  int32_t mask_cols, hq, group, splits, chunk, page_shift;
  float scale_log2;
};

template <typename T> struct IsHalf { static constexpr bool value = false; };
template <> struct IsHalf<__half> { static constexpr bool value = true; };

#ifdef __CUDACC__
// Tokens per split of a sequence: the launch's, or more where the sequence is longer than the host's bound said.
__device__ __forceinline__ int kv_attend_chunk(const KvAttendParams& p, int len) {
  const int need = (len + p.splits - 1) / p.splits;
  return max(p.chunk, (need + 127) / 128 * 128);
}
__device__ __forceinline__ float kv_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// four 8-bit codes -> two fp16 pairs (bytes 0, 1 and 2, 3), exactly
template <int FMT> __device__ __forceinline__ void kv_bytes(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (FMT == GL_KV_FP8) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
  } else {
    // byte + 128 in the low bits of fp16 1024: 1152 + code
    const uint32_t u = w ^ 0x80808080u;
    const __half2 bias = __half2half2(__ushort_as_half(0x6480));
    uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), bias), y = __hsub2(*reinterpret_cast<__half2*>(&b), bias);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  }
}
// bits 0..3 and 16..19 -> the fp16 pair (code - zero); `zero` holds fp16 1024 + zero twice
__device__ __forceinline__ uint32_t kv_nibbles(uint32_t w, uint32_t zero) {
  uint32_t u = (w & 0x000f000fu) | 0x64006400u;
  const __half2 x = __hsub2(*reinterpret_cast<__half2*>(&u), *reinterpret_cast<__half2*>(&zero));
  return *reinterpret_cast<const uint32_t*>(&x);
}
// a / l, rounded once to 16 bits; a row that saw nothing (l = 0) gives zeros
template <typename T> __device__ __forceinline__ void kv_store4(T* dst, float4 a, float l) {
  const float r = l == 0.f ? 0.f : 1.f / l;
  uint32_t lo, hi;
  if constexpr (IsHalf<T>::value) {
    const __half2 x = __floats2half2_rn(a.x * r, a.y * r), y = __floats2half2_rn(a.z * r, a.w * r);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  } else {
    const __nv_bfloat162 x = __floats2bfloat162_rn(a.x * r, a.y * r), y = __floats2bfloat162_rn(a.z * r, a.w * r);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  }
  *reinterpret_cast<uint2*>(dst) = make_uint2(lo, hi);
}
#endif
