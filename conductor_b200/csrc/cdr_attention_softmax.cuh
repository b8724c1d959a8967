// Softmax arithmetic of the tensor-memory attention kernels (cdr_attention.cu, cdr_tile_attention.cu): one
// query row per thread, scores read from and weights written to tensor memory.
#pragma once

#include <math.h>

#include "cdr_common.cuh"
#include "cdr_sm100.cuh"

namespace cdr {

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

#ifndef CDR_ATT_EMU
#define CDR_ATT_EMU 0   // pairs of every 8 whose exp2 runs on the FMA pipes (0: measured best on this kernel)
#endif

// ---- two fp32 lanes per instruction (fma/add/sub .f32x2) and the three-input max of sm_100
__device__ __forceinline__ uint64_t pack2(float a, float b) { uint64_t r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) { uint64_t d; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c)); return d; }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) { uint64_t d; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b)); return d; }
__device__ __forceinline__ uint64_t sub2(uint64_t a, uint64_t b) { uint64_t d; asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b)); return d; }
__device__ __forceinline__ float max3(float a, float b, float c) { float d; asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c)); return d; }

// 2^x for a pair on the FMA pipes instead of the special-function unit: x = n + f with n the
// nearest integer (magic-number rounding) and f in [-0.5, 0.5]; 2^f by a cubic (max relative error
// 7.5e-5, far inside the 2^-9 of the 16-bit P it feeds); n goes straight into the exponent field.
// Inputs are clamped to -125 so the exponent cannot wrap.
__device__ __forceinline__ void poly_exp2_pair(uint64_t x, float& p0, float& p1) {
  float x0, x1;
  unpack2(x, x0, x1);
  x = pack2(fmaxf(x0, -125.0f), fmaxf(x1, -125.0f));
  const uint64_t magic = pack2(12582912.0f, 12582912.0f);
  const uint64_t t = add2(x, magic);
  const uint64_t f = sub2(x, sub2(t, magic));
  uint64_t r = fma2(pack2(0.055171459913253784f, 0.055171459913253784f), f, pack2(0.2426108568906784f, 0.2426108568906784f));
  r = fma2(r, f, pack2(0.6932609677314758f, 0.6932609677314758f));
  r = fma2(r, f, pack2(0.9999281167984009f, 0.9999281167984009f));
  float t0, t1, r0, r1;
  unpack2(t, t0, t1);
  unpack2(r, r0, r1);
  p0 = __uint_as_float(__float_as_uint(r0) + (__float_as_uint(t0) << 23));
  p1 = __uint_as_float(__float_as_uint(r1) + (__float_as_uint(t1) << 23));
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack_pair(float a, float b) {
  if (BF16) { __nv_bfloat162 t = __floats2bfloat162_rn(a, b); return *reinterpret_cast<uint32_t*>(&t); }
  __half2 t = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&t);
}

// P = exp2(s*c - m) for one row's 128 scores, packed to 16-bit pairs and stored over the S columns the
// row just read (`p_taddr`); row sums accumulate in two fp32 lanes.  EMU of every 8 pairs take the polynomial path,
// the rest the special-function unit.
// With WITH_MAX the maximum of the raw scores is accumulated alongside (four independent chains) and returned.
template <bool BF16, int EMU, bool WITH_MAX>
__device__ __forceinline__ float store_p(uint32_t (&sr)[4][32], float scale_log2, float neg_m, float& l0, float& l1, uint32_t p_taddr) {
  const uint64_t scale2 = pack2(scale_log2, scale_log2), negm2 = pack2(neg_m, neg_m);
  uint64_t lsum4[4] = {pack2(l0, l1), pack2(0.0f, 0.0f), pack2(0.0f, 0.0f), pack2(0.0f, 0.0f)};   // independent chains
  float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t pw[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float p0, p1;
      const uint64_t x = fma2(pack2(__uint_as_float(sr[c][2 * i]), __uint_as_float(sr[c][2 * i + 1])), scale2, negm2);
      if (WITH_MAX) mx[i & 1] = max3(mx[i & 1], __uint_as_float(sr[c][2 * i]), __uint_as_float(sr[c][2 * i + 1]));
      if ((i & 7) < EMU) {
        poly_exp2_pair(x, p0, p1);
      } else {
        float x0, x1;
        unpack2(x, x0, x1);
        p0 = fast_exp2(x0);
        p1 = fast_exp2(x1);
      }
      lsum4[i & 3] = add2(lsum4[i & 3], pack2(p0, p1));
      pw[i] = pack_pair<BF16>(p0, p1);
    }
    sm100::tmem_st16(p_taddr + c * 16, pw);
  }
  unpack2(add2(add2(lsum4[0], lsum4[1]), add2(lsum4[2], lsum4[3])), l0, l1);
  return fmaxf(mx[0], mx[1]);
}

}  // namespace cdr
