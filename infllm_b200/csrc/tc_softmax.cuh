// What the tensor-core kernels' softmax warps and waits are made of: bounded waits that the roles of a CTA give up together,
// exponentials to base 2, and Blackwell's packed fp32 arithmetic.
#pragma once
#include "tc_common.cuh"

namespace infllm {

using namespace tc;

__device__ __forceinline__ void record_error(int* err, int code, int where) {
  if (atomicCAS(&err[0], 0, code) == 0) {
    err[1] = where;
    err[2] = blockIdx.x;
    err[3] = blockIdx.y;
  }
}

// wait that also gives up when another role of the CTA has already failed
__device__ __forceinline__ bool wait_or_abort(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* err,
                                              int where) {
  for (uint32_t i = 0; i < kSpinLimit; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*abort_flag) return false;
    if (i > 64) __nanosleep(i > 4096 ? 256 : 32);
  }
  *abort_flag = 1;
  record_error(err, kErrWaitTimeout, where);
  return false;
}

// the same for a whole (converged) warp, whose lanes go on or give up together.  Nearly always the phase has passed or is about
// to: one look, in straight code, before the loop, in which lanes could part (75 cycles a wait instead of 110; four such waits are in
// the way of a key tile: 512 queries by 4608 + 2688 keys 5 % less)
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* err, int where) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  return __all_sync(0xffffffffu, wait_or_abort(bar, parity, abort_flag, err, where));
}

__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Blackwell's packed fp32 pairs and three-input maximum: half the instructions of the scalar forms
__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float2 ffma2(float a0, float a1, float2 b, float2 c) {
  float2 d;
  asm("{ .reg .b64 ra, rb, rc, rd; mov.b64 ra, {%2,%3}; mov.b64 rb, {%4,%5}; mov.b64 rc, {%6,%7}; "
      "fma.rn.f32x2 rd, ra, rb, rc; mov.b64 {%0,%1}, rd; }"
      : "=f"(d.x), "=f"(d.y) : "f"(a0), "f"(a1), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 fmul2(float2 a, float2 b) {
  float2 d;
  asm("{ .reg .b64 ra, rb, rd; mov.b64 ra, {%2,%3}; mov.b64 rb, {%4,%5}; mul.rn.f32x2 rd, ra, rb; mov.b64 {%0,%1}, rd; }"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 fadd2(float2 a, float2 b) {
  float2 d;
  asm("{ .reg .b64 ra, rb, rd; mov.b64 ra, {%2,%3}; mov.b64 rb, {%4,%5}; add.rn.f32x2 rd, ra, rb; mov.b64 {%0,%1}, rd; }"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// exp2 of a pair on the FMA and integer pipes (the special-function unit does 16 per clock per SM, which bounds the
// softmax when every exponential goes there): x = n + f with n the nearest integer (magic-number rounding) and f in
// [-0.5, 0.5], 2^f by a polynomial whose relative error was minimised over that interval (least squares on Chebyshev
// points), times 2^n.  A NaN stays one; arguments below -126, those of masked keys too, give 2^-126.
//   cubic    7.5e-5: a twentieth of the rounding of a bf16 P, a third to a sixth of that of an fp16 P
//   quartic  2.6e-6
//   quintic  2e-7 as evaluated in fp32, which is what ex2.approx has: where exp2f was
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
template <int kDegree>
__device__ __forceinline__ float2 ex2_poly2(float2 x) {
  static_assert(kDegree >= 3 && kDegree <= 5, "");
  x.x = max_nan(x.x, -126.f);
  x.y = max_nan(x.y, -126.f);
  const float2 magic = make_float2(12582912.f, 12582912.f), neg_magic = make_float2(-12582912.f, -12582912.f);
  const float2 t = fadd2(x, magic);
  const float2 n = fadd2(t, neg_magic);
  const float2 f = fadd2(x, make_float2(-n.x, -n.y));
  auto c2 = [](float c) { return make_float2(c, c); };
  float2 p;
  if (kDegree == 3) {
    p = ffma2(f.x, f.y, c2(0.05517167f), c2(0.24261113f));
    p = ffma2(p.x, p.y, f, c2(0.69326097f));
    p = ffma2(p.x, p.y, f, c2(0.99992806f));
  } else if (kDegree == 4) {
    p = ffma2(f.x, f.y, c2(0.0095701022f), c2(0.055917859f));
    p = ffma2(p.x, p.y, f, c2(0.24024744f));
    p = ffma2(p.x, p.y, f, c2(0.69312179f));
    p = ffma2(p.x, p.y, f, c2(0.99999928f));
  } else {
    p = ffma2(f.x, f.y, c2(0.00132669706f), c2(0.00967545994f));
    p = ffma2(p.x, p.y, f, c2(0.0555074252f));
    p = ffma2(p.x, p.y, f, c2(0.240221217f));
    p = ffma2(p.x, p.y, f, c2(0.693146944f));
    p = ffma2(p.x, p.y, f, c2(1.00000012f));
  }
  // a product, not an addition to the exponent's bits: that would make a number of a NaN
  return fmul2(p, make_float2(__int_as_float((__float_as_int(t.x) << 23) + 0x3f800000),
                              __int_as_float((__float_as_int(t.y) << 23) + 0x3f800000)));
}

constexpr int kPolyEvery = 8;
// exponentials of 32 columns of a row, packed; sums into rs
template <typename T, int kDegree>
__device__ __forceinline__ void exp_chunk(const float2* a, float2* rs, uint32_t* pk) {
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    float2 p;
    if (k % kPolyEvery == kPolyEvery - 1) {
      p = ex2_poly2<kDegree>(a[k]);  // one pair in kPolyEvery off the special-function unit
    } else {
      p = make_float2(ex2_approx(a[k].x), ex2_approx(a[k].y));
    }
    rs[k & 3] = fadd2(rs[k & 3], p);
    typename Act<T>::T2 v = Act<T>::from_f2(p.x, p.y);
    pk[k] = *reinterpret_cast<uint32_t*>(&v);
  }
}
// 32 columns of scores into exponents; what they were loaded into may be loaded into again behind it
__device__ __forceinline__ void arg_chunk(const float* s, float sc, float neg_m, float2* a) {
  const float2 sc2 = make_float2(sc, sc), nm2 = make_float2(neg_m, neg_m);
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    a[k] = ffma2(s[2 * k], s[2 * k + 1], sc2, nm2);
    asm volatile("" : "+f"(a[k].x), "+f"(a[k].y));
  }
}
__device__ __forceinline__ void max_chunk(const float* s, float* mx) {
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    mx[0] = fmax3(mx[0], s[i], s[i + 1]);
    mx[1] = fmax3(mx[1], s[i + 2], s[i + 3]);
    mx[2] = fmax3(mx[2], s[i + 4], s[i + 5]);
    mx[3] = fmax3(mx[3], s[i + 6], s[i + 7]);
  }
}

}  // namespace infllm
