// Arithmetic of the tcgen05 attention kernels' softmax warps: two floats an instruction, and powers of two on the special-function unit or on
// the multiply-add units.
#pragma once
#include "common.cuh"

namespace packed {

// 2^x by the special-function unit (relative error about 2^-22; 2^-inf = 0)
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
typedef unsigned long long f2;                            // two packed floats
__device__ __forceinline__ f2 pack2(float lo, float hi) {
    f2 v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
__device__ __forceinline__ void unpack2(f2 v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
    f2 v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
    f2 v;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
    f2 v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
// The larger of two numbers, or NaN where one of them is NaN (fmaxf gives the other).
__device__ __forceinline__ float max_or_nan(float a, float b) {
    float v;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(v) : "f"(a), "f"(b));
    return v;
}
// 2^x for two numbers on the multiply-add units, x at most 127: x = n + f with n whole and |f| <= 1/2, a polynomial of degree 5 for 2^f
// (least worst relative error over [-1/2, 1/2], fitted by Lawson's iteration: 7.5e-8, 2.1e-7 with the roundings, as much as the
// special-function unit's) times 2^n.  As with the unit, NaN gives NaN, and what lies below -127 gives 0 (n = -127 makes the factor's
// bits all zero).  (n is not added to the polynomial's exponent, which would be one multiplication less: on a NaN's bits that gives a number.)
__device__ __forceinline__ void ex2_pair(f2 x, float& a, float& b) {
    auto both = [](float v) { return pack2(v, v); };
    float xa, xb;
    unpack2(x, xa, xb);
    x = pack2(max_or_nan(xa, -127.f), max_or_nan(xb, -127.f));
    const f2 n = add2(x, both(12582912.f));                // 1.5 * 2^23: n stands in the low bits
    const f2 f = fma2(add2(n, both(-12582912.f)), both(-1.f), x);
    f2 p = fma2(both(0.00132764445f), f, both(0.00967553724f));
    p = fma2(p, f, both(0.0555071346f));
    p = fma2(p, f, both(0.240221202f));
    p = fma2(p, f, both(0.693146944f));
    p = fma2(p, f, both(1.00000012f));
    float na, nb;
    unpack2(n, na, nb);
    const f2 two_n = pack2(__int_as_float((__float_as_int(na) << 23) + 0x3f800000), __int_as_float((__float_as_int(nb) << 23) + 0x3f800000));
    unpack2(mul2(p, two_n), a, b);
}
__device__ __forceinline__ unsigned pack_bf16(float a, float b) {
    __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *(unsigned*)&v;
}

}  // namespace packed
