// Two fp32 values in a 64-bit register pair and the instructions that work on both.
#pragma once
#include "sm100_ptx.cuh"

namespace gdn {
namespace pairs {

using f2 = unsigned long long;
__device__ __forceinline__ f2 pk(float lo, float hi) {
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ f2 pk(uint32_t lo, uint32_t hi) { return pk(__uint_as_float(lo), __uint_as_float(hi)); }
__device__ __forceinline__ void unpk(f2 v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
    f2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
    f2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
    f2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint32_t pack2(f2 v) {
    float lo, hi;
    unpk(v, lo, hi);
    return ptx::pack_bf16(lo, hi);
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// u / (1 + e^-u)
__device__ __forceinline__ f2 silu2(f2 u) {
    float a, b;
    unpk(mul2(u, pk(-1.4426950408889634f, -1.4426950408889634f)), a, b);
    unpk(add2(pk(ex2(a), ex2(b)), pk(1.f, 1.f)), a, b);
    return mul2(u, pk(rcp(a), rcp(b)));
}

}  // namespace pairs
}  // namespace gdn
