// Two float32 operations an instruction (fma.rn.f32x2 and its kin), the three-input maximum, the hardware's 2^x, and quotients of small
// numbers: kernels whose warps are bound by the instructions they issue do their arithmetic with these.
#pragma once

#include "common.cuh"

namespace {

__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ unsigned long long pack2(float lo, float hi) {
    unsigned long long v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
__device__ __forceinline__ void unpack2(unsigned long long v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b) {
    unsigned long long d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
    unsigned long long d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// x / d and x % d of numbers up to 2^22: a quotient by the reciprocal, put right where it is one off.
struct ByDivisor {
    int d;
    float inv;
    __device__ __forceinline__ explicit ByDivisor(int n) : d(n), inv(1.0f / (float)n) {}
    __device__ __forceinline__ int2 operator()(int x) const {
        int q = (int)((float)x * inv), r = x - q * d;
        if (r < 0) { --q; r += d; }
        if (r >= d) { ++q; r -= d; }
        return make_int2(q, r);
    }
};

}  // namespace
