// Arithmetic on two floats at once: one instruction issued for both, each rounded as by itself (but a product that is only added to something may be contracted with the sum).
#pragma once

namespace seera {

struct __align__(8) Two { float x, y; };
__device__ __forceinline__ unsigned long long bits(Two a) { return *reinterpret_cast<unsigned long long *>(&a); }
__device__ __forceinline__ Two two(unsigned long long b) { return *reinterpret_cast<Two *>(&b); }
__device__ __forceinline__ Two both(float x) { return Two{x, x}; }
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
    unsigned long long d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(bits(a)), "l"(bits(b)), "l"(bits(c)));
    return two(d);
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
    unsigned long long d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits(a)), "l"(bits(b)));
    return two(d);
}
__device__ __forceinline__ Two add2(Two a, Two b) {
    unsigned long long d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits(a)), "l"(bits(b)));
    return two(d);
}
__device__ __forceinline__ Two less2(Two a, Two b) { return fma2(b, both(-1.f), a); }       // a - b

}  // namespace seera
