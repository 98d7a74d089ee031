// The logistic function to full relative precision on both sides.
#pragma once

namespace seera {

// 1 / (1 + e^|x|), the smaller of sigmoid(x) and 1 - sigmoid(x), with the sign of x.
// 1 / (1 + 2^t) with t = |x| log2 e; what t's rounding loses, up to |x| 2^-24 of the power, is made good by a factor of 1 + ln 2 times it (the
// constant's own loses |x| 2^-26).  The two approximate instructions are off by at most 2^-22 and 2^-23: half the instructions that expf and a
// division take, and instructions bound the kernels that use it next to the bytes.  Beyond 88 the power would leave the range: the result is 0 there, and
// below the smallest normal number anyway.
__device__ __forceinline__ float sigmoid_less(float x) {
    float a, e, s;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(fabsf(x)), "f"(88.f));
    const float t = a * 1.44269502f, lost = fmaf(a, 1.44269502f, -t);
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
    e = fmaf(e, lost * 0.693147182f, e);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.f + e));
    return copysignf(s, x);
}

}  // namespace seera
