// Packed fp32 arithmetic.
#pragma once

#include <cuda_runtime.h>

namespace o1d {

// Two fp32 numbers that one instruction works on (fma.rn.f32x2 and the like): kernels that use them are bound by
// instruction issue, and a packed instruction takes one slot for two values.  Each half is rounded as the scalar instruction rounds.
struct F2 { unsigned long long v; };
__device__ __forceinline__ F2 two(float a, float b) { F2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ F2 both(float a) { return two(a, a); }
__device__ __forceinline__ float2 apart(F2 a) { float2 r; asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v)); return r; }
__device__ __forceinline__ F2 add2(F2 a, F2 b) { F2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }
__device__ __forceinline__ F2 mul2(F2 a, F2 b) { F2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) { F2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v)); return r; }

}  // namespace o1d
