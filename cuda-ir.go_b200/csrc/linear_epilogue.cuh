// linear_epilogue.cuh - what the linear and gated kernels do with an
// accumulator: the activations and their derivatives, and the loads and stores
// of a row's 32 consecutive columns in 16 or 32 bits.
//
// Everything is computed in fp32 and rounded once, to nearest, when it is
// stored.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "../../include/cudair_b200.h"
#include "linear_internal.h"

namespace cudair {
namespace ffn {

// ---- activations ---------------------------------------------------------------
//
//   relu       max(z, 0), a NaN kept
//   silu       z s(z), s(z) = 1 / (1 + e^-z)
//   gelu       z P(z), P the normal distribution's integral
//   gelu_tanh  z (1 + tanh(y)) / 2 with y = sqrt(2/pi) (z + 0.044715 z^3),
//              computed as z s(2y), which is the same and does not cancel
//
// An epilogue warp runs 32 columns of these alone on its scheduler, so their
// length is the epilogue's: with expf, an IEEE division and normcdff a
// 256-column tile took 18 us (silu, 256 x 1024 outputs; 40 us where the
// division leaves its fast path) against 2 us without an activation.  So the
// power of two and the reciprocal are one hardware instruction each: 2^-22 of
// the value, with the argument's rounding |z| 2^-23 more for e^z; results below
// 2^-126 become 0.

constexpr float kGeluC = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kGeluB = 0.044715f;

__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rcp_fast(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
constexpr float kLog2E = 1.4426950408889634f;

__device__ __forceinline__ float sigmoid(float z) { return rcp_fast(1.0f + exp2_fast(-kLog2E * z)); }
// sigmoid(2y) of gelu_tanh, from z and z^2: the constants of 2y and of e^-2y in one.
__device__ __forceinline__ float gelu_tanh_sigmoid(float z, float z2) {
    return rcp_fast(1.0f + exp2_fast(z * fmaf(-kLog2E * kGeluC * kGeluB, z2, -kLog2E * kGeluC)));
}

// The normal distribution's upper tail at u >= 0 is T(u) = E R with E = e^(-u^2 / 2)
// and R = e^(u^2 / 2) erfc(u / sqrt(2)) / 2, which falls from 1/2 like 1 / u: R is
// t times a polynomial in t = 1 / (1 + q u).  q and the coefficients were fitted
// here, by least squares reweighted until the largest relative error over
// 0 <= u <= 13.4 (E is 0 beyond) was level: 6.3e-7, 9e-7 evaluated in fp32.  So
// gelu keeps its relative accuracy for negative z, where it is -|z| T: there
// the exponent's rounding adds u^2 2^-24.  Two terms more than a fit of erfc's
// absolute error needs (which is 1e-2 of gelu's value at -8): 8192 x 14336 x 512
// with bias and gelu 188.6 -> 190.5 us.
constexpr float kTailQ = 0.265f;
__device__ constexpr float kTail[7] = {0.10559984f, 0.10783678f, 0.082946599f, 0.14249332f, -0.066362917f, 0.19527312f,
                                       -0.067787044f};

// P(z) and E = e^(-z^2 / 2).
__device__ __forceinline__ void normal_integral(float z, float &P, float &E) {
    E = exp2_fast(-0.5f * kLog2E * z * z);
    const float t = rcp_fast(fmaf(kTailQ, fabsf(z), 1.0f));
    float h = kTail[6];
#pragma unroll
    for (int k = 5; k >= 0; --k) h = fmaf(t, h, kTail[k]);
    h *= t * E;
    P = z < 0.0f ? h : 1.0f - h;
}

// ---- two values at a time --------------------------------------------------------
//
// fma, mul and add on pairs of fp32 values are one instruction each on sm_100,
// rounded as the single ones.  An epilogue's instructions are half of its time, so
// its activations work on pairs (a chunk of 32 columns with gelu: 22 instructions a
// value one by one, 10 in pairs; what remains is the two hardware functions).

struct Pair {
    uint64_t v;
};
__device__ __forceinline__ Pair pair(float lo, float hi) {
    Pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ Pair pair(float both) { return pair(both, both); }
__device__ __forceinline__ void unpair(Pair p, float &lo, float &hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(p.v));
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Pair exp2_fast2(Pair p) {
    float a, b;
    unpair(p, a, b);
    return pair(exp2_fast(a), exp2_fast(b));
}
__device__ __forceinline__ Pair rcp_fast2(Pair p) {
    float a, b;
    unpair(p, a, b);
    return pair(rcp_fast(a), rcp_fast(b));
}
// max(z, 0), a NaN kept.
__device__ __forceinline__ float relu(float z) {
    float r;
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(z));
    return r;
}

// z held above -1e18 and below 1e18, a NaN kept.  There the activations and their
// derivatives have reached their limits in fp32, and an infinite z gives no 0
// times infinity.  (Its square is finite too.)
constexpr float kFar = 1e18f;
__device__ __forceinline__ float above(float z) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(z), "f"(-kFar));
    return r;
}
__device__ __forceinline__ float below(float z) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(z), "f"(kFar));
    return r;
}

// act(a), act(b) in place.  gelu: z P(z) = max(z, 0) - |z| T, T the upper tail at
// |z| that normal_integral computes.
template <int ACT>
__device__ __forceinline__ void act_pair(float &a, float &b) {
    if (ACT == CUDAIR_ACT_RELU) {
        a = relu(a);
        b = relu(b);
    } else if (ACT == CUDAIR_ACT_SILU) {
        const Pair z = pair(above(a), above(b));
        const Pair e = exp2_fast2(mul2(z, pair(-kLog2E)));
        unpair(mul2(z, rcp_fast2(add2(e, pair(1.0f)))), a, b);
    } else if (ACT == CUDAIR_ACT_GELU_TANH) {
        const Pair z = pair(above(a), above(b));
        const Pair y = fma2(mul2(z, z), pair(-kLog2E * kGeluC * kGeluB), pair(-kLog2E * kGeluC));
        unpair(mul2(z, rcp_fast2(add2(exp2_fast2(mul2(z, y)), pair(1.0f)))), a, b);
    } else if (ACT == CUDAIR_ACT_GELU) {
        const Pair u = pair(fminf(fabsf(a), kFar), fminf(fabsf(b), kFar));
        const Pair E = exp2_fast2(mul2(mul2(u, pair(-0.5f * kLog2E)), u));
        const Pair t = rcp_fast2(fma2(u, pair(kTailQ), pair(1.0f)));
        Pair h = pair(kTail[6]);
#pragma unroll
        for (int k = 5; k >= 0; --k) h = fma2(t, h, pair(kTail[k]));
        h = mul2(h, mul2(t, E));
        unpair(fma2(mul2(u, pair(-1.0f)), h, pair(relu(a), relu(b))), a, b);
    }
}

// The value and the derivative at z.
template <int ACT>
__device__ __forceinline__ void act_both(float z, float &value, float &grad) {
    if (ACT == CUDAIR_ACT_RELU) {
        value = relu(z);
        grad = z <= 0.0f ? 0.0f : 1.0f;
    } else if (ACT == CUDAIR_ACT_SILU) {
        z = above(z);
        const float s = sigmoid(z);
        value = z * s;
        grad = s * (1.0f + below(z) * (1.0f - s));
    } else if (ACT == CUDAIR_ACT_GELU) {
        float P, E;
        z = above(z);
        normal_integral(z, P, E);
        value = z * P;
        grad = P + below(z) * (0.3989422804014327f * E);
    } else if (ACT == CUDAIR_ACT_GELU_TANH) {
        z = above(z);
        const float z2 = z * z;
        const float s = gelu_tanh_sigmoid(z, z2);
        value = z * s;
        // s (1 - s) is zero where s is 0 or 1; z^2 may be infinite there (z is not held from above).
        const float w = s - s * s;
        grad = w == 0.0f ? s : s + w * (z * fmaf(3.0f * kGeluB * kGeluC, z2, kGeluC));
    } else {
        value = z;
        grad = 1.0f;
    }
}

// Calls f with the activation as a compile-time constant: the choice is made
// once per block of elements, not per element.
template <int V>
struct ActTag {
    static constexpr int value = V;
};
template <class F>
__device__ __forceinline__ void with_act(int act, F &&f) {
    switch (act) {
        case CUDAIR_ACT_RELU: f(ActTag<CUDAIR_ACT_RELU>{}); break;
        case CUDAIR_ACT_GELU: f(ActTag<CUDAIR_ACT_GELU>{}); break;
        case CUDAIR_ACT_GELU_TANH: f(ActTag<CUDAIR_ACT_GELU_TANH>{}); break;
        case CUDAIR_ACT_SILU: f(ActTag<CUDAIR_ACT_SILU>{}); break;
        default: f(ActTag<CUDAIR_ACT_NONE>{}); break;
    }
}

// ---- 16-bit conversions ----------------------------------------------------------

__device__ __forceinline__ float from16(uint16_t h, bool bf16) {
    return bf16 ? __uint_as_float(static_cast<uint32_t>(h) << 16) : __half2float(__ushort_as_half(h));
}
__device__ __forceinline__ uint16_t to16(float f, bool bf16) {
    return bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(f)) : __half_as_ushort(__float2half_rn(f));
}
__device__ __forceinline__ void unpack16(uint32_t w, bool bf16, float &lo, float &hi) {
    if (bf16) {
        lo = __uint_as_float(w << 16);
        hi = __uint_as_float(w & 0xFFFF0000u);
    } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
        lo = f.x;
        hi = f.y;
    }
}
__device__ __forceinline__ uint32_t pack16(float lo, float hi, bool bf16) {
    if (bf16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// ---- global memory, 32 or 16 bytes at a time ----------------------------------------

__device__ __forceinline__ void st_v8(void *p, const uint32_t *w) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]),
                 "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}
__device__ __forceinline__ void st_v4(void *p, const uint32_t *w) {
    asm volatile("st.global.v4.b32 [%0], {%1, %2, %3, %4};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                 "r"(w[3])
                 : "memory");
}
__device__ __forceinline__ void ld_v8(const void *p, uint32_t *w) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]),
                   "=r"(w[7])
                 : "l"(p)
                 : "memory");
}
__device__ __forceinline__ void ld_v4(const void *p, uint32_t *w) {
    asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "l"(p)
                 : "memory");
}

// A row-major matrix that an epilogue reads or writes.
struct Mat {
    void *p;        // nullptr: absent
    long long ld;   // elements
    int f32;        // 32-bit elements, else 16-bit of the operands' type
    int wide;       // base and pitch are multiples of 32 bytes, else of 16
};

inline Mat mat_of(const OutMat &m) {
    const uint64_t bytes = m.f32 ? 4 : 2;
    Mat r;
    r.p = m.p;
    r.ld = static_cast<long long>(m.ld);
    r.f32 = m.f32;
    r.wide = ((reinterpret_cast<uintptr_t>(m.p) | (static_cast<uint64_t>(m.ld) * bytes)) & 31u) == 0;
    return r;
}

// One row's 32 columns from col (a multiple of 32, below N): whole 32-byte
// sectors where the matrix allows it, else 16 bytes at a time; the columns of
// a last block that ends inside it one by one, none beyond N touched.
__device__ __forceinline__ void store_row32(const Mat &m, long long row, int col, int N, bool bf16,
                                            const float (&v)[32]) {
    if (m.f32) {
        float *p = static_cast<float *>(m.p) + row * m.ld + col;
        if (col + 32 <= N) {
            uint32_t w[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) w[j] = __float_as_uint(v[j]);
            if (m.wide) {
#pragma unroll
                for (int j = 0; j < 4; ++j) st_v8(p + 8 * j, w + 8 * j);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) st_v4(p + 4 * j, w + 4 * j);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (col + j < N) p[j] = v[j];
        }
    } else {
        uint16_t *p = static_cast<uint16_t *>(m.p) + row * m.ld + col;
        if (col + 32 <= N) {
            uint32_t w[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = pack16(v[2 * j], v[2 * j + 1], bf16);
            if (m.wide) {
                st_v8(p, w);
                st_v8(p + 16, w + 8);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) st_v4(p + 8 * j, w + 4 * j);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (col + j < N) p[j] = to16(v[j], bf16);
        }
    }
}

// One row's 32 columns as they lie in memory (16 words of 16-bit values, or
// 32), so that the loads can be issued long before the values are needed.
struct Row32 {
    uint32_t w[32];
};
__device__ __forceinline__ void fetch_row32(const Mat &m, long long row, int col, int N, Row32 &r) {
    if (m.f32) {
        const float *p = static_cast<const float *>(m.p) + row * m.ld + col;
        if (col + 32 <= N) {
            if (m.wide) {
#pragma unroll
                for (int j = 0; j < 4; ++j) ld_v8(p + 8 * j, r.w + 8 * j);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) ld_v4(p + 4 * j, r.w + 4 * j);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) r.w[j] = col + j < N ? __float_as_uint(p[j]) : 0u;
        }
    } else {
        const uint16_t *p = static_cast<const uint16_t *>(m.p) + row * m.ld + col;
        if (col + 32 <= N) {
            if (m.wide) {
                ld_v8(p, r.w);
                ld_v8(p + 16, r.w + 8);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) ld_v4(p + 8 * j, r.w + 4 * j);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j)
                r.w[j] = (col + 2 * j < N ? p[2 * j] : 0u) | (col + 2 * j + 1 < N ? p[2 * j + 1] : 0u) << 16;
        }
    }
}
__device__ __forceinline__ void add_row32(const Row32 &r, bool f32, bool bf16, float (&v)[32]) {
    if (f32) {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] += __uint_as_float(r.w[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            float lo, hi;
            unpack16(r.w[j], bf16, lo, hi);
            unpair(add2(pair(v[2 * j], v[2 * j + 1]), pair(lo, hi)), v[2 * j], v[2 * j + 1]);
        }
    }
}

}  // namespace ffn
}  // namespace cudair
