// sp_q8_attn.cuh — arguments, work split and workspace shared by the
// attention kernels over the 8-bit cache.
#pragma once

#include "sp_q8.cuh"

namespace q8 {

struct AttnArgs {
    Layer l;
    Batch b;
    const void *q;
    void *out;
    float *lse;                      // NULL: not wanted
    long long q_stride, out_stride;  // elements between tokens
    int n_q_heads, group;
    float scale;                     // logit scale
    int causal, window;
    int few_rows;                    // entries of up to so many rows (new tokens x group) are the
                                     // few-row kernel's, the others the many-row kernel's
    unsigned int *counters;          // [kMaxCtas], zero between calls
    float *partials;
};

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kNone = -3.402823466e38f;    // running maximum of a row that has seen nothing

// --- work split -------------------------------------------------------
// A call's tiles of positions, laid end to end over its units of work, are
// cut into equal runs, one for each CTA, whatever the lengths; a unit that
// falls into several runs leaves a partial result (maximum, sum, weighted
// values) for each, and the CTA that finishes last joins them in run order,
// so results do not depend on the order of arrival.
struct Runs {
    unsigned total, n, q, r;         // tiles, CTAs with work, tiles of a run (the first r have one more)
};

__device__ __forceinline__ Runs runs_of(unsigned total, unsigned grid)
{
    Runs s;
    s.total = total;
    s.n = min(total, grid);
    s.q = s.n ? total / s.n : 0;
    s.r = s.n ? total - s.q * s.n : 0;
    return s;
}
__device__ __forceinline__ unsigned run_begin(const Runs &s, unsigned i) { return i * s.q + min(i, s.r); }
__device__ __forceinline__ unsigned run_of_tile(const Runs &s, unsigned t)
{
    const unsigned cut = s.r * (s.q + 1);
    return t < cut ? t / (s.q + 1) : s.r + (t - cut) / s.q;
}

// --- small things -----------------------------------------------------
__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x)
{
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 1 / x to the last place, for x whose reciprocal is a normal number.
__device__ __forceinline__ float rcp(float x)
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Four codes (bytes 0..3 of x) as fp16 pairs, lo = (0, 1) and hi = (2, 3),
// exactly.
//   int8: q + 128 placed in the low mantissa of 1024, then 1152 taken off:
//   finite for every byte.  8.5 cycles for a warp.
//   e4m3: the conversion instruction, 4.1 cycles (moving the fields by shifts
//   and masks takes 12.4); the two NaN codes stay NaN, so codes past a
//   sequence's end are not left in V.
template <int FMT>
__device__ __forceinline__ void unpack4(uint32_t x, uint32_t &lo, uint32_t &hi)
{
    if constexpr (FMT == SP_Q8_INT8) {
        x ^= 0x80808080u;
        const uint32_t a = __byte_perm(x, 0x64646464u, 0x4140), b = __byte_perm(x, 0x64646464u, 0x4342);
        const __half2 c = __half2half2(__ushort_as_half(0x6480));       // 1152
        const __half2 u = __hsub2(*reinterpret_cast<const __half2 *>(&a), c);
        const __half2 v = __hsub2(*reinterpret_cast<const __half2 *>(&b), c);
        lo = *reinterpret_cast<const uint32_t *>(&u);
        hi = *reinterpret_cast<const uint32_t *>(&v);
    } else {
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
            : "=r"(lo), "=r"(hi) : "r"(x));
    }
}

// 2^-e and 2^e for a row of queries whose largest magnitude is top, e its
// exponent: scaled rows fit fp16 whatever their type's range.
__device__ __forceinline__ void row_scale(float top, float &down, float &up)
{
    const unsigned E = (__float_as_uint(top) >> 23) & 0xff;
    const unsigned F = top > 0.0f && E < 255 ? min(max(E, 1u), 253u) : 127u;
    down = __uint_as_float((254u - F) << 23);
    up = __uint_as_float(F << 23);
}

size_t split_bytes(int sm_count);                                    // sp_q8_attn_many.cu
int launch_many(const AttnArgs &a, int format, int dtype, int hd, int sms, cudaStream_t s);

}  // namespace q8
