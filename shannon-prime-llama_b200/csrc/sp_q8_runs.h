// sp_q8_runs.h — how the many-row attention over the 8-bit cache cuts its tiles
// into runs; plain C++ too, for the host.
#pragma once

#ifdef __CUDACC__
#define SP_Q8_HD __host__ __device__ __forceinline__
#else
#define SP_Q8_HD inline
#endif

namespace q8 {

// `total` tiles cut into equal runs, one for each of `n` CTAs (the first r have
// a tile more).  A prompt of a million tokens has more than 2^32 tiles (they go
// with its square), so places among all tiles are 64-bit; a run's own length
// and what lies near it stay within 31 bits (2^31 tiles of one CTA are hours),
// and are compared by their difference in 32.
struct LongRuns {
    unsigned n, q, r;
};

SP_Q8_HD LongRuns long_runs_of(unsigned long long total, unsigned grid)
{
    LongRuns s;
    s.n = total < grid ? (unsigned)total : grid;
    s.q = s.n ? (unsigned)(total / s.n) : 0;
    s.r = s.n ? (unsigned)(total - (unsigned long long)s.q * s.n) : 0;
    return s;
}
SP_Q8_HD unsigned long long run_begin(const LongRuns &s, unsigned i)
{
    return (unsigned long long)i * s.q + (i < s.r ? i : s.r);
}
SP_Q8_HD unsigned run_of_tile(const LongRuns &s, unsigned long long t)
{
    const unsigned long long cut = (unsigned long long)s.r * (s.q + 1ull);
    return t < cut ? (unsigned)(t / (s.q + 1ull)) : s.r + (unsigned)((t - cut) / s.q);
}

// a - b of two places near one another, of which only the low 32 bits are kept.
SP_Q8_HD int apart(unsigned a, unsigned b) { return (int)(a - b); }

}  // namespace q8
