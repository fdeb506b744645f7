// sp_rope.cu — rotary positions with several axes (shannon_prime_q8.h).
//
// Each pair (x, y) of a head's first rot_dim elements turns by
// a = pos[axis] * f, f a 32-bit float: the tables of frequencies that models
// are trained with are such, and at position 1e5 the formula's own frequencies
// turn by up to 3e-3 radians more or less.  The angle is kept as a fraction of a
// turn in 64-bit fixed point: f / 2 pi times 2^64 is rounded once on the host,
// and the low 64 bits of position * phase are the fraction, reduced exactly
// however far the position is (a 32-bit product of position and frequency is
// off by another 4e-3 radians there).  Its top 32 bits go through sincospif.
#include "sp_internal.cuh"
#include "sp_q8.cuh"

#include <atomic>
#include <math.h>
#include <string.h>

extern "C" int sp_rope_axes_init(sp_rope_axes_t *ra, int head_dim, int rot_dim, int pairing, int n_axes,
                                 const int *sections, int flags, double theta, const float *freq_factors)
{
    sp_clear_error();
    if (!ra || !sections) return sp_set_error(SP_ERR_ARG, "rope_axes_init: NULL argument");
    memset(ra, 0, sizeof(*ra));
    if (head_dim <= 0 || head_dim > SP_MAX_HEAD_DIM || head_dim % 8)
        return sp_set_error(SP_ERR_UNSUPPORTED, "rope_axes_init: head_dim %d is not a multiple of 8 in [8,%d]", head_dim,
                            SP_MAX_HEAD_DIM);
    if (rot_dim <= 0 || rot_dim > head_dim || rot_dim % 16)
        return sp_set_error(SP_ERR_UNSUPPORTED, "rope_axes_init: rot_dim %d is not a multiple of 16 in [16,%d]", rot_dim,
                            head_dim);
    if (pairing != SP_ROPE_ADJACENT && pairing != SP_ROPE_HALVES)
        return sp_set_error(SP_ERR_ARG, "rope_axes_init: pairing %d", pairing);
    if (n_axes < 1 || n_axes > SP_ROPE_MAX_AXES)
        return sp_set_error(SP_ERR_ARG, "rope_axes_init: %d axes, 1 to %d are possible", n_axes, SP_ROPE_MAX_AXES);
    if (flags & ~(SP_ROPE_INTERLEAVED | SP_ROPE_AXIS_LADDER))
        return sp_set_error(SP_ERR_ARG, "rope_axes_init: unknown flags %d", flags);
    if (!(theta > 0.0) || !isfinite(theta)) return sp_set_error(SP_ERR_ARG, "rope_axes_init: theta %g", theta);
    const int n_pairs = rot_dim / 2;
    long long sum = 0;
    for (int a = 0; a < n_axes; a++) {
        if (sections[a] < 0) return sp_set_error(SP_ERR_ARG, "rope_axes_init: section %d has %d pairs", a, sections[a]);
        sum += sections[a];
    }
    if (sum != n_pairs)
        return sp_set_error(SP_ERR_ARG, "rope_axes_init: the sections have %lld pairs, rot_dim %d has %d", sum, rot_dim,
                            n_pairs);
    sp_rope_axes_t plan = {head_dim, rot_dim, n_axes, pairing, {}, {}};      // *ra stays empty where a frequency is refused
    int used[SP_ROPE_MAX_AXES] = {0, 0, 0, 0};
    int a = 0;
    for (int i = 0; i < n_pairs; i++) {
        while (used[a] == sections[a]) a = (a + 1) % n_axes;
        const double e = flags & SP_ROPE_AXIS_LADDER ? (double)used[a] / sections[a] : 2.0 * i / rot_dim;
        double f = pow(theta, -e);
        if (freq_factors) {
            if (!isfinite(freq_factors[i]) || freq_factors[i] == 0.0f)
                return sp_set_error(SP_ERR_ARG, "rope_axes_init: factor %d is %g", i, (double)freq_factors[i]);
            f /= (double)freq_factors[i];
        }
        f = (double)(float)f;
        if (!isfinite(f)) return sp_set_error(SP_ERR_ARG, "rope_axes_init: frequency %d is past 32-bit floats", i);
        // whole turns for each step do not matter at whole positions
        double turn = f / 6.283185307179586476925;
        turn -= floor(turn);
        plan.phase[i] = turn >= 1.0 ? 0 : (uint64_t)ldexp(turn, 64);
        plan.axis[i] = (uint8_t)a;
        used[a]++;
        if (flags & SP_ROPE_INTERLEAVED) a = (a + 1) % n_axes;
    }
    *ra = plan;
    return SP_OK;
}

namespace {

constexpr int kRopeThreads = 256;

struct RopeHalf {
    const void *in;
    void *out;
    long long in_stride, out_stride;   // elements between tokens
    int heads;
};

// The plan with room for PAIRS pairs: a launch copies its arguments, and 64
// pairs (head_dim 128) are a quarter of what the largest head has.
template <int PAIRS>
struct RopeArgs {
    int hd, rot;
    uint64_t phase[PAIRS];
    uint8_t axis[PAIRS];
    const int *pos;
    RopeHalf h[2];
    int n_tokens;
    int tokens_per_cta;
    int inverse;
};

template <typename T>
__device__ __forceinline__ void load8(const T *p, float (&x)[8])
{
    if constexpr (sizeof(T) == 4) {
        const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
        const uint4 w = *reinterpret_cast<const uint4 *>(p);
        const T *e = reinterpret_cast<const T *>(&w);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = sp_load_as_float(e, i);
    }
}

__device__ __forceinline__ void put(float *p, float v) { *p = v; }
__device__ __forceinline__ void put(__half *p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

template <typename T>
__device__ __forceinline__ void store8(T *p, const float (&x)[8])
{
    constexpr int kVecs = sizeof(T) == 4 ? 2 : 1;
    uint4 w[kVecs];
    T *e = reinterpret_cast<T *>(w);
#pragma unroll
    for (int i = 0; i < 8; i++) put(e + i, x[i]);
#pragma unroll
    for (int i = 0; i < kVecs; i++) reinterpret_cast<uint4 *>(p)[i] = w[i];
}

// A CTA takes tokens_per_cta tokens: first its threads share their cosines
// and sines (one sincospif for each pair and token, not for each head), then
// every thread rotates units of 8 adjacent elements, or 8 elements and their
// partners half a rotation away, of any token and head.  Memory bounds it: the
// 336 MB of 16421 tokens with 32 and 8 heads of 128 in bf16 take 62 us, 83% of
// the copy rate (one token for each CTA: 68 us); a step's few tokens take as long
// as a launch, and a CTA for each token puts them on the most SMs.
template <typename T, int PAIRING, int PAIRS>
__global__ void __launch_bounds__(kRopeThreads) k_rope_axes(const __grid_constant__ RopeArgs<PAIRS> a)
{
    extern __shared__ __align__(16) float2 cs[];       // [tokens][pairs]
    q8::begin();
    const int n_pairs = a.rot / 2, hd = a.hd, rot = a.rot;
    const int t0 = blockIdx.x * a.tokens_per_cta;
    const int n_t = min(a.tokens_per_cta, a.n_tokens - t0);
    for (int i = threadIdx.x; i < n_t * n_pairs; i += kRopeThreads) {
        const int t = i / n_pairs, p = i - t * n_pairs;
        const long long pos = a.pos[(long long)a.axis[p] * a.n_tokens + t0 + t];
        const uint64_t turn = (uint64_t)pos * a.phase[p];
        float s, c;
        sincospif((float)(int)(turn >> 32) * 0x1p-31f, &s, &c);
        cs[i] = make_float2(c, a.inverse ? -s : s);
    }
    __syncthreads();
    const int rot_units = PAIRING == SP_ROPE_ADJACENT ? rot / 8 : rot / 16;
    const int units = rot_units + (hd - rot) / 8;       // the rest of a head passes through
    const int heads = a.h[0].heads + a.h[1].heads;
    const int n = n_t * heads * units;
    for (int i = threadIdx.x; i < n; i += kRopeThreads) {
        const int row = i / units, u = i - row * units;
        const int t = row / heads;
        int head = row - t * heads;
        const int w = head >= a.h[0].heads;
        if (w) head -= a.h[0].heads;
        const RopeHalf &h = a.h[w];
        const T *in = static_cast<const T *>(h.in) + (long long)(t0 + t) * h.in_stride + head * hd;
        T *out = static_cast<T *>(h.out) + (long long)(t0 + t) * h.out_stride + head * hd;
        if (u >= rot_units) {
            const int e = rot + 8 * (u - rot_units);
            if (in != out) {
                float x[8];
                load8(in + e, x);
                store8(out + e, x);
            }
        } else if (PAIRING == SP_ROPE_ADJACENT) {
            float x[8], y[8];
            load8(in + 8 * u, x);
            const float4 *f = reinterpret_cast<const float4 *>(cs + t * n_pairs + 4 * u);
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const float4 v = f[j];
                y[4 * j] = x[4 * j] * v.x - x[4 * j + 1] * v.y;
                y[4 * j + 1] = x[4 * j] * v.y + x[4 * j + 1] * v.x;
                y[4 * j + 2] = x[4 * j + 2] * v.z - x[4 * j + 3] * v.w;
                y[4 * j + 3] = x[4 * j + 2] * v.w + x[4 * j + 3] * v.z;
            }
            store8(out + 8 * u, y);
        } else {
            float x[8], y[8], lo[8], hi[8];
            load8(in + 8 * u, x);
            load8(in + rot / 2 + 8 * u, y);
            const float4 *f = reinterpret_cast<const float4 *>(cs + t * n_pairs + 8 * u);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float4 v = f[j];
                lo[2 * j] = x[2 * j] * v.x - y[2 * j] * v.y;
                hi[2 * j] = x[2 * j] * v.y + y[2 * j] * v.x;
                lo[2 * j + 1] = x[2 * j + 1] * v.z - y[2 * j + 1] * v.w;
                hi[2 * j + 1] = x[2 * j + 1] * v.w + y[2 * j + 1] * v.z;
            }
            store8(out + 8 * u, lo);
            store8(out + rot / 2 + 8 * u, hi);
        }
    }
}

template <typename T, int PAIRS>
int launch_pairs(const sp_rope_axes_t *ra, RopeArgs<PAIRS> &a, unsigned grid, size_t smem, cudaStream_t s)
{
    a.hd = ra->head_dim;
    a.rot = ra->rot_dim;
    memcpy(a.phase, ra->phase, sizeof(a.phase));
    memcpy(a.axis, ra->axis, sizeof(a.axis));
    return q8::launch("rope_axes launch", ra->pairing == SP_ROPE_ADJACENT ? k_rope_axes<T, SP_ROPE_ADJACENT, PAIRS> : k_rope_axes<T, SP_ROPE_HALVES, PAIRS>,
                      grid, kRopeThreads, smem, s, a);
}

template <int PAIRS>
int launch(const sp_rope_axes_t *ra, RopeArgs<PAIRS> &a, int dtype, unsigned grid, size_t smem, cudaStream_t s)
{
    if (dtype == SP_DTYPE_F32) return launch_pairs<float>(ra, a, grid, smem, s);
    if (dtype == SP_DTYPE_F16) return launch_pairs<__half>(ra, a, grid, smem, s);
    return launch_pairs<__nv_bfloat16>(ra, a, grid, smem, s);
}

}  // namespace

extern "C" int sp_cuda_rope_axes(const sp_rope_axes_t *ra, const int *d_pos, int n_tokens, const void *d_q,
                                 long long q_stride, int n_q_heads, void *d_q_out, long long q_out_stride,
                                 const void *d_k, long long k_stride, int n_k_heads, void *d_k_out,
                                 long long k_out_stride, int dtype, int inverse, void *stream)
{
    sp_clear_error();
    if (!ra || ra->head_dim <= 0) return sp_set_error(SP_ERR_ARG, "rope_axes: no plan");
    if (dtype != SP_DTYPE_F32 && dtype != SP_DTYPE_F16 && dtype != SP_DTYPE_BF16)
        return sp_set_error(SP_ERR_ARG, "rope_axes: dtype %d", dtype);
    if (n_tokens < 0) return sp_set_error(SP_ERR_ARG, "rope_axes: %d tokens", n_tokens);
    if (!d_q != !d_q_out || !d_k != !d_k_out) return sp_set_error(SP_ERR_ARG, "rope_axes: an input without its output");
    RopeHalf halves[2] = {{d_q, d_q_out, q_stride, q_out_stride, d_q ? n_q_heads : 0},
                          {d_k, d_k_out, k_stride, k_out_stride, d_k ? n_k_heads : 0}};
    const long long el = dtype == SP_DTYPE_F32 ? 4 : 2;
    for (RopeHalf &h : halves) {
        if (!h.in) continue;
        const long long row = (long long)h.heads * ra->head_dim;
        if (h.heads < 1 || h.heads > 65536) return sp_set_error(SP_ERR_ARG, "rope_axes: %d heads", h.heads);
        if (h.in_stride == 0) h.in_stride = row;
        if (h.out_stride == 0) h.out_stride = row;
        if (h.in_stride < row || h.out_stride < row)
            return sp_set_error(SP_ERR_ARG, "rope_axes: a token's stride is less than its rows");
        if (((uintptr_t)h.in | (uintptr_t)h.out | (uintptr_t)(h.in_stride * el) | (uintptr_t)(h.out_stride * el)) % 16)
            return sp_set_error(SP_ERR_ARG, "rope_axes: pointers and strides must be multiples of 16 bytes");
        if (h.in == h.out && h.in_stride != h.out_stride)
            return sp_set_error(SP_ERR_ARG, "rope_axes: in place with two strides");
    }
    if (n_tokens == 0 || (!d_q && !d_k)) return SP_OK;
    if (!d_pos) return sp_set_error(SP_ERR_ARG, "rope_axes: no positions");
    const int n_pairs = ra->rot_dim / 2;
    // As many tokens for a CTA as give each thread one sincospif, where there
    // are CTAs for all the SMs' threads even so; below that a CTA for each token.
    const int each = kRopeThreads / n_pairs > 1 && n_tokens >= 2048 ? kRopeThreads / n_pairs : 1;
    const unsigned grid = (unsigned)((n_tokens + each - 1) / each);
    const size_t smem = sizeof(float2) * n_pairs * each;
    cudaStream_t s = (cudaStream_t)stream;
    auto go = [&](auto &a) {
        a.pos = d_pos;
        a.h[0] = halves[0];
        a.h[1] = halves[1];
        a.n_tokens = n_tokens;
        a.tokens_per_cta = each;
        a.inverse = inverse;
        return launch(ra, a, dtype, grid, smem, s);
    };
    if (n_pairs <= 64) {
        RopeArgs<64> a;
        return go(a);
    }
    RopeArgs<SP_MAX_HEAD_DIM / 2> a;
    return go(a);
}
