// sp_q8.cu — the 8-bit cache (shannon_prime_q8.h): lifecycle, the quantising
// write and the read back.
#include "sp_q8.cuh"

#include <string.h>

namespace q8 {
size_t attn_workspace_bytes(int sm_count, int head_dim);   // sp_q8_attn.cu

static int check_cache(const sp_cuda_q8_cache_t *qc, int layer, const char *what)
{
    if (!qc || !qc->d_k_cache) return sp_set_error(SP_ERR_ARG, "%s: cache not initialised", what);
    if (layer < 0 || layer >= qc->config.n_layers) return sp_set_error(SP_ERR_ARG, "%s: layer %d out of range", what, layer);
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess || dev != qc->device)
        return sp_set_error(SP_ERR_ARG, "%s: the cache is on device %d, the current device is %d", what, qc->device, dev);
    return SP_OK;
}

int check_batch(const sp_cuda_q8_cache_t *qc, int layer, const sp_cuda_q8_batch_t *b, const char *what)
{
    int rc = check_cache(qc, layer, what);
    if (rc) return rc;
    if (!b) return sp_set_error(SP_ERR_ARG, "%s: no batch", what);
    if (b->n_seqs < 0 || b->n_tokens < 0 || b->max_new < 0 || b->max_kv < 0 || b->max_kv > qc->max_seq_len)
        return sp_set_error(SP_ERR_ARG, "%s: batch of %d entries, %d tokens, max_new %d, max_kv %d (cache: %d positions)",
                            what, b->n_seqs, b->n_tokens, b->max_new, b->max_kv, qc->max_seq_len);
    if (!b->d_seq && b->n_seqs > qc->n_seqs)
        return sp_set_error(SP_ERR_ARG, "%s: %d entries for %d sequences", what, b->n_seqs, qc->n_seqs);
    if (b->n_seqs > 0 && (!b->d_cu || !b->d_kv_len)) return sp_set_error(SP_ERR_ARG, "%s: batch without its arrays", what);
    return SP_OK;
}

}  // namespace q8

// ---------------------------------------------------------- lifecycle --

extern "C" int sp_cuda_q8_cache_init(sp_cuda_q8_cache_t *qc, const sp_config_t *cfg, int format, int block_tokens,
                                     int n_seqs, int max_seq_len, void *stream)
{
    sp_clear_error();
    if (!qc || !cfg) return sp_set_error(SP_ERR_ARG, "q8_cache_init: NULL argument");
    memset(qc, 0, sizeof(*qc));
    if (cfg->n_layers <= 0 || cfg->n_heads_kv <= 0 || cfg->n_heads_kv > 32767 || n_seqs <= 0 || max_seq_len <= 0 ||
        max_seq_len > (1 << 30))
        return sp_set_error(SP_ERR_ARG, "q8_cache_init: bad dims");
    if (cfg->head_dim != 64 && cfg->head_dim != 128 && cfg->head_dim != 256)
        return sp_set_error(SP_ERR_UNSUPPORTED, "q8_cache_init: head_dim %d is not 64, 128 or 256", cfg->head_dim);
    if (format != SP_Q8_INT8 && format != SP_Q8_E4M3) return sp_set_error(SP_ERR_ARG, "q8_cache_init: format %d", format);
    if (block_tokens != 16 && block_tokens != 32 && block_tokens != 64 && block_tokens != 128)
        return sp_set_error(SP_ERR_UNSUPPORTED, "q8_cache_init: blocks of %d tokens, not 16, 32, 64 or 128", block_tokens);
    const long long slots = (long long)cfg->n_layers * n_seqs * cfg->n_heads_kv;
    if (slots > 0x7fffffff) return sp_set_error(SP_ERR_ARG, "q8_cache_init: bad dims");
    qc->config = *cfg;
    qc->format = format;
    qc->block_tokens = block_tokens;
    qc->n_seqs = n_seqs;
    qc->max_seq_len = (max_seq_len + 127) & ~127;
    qc->stream = stream;
    qc->n_slots = (int)slots;
    int rc = SP_OK;
    if ((rc = sp_check_cuda(cudaGetDevice(&qc->device), "q8_cache_init device")) ||
        (rc = sp_check_cuda(cudaDeviceGetAttribute(&qc->sm_count, cudaDevAttrMultiProcessorCount, qc->device),
                            "q8_cache_init device")))
        return rc;
    // One allocation, in the order of the fields; every part on a 256-byte boundary.
    auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
    const size_t codes = up((size_t)slots * qc->max_seq_len * cfg->head_dim);
    const size_t scales = up((size_t)slots * (qc->max_seq_len / block_tokens) * sizeof(float));
    qc->attn_ws_bytes = up(q8::attn_workspace_bytes(qc->sm_count, cfg->head_dim));
    char *base = nullptr;
    if ((rc = sp_check_cuda(cudaMalloc(&base, 2 * codes + 2 * scales + 256 + qc->attn_ws_bytes), "cudaMalloc q8 cache")))
        return rc;
    qc->d_k_cache = base;
    qc->d_v_cache = base + codes;
    qc->d_k_scale = (float *)(base + 2 * codes);
    qc->d_v_scale = (float *)(base + 2 * codes + scales);
    qc->d_status = (unsigned int *)(base + 2 * codes + 2 * scales);
    qc->d_attn_ws = base + 2 * codes + 2 * scales + 256;
    // of the workspace only the counters at its start have to be zero
    if ((rc = sp_check_cuda(cudaMemset(base, 0, 2 * codes + 2 * scales + 256 + q8::kCounterBytes), "q8_cache_init")) ||
        (rc = sp_check_cuda(cudaDeviceSynchronize(), "q8_cache_init"))) {
        sp_cuda_q8_cache_free(qc);
        return rc;
    }
    return SP_OK;
}

extern "C" void sp_cuda_q8_cache_free(sp_cuda_q8_cache_t *qc)
{
    if (!qc) return;
    cudaFree(qc->d_k_cache);
    qc->d_k_cache = qc->d_v_cache = nullptr;
    qc->d_k_scale = qc->d_v_scale = nullptr;
    qc->d_attn_ws = nullptr;
    qc->d_status = nullptr;
}

extern "C" int sp_cuda_q8_status(const sp_cuda_q8_cache_t *qc, unsigned int *status_out, int clear, void *stream)
{
    sp_clear_error();
    if (!qc || !qc->d_status || !status_out) return sp_set_error(SP_ERR_ARG, "q8_status: NULL argument");
    cudaStream_t s = (cudaStream_t)stream;
    int rc = sp_check_cuda(cudaMemcpyAsync(status_out, qc->d_status, 4, cudaMemcpyDeviceToHost, s), "q8_status");
    if (!rc && clear) rc = sp_check_cuda(cudaMemsetAsync(qc->d_status, 0, 4, s), "q8_status");
    if (!rc) rc = sp_check_cuda(cudaStreamSynchronize(s), "q8_status");
    return rc;
}

// --------------------------------------------------------------- write --

namespace {

struct WriteHalf {
    const void *in;      // [n_tokens][heads][hd], NULL: skipped
    uint8_t *codes;
    float *scale;
};

struct WriteArgs {
    WriteHalf h[2];
    q8::Batch b;
    long long token_stride;    // elements
    int heads, max_seq, block_log2;
    int slots, slots_each;     // (half, head) pairs of a block, and how many of them a CTA takes in turn
};

template <typename T>
struct Raw8 {                  // 8 input elements as they are in memory
    uint4 w[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ float raw_at(const Raw8<T> &r, int i)
{
    return sp_load_as_float(reinterpret_cast<const T *>(r.w), i);
}

// The largest magnitude of 8 inputs and `top`; NaN if any is NaN.
__device__ __forceinline__ float max_nan(float a, float b)
{
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
template <typename T>
struct Top;
template <>
struct Top<float> {
    float v = 0.0f;
    __device__ __forceinline__ void add(const Raw8<float> &r)
    {
#pragma unroll
        for (int i = 0; i < 8; i++) v = max_nan(v, fabsf(raw_at(r, i)));
    }
    __device__ __forceinline__ float value() const { return v; }
};
template <>
struct Top<__half> {
    __half2 v = __float2half2_rn(0.0f);
    __device__ __forceinline__ void add(const Raw8<__half> &r)
    {
        const __half2 *x = reinterpret_cast<const __half2 *>(r.w);
#pragma unroll
        for (int i = 0; i < 4; i++) v = __hmax2_nan(v, __habs2(x[i]));
    }
    __device__ __forceinline__ float value() const { return max_nan(__low2float(v), __high2float(v)); }
};
template <>
struct Top<__nv_bfloat16> {
    __nv_bfloat162 v = __float2bfloat162_rn(0.0f);
    __device__ __forceinline__ void add(const Raw8<__nv_bfloat16> &r)
    {
        const __nv_bfloat162 *x = reinterpret_cast<const __nv_bfloat162 *>(r.w);
#pragma unroll
        for (int i = 0; i < 4; i++) v = __hmax2_nan(v, __habs2(x[i]));
    }
    __device__ __forceinline__ float value() const { return max_nan(__low2float(v), __high2float(v)); }
};

// Codes of 8 values already in units of the scale; CHECKED: they may be NaN or
// pass the largest code by more than rounding.
template <int FMT, bool CHECKED>
__device__ __forceinline__ uint2 encode8(float (&x)[8])
{
    uint2 r;
    if (CHECKED) {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = x[i] == x[i] ? x[i] : 0.0f;
    }
    if constexpr (FMT == SP_Q8_INT8) {
        // adding 1.5 * 2^23 rounds to a whole number, ties to even, which then
        // stands in the low bits
        uint32_t q[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if (CHECKED) x[i] = fmaxf(fminf(x[i], 127.0f), -127.0f);
            q[i] = __float_as_uint(__fadd_rn(x[i], 12582912.0f));
        }
        r.x = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
        r.y = __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410);
    } else {
        uint32_t p[4];
#pragma unroll
        for (int i = 0; i < 4; i++)
            p[i] = __nv_cvt_float2_to_fp8x2(make_float2(x[2 * i], x[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
        r.x = __byte_perm(p[0], p[1], 0x5410);
        r.y = __byte_perm(p[2], p[3], 0x5410);
    }
    return r;
}

// One CTA for one block of one sequence, and in it one (half, head) pair after
// another; block * HD / 32 threads, each with four groups of 8 adjacent
// elements, so the input is read once and stays in registers while the CTA
// finds its maximum.  The next pair's input is on its way meanwhile.  (A cluster
// of CTAs of 256 threads for the larger blocks, joining their maxima through
// shared memory, took 1.4 times as long.)
//
// Memory and the chain load, maximum, barrier, codes, store bound it: 33042
// tokens of prompts in bf16 (8 heads of 128, blocks of 32, e4m3; 195 MB) take 39
// us, 76% of the copy rate; 8192 in 32 bits (16 heads of 256, blocks of 128,
// int8; 336 MB) 63 us, 81%.  With places and masks found anew for each pair and
// maxima joined by shuffles 47 and 77 us; one pair for each CTA, without the
// next one's input on its way, 68 and 104 us.  Single tokens of 16 sequences
// take 5.1 us back to back, most of it the call.
template <typename T, int FMT, int HD, int THREADS>
__global__ void __launch_bounds__(THREADS) k_q8_write(const __grid_constant__ WriteArgs a)
{
    constexpr int kPerToken = HD / 8;
    constexpr bool kAhead = sizeof(T) == 2 || THREADS < 1024;   // 1024 threads have 64 registers
    const int unit = blockIdx.x;
    q8::begin();

    // which sequence and block: a running sum of the blocks that each entry touches
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int blk = -1, before = 0;
    q8::Entry e = {0, 0, 0, 0};
    for (int base = 0; base < a.b.n_seqs && blk < 0; base += 32) {
        q8::Entry m = {0, 0, 0, 0};
        int n = 0;
        if (base + lane < a.b.n_seqs) {
            m = q8::entry(a.b, base + lane);
            if (m.n > m.kv_len) {                // a write cannot begin before position 0
                if (a.b.status) atomicOr(a.b.status, 1u);
                m.n = 0;
            }
            if (m.n > 0) n = ((m.kv_len - 1) >> a.block_log2) - ((m.kv_len - m.n) >> a.block_log2) + 1;
        }
        int upto = n;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += o;
        }
        const bool mine = unit >= before + upto - n && unit < before + upto;
        const unsigned who = __ballot_sync(0xffffffffu, mine);
        if (who) {
            const int src = __ffs(who) - 1;
            e.seq = __shfl_sync(0xffffffffu, m.seq, src);
            e.q0 = __shfl_sync(0xffffffffu, m.q0, src);
            e.n = __shfl_sync(0xffffffffu, m.n, src);
            e.kv_len = __shfl_sync(0xffffffffu, m.kv_len, src);
            blk = unit - (before + __shfl_sync(0xffffffffu, upto - n, src)) + ((e.kv_len - e.n) >> a.block_log2);
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (blk < 0) return;                         // the grid is an upper bound

    const int p0 = e.kv_len - e.n, lo = blk << a.block_log2;
    const bool keeps = p0 > lo;                  // older positions stay in this block
    const int s0 = blockIdx.y * a.slots_each, s1 = min(s0 + a.slots_each, a.slots);
    // maxima of the warps, which as bits are in the order of whole numbers; of two
    // pairs in turn, so that one barrier for each pair is enough
    __shared__ __align__(16) unsigned tops[2][THREADS / 32 < 4 ? 4 : THREADS / 32];
    if (warps < 4 && threadIdx.x < 8 && (threadIdx.x & 3) >= warps) tops[threadIdx.x >> 2][threadIdx.x & 3] = 0;

    // this thread's groups: of the tokens row, row + step, ..., the ones to be written
    const int row = threadIdx.x / kPerToken, step = blockDim.x / kPerToken;
    unsigned has = 0;
#pragma unroll
    for (int c = 0; c < 4; c++)
        if (lo + row + c * step >= p0 && lo + row + c * step < e.kv_len) has |= 1u << c;
    const long long in_at = (long long)(e.q0 + lo + row - p0) * a.token_stride + threadIdx.x % kPerToken * 8;
    const long long in_step = (long long)step * a.token_stride;
    int half = s0 / a.heads, head = s0 - half * a.heads, next_half = half, next_head = head;
    auto load = [&](Raw8<T>(&raw)[4]) {
        const T *src = static_cast<const T *>(a.h[next_half].in) + in_at + next_head * HD;
#pragma unroll
        for (int c = 0; c < 4; c++, src += in_step) {
            if (has >> c & 1) {
#pragma unroll
                for (int i = 0; i < (int)sizeof(T) / 2; i++) raw[c].w[i] = __ldcs(reinterpret_cast<const uint4 *>(src) + i);
            }
        }
        if (++next_head == a.heads) {
            next_head = 0;
            next_half++;
        }
    };
    auto one = [&](const Raw8<T>(&raw)[4], Raw8<T>(&next)[4], int slot) {
        const int odd = slot & 1;
        const WriteHalf &h = a.h[half];
        const long long at = (long long)e.seq * a.heads + head;
        uint8_t *codes = h.codes + (at * a.max_seq + lo) * HD;
        float *scale = h.scale + at * (a.max_seq >> a.block_log2) + blk;
        if (++head == a.heads) {
            head = 0;
            half++;
        }
        const float old = keeps ? *scale : 0.0f;
        if (kAhead && slot + 1 < s1) load(next);
        Top<T> most;
#pragma unroll
        for (int c = 0; c < 4; c++)
            if (has >> c & 1) most.add(raw[c]);
        // infinities and NaN do not count
        float top = most.value();
        bool odd_values = !(top <= 3.402823466e38f);
        if (odd_values) {
            top = 0.0f;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                if (has >> c & 1) {
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float m = fabsf(raw_at(raw[c], i));
                        if (m <= 3.402823466e38f) top = fmaxf(top, m);
                    }
                }
            }
        }
        const unsigned warp_top = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
        if (lane == 0) tops[odd][warp] = warp_top;
        odd_values = __syncthreads_or(odd_values);
        unsigned all_top = 0;
        for (int i = 0; i < warps; i += 4) {
            const uint4 w = *reinterpret_cast<const uint4 *>(&tops[odd][i]);
            all_top = max(max(all_top, max(w.x, w.y)), max(w.z, w.w));
        }
        top = __uint_as_float(all_top);

        float s = fminf(fmaxf(__fmul_rn(top, 1.0f / q8::code_max(FMT)), q8::kScaleMin), q8::kScaleMax);
        const bool grown = keeps && s > old;
        s = fmaxf(s, old);
        const float inv = __frcp_rn(s);
        // values this CTA has that are NaN or out of the codes' range
        const bool checked = odd_values || !(top * inv < q8::code_max(FMT) + 0.25f);
        if (threadIdx.x == 0) *scale = s;            // all have read the old one: the barrier above
#pragma unroll
        for (int c = 0; c < 4; c++) {
            uint2 *dst = reinterpret_cast<uint2 *>(codes) + c * blockDim.x + threadIdx.x;
            float x[8];
            if (has >> c & 1) {
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = __fmul_rn(raw_at(raw[c], i), inv);
                *dst = checked ? encode8<FMT, true>(x) : encode8<FMT, false>(x);
            } else if (grown && lo + row + c * step < p0) {
                const float ratio = __fdiv_rn(old, s);
                const uint2 w = *dst;
                const uint8_t *b = reinterpret_cast<const uint8_t *>(&w);
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = __fmul_rn(q8::decode1<FMT>(b[i]), ratio);
                *dst = encode8<FMT, true>(x);
            }
        }
    };
    Raw8<T> x[4], y[4];
    if (kAhead) {
        load(x);
        for (int slot = s0; slot < s1; slot += 2) {
            one(x, y, slot);
            if (slot + 1 < s1) one(y, x, slot + 1);
        }
    } else {
        for (int slot = s0; slot < s1; slot++) {
            load(x);
            one(x, x, slot);
        }
    }
}

template <typename T, int FMT, int HD>
int launch_write_hd(const WriteArgs &a, dim3 grid, int threads, cudaStream_t s)
{
    if (threads <= 256) return q8::launch("q8_write launch", k_q8_write<T, FMT, HD, 256>, grid, threads, 0, s, a);
    if constexpr (HD >= 128) {
        if (threads == 512) return q8::launch("q8_write launch", k_q8_write<T, FMT, HD, 512>, grid, threads, 0, s, a);
    }
    if constexpr (HD == 256) {
        if (threads == 1024) return q8::launch("q8_write launch", k_q8_write<T, FMT, HD, 1024>, grid, threads, 0, s, a);
    }
    return SP_ERR_UNSUPPORTED;
}

template <typename T, int FMT>
int launch_write(const WriteArgs &a, int hd, dim3 grid, int threads, cudaStream_t s)
{
    if (hd == 64) return launch_write_hd<T, FMT, 64>(a, grid, threads, s);
    if (hd == 128) return launch_write_hd<T, FMT, 128>(a, grid, threads, s);
    return launch_write_hd<T, FMT, 256>(a, grid, threads, s);
}

template <int FMT>
int launch_write_of(const WriteArgs &a, int dtype, int hd, dim3 grid, int threads, cudaStream_t s)
{
    if (dtype == SP_DTYPE_F32) return launch_write<float, FMT>(a, hd, grid, threads, s);
    if (dtype == SP_DTYPE_F16) return launch_write<__half, FMT>(a, hd, grid, threads, s);
    return launch_write<__nv_bfloat16, FMT>(a, hd, grid, threads, s);
}

}  // namespace

extern "C" int sp_cuda_q8_write_kv_tokens(sp_cuda_q8_cache_t *qc, int layer, const sp_cuda_q8_batch_t *batch,
                                          const void *d_k, const void *d_v, long long token_stride, int dtype)
{
    sp_clear_error();
    int rc = q8::check_batch(qc, layer, batch, "q8_write");
    if (rc) return rc;
    if (dtype != SP_DTYPE_F32 && dtype != SP_DTYPE_F16 && dtype != SP_DTYPE_BF16)
        return sp_set_error(SP_ERR_ARG, "q8_write: dtype %d", dtype);
    const int H = qc->config.n_heads_kv, hd = qc->config.head_dim;
    const long long el = dtype == SP_DTYPE_F32 ? 4 : 2;
    if (token_stride == 0) token_stride = (long long)H * hd;
    if (token_stride < (long long)H * hd)
        return sp_set_error(SP_ERR_ARG, "q8_write: a token's stride is less than its rows");
    if (((uintptr_t)d_k | (uintptr_t)d_v | (uintptr_t)(token_stride * el)) % 16)
        return sp_set_error(SP_ERR_ARG, "q8_write: pointers and strides must be multiples of 16 bytes");
    if (batch->n_tokens == 0 || batch->n_seqs == 0 || batch->max_new == 0 || (!d_k && !d_v)) return SP_OK;

    const q8::Layer l = q8::layer_of(qc, layer);
    WriteArgs a;
    a.b = q8::batch_of(qc, batch);
    a.token_stride = token_stride;
    a.heads = H;
    a.max_seq = l.max_seq;
    a.block_log2 = l.block_log2;
    int n = 0;
    if (d_k) a.h[n++] = {d_k, const_cast<uint8_t *>(l.k), const_cast<float *>(l.k_scale)};
    if (d_v) a.h[n++] = {d_v, const_cast<uint8_t *>(l.v), const_cast<float *>(l.v_scale)};
    // Blocks touched at most: an entry's tokens may begin and end inside one.
    const long long B = qc->block_tokens;
    const long long each = batch->n_seqs * ((batch->max_new + B - 2) / B + 1);
    const long long all = batch->n_tokens / B + 2ll * batch->n_seqs;
    const long long units = each < all ? each : all;
    if (units > 0x7fffffff / 4) return sp_set_error(SP_ERR_ARG, "q8_write: %lld blocks in one call", units);
    a.slots = n * H;
    const int threads = (int)(B * hd / 32);
    // Pairs in turn where there are blocks enough to fill the SMs' threads more
    // than twice over (prompts of the kernel's comment: 39 us for 6 in turn, 45 for
    // 2; its 32-bit inputs: 63 us for 7, 66 for 2, 69 for 1): a step of single
    // tokens wants a CTA for each instead.
    long long in_turn = units * a.slots * threads / (2048ll * qc->sm_count);
    in_turn = in_turn < 1 ? 1 : in_turn > 16 ? 16 : in_turn;
    a.slots_each = (int)(in_turn < a.slots ? in_turn : a.slots);
    const dim3 grid((unsigned)units, (a.slots + a.slots_each - 1) / a.slots_each);
    cudaStream_t s = (cudaStream_t)qc->stream;
    return qc->format == SP_Q8_INT8 ? launch_write_of<SP_Q8_INT8>(a, dtype, hd, grid, threads, s)
                                    : launch_write_of<SP_Q8_E4M3>(a, dtype, hd, grid, threads, s);
}

// ---------------------------------------------------------------- read --

namespace {

constexpr int kReadThreads = 256, kReadUnits = 4;

struct ReadArgs {
    const uint8_t *codes;          // of the sequence's first head
    const float *scale;
    void *out;
    int heads, max_seq, hd_log2, block_log2, start;
    unsigned n;                    // units of a head
};

// The values of 8 codes (4 of them where x.y is not given).
template <int FMT, int E>
__device__ __forceinline__ void decode8(uint2 c, float (&x)[8])
{
#pragma unroll
    for (int w = 0; w < E / 4; w++) {
        const uint32_t v = w ? c.y : c.x;
        if constexpr (FMT == SP_Q8_INT8) {
            // q + 128 in the low bits of 2^23
            const uint32_t u = v ^ 0x80808080u;
#pragma unroll
            for (int i = 0; i < 4; i++)
                x[4 * w + i] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7540 + i)) - 8388736.0f;
        } else {
            uint32_t a, b;
            asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
                : "=r"(a), "=r"(b) : "r"(v));
            const float2 p = __half22float2(*reinterpret_cast<const __half2 *>(&a)), q = __half22float2(*reinterpret_cast<const __half2 *>(&b));
            x[4 * w] = p.x; x[4 * w + 1] = p.y; x[4 * w + 2] = q.x; x[4 * w + 3] = q.y;
        }
    }
}

// A row of CTAs for each head.  Each thread turns kReadUnits units of codes (16
// bytes of values each) into values; a warp's loads and stores of one unit are
// contiguous within a position.  Memory bounds it: 32768 positions of 8 heads
// of 128, K and V, 201 MB with their values in bf16, in 36 to 41 us, 75 to 85% of
// the copy rate (a unit for each thread, heads in turn within a position: 97 us).
template <typename T, int FMT>
__global__ void __launch_bounds__(kReadThreads) k_q8_read(const __grid_constant__ ReadArgs a)
{
    constexpr int E = 16 / sizeof(T);              // codes of a unit
    q8::begin();
    const int unit_log2 = a.hd_log2 - (E == 8 ? 3 : 2);
    const int head = blockIdx.y;
    const uint8_t *codes = a.codes + (((long long)head * a.max_seq + a.start) << a.hd_log2);
    const float *scale = a.scale + (long long)head * (a.max_seq >> a.block_log2);
    char *out = (char *)a.out + ((long long)head << a.hd_log2) * sizeof(T);
    const long long row_bytes = ((long long)a.heads << a.hd_log2) * sizeof(T);
    uint2 c[kReadUnits];
    float s[kReadUnits];
    const unsigned u0 = blockIdx.x * (kReadThreads * kReadUnits) + threadIdx.x;
#pragma unroll
    for (int k = 0; k < kReadUnits; k++) {
        const unsigned u = u0 + k * kReadThreads;
        if (u < a.n) {
            if constexpr (E == 8) c[k] = __ldcs(reinterpret_cast<const uint2 *>(codes) + u);
            else c[k].x = __ldcs(reinterpret_cast<const unsigned *>(codes) + u);
            s[k] = scale[(a.start + (u >> unit_log2)) >> a.block_log2];
        }
    }
#pragma unroll
    for (int k = 0; k < kReadUnits; k++) {
        const unsigned u = u0 + k * kReadThreads;
        if (u < a.n) {
            float v[8];
            decode8<FMT, E>(c[k], v);
            uint4 w;
            T *x = reinterpret_cast<T *>(&w);
#pragma unroll
            for (int i = 0; i < E; i++) x[i] = T(v[i] * s[k]);
            const unsigned t = u >> unit_log2;
            __stcs(reinterpret_cast<uint4 *>(out + t * row_bytes) + (u - (t << unit_log2)), w);
        }
    }
}

template <int FMT>
int launch_read(const ReadArgs &a, int dtype, cudaStream_t s)
{
    const dim3 grid((a.n + kReadThreads * kReadUnits - 1) / (kReadThreads * kReadUnits), a.heads);
    return q8::launch("q8_read launch", dtype == SP_DTYPE_F32 ? k_q8_read<float, FMT> : dtype == SP_DTYPE_F16 ? k_q8_read<__half, FMT> : k_q8_read<__nv_bfloat16, FMT>,
                      grid, kReadThreads, 0, s, a);
}

}  // namespace

extern "C" int sp_cuda_q8_read_kv_tokens(const sp_cuda_q8_cache_t *qc, int which, int layer, int seq, int start_pos,
                                         int n_tok, void *d_out, int dtype)
{
    sp_clear_error();
    int rc = q8::check_cache(qc, layer, "q8_read");
    if (rc) return rc;
    if (which != 0 && which != 1) return sp_set_error(SP_ERR_ARG, "q8_read: which must be 0 (K) or 1 (V)");
    if (dtype != SP_DTYPE_F32 && dtype != SP_DTYPE_F16 && dtype != SP_DTYPE_BF16)
        return sp_set_error(SP_ERR_ARG, "q8_read: dtype %d", dtype);
    if (seq < 0 || seq >= qc->n_seqs) return sp_set_error(SP_ERR_ARG, "q8_read: sequence %d out of range", seq);
    if (start_pos < 0 || n_tok < 0 || (long long)start_pos + n_tok > qc->max_seq_len)
        return sp_set_error(SP_ERR_ARG, "q8_read: %d positions from %d are outside the cache", n_tok, start_pos);
    if (n_tok == 0) return SP_OK;
    if (!d_out || (uintptr_t)d_out % 16) return sp_set_error(SP_ERR_ARG, "q8_read: the output must be 16-byte aligned");
    const q8::Layer l = q8::layer_of(qc, layer);
    const int hd = qc->config.head_dim, hd_log2 = hd == 64 ? 6 : hd == 128 ? 7 : 8;
    const long long slot = (long long)seq * l.heads;
    const uint8_t *codes = (which ? l.v : l.k) + slot * l.max_seq * hd;
    const float *scale = (which ? l.v_scale : l.k_scale) + slot * (l.max_seq >> l.block_log2);
    const int el = dtype == SP_DTYPE_F32 ? 4 : 2;
    const int per = hd * el / 16;                    // units of a position and head
    cudaStream_t s = (cudaStream_t)qc->stream;
    // as many positions at a time as 32-bit unit numbers reach
    const int most = 0x7fffffff / per;
    for (long long t = 0; t < n_tok; t += most) {
        ReadArgs a = {codes, scale, (char *)d_out + t * per * l.heads * 16, l.heads, l.max_seq, hd_log2, l.block_log2,
                      (int)(start_pos + t), (unsigned)((n_tok - t < most ? n_tok - t : most) * per)};
        rc = qc->format == SP_Q8_INT8 ? launch_read<SP_Q8_INT8>(a, dtype, s) : launch_read<SP_Q8_E4M3>(a, dtype, s);
        if (rc) return rc;
    }
    return SP_OK;
}
