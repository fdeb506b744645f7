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
    if (cfg->n_layers <= 0 || cfg->n_heads_kv <= 0 || n_seqs <= 0 || max_seq_len <= 0 || max_seq_len > (1 << 30))
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
    const size_t codes = (size_t)slots * qc->max_seq_len * cfg->head_dim;
    const size_t scales = (size_t)slots * (qc->max_seq_len / block_tokens) * sizeof(float);
    qc->attn_ws_bytes = q8::attn_workspace_bytes(qc->sm_count, cfg->head_dim);
    if ((rc = sp_check_cuda(cudaMalloc(&qc->d_k_cache, codes), "cudaMalloc q8 K")) ||
        (rc = sp_check_cuda(cudaMalloc(&qc->d_v_cache, codes), "cudaMalloc q8 V")) ||
        (rc = sp_check_cuda(cudaMalloc(&qc->d_k_scale, scales), "cudaMalloc q8 K scales")) ||
        (rc = sp_check_cuda(cudaMalloc(&qc->d_v_scale, scales), "cudaMalloc q8 V scales")) ||
        (rc = sp_check_cuda(cudaMalloc(&qc->d_attn_ws, qc->attn_ws_bytes), "cudaMalloc q8 workspace")) ||
        (rc = sp_check_cuda(cudaMalloc(&qc->d_status, 16), "cudaMalloc q8 status")) ||
        (rc = sp_check_cuda(cudaMemset(qc->d_k_cache, 0, codes), "q8_cache_init")) ||
        (rc = sp_check_cuda(cudaMemset(qc->d_v_cache, 0, codes), "q8_cache_init")) ||
        (rc = sp_check_cuda(cudaMemset(qc->d_k_scale, 0, scales), "q8_cache_init")) ||
        (rc = sp_check_cuda(cudaMemset(qc->d_v_scale, 0, scales), "q8_cache_init")) ||
        (rc = sp_check_cuda(cudaMemset(qc->d_attn_ws, 0, qc->attn_ws_bytes), "q8_cache_init")) ||
        (rc = sp_check_cuda(cudaMemset(qc->d_status, 0, 16), "q8_cache_init")) ||
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
    cudaFree(qc->d_v_cache);
    cudaFree(qc->d_k_scale);
    cudaFree(qc->d_v_scale);
    cudaFree(qc->d_attn_ws);
    cudaFree(qc->d_status);
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

// Codes of 8 values already in units of the scale.
template <int FMT>
__device__ __forceinline__ uint2 encode8(const float (&x)[8])
{
    uint2 r;
    if constexpr (FMT == SP_Q8_INT8) {
        // adding 1.5 * 2^23 rounds to a whole number, ties to even, which then
        // stands in the low bits
        uint32_t q[8];
#pragma unroll
        for (int i = 0; i < 8; i++)
            q[i] = __float_as_uint(__fadd_rn(fmaxf(fminf(x[i], 127.0f), -127.0f), 12582912.0f));
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

// One CTA for one block of one sequence, head and half; block * HD / 32
// threads, each with four groups of 8 adjacent elements, so the block's input
// is read once and stays in registers while its maximum is found.
template <typename T, int FMT, int HD>
__global__ void __launch_bounds__(1024) k_q8_write(const __grid_constant__ WriteArgs a)
{
    constexpr int kPerToken = HD / 8;
    const WriteHalf &h = a.h[blockIdx.y];
    const int unit = blockIdx.x / a.heads, head = blockIdx.x - unit * a.heads;
    const int B = 1 << a.block_log2;

    // which sequence and block: a running sum of the blocks that each entry touches
    const int lane = threadIdx.x & 31;
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
    const long long slot = (long long)e.seq * a.heads + head;
    uint8_t *codes = h.codes + (slot * a.max_seq + lo) * HD;
    float *scale = h.scale + slot * (a.max_seq >> a.block_log2) + blk;
    const bool keeps = p0 > lo;                  // older positions stay in this block
    const float old = keeps ? *scale : 0.0f;

    Raw8<T> raw[4];
    float top = 0.0f;
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const int g = c * blockDim.x + threadIdx.x;
        const int pos = lo + g / kPerToken;
        if (pos >= p0 && pos < e.kv_len) {
            const T *src = static_cast<const T *>(h.in) + (long long)(e.q0 + pos - p0) * a.token_stride + head * HD +
                           (g % kPerToken) * 8;
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; i++) raw[c].w[i] = reinterpret_cast<const uint4 *>(src)[i];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float m = fabsf(raw_at(raw[c], i));
                if (m <= 3.402823466e38f) top = fmaxf(top, m);    // neither infinity nor NaN
            }
        }
    }
    __shared__ float tops[32];
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    if (lane == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
    top = 0.0f;
    for (int i = 0; i < (int)(blockDim.x >> 5); i++) top = fmaxf(top, tops[i]);

    float s = fminf(fmaxf(__fmul_rn(top, 1.0f / q8::code_max(FMT)), q8::kScaleMin), q8::kScaleMax);
    const bool grown = keeps && s > old;
    s = fmaxf(s, old);
    const float inv = __frcp_rn(s), ratio = __fdiv_rn(old, s);
    if (threadIdx.x == 0) *scale = s;            // all have read the old one: the barrier above
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const int g = c * blockDim.x + threadIdx.x;
        const int pos = lo + g / kPerToken;
        uint2 *dst = reinterpret_cast<uint2 *>(codes + (long long)g * 8);
        float x[8];
        if (pos >= p0 && pos < e.kv_len) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float v = __fmul_rn(raw_at(raw[c], i), inv);
                x[i] = v == v ? v : 0.0f;
            }
            *dst = encode8<FMT>(x);
        } else if (grown && pos < p0) {
            const uint2 w = *dst;
            const uint8_t *b = reinterpret_cast<const uint8_t *>(&w);
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = __fmul_rn(q8::decode1<FMT>(b[i]), ratio);
            *dst = encode8<FMT>(x);
        }
    }
}

template <typename T, int FMT>
void launch_write(const WriteArgs &a, int hd, dim3 grid, int threads, cudaStream_t s)
{
    if (hd == 64) k_q8_write<T, FMT, 64><<<grid, threads, 0, s>>>(a);
    else if (hd == 128) k_q8_write<T, FMT, 128><<<grid, threads, 0, s>>>(a);
    else k_q8_write<T, FMT, 256><<<grid, threads, 0, s>>>(a);
}

template <int FMT>
void launch_write_of(const WriteArgs &a, int dtype, int hd, dim3 grid, int threads, cudaStream_t s)
{
    if (dtype == SP_DTYPE_F32) launch_write<float, FMT>(a, hd, grid, threads, s);
    else if (dtype == SP_DTYPE_F16) launch_write<__half, FMT>(a, hd, grid, threads, s);
    else launch_write<__nv_bfloat16, FMT>(a, hd, grid, threads, s);
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
    const long long units = (each < all ? each : all) * H;
    if (units > 0x7fffffff) return sp_set_error(SP_ERR_ARG, "q8_write: %lld blocks in one call", units);
    const dim3 grid((unsigned)units, n);
    const int threads = (int)(B * hd / 32);
    cudaStream_t s = (cudaStream_t)qc->stream;
    if (qc->format == SP_Q8_INT8) launch_write_of<SP_Q8_INT8>(a, dtype, hd, grid, threads, s);
    else launch_write_of<SP_Q8_E4M3>(a, dtype, hd, grid, threads, s);
    return sp_check_cuda(cudaGetLastError(), "q8_write launch");
}

// ---------------------------------------------------------------- read --

namespace {

constexpr int kReadThreads = 256;

// Each thread turns four codes into four values; a warp's loads and stores
// are contiguous.
template <typename T, int FMT>
__global__ void __launch_bounds__(kReadThreads)
k_q8_read(const uint8_t *codes, const float *scale, int heads, int max_seq, int hd_log2, int block_log2, int start,
          long long n, T *out)
{
    for (long long i = (long long)blockIdx.x * kReadThreads + threadIdx.x; i < n; i += (long long)gridDim.x * kReadThreads) {
        const long long el = i * 4, row = el >> hd_log2;
        const int d = (int)(el - (row << hd_log2));
        const int t = (int)(row / heads), head = (int)(row - (long long)t * heads);
        const int pos = start + t;
        const uchar4 c = *reinterpret_cast<const uchar4 *>(codes + ((((long long)head * max_seq + pos) << hd_log2) + d));
        const float s = scale[(long long)head * (max_seq >> block_log2) + (pos >> block_log2)];
        const float x[4] = {q8::decode1<FMT>(c.x) * s, q8::decode1<FMT>(c.y) * s, q8::decode1<FMT>(c.z) * s,
                            q8::decode1<FMT>(c.w) * s};
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4 *>(out + el) = make_float4(x[0], x[1], x[2], x[3]);
        } else {
            uint2 w;
            T *e = reinterpret_cast<T *>(&w);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if constexpr (sizeof(T) == 2) e[j] = T(x[j]);
            }
            *reinterpret_cast<uint2 *>(out + el) = w;
        }
    }
}

template <int FMT>
void launch_read(const uint8_t *codes, const float *scale, int heads, int max_seq, int hd_log2, int block_log2, int start,
                 long long n, void *out, int dtype, unsigned grid, cudaStream_t s)
{
    if (dtype == SP_DTYPE_F32)
        k_q8_read<float, FMT><<<grid, kReadThreads, 0, s>>>(codes, scale, heads, max_seq, hd_log2, block_log2, start, n, (float *)out);
    else if (dtype == SP_DTYPE_F16)
        k_q8_read<__half, FMT><<<grid, kReadThreads, 0, s>>>(codes, scale, heads, max_seq, hd_log2, block_log2, start, n, (__half *)out);
    else
        k_q8_read<__nv_bfloat16, FMT><<<grid, kReadThreads, 0, s>>>(codes, scale, heads, max_seq, hd_log2, block_log2, start, n,
                                                                  (__nv_bfloat16 *)out);
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
    const long long n = (long long)n_tok * l.heads * hd / 4;
    const long long ctas = (n + kReadThreads - 1) / kReadThreads;
    const unsigned grid = (unsigned)(ctas < 0x7fffffff ? ctas : 0x7fffffff);
    cudaStream_t s = (cudaStream_t)qc->stream;
    if (qc->format == SP_Q8_INT8)
        launch_read<SP_Q8_INT8>(codes, scale, l.heads, l.max_seq, hd_log2, l.block_log2, start_pos, n, d_out, dtype, grid, s);
    else
        launch_read<SP_Q8_E4M3>(codes, scale, l.heads, l.max_seq, hd_log2, l.block_log2, start_pos, n, d_out, dtype, grid, s);
    return sp_check_cuda(cudaGetLastError(), "q8_read launch");
}
