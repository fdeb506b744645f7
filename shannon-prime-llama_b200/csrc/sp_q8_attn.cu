// sp_q8_attn.cu — attention over the 8-bit cache (shannon_prime_q8.h).
#include "sp_q8.cuh"

#include <math.h>

namespace q8 {
size_t attn_workspace_bytes(int sm_count, int head_dim)
{
    (void)sm_count;
    (void)head_dim;
    return 256;
}
}  // namespace q8

namespace {

struct AttnArgs {
    q8::Layer l;
    q8::Batch b;
    const void *q;
    void *out;
    float *lse;
    long long q_stride, out_stride;
    int n_q_heads, group;
    float scale;
    int causal, window;
};

// One warp for each (token, query head): one pass over the positions that the
// token sees with a running maximum and sum, a lane holding every 32nd
// element of the head.
template <typename T, int FMT, int HD>
__global__ void __launch_bounds__(128) k_q8_attn_rows(const __grid_constant__ AttnArgs a)
{
    const long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    const int t = (int)(unit / a.n_q_heads), g = (int)(unit - (long long)t * a.n_q_heads);
    if (t >= a.b.n_tokens) return;
    q8::Entry e = {0, 0, 0, 0};
    for (int i = 0; i < a.b.n_seqs; i++) {
        const q8::Entry m = q8::entry(a.b, i);
        if (m.n > 0 && t >= m.q0 && t < m.q0 + m.n) { e = m; break; }
    }
    if (e.n == 0) return;
    const int pos = e.kv_len - e.n + t - e.q0;
    const int end = a.causal ? pos + 1 : e.kv_len;
    const int begin = a.window > 0 && pos - a.window + 1 > 0 ? pos - a.window + 1 : 0;
    const long long slot = (long long)e.seq * a.l.heads + g / a.group;
    const uint8_t *k = a.l.k + slot * a.l.max_seq * HD, *v = a.l.v + slot * a.l.max_seq * HD;
    const float *ks = a.l.k_scale + slot * (a.l.max_seq >> a.l.block_log2);
    const float *vs = a.l.v_scale + slot * (a.l.max_seq >> a.l.block_log2);
    const T *q = static_cast<const T *>(a.q) + t * a.q_stride + g * HD;
    float qr[HD / 32], acc[HD / 32], m = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < HD / 32; i++) {
        qr[i] = sp_load_as_float(q, lane + 32 * i) * a.scale;
        acc[i] = 0.0f;
    }
    for (int j = begin; j < end; j++) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < HD / 32; i++) s += qr[i] * q8::decode1<FMT>(k[(long long)j * HD + lane + 32 * i]);
#pragma unroll
        for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        s *= ks[j >> a.l.block_log2];
        const float top = fmaxf(m, s), fix = expf(m - top), p = expf(s - top);
        m = top;
        sum = sum * fix + p;
        const float w = p * vs[j >> a.l.block_log2];
#pragma unroll
        for (int i = 0; i < HD / 32; i++)
            acc[i] = acc[i] * fix + w * q8::decode1<FMT>(v[(long long)j * HD + lane + 32 * i]);
    }
    T *out = static_cast<T *>(a.out) + t * a.out_stride + g * HD;
    const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
    for (int i = 0; i < HD / 32; i++) out[lane + 32 * i] = T(acc[i] * inv);
    if (a.lse && lane == 0) a.lse[(long long)t * a.n_q_heads + g] = m + logf(sum);
}

template <typename T, int FMT>
void launch_rows(const AttnArgs &a, int hd, unsigned grid, cudaStream_t s)
{
    if (hd == 64) k_q8_attn_rows<T, FMT, 64><<<grid, 128, 0, s>>>(a);
    else if (hd == 128) k_q8_attn_rows<T, FMT, 128><<<grid, 128, 0, s>>>(a);
    else k_q8_attn_rows<T, FMT, 256><<<grid, 128, 0, s>>>(a);
}

}  // namespace

extern "C" int sp_cuda_q8_attn(const sp_cuda_q8_cache_t *qc, int layer, const sp_cuda_q8_batch_t *batch, const void *d_q,
                               long long q_stride, int n_q_heads, int dtype, float logit_scale, int causal, int window,
                               void *d_out, long long out_stride, float *d_lse, void *stream)
{
    sp_clear_error();
    int rc = q8::check_batch(qc, layer, batch, "q8_attn");
    if (rc) return rc;
    if (dtype != SP_DTYPE_F16 && dtype != SP_DTYPE_BF16)
        return sp_set_error(SP_ERR_UNSUPPORTED, "q8_attn: dtype %d, not fp16 or bf16", dtype);
    const int H = qc->config.n_heads_kv, hd = qc->config.head_dim;
    if (n_q_heads <= 0 || n_q_heads % H || n_q_heads / H > 128)
        return sp_set_error(SP_ERR_ARG, "q8_attn: %d query heads for %d KV heads", n_q_heads, H);
    if (!isfinite(logit_scale)) return sp_set_error(SP_ERR_ARG, "q8_attn: logit scale %g", (double)logit_scale);
    if (window < 0 || (window && !causal)) return sp_set_error(SP_ERR_ARG, "q8_attn: window %d", window);
    if (q_stride == 0) q_stride = (long long)n_q_heads * hd;
    if (out_stride == 0) out_stride = (long long)n_q_heads * hd;
    if (q_stride < (long long)n_q_heads * hd || out_stride < (long long)n_q_heads * hd)
        return sp_set_error(SP_ERR_ARG, "q8_attn: a token's stride is less than its rows");
    if (batch->n_tokens == 0 || batch->n_seqs == 0 || batch->max_new == 0) return SP_OK;
    if (!d_q || !d_out) return sp_set_error(SP_ERR_ARG, "q8_attn: NULL argument");
    if (((uintptr_t)d_q | (uintptr_t)d_out | (uintptr_t)(q_stride * 2) | (uintptr_t)(out_stride * 2)) % 16 || (uintptr_t)d_lse % 4)
        return sp_set_error(SP_ERR_ARG, "q8_attn: pointers and strides must be multiples of 16 bytes");
    AttnArgs a = {q8::layer_of(qc, layer), q8::batch_of(qc, batch), d_q, d_out, d_lse, q_stride, out_stride,
                  n_q_heads, n_q_heads / H, logit_scale, causal, window};
    const long long units = (long long)batch->n_tokens * n_q_heads;
    if (units > 0x7fffffff) return sp_set_error(SP_ERR_ARG, "q8_attn: %lld rows in one call", units);
    const unsigned grid = (unsigned)((units + 3) / 4);
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == SP_DTYPE_F16) {
        if (qc->format == SP_Q8_INT8) launch_rows<__half, SP_Q8_INT8>(a, hd, grid, s);
        else launch_rows<__half, SP_Q8_E4M3>(a, hd, grid, s);
    } else {
        if (qc->format == SP_Q8_INT8) launch_rows<__nv_bfloat16, SP_Q8_INT8>(a, hd, grid, s);
        else launch_rows<__nv_bfloat16, SP_Q8_E4M3>(a, hd, grid, s);
    }
    return sp_check_cuda(cudaGetLastError(), "q8_attn launch");
}
