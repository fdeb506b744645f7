// sp_q8_attn_many.cu — attention over the 8-bit cache for many rows (prompts
// and chunks of prompts).
#include "sp_q8_attn.cuh"

namespace {

using namespace q8;

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
    Entry e = {0, 0, 0, 0};
    for (int i = 0; i < a.b.n_seqs; i++) {
        const Entry m = entry(a.b, i);
        if (m.n > 0 && t >= m.q0 && t < m.q0 + m.n) { e = m; break; }
    }
    if ((long long)e.n * a.group <= a.few_rows) return;
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
        for (int i = 0; i < HD / 32; i++) s += qr[i] * decode1<FMT>(k[(long long)j * HD + lane + 32 * i]);
#pragma unroll
        for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        s *= ks[j >> a.l.block_log2];
        const float top = fmaxf(m, s), fix = expf(m - top), p = expf(s - top);
        m = top;
        sum = sum * fix + p;
        const float w = p * vs[j >> a.l.block_log2];
#pragma unroll
        for (int i = 0; i < HD / 32; i++)
            acc[i] = acc[i] * fix + w * decode1<FMT>(v[(long long)j * HD + lane + 32 * i]);
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

namespace q8 {
int launch_many(const AttnArgs &a, int format, int dtype, int hd, int sms, cudaStream_t s)
{
    (void)sms;
    const long long units = (long long)a.b.n_tokens * a.n_q_heads;
    if (units > 0x7fffffff) return sp_set_error(SP_ERR_ARG, "q8_attn: %lld rows in one call", units);
    const unsigned grid = (unsigned)((units + 3) / 4);
    if (dtype == SP_DTYPE_F16) {
        if (format == SP_Q8_INT8) launch_rows<__half, SP_Q8_INT8>(a, hd, grid, s);
        else launch_rows<__half, SP_Q8_E4M3>(a, hd, grid, s);
    } else {
        if (format == SP_Q8_INT8) launch_rows<__nv_bfloat16, SP_Q8_INT8>(a, hd, grid, s);
        else launch_rows<__nv_bfloat16, SP_Q8_E4M3>(a, hd, grid, s);
    }
    return sp_check_cuda(cudaGetLastError(), "q8_attn launch");
}
}  // namespace q8
