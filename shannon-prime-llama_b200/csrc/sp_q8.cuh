// sp_q8.cuh — what the kernels of the 8-bit cache share (shannon_prime_q8.h).
#pragma once

#include "sp_internal.cuh"
#include "shannon_prime_q8.h"

#include <cuda_fp8.h>

namespace q8 {

constexpr int kMaxCtas = 1024;               // most CTAs of an attention grid
constexpr size_t kCounterBytes = kMaxCtas * sizeof(unsigned);   // at the start of its workspace

constexpr float kScaleMin = 0x1p-40f, kScaleMax = 0x1p40f;

__host__ __device__ constexpr float code_max(int format) { return format == SP_Q8_INT8 ? 127.0f : 448.0f; }

// Every kernel of this tier is launched as a programmatic dependent: the next
// one's CTAs are placed while the last one's finish (about 2 us of a step's short
// kernels).  begin() stands before any access to memory: it waits until all
// earlier work of the stream is over and seen, and only then lets the next
// kernel be placed, so nothing that starts early finds unfinished work behind it.
__device__ __forceinline__ void begin()
{
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

template <typename... P, typename... A>
int launch(const char *what, void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t s, const A &...a)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return sp_check_cuda(cudaLaunchKernelEx(&cfg, kernel, a...), what);
}

// One layer of a cache.
struct Layer {
    const uint8_t *k, *v;          // [n_seqs][heads][max_seq][hd]
    const float *k_scale, *v_scale;  // [n_seqs][heads][max_seq / block]
    int n_seqs, heads, max_seq;
    int block_log2;
};

inline Layer layer_of(const sp_cuda_q8_cache_t *qc, int layer)
{
    Layer l;
    const long long per = (long long)qc->n_seqs * qc->config.n_heads_kv * qc->max_seq_len;
    l.k = (const uint8_t *)qc->d_k_cache + layer * per * qc->config.head_dim;
    l.v = (const uint8_t *)qc->d_v_cache + layer * per * qc->config.head_dim;
    l.k_scale = qc->d_k_scale + layer * (per / qc->block_tokens);
    l.v_scale = qc->d_v_scale + layer * (per / qc->block_tokens);
    l.n_seqs = qc->n_seqs;
    l.heads = qc->config.n_heads_kv;
    l.max_seq = qc->max_seq_len;
    l.block_log2 = 0;
    while ((1 << l.block_log2) < qc->block_tokens) l.block_log2++;
    return l;
}

// The batch as the kernels see it, with the cache's number of sequences.
struct Batch {
    int n_seqs, n_tokens, max_new, max_kv, cache_seqs;
    const int *seq, *cu, *kv_len;
    unsigned int *status;
};

inline Batch batch_of(const sp_cuda_q8_cache_t *qc, const sp_cuda_q8_batch_t *b)
{
    return {b->n_seqs, b->n_tokens, b->max_new, b->max_kv, qc->n_seqs, b->d_seq, b->d_cu, b->d_kv_len, qc->d_status};
}

// Host-side checks of a batch (sp_q8.cu).
int check_batch(const sp_cuda_q8_cache_t *qc, int layer, const sp_cuda_q8_batch_t *b, const char *what);

// Entry i of the batch; n == 0 where it has no tokens or is out of range (the
// status word then says so).
struct Entry {
    int seq, q0, n, kv_len;
};

__device__ __forceinline__ Entry entry(const Batch &b, int i)
{
    Entry e;
    e.seq = b.seq ? b.seq[i] : i;
    e.q0 = b.cu[i];
    const int q1 = b.cu[i + 1];
    e.kv_len = b.kv_len[i];
    e.n = q1 - e.q0;
    const bool ok = e.q0 >= 0 && e.q0 <= q1 && q1 <= b.n_tokens && e.n <= b.max_new && e.kv_len >= 0 &&
                    e.kv_len <= b.max_kv && e.seq >= 0 && e.seq < b.cache_seqs;
    if (!ok) {
        if (b.status) atomicOr(b.status, 1u);
        e.n = 0;
        e.kv_len = 0;
        e.seq = 0;
        e.q0 = 0;
    }
    return e;
}

// The value of one code.
template <int FMT>
__device__ __forceinline__ float decode1(uint8_t c)
{
    if constexpr (FMT == SP_Q8_INT8) return (float)(int8_t)c;
    else return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}

}  // namespace q8
