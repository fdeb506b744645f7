// sp_q8_attn.cu — attention over the 8-bit cache (shannon_prime_q8.h): the
// entry point and the kernel for few rows (single tokens, draft tokens).
#include "sp_q8_attn.cuh"

#include <math.h>

#include <atomic>

namespace {

using namespace q8;

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kTile = 16 * kWarps;       // positions of a tile: 16 for each warp

__device__ __forceinline__ void copy_async16(uint32_t dst, const uint8_t *src)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x)
{
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// Tiles of one (entry, KV head): the positions that any of its rows sees, from
// a multiple of 16 on.  At least one, so that rows that see nothing are written.
struct Unit0 {
    int start, end, tiles;
};
__device__ __forceinline__ Unit0 unit_of(const AttnArgs &a, const Entry &e)
{
    Unit0 u = {0, e.kv_len, 0};
    if (e.n <= 0 || (long long)e.n * a.group > a.few_rows) return u;
    const int first = e.kv_len - e.n;
    if (a.window > 0 && first - a.window + 1 > 0) u.start = (first - a.window + 1) & ~15;
    u.tiles = max(1, (u.end - u.start + kTile - 1) / kTile);
    return u;
}

// A warp's stage: 16 rows of K and of V as they are in memory, rows a little
// apart so that the fragments' reads fall on different banks.
template <int HD>
struct Stage {
    static constexpr int KPitch = HD + 16, VPitch = HD + 16;
    static constexpr int Bytes = 16 * (KPitch + VPitch);
};

template <int HD, int NT, int STAGES>
struct FewSmem {
    unsigned char ring[kWarps][STAGES][Stage<HD>::Bytes];
    uint2 q[NT][HD / 16][32];                 // query fragments, one 8-byte word a lane
    float mul[8 * NT];                        // each row's factor of the scores, in base 2
    float m[kWarps][8 * NT], l[kWarps][8 * NT];
    float o[4][8 * NT][HD + 4];               // + 4: rows on different banks
    unsigned scan[kWarps], found[3];
    int last;
};

// Rows of a unit are its new tokens times the query heads that share the KV
// head, up to 8 NT of them.  A warp takes 16 positions at a time and works on
// the transposed problem, S' = K q' and O' += V' P, so that positions and head
// dimensions fill the 16-row side of mma.sync.m16n8k16 and the few rows its
// 8-column side.  Codes go from memory to registers in the order in which the
// fragments need them (a dimension's place in the product is free as long as
// the queries have the same), become fp16 there, exactly, and meet fp16
// queries scaled by a power of two to fit.  The score fragment becomes the
// weight fragment by one movmatrix.
//
// Softmax in base 2 with the block's V scale folded into the exponent: weights
// are w = 2^(s + log2 vs - m), m a running maximum of s + log2 vs (raised only
// when a score passes it by 2^8, so w <= 2^8 and seldom rescaled); they are
// rounded to fp16 for the product alone, relative to what they contribute,
// and the sum of the unscaled weights is kept beside them in 32 bits as
// sum w / vs.
//
// Measured: 16 sequences of 5693 to 32768 positions, one token each, 32 query
// heads on 8 of 128 dimensions, e4m3: 118 us for 653 MB, 5.5 TB/s (84% of the
// card's copy rate): memory bounds it, and what is left is the start of the
// runs and their join.  With up to 32 rows (4 draft tokens, 32 query heads on 4
// of 64 dimensions, int8; 48 sequences of 1296 to 9005) the 129 MB take 73 us:
// about 470 instructions of a warp for 16 positions, issued in half of the
// cycles by the 16 warps that the registers of 32 rows' accumulators leave an
// SM.  Copies go into a ring for each warp, without a barrier in the loop: loads
// straight into registers, a tile ahead, took 137 us and 86 us.
template <typename T, int FMT, int HD, int NT, int STAGES, int CTAS>
__global__ void __launch_bounds__(kThreads, CTAS) k_q8_attn_few(const __grid_constant__ AttnArgs a)
{
    constexpr int KS = HD / 16;               // k-steps of the scores, 32-bit code words of a K row in a lane
    constexpr int VW = HD / 32;               // code words of a V row in a lane
    // what does not fit beside the accumulators is read from shared memory again
    // for each tile (kept in registers it spills: draft tokens 73 -> 76 us)
    constexpr bool kQInRegs = NT * KS <= 8, kMulInRegs = kQInRegs || CTAS == 1;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    FewSmem<HD, NT, STAGES> &sm = *reinterpret_cast<FewSmem<HD, NT, STAGES> *>(smem_raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
    const int H = a.l.heads, G = a.group;
    begin();

    // ---- this CTA's run of tiles: sum over all entries, then the entry it begins in
    unsigned total = 0;
    for (int base = 0; base < a.b.n_seqs; base += kThreads) {
        unsigned t = 0;
        if (base + tid < a.b.n_seqs) t = unit_of(a, entry(a.b, base + tid)).tiles * H;
#pragma unroll
        for (int d = 16; d; d >>= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
        if (lane == 0) sm.scan[warp] = t;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kWarps; i++) total += sm.scan[i];
        __syncthreads();
    }
    const Runs runs = runs_of(total, gridDim.x);
    if (blockIdx.x >= runs.n) return;
    unsigned t = run_begin(runs, blockIdx.x);
    const unsigned t_begin = t, t_end = run_begin(runs, blockIdx.x + 1);
    unsigned before = 0;
    for (int base = 0; base < a.b.n_seqs; base += kThreads) {
        unsigned n = 0;
        if (base + tid < a.b.n_seqs) n = unit_of(a, entry(a.b, base + tid)).tiles * H;
        unsigned upto = n;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const unsigned o = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += o;
        }
        if (lane == 31) sm.scan[warp] = upto;
        __syncthreads();
        unsigned sum = 0;
#pragma unroll
        for (int i = 0; i < kWarps; i++) {
            if (i < warp) upto += sm.scan[i];
            sum += sm.scan[i];
        }
        upto += before;
        if (t >= upto - n && t < upto) {
            sm.found[0] = base + tid;
            sm.found[1] = upto - n;
        }
        before += sum;
        __syncthreads();
        if (t < before) break;
    }
    int ei = sm.found[0];
    unsigned entry_t = sm.found[1];           // the entry's first tile
    Entry e = entry(a.b, ei);
    Unit0 u = unit_of(a, e);

    while (t < t_end) {
        while (t >= entry_t + u.tiles * H) {  // on to the next entry that has tiles
            entry_t += u.tiles * H;
            e = entry(a.b, ++ei);
            u = unit_of(a, e);
        }
        const int head = (t - entry_t) / u.tiles;
        const unsigned unit_t = entry_t + head * u.tiles;
        const int k0 = t - unit_t, k1 = min((unsigned)u.tiles, t_end - unit_t);
        const int rows = e.n * G, first = e.kv_len - e.n;
        const long long slot = (long long)e.seq * H + head;
        const uint8_t *kp = a.l.k + slot * a.l.max_seq * HD, *vp = a.l.v + slot * a.l.max_seq * HD;
        const float *ksp = a.l.k_scale + slot * (a.l.max_seq >> a.l.block_log2);
        const float *vsp = a.l.v_scale + slot * (a.l.max_seq >> a.l.block_log2);

        // ---- the warp's ring: 16 positions a stage, copied a few stages ahead
        using St = Stage<HD>;
        constexpr int kChunks = HD / 16, kRows = 32 / kChunks;           // 16-byte pieces of a row, rows at a time
        const uint32_t ring = (uint32_t)__cvta_generic_to_shared(sm.ring[warp]) + lane / kChunks * St::KPitch + lane % kChunks * 16;
        const uint8_t *kf, *vf;                // this lane's next pieces
        auto fetch = [&](int st) {
            const uint32_t dk = ring + st * St::Bytes, dv = dk + 16 * St::KPitch;
#pragma unroll
            for (int r = 0; r < 16; r += kRows) {
                copy_async16(dk + r * St::KPitch, kf + r * HD);
                copy_async16(dv + r * St::VPitch, vf + r * HD);
            }
            kf += kTile * HD;
            vf += kTile * HD;
        };
        // dimension of code word i of a V row
        auto dim_of = [&](int i) { return HD == 64 ? 8 * g + 4 * i : 128 * (i / 4) + 16 * g + 4 * (i % 4); };

        int j0 = u.start + k0 * kTile + 16 * warp;
        const int j_stop = min(u.end, u.start + k1 * kTile);
        int jf = j0;                           // next positions to fetch
        kf = kp + (long long)(j0 + lane / kChunks) * HD + lane % kChunks * 16;
        vf = vp + (long long)(j0 + lane / kChunks) * HD + lane % kChunks * 16;
        float ks[STAGES], vs[STAGES];          // scales of the stages in flight, oldest first
#pragma unroll
        for (int i = 0; i < STAGES; i++) {
            ks[i] = 0.0f;
            vs[i] = 1.0f;
            if (jf < j_stop) {
                fetch(i);
                ks[i] = ksp[jf >> a.l.block_log2];
                vs[i] = vsp[jf >> a.l.block_log2];
            }
            copy_commit();
            jf += kTile;
        }
        int st = 0;

        // ---- queries: scaled to fp16, in fragment order
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const int row = 8 * n + warp;
            constexpr int E = HD / 32;
            float x[E], top = 0.0f;
            if (row < rows) {
                const T *q = static_cast<const T *>(a.q) + (long long)(e.q0 + row / G) * a.q_stride + (head * G + row % G) * HD;
#pragma unroll
                for (int i = 0; i < E; i++) {
                    x[i] = sp_load_as_float(q, lane + 32 * i);
                    top = fmaxf(top, fabsf(x[i]));
                }
            } else {
#pragma unroll
                for (int i = 0; i < E; i++) x[i] = 0.0f;
            }
#pragma unroll
            for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            float down, up;
            row_scale(top, down, up);
            if (lane == 0) sm.mul[row] = a.scale * kLog2e * up;
#pragma unroll
            for (int i = 0; i < E; i++) {
                const int d = lane + 32 * i, s = d / 64 * 4 + d % 16 / 4;
                reinterpret_cast<__half *>(&sm.q[n][s][4 * warp + d % 64 / 16])[d % 4] = __float2half_rn(x[i] * down);
            }
        }
        __syncthreads();

        uint2 qr[kQInRegs ? NT : 1][kQInRegs ? KS : 1];
        if constexpr (kQInRegs) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int s = 0; s < KS; s++) qr[n][s] = sm.q[n][s][lane];
        }
        float mul[kMulInRegs ? NT : 1][2], m[NT][2], l[NT][2];
        // the positions that a row sees: kept with 8 rows, found again where a mask
        // asks for them with more, whose registers then hold two CTAs on an SM
        int hi[2], lo[2];
        auto limits = [&](int n, int i, int &h, int &w) {
            const int pos = first + (8 * n + 2 * c + i) / G;
            h = a.causal ? pos : e.kv_len - 1;
            w = a.window > 0 ? pos - a.window + 1 : 0;
        };
        if (NT == 1) {
            limits(0, 0, hi[0], lo[0]);
            limits(0, 1, hi[1], lo[1]);
        }
        const int hi_min = a.causal ? first : e.kv_len - 1;
        const int lo_max = a.window > 0 ? e.kv_len - a.window : 0;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                if (kMulInRegs) mul[kMulInRegs ? n : 0][i] = sm.mul[8 * n + 2 * c + i];
                m[n][i] = kNone;
                l[n][i] = 0.0f;
            }
        float o[NT][2 * VW][4];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 2 * VW; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) o[n][i][j] = 0.0f;

        for (; j0 < j_stop; j0 += kTile) {
            copy_wait<STAGES - 1>();
            __syncwarp();
            const unsigned char *stage = sm.ring[warp][st];
            // ---- scores of 16 positions
            float s[NT][4];
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int j = 0; j < 4; j++) s[n][j] = 0.0f;
#pragma unroll
            for (int q = 0; q < KS / 4; q++) {
                uint4 w[2];
#pragma unroll
                for (int r = 0; r < 2; r++) w[r] = *reinterpret_cast<const uint4 *>(stage + (g + 8 * r) * St::KPitch + 64 * q + 16 * c);
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const int i = 4 * q + x;
                    uint32_t f[4];
                    unpack4<FMT>(reinterpret_cast<const uint32_t *>(&w[0])[x], f[0], f[2]);
                    unpack4<FMT>(reinterpret_cast<const uint32_t *>(&w[1])[x], f[1], f[3]);
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        const uint2 b = kQInRegs ? qr[kQInRegs ? n : 0][kQInRegs ? i : 0] : sm.q[n][i][lane];
                        mma(s[n], f, b.x, b.y);
                    }
                }
            }
            const float k_scale = ks[0], v_scale = fmaxf(vs[0], kScaleMin);
#pragma unroll
            for (int i = 0; i + 1 < STAGES; i++) {
                ks[i] = ks[i + 1];
                vs[i] = vs[i + 1];
            }
            if (jf < j_stop) {
                ks[STAGES - 1] = ksp[jf >> a.l.block_log2];
                vs[STAGES - 1] = vsp[jf >> a.l.block_log2];
            }

            // ---- weights
            const float lv = lg2(v_scale), iv = rcp(v_scale);
            const bool all = j0 + 15 <= hi_min && j0 >= lo_max;     // nothing is masked
            bool over = false;
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const float f = k_scale * (kMulInRegs ? mul[kMulInRegs ? n : 0][i] : sm.mul[8 * n + 2 * c + i]);
                    s[n][i] = fmaf(s[n][i], f, lv);
                    s[n][2 + i] = fmaf(s[n][2 + i], f, lv);
                    if (!all) {
                        const int j = j0 + g;
                        if (NT > 1) limits(n, i, hi[i], lo[i]);
                        if (j > hi[i] || j < lo[i]) s[n][i] = -INFINITY;
                        if (j + 8 > hi[i] || j + 8 < lo[i]) s[n][2 + i] = -INFINITY;
                    }
                    over |= fmaxf(s[n][i], s[n][2 + i]) > m[n][i] + 8.0f;
                }
            if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        float top = fmaxf(s[n][i], s[n][2 + i]);
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                        top = fmaxf(top, m[n][i]);
                        const float fix = ex2(m[n][i] - top);
                        m[n][i] = top;
                        l[n][i] *= fix;
#pragma unroll
                        for (int x = 0; x < 2 * VW; x++) {
                            o[n][x][i] *= fix;
                            o[n][x][2 + i] *= fix;
                        }
                    }
            }
            uint32_t p[NT][2];
#pragma unroll
            for (int n = 0; n < NT; n++) {
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    s[n][i] = ex2(s[n][i] - m[n][i]);
                    s[n][2 + i] = ex2(s[n][2 + i] - m[n][i]);
                    l[n][i] = fmaf(s[n][i] + s[n][2 + i], iv, l[n][i]);
                }
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    const __half2 h = __floats2half2_rn(s[n][2 * r], s[n][2 * r + 1]);
                    p[n][r] = transpose8x8(*reinterpret_cast<const uint32_t *>(&h));
                }
            }
            // ---- values
            {
                constexpr int kWide = HD == 64 ? 2 : 4;        // code words of a lane's run of a row
                const unsigned char *vst = stage + 16 * St::KPitch + 2 * c * St::VPitch + 4 * kWide * g;
#pragma unroll
                for (int q = 0; q < VW / kWide; q++) {
                    uint32_t w[4][kWide];
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const unsigned char *p8 = vst + ((r & 1) + 8 * (r >> 1)) * St::VPitch + 128 * q;
                        if constexpr (kWide == 2) *reinterpret_cast<uint2 *>(w[r]) = *reinterpret_cast<const uint2 *>(p8);
                        else *reinterpret_cast<uint4 *>(w[r]) = *reinterpret_cast<const uint4 *>(p8);
                        // codes past the end may be NaN, which a weight of 0 does not undo
                        if (FMT == SP_Q8_E4M3 && j0 + 15 >= e.kv_len && j0 + 2 * c + (r & 1) + 8 * (r >> 1) >= e.kv_len) {
#pragma unroll
                            for (int x = 0; x < kWide; x++) w[r][x] = 0;
                        }
                    }
#pragma unroll
                    for (int x = 0; x < kWide; x++) {
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const int i = kWide * q + x;
                            uint32_t f[4];
                            const unsigned pick = h ? 0x7362 : 0x5140;     // a dimension of two positions side by side
                            unpack4<FMT>(__byte_perm(w[0][x], w[1][x], pick), f[0], f[1]);
                            unpack4<FMT>(__byte_perm(w[2][x], w[3][x], pick), f[2], f[3]);
#pragma unroll
                            for (int n = 0; n < NT; n++) mma(o[n][2 * i + h], f, p[n][0], p[n][1]);
                        }
                    }
                }
            }
            __syncwarp();                      // all lanes have read the stage
            if (jf < j_stop) fetch(st);
            copy_commit();
            jf += kTile;
            st = st + 1 == STAGES ? 0 : st + 1;
        }

        // ---- the warps' results into one: rows lie in shared memory in the
        // order (even rows, odd rows) of each 8, so a quarter warp's 16-byte
        // stores fall on different banks
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], d);
                if (g == 0) {
                    sm.m[warp][8 * n + 2 * c + i] = m[n][i];
                    sm.l[warp][8 * n + 2 * c + i] = l[n][i];
                }
            }
        __syncthreads();
        float fix[NT][2];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                float top = kNone;
#pragma unroll
                for (int w = 0; w < kWarps; w++) top = fmaxf(top, sm.m[w][8 * n + 2 * c + i]);
                fix[n][i] = ex2(m[n][i] - top);
            }
#pragma unroll
        for (int half = 1; half >= 0; half--) {
            if ((warp >> 2) == half) {
                float(*dst)[HD + 4] = sm.o[warp & 3];
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int x = 0; x < VW; x++)
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            float4 *at = reinterpret_cast<float4 *>(&dst[8 * n + c + 4 * i][dim_of(x)]);
                            float4 v = make_float4(o[n][2 * x][i] * fix[n][i], o[n][2 * x][2 + i] * fix[n][i],
                                                   o[n][2 * x + 1][i] * fix[n][i], o[n][2 * x + 1][2 + i] * fix[n][i]);
                            if (half == 0) {
                                const float4 w = *at;
                                v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
                            }
                            *at = v;
                        }
            }
            __syncthreads();
        }

        // ---- the unit's result, or this run's part of it
        const bool whole = k0 == 0 && k1 == u.tiles;
        const unsigned run0 = run_of_tile(runs, unit_t), run1 = run_of_tile(runs, unit_t + u.tiles - 1);
        constexpr int kSlot = 8 * NT * (HD + 2);
        auto finish = [&](int row, int d, float4 v, float top, float sum) {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;      // a sum that is NaN stays
            T w[4] = {T(v.x * inv), T(v.y * inv), T(v.z * inv), T(v.w * inv)};
            const long long tok = e.q0 + row / G;
            const int qh = head * G + row % G;
            *reinterpret_cast<uint2 *>(static_cast<T *>(a.out) + tok * a.out_stride + qh * HD + d) = *reinterpret_cast<uint2 *>(w);
            if (a.lse && d == 0) a.lse[tok * a.n_q_heads + qh] = sum == 0.0f ? -INFINITY : kLn2 * (top + lg2(sum));
        };
        // slots: a run has at most one unit that began before it and one that goes on after it
        float *part = a.partials + (2 * blockIdx.x + (unit_t >= t_begin)) * kSlot;
        for (int i = tid; i < rows * (HD / 4); i += kThreads) {
            const int row = i / (HD / 4), d = i % (HD / 4) * 4, at = (row & ~7) + (row & 7) / 2 + 4 * (row & 1);
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const float4 x = *reinterpret_cast<const float4 *>(&sm.o[w][at][d]);
                v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
            }
            float top = kNone, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; w++) top = fmaxf(top, sm.m[w][row]);
#pragma unroll
            for (int w = 0; w < kWarps; w++) sum += sm.l[w][row] * ex2(sm.m[w][row] - top);
            if (whole) {
                finish(row, d, v, top, sum);
            } else {
                __stcg(reinterpret_cast<float4 *>(part + row * HD + d), v);
                if (d == 0) __stcg(reinterpret_cast<float2 *>(part + 8 * NT * HD + 2 * row), make_float2(top, sum));
            }
        }
        if (!whole) {
            __threadfence();
            __syncthreads();
            if (tid == 0) sm.last = atomicAdd(a.counters + run0, 1u) == run1 - run0;
            __syncthreads();
            if (sm.last) {
                __threadfence();
                if (tid == 0) a.counters[run0] = 0;
                auto slot_of = [&](unsigned r) { return a.partials + (2 * r + (run_begin(runs, r) <= unit_t)) * kSlot; };
                for (int i = tid; i < rows * (HD / 4); i += kThreads) {
                    const int row = i / (HD / 4), d = i % (HD / 4) * 4;
                    float top = kNone, sum = 0.0f;
                    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    for (unsigned r = run0; r <= run1; r += 8) {
                        float2 ml[8];
                        float4 x[8];
                        float up = top;
#pragma unroll
                        for (int k = 0; k < 8; k++) {
                            ml[k] = make_float2(kNone, 0.0f);
                            x[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            if (r + k <= run1) {
                                const float *q = slot_of(r + k);
                                ml[k] = __ldcg(reinterpret_cast<const float2 *>(q + 8 * NT * HD + 2 * row));
                                x[k] = __ldcg(reinterpret_cast<const float4 *>(q + row * HD + d));
                            }
                        }
#pragma unroll
                        for (int k = 0; k < 8; k++) up = fmaxf(up, ml[k].x);
                        const float old = ex2(top - up);
                        sum *= old;
                        v.x *= old; v.y *= old; v.z *= old; v.w *= old;
#pragma unroll
                        for (int k = 0; k < 8; k++) {
                            const float f = ex2(ml[k].x - up);
                            sum = fmaf(ml[k].y, f, sum);
                            v.x = fmaf(x[k].x, f, v.x);
                            v.y = fmaf(x[k].y, f, v.y);
                            v.z = fmaf(x[k].z, f, v.z);
                            v.w = fmaf(x[k].w, f, v.w);
                        }
                        top = up;
                    }
                    finish(row, d, v, top, sum);
                }
            }
        }
        t = unit_t + k1;
        __syncthreads();                       // shared memory is free for the next unit
    }
}

template <typename T, int FMT, int HD, int NT>
int launch_few(const AttnArgs &a, int sms, unsigned tiles, cudaStream_t s)
{
    // CTAs on an SM: what the registers of 256 threads allow without spilling;
    // stages: what shared memory then holds
    constexpr int CTAS = HD == 256 || NT * HD == 512 ? 1 : NT * HD <= 64 ? 3 : 2;
    constexpr int STAGES = HD == 256 || (HD == 64 && NT == 4) || (HD == 128 && NT < 4) ? 2 : 3;
    auto kernel = k_q8_attn_few<T, FMT, HD, NT, STAGES, CTAS>;
    constexpr int smem = sizeof(FewSmem<HD, NT, STAGES>);
    static std::atomic<unsigned long long> ready{0};      // devices whose attribute is set
    int dev = 0;
    cudaGetDevice(&dev);
    if (smem > 48 * 1024 && !(ready.load(std::memory_order_acquire) >> (dev & 63) & 1)) {
        const int rc = sp_check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem),
                                     "q8_attn shared memory");
        if (rc) return rc;
        if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_release);
    }
    unsigned grid = (unsigned)(sms * CTAS);
    if (grid > (unsigned)kMaxCtas) grid = kMaxCtas;
    if (grid > tiles) grid = tiles;
    return q8::launch("q8_attn launch", kernel, grid, kThreads, smem, s, a);
}

template <typename T, int FMT>
int launch_few_of(const AttnArgs &a, int hd, int nt, int sms, unsigned tiles, cudaStream_t s)
{
    if (hd == 64) return nt == 1 ? launch_few<T, FMT, 64, 1>(a, sms, tiles, s) : nt == 2 ? launch_few<T, FMT, 64, 2>(a, sms, tiles, s)
                                                                                          : launch_few<T, FMT, 64, 4>(a, sms, tiles, s);
    if (hd == 128) return nt == 1 ? launch_few<T, FMT, 128, 1>(a, sms, tiles, s) : nt == 2 ? launch_few<T, FMT, 128, 2>(a, sms, tiles, s)
                                                                                            : launch_few<T, FMT, 128, 4>(a, sms, tiles, s);
    return nt == 1 ? launch_few<T, FMT, 256, 1>(a, sms, tiles, s) : launch_few<T, FMT, 256, 2>(a, sms, tiles, s);
}

}  // namespace

namespace q8 {
// Counters, the many-row kernel's list of split units, then the partial
// results of the larger grid: two slots for each CTA of up to 32 rows at up
// to three CTAs an SM, or of 256 rows at one.
size_t attn_workspace_bytes(int sm_count, int head_dim)
{
    const size_t few = (size_t)2 * 3 * sm_count * 32 * (head_dim + 2) * sizeof(float);
    const size_t many = (size_t)2 * sm_count * 256 * (head_dim + 2) * sizeof(float);
    return kCounterBytes + split_bytes(sm_count) + (few > many ? few : many);
}
}  // namespace q8

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
    // past the cache's length a window hides nothing; so bounded, position - window
    // stays in 32 bits for tokens before the first position too
    if (window > qc->max_seq_len) window = qc->max_seq_len;
    if (q_stride == 0) q_stride = (long long)n_q_heads * hd;
    if (out_stride == 0) out_stride = (long long)n_q_heads * hd;
    if (q_stride < (long long)n_q_heads * hd || out_stride < (long long)n_q_heads * hd)
        return sp_set_error(SP_ERR_ARG, "q8_attn: a token's stride is less than its rows");
    if (batch->n_tokens == 0 || batch->n_seqs == 0 || batch->max_new == 0) return SP_OK;
    if (!d_q || !d_out) return sp_set_error(SP_ERR_ARG, "q8_attn: NULL argument");
    if (((uintptr_t)d_q | (uintptr_t)d_out | (uintptr_t)(q_stride * 2) | (uintptr_t)(out_stride * 2)) % 16 || (uintptr_t)d_lse % 4)
        return sp_set_error(SP_ERR_ARG, "q8_attn: pointers and strides must be multiples of 16 bytes");
    const int G = n_q_heads / H;
    // rows of an entry are counted in 32 bits; a tensor of so many has 275 GB
    if ((long long)(batch->max_new < batch->n_tokens ? batch->max_new : batch->n_tokens) * G > 0x7fffffff)
        return sp_set_error(SP_ERR_ARG, "q8_attn: %d tokens of %d query heads for a KV head in one entry", batch->max_new, G);
    AttnArgs a = {q8::layer_of(qc, layer), q8::batch_of(qc, batch), d_q, d_out, d_lse, q_stride, out_stride,
                  n_q_heads, G, logit_scale, causal, window, 0, (unsigned int *)qc->d_attn_ws,
                  (float *)((char *)qc->d_attn_ws + kCounterBytes + q8::split_bytes(qc->sm_count))};
    const long long tiles = (long long)batch->n_seqs * H * (batch->max_kv / kTile + 2);
    const long long rows = (long long)batch->max_new * G;
    if (tiles > 0x7fffffff) return sp_set_error(SP_ERR_ARG, "q8_attn: %lld tiles in one call", tiles);
    // The few-row kernel takes entries of up to 8, 16 or 32 rows (32 only where
    // the accumulators of head_dim 256 do not fill the registers).  Where the
    // batch has longer entries it takes those of one token or so, and the
    // many-row kernel the others.
    const int most = hd == 256 ? 16 : 32;
    const long long take = rows <= most ? rows : G;
    const int nt = take <= 8 ? 1 : take <= 16 ? 2 : take <= most ? 4 : 0;
    a.few_rows = 8 * nt;
    cudaStream_t s = (cudaStream_t)stream;
    const bool i8 = qc->format == SP_Q8_INT8;
    if (nt) {
        if (dtype == SP_DTYPE_F16)
            rc = i8 ? launch_few_of<__half, SP_Q8_INT8>(a, hd, nt, qc->sm_count, (unsigned)tiles, s)
                    : launch_few_of<__half, SP_Q8_E4M3>(a, hd, nt, qc->sm_count, (unsigned)tiles, s);
        else
            rc = i8 ? launch_few_of<__nv_bfloat16, SP_Q8_INT8>(a, hd, nt, qc->sm_count, (unsigned)tiles, s)
                    : launch_few_of<__nv_bfloat16, SP_Q8_E4M3>(a, hd, nt, qc->sm_count, (unsigned)tiles, s);
        if (rc) return rc;
    }
    if (rows > a.few_rows) rc = q8::launch_many(a, qc->format, dtype, hd, qc->sm_count, s);
    return rc;
}
