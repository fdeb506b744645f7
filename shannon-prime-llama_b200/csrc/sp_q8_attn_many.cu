// sp_q8_attn_many.cu — attention over the 8-bit cache for many rows (prompts
// and chunks of prompts) on the 5th-generation tensor cores.
//
// Rows of a unit of work are its tokens times the query heads that share the
// KV head, 256 at a time (128 at head_dim 256), against tiles of 128 (64)
// positions:
//     S = Q K'      both from shared memory, into tensor memory
//     P = 2^(S f + log2 vs - m), by the rows' own threads, back into the
//         columns of S as fp16 (the softmax of sp_q8_attn.cu)
//     O += P V      P from tensor memory, V from shared memory
// Codes become fp16 once for all 256 rows: seven warps (eleven at head_dim 256)
// load them, unpack them in registers and store them in the core-matrix layout
// (8 rows of 16 bytes) that serves K as the K-major and V as the MN-major
// operand.  One thread issues the products; while a softmax warpgroup works on
// its 128 rows, the tensor cores work on the other 128.
//
// Measured: a causal prompt of 8192 tokens, 32 query heads on 8 of 128
// dimensions, e4m3 and bf16, takes 711 us, 773 TFLOP/s (47% of the library's
// plain product); chunks of 202 to 1021 tokens on up to 7570 positions, 16 query
// heads on 2 of 256, int8, window 4096, 270 us, 685 TFLOP/s.  What bounds it is
// the chain of a 128-row tile: scores, softmax (one row a thread, about 1950
// cycles for 128 positions with two warps on each scheduler), store of the
// weights (700), P V and the next scores (1400).  A tile of both halves takes
// 3900 cycles, the products 2100 of them.  Tensor memory is full (two scores,
// two outputs), so the next scores cannot be computed earlier: in halves of 64
// columns, one of them ahead, the prompt took 994 us, since products of 64
// columns cost 3/4 of those of 128.  The same prompt in 64 dimensions takes 577
// us, 476 TFLOP/s: products are half as long, the rest of the chain is not, and the
// powers of two alone keep the special-function units busy for 231 us (a polynomial
// for a quarter or an eighth of them changed nothing).  The beginning and end of a unit (queries,
// output) take about 12000 cycles, a tenth of the prompt's time.
#include "sp_q8_attn.cuh"
#include "sp_q8_runs.h"
#include "sp_bulk.cuh"

#include <atomic>
#include <type_traits>

namespace {

using namespace q8;

template <int HD>
struct Shape {
    static constexpr int NQ = HD == 256 ? 1 : 2;       // 128-row tiles of queries
    static constexpr int BN = HD == 256 ? 64 : 128;    // positions of a tile
    static constexpr int ROWS = 128 * NQ;
    static constexpr int SoftWarps = 4 * NQ, ConvWarps = 15 - SoftWarps;
    static constexpr int Threads = 32 * (SoftWarps + ConvWarps + 1);   // the last warp issues the products
    static constexpr int ColO = 256;                   // S (and P) at 128 i or 64 (k & 1), O at 256 + HD i
    // Operands lie in core matrices of 8 rows of 16 bytes, the next 8 dimensions'
    // Core bytes on: 16 more than a core matrix has, so that the stores of 4
    // lanes for each row, whose loads are then 64 contiguous bytes, fall on
    // different banks.  Products run at the same rate as without the gap.
    static constexpr int Core = 144, Rows8 = HD / 8 * Core;
    static constexpr int StageB = BN / 8 * Rows8, QB = 16 * Rows8;
    static constexpr int SlotFloats = ROWS * (HD + 2);
};

template <int HD>
struct ManySmem {
    unsigned char q[Shape<HD>::NQ][Shape<HD>::QB];
    unsigned char k[2][Shape<HD>::StageB], v[2][Shape<HD>::StageB];
    unsigned long long q_full[2], k_full[2], k_free[2], v_full[2], v_free[2], s_full[2], p_full[2], pv_done[2], end;
    float4 scales[4][Shape<HD>::BN / 16];              // of four tiles in turn: K scale, log2 of V's, 1 / V's
    unsigned long long tiles[256], total;              // of each entry of a chunk; of the entries so far
    unsigned long long found_t;
    int found;
    uint32_t tmem;
    int abort;
};

// What the join kernel needs of a unit that falls into several runs; kept by
// the run in which the unit begins.
struct Split {
    int valid, q0, row0, rows, head;
    unsigned run0, run1;
};

// --- tensor core and tensor memory --------------------------------------
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

#define Q8_R8(b) "=r"(v[b]), "=r"(v[b + 1]), "=r"(v[b + 2]), "=r"(v[b + 3]), "=r"(v[b + 4]), "=r"(v[b + 5]), "=r"(v[b + 6]), "=r"(v[b + 7])
__device__ __forceinline__ void tmem_ld32(uint32_t at, uint32_t (&v)[32])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
                 "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : Q8_R8(0), Q8_R8(8), Q8_R8(16), Q8_R8(24) : "r"(at));
}
#undef Q8_R8
#define Q8_R8(b) "r"(v[b]), "r"(v[b + 1]), "r"(v[b + 2]), "r"(v[b + 3]), "r"(v[b + 4]), "r"(v[b + 5]), "r"(v[b + 6]), "r"(v[b + 7])
__device__ __forceinline__ void tmem_ld16(uint32_t at, uint32_t (&v)[16])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
                   "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(at));
}
// With its wait.
__device__ __forceinline__ void tmem_ld8(uint32_t at, uint32_t (&v)[8])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=&r"(v[0]), "=&r"(v[1]), "=&r"(v[2]), "=&r"(v[3]), "=&r"(v[4]), "=&r"(v[5]), "=&r"(v[6]), "=&r"(v[7])
                 : "r"(at) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t (&v)[16])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(at), Q8_R8(0), Q8_R8(8) : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t at, const uint32_t (&v)[8])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(at), Q8_R8(0) : "memory");
}
#undef Q8_R8

// Waits for the loads so far; their registers are named so that no use of them
// moves before the wait.
#define Q8_R8(b) "+r"(v[b]), "+r"(v[b + 1]), "+r"(v[b + 2]), "+r"(v[b + 3]), "+r"(v[b + 4]), "+r"(v[b + 5]), "+r"(v[b + 6]), "+r"(v[b + 7])
__device__ __forceinline__ void wait_ld16(uint32_t (&v)[16])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;" : Q8_R8(0), Q8_R8(8) :: "memory");
}
__device__ __forceinline__ void wait_ld32(uint32_t (&v)[32])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;" : Q8_R8(0), Q8_R8(8), Q8_R8(16), Q8_R8(24) :: "memory");
}
#undef Q8_R8

// Two 32-bit sums or products at a time.
struct F2 {
    float x, y;
};
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c)
{
    F2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b)
{
    F2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
// Shared-memory operand without swizzle, in core matrices of 8 rows of 16
// bytes: lbo bytes between core matrices along K, sbo along M or N (for both
// the K-major and the MN-major operands).
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t lbo, uint32_t sbo)
{
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)((lbo >> 4) & 0x3FFFu) << 16 |
           (uint64_t)((sbo >> 4) & 0x3FFFu) << 32 | (uint64_t)1 << 46;
}

// fp16 x fp16 -> fp32, M = 128.  A whole warp comes here and one elected lane
// issues: the operands then stay in uniform registers (65 cycles for a product
// of 128 x 128 x 16, against 122 to 200 from inside a one-lane branch).
constexpr uint32_t instr(int n, bool b_mn)
{
    return (1u << 4) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t i, uint32_t add)
{
    asm volatile("{\n\t.reg .pred p, e;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %3, 0;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %4, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(add), "r"(i)
                 : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t i, uint32_t add)
{
    asm volatile("{\n\t.reg .pred p, e;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %3, 0;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %4, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(add), "r"(i)
                 : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar)
{
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
                 "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void arrive(uint32_t bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Waits for a phase; false once any wait of this CTA has run out (2 s).
__device__ __forceinline__ bool wait_slow(uint32_t bar, uint32_t parity, int *abort, unsigned int *status)
{
    const unsigned long long t0 = spb::global_ns();
    for (;;) {
        for (int i = 0; i < 64; i++)
            if (spb::mbar_try_wait(bar, parity)) return true;
        if (*(volatile int *)abort) return false;
        if (spb::global_ns() - t0 > spb::kWaitLimitNs) break;
    }
    *(volatile int *)abort = 1;
    if (status) atomicOr(status, 2u);
    return false;
}

// --- units: (entry, KV head, tile of rows) ------------------------------
struct Rows {
    int row0, rows, start, tiles;
};

template <int HD>
__device__ __forceinline__ int row_tiles(const AttnArgs &a, const Entry &e)
{
    const long long r = (long long)e.n * a.group;
    return r <= a.few_rows ? 0 : (int)((r + Shape<HD>::ROWS - 1) / Shape<HD>::ROWS);
}

template <int HD>
__device__ __forceinline__ Rows rows_of(const AttnArgs &a, const Entry &e, int qt)
{
    constexpr int BN = Shape<HD>::BN;
    Rows r;
    r.row0 = qt * Shape<HD>::ROWS;
    r.rows = min(Shape<HD>::ROWS, e.n * a.group - r.row0);
    const int first = e.kv_len - e.n;
    const int lo = first + r.row0 / a.group, hi = first + (r.row0 + r.rows - 1) / a.group;
    const int end = a.causal ? hi + 1 : e.kv_len;
    r.start = a.window > 0 && lo - a.window + 1 > 0 ? (lo - a.window + 1) / BN * BN : 0;
    r.tiles = max(1, (end - r.start + BN - 1) / BN);
    return r;
}

// Token and query head (of the KV head's) of the unit's row rr: one division for
// the unit, then a multiplication each (exact for rr + group < 2^32 / group).
struct RowMap {
    int t0, r0, group;
    unsigned inv;
    __device__ __forceinline__ RowMap(int row0, int g) : group(g), inv(0xffffffffu / g + 1)
    {
        t0 = row0 / g;
        r0 = row0 - t0 * g;
    }
    __device__ __forceinline__ void at(int rr, int &token, int &head) const
    {
        const unsigned y = r0 + rr, q = group == 1 ? y : __umulhi(y, inv);
        token = t0 + q;
        head = y - q * group;
    }
};

// Walks the units of a run: every role goes through the same ones.
template <int HD>
struct Walk {
    Entry e;
    int ei, qt, n_qt, head;
    unsigned t, t_end, unit_t;      // next tile, end of the run, first tile of the unit: their low 32 bits
    Rows r;
    __device__ __forceinline__ bool more() const { return apart(t_end, t) > 0; }
    __device__ __forceinline__ int k0() const { return t - unit_t; }
    __device__ __forceinline__ int k1() const { return min((unsigned)r.tiles, t_end - unit_t); }
    __device__ __forceinline__ void next(const AttnArgs &a)
    {
        t = unit_t + k1();
        if (!more()) return;
        unit_t += r.tiles;
        if (++qt == n_qt) {
            qt = 0;
            if (++head == a.l.heads) {
                head = 0;
                do {
                    e = entry(a.b, ++ei);
                    n_qt = row_tiles<HD>(a, e);
                } while (n_qt == 0);
            }
        }
        r = rows_of<HD>(a, e, qt);
    }
};

template <typename T, int FMT, int HD>
__global__ void __launch_bounds__(Shape<HD>::Threads, 1) k_q8_attn_many(const __grid_constant__ AttnArgs a)
{
    using S = Shape<HD>;
    constexpr int NQ = S::NQ, BN = S::BN;
    extern __shared__ __align__(128) unsigned char smem_raw[];
    ManySmem<HD> &sm = *reinterpret_cast<ManySmem<HD> *>(smem_raw);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    constexpr int kWarps = S::Threads / 32;
    begin();
    Split *splits = reinterpret_cast<Split *>(a.counters + kMaxCtas) + blockIdx.x;
    if (tid == 0) splits->valid = 0;

    // ---- this CTA's run: tiles of one head of each entry (a warp for an entry, a lane for
    // a tile of rows), their sum, and the entry in which the run begins
    LongRuns runs;
    unsigned long long before = 0;
    for (int pass = 0; pass < 2; pass++) {
        before = 0;
        for (int base = 0; base < a.b.n_seqs; base += 256) {
            const int n = min(256, a.b.n_seqs - base);
            for (int i = warp; i < n; i += kWarps) {
                const Entry e = entry(a.b, base + i);
                const int nq = row_tiles<HD>(a, e);
                unsigned long long sum = 0;
                for (int q = lane; q < nq; q += 32) sum += rows_of<HD>(a, e, q).tiles;
#pragma unroll
                for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                if (lane == 0) sm.tiles[i] = sum * a.l.heads;
            }
            __syncthreads();
            if (warp == 0) {
                for (int i = 0; i < n; i += 32) {
                    const unsigned long long x = i + lane < n ? sm.tiles[i + lane] : 0;
                    unsigned long long upto = x;
#pragma unroll
                    for (int d = 1; d < 32; d <<= 1) {
                        const unsigned long long o = __shfl_up_sync(0xffffffffu, upto, d);
                        if (lane >= d) upto += o;
                    }
                    if (pass) {
                        const unsigned long long t = run_begin(runs, blockIdx.x);
                        if (t >= before + upto - x && t < before + upto) {
                            sm.found = base + i + lane;
                            sm.found_t = before + upto - x;
                        }
                    }
                    before += __shfl_sync(0xffffffffu, upto, 31);
                }
                if (lane == 0) sm.total = before;
            }
            __syncthreads();
            before = sm.total;
            __syncthreads();
        }
        if (pass == 0) {
            runs = long_runs_of(before, gridDim.x);
            if (blockIdx.x >= runs.n) return;
        }
    }
    Walk<HD> w;
    w.t = (unsigned)run_begin(runs, blockIdx.x);
    w.t_end = (unsigned)run_begin(runs, blockIdx.x + 1);
    w.ei = sm.found;
    w.e = entry(a.b, w.ei);
    w.n_qt = row_tiles<HD>(a, w.e);
    {
        // the head, then the tile of rows, in which the run begins
        unsigned long long each = 0;
        for (int q = lane; q < w.n_qt; q += 32) each += rows_of<HD>(a, w.e, q).tiles;
#pragma unroll
        for (int d = 16; d; d >>= 1) each += __shfl_xor_sync(0xffffffffu, each, d);
        const unsigned long long in = run_begin(runs, blockIdx.x) - sm.found_t;
        w.head = (int)(in / each);
        const unsigned long long off = in - w.head * each;
        unsigned long long pre = 0;
        w.qt = 0;
        w.unit_t = 0;
        for (int base = 0; base < w.n_qt; base += 32) {
            const unsigned x = base + lane < w.n_qt ? rows_of<HD>(a, w.e, base + lane).tiles : 0;
            unsigned upto = x;               // of 32 tiles of rows, with at most 2^24 tiles of positions each
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const unsigned o = __shfl_up_sync(0xffffffffu, upto, d);
                if (lane >= d) upto += o;
            }
            const unsigned who = __ballot_sync(0xffffffffu, off >= pre + upto - x && off < pre + upto);
            if (who) {
                const int src = __ffs(who) - 1;
                w.qt = base + src;
                w.unit_t = w.t - (unsigned)(off - (pre + __shfl_sync(0xffffffffu, upto - x, src)));
            }
            pre += __shfl_sync(0xffffffffu, upto, 31);
        }
        w.r = rows_of<HD>(a, w.e, w.qt);
    }

    if (tid == 0) {
        for (int i = 0; i < 2; i++) {
            spb::mbar_init(spb::smem_u32(&sm.q_full[i]), 4);
            spb::mbar_init(spb::smem_u32(&sm.k_full[i]), S::ConvWarps);
            spb::mbar_init(spb::smem_u32(&sm.k_free[i]), 1);
            spb::mbar_init(spb::smem_u32(&sm.v_full[i]), S::ConvWarps);
            spb::mbar_init(spb::smem_u32(&sm.v_free[i]), 1);
            spb::mbar_init(spb::smem_u32(&sm.s_full[i]), 1);
            spb::mbar_init(spb::smem_u32(&sm.p_full[i]), 4);
            spb::mbar_init(spb::smem_u32(&sm.pv_done[i]), 1);
        }
        spb::mbar_init(spb::smem_u32(&sm.end), 1);
        spb::mbar_init_fence();
        sm.abort = 0;
    }
    constexpr int kMmaWarp = S::SoftWarps + S::ConvWarps;
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(spb::smem_u32(&sm.tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, sm.tmem, 0);
    auto wait = [&](unsigned long long &bar, unsigned n) {      // a whole warp, for the end of phase n
        const uint32_t b = spb::smem_u32(&bar);
        return __all_sync(0xffffffffu, spb::mbar_try_wait(b, n & 1) || wait_slow(b, n & 1, &sm.abort, a.b.status)) != 0;
    };

    if (warp < S::SoftWarps) {
        // ================= softmax: one thread for each row =================
        const int i = warp >> 2, r = tid & 127;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t t_o = tmem + lanes + S::ColO + HD * i;
        unsigned done = 0;                                      // tiles so far, of all units
        // For the values of tile n.  With two buffers of scores a warp may be two
        // products ahead of the tensor cores, and a barrier tells only neighbouring
        // phases apart: the buffers have a barrier each.
        auto wait_values = [&](unsigned n) { return NQ == 2 ? wait(sm.pv_done[i], n) : wait(sm.pv_done[n & 1], n >> 1); };
        for (; w.more(); w.next(a)) {
            const RowMap map(w.r.row0, a.group);
            const bool real = 128 * i + r < w.r.rows;
            int tok, qh;
            map.at(128 * i + r, tok, qh);
            const int pos = w.e.kv_len - w.e.n + tok;
            tok += w.e.q0;
            qh += w.head * a.group;
            // ---- the warp's 32 rows of queries, 8 rows x 4 runs of 8 dimensions at a
            // time, into the operand's places as they are; then a thread for each
            // row scales its own to fp16
            float mul, top = 0.0f;
            unsigned char *own = sm.q[i] + (warp & 3) * 4 * S::Rows8;
#pragma unroll 1
            for (int n = 0; n < 4; n++) {
                const int rr = 128 * i + 32 * (warp & 3) + 8 * n + (lane >> 2);
                int t, h;
                map.at(rr, t, h);
                const T *q = static_cast<const T *>(a.q) + (w.e.q0 + t) * a.q_stride + (w.head * a.group + h) * HD + (lane & 3) * 8;
                const uint32_t dst = spb::smem_u32(own + n * S::Rows8 + (lane & 3) * S::Core + (lane >> 2) * 16), bytes = rr < w.r.rows ? 16 : 0;
#pragma unroll
                for (int c = 0; c < HD / 32; c++)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + 4 * S::Core * c),
                                 "l"(bytes ? q + 32 * c : static_cast<const T *>(a.q)), "r"(bytes) : "memory");
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            __syncwarp();
            {
                unsigned char *mine = own + (lane >> 3) * S::Rows8 + (lane & 7) * 16;
#pragma unroll 4
                for (int c = 0; c < HD / 8; c++) {
                    const uint4 x = *reinterpret_cast<const uint4 *>(mine + S::Core * c);
#pragma unroll
                    for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(sp_load_as_float(reinterpret_cast<const T *>(&x), j)));
                }
                float down, up;
                row_scale(top, down, up);
                mul = fabsf(a.scale) * kLog2e * up;
                if (a.scale < 0.0f) down = -down;
#pragma unroll 2
                for (int c = 0; c < HD / 8; c++) {
                    const uint4 x = *reinterpret_cast<const uint4 *>(mine + S::Core * c);
                    __half h[8];
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        h[j] = __float2half_rn(sp_load_as_float(reinterpret_cast<const T *>(&x), j) * down);
                    *reinterpret_cast<uint4 *>(mine + S::Core * c) = *reinterpret_cast<const uint4 *>(h);
                }
            }
            spb::fence_proxy_async();
            __syncwarp();
            if (lane == 0) arrive(spb::smem_u32(&sm.q_full[i]));
            const int hi = !real ? 0x7fffffff : a.causal ? pos : w.e.kv_len - 1;
            const int lo = real && a.window > 0 ? pos - a.window + 1 : 0;
            float m = kNone, l = 0.0f;
            const int k0 = w.k0(), k1 = w.k1();
            for (int k = k0; k < k1; k++, done++) {
                const int j0 = w.r.start + k * BN;
                const float4 *sc = sm.scales[done & 3];
                const bool all = __all_sync(0xffffffffu, j0 + BN - 1 <= hi && j0 >= lo);
                const int buf = NQ == 2 ? i : (int)(done & 1);
                const uint32_t t_s = tmem + lanes + (NQ == 2 ? 128 : 64) * buf;
                if (!wait(sm.s_full[buf], NQ == 2 ? done : done >> 1)) goto out;
                fence_after();
                // ---- 32 positions' weights by the maximum so far.  True where 16 of them
                // sum up to more than 2^12, which no weight passes otherwise (well inside
                // fp16): the maximum is too small.
                auto weights = [&](const uint32_t(&u)[32], int c, uint32_t(&p)[16], float &sum) {
                    bool over = false;
                    sum = 0.0f;
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const float4 now = sc[2 * c + h];
                        const float fg = now.x * mul, off = now.y - m;
                        F2 part = {0.0f, 0.0f};
#pragma unroll
                        for (int j = 8 * h; j < 8 * h + 8; j++) {
                            F2 x = fma2({__uint_as_float(u[2 * j]), __uint_as_float(u[2 * j + 1])}, {fg, fg}, {off, off});
                            x.x = ex2(x.x);
                            x.y = ex2(x.y);
                            part = add2(part, x);
                            const __half2 hw = __floats2half2_rn(x.x, x.y);
                            p[j] = *reinterpret_cast<const uint32_t *>(&hw);
                        }
                        over |= part.x + part.y > 4096.0f;
                        sum = fmaf(part.x + part.y, now.z, sum);
                    }
                    return over;
                };
                // ---- the same where positions are masked or the maximum has to grow: it is
                // found first, and what the products so far have summed, and this tile's
                // weights before these (rounded a second time), shrink.  Exponents are
                // differences of the numbers that the maximum was taken of: in one sum with
                // scale and maximum, as above, the largest key's own is off by as much as the
                // maximum was rounded, 2^5 at logits of 1e9.
                auto careful = [&](int c) {
                    float top = kNone;
#pragma unroll 1
                    for (int h = 2 * c; h < 2 * c + 2; h++) {
                        const float fg = sc[h].x * mul, lg = sc[h].y;
                        uint32_t v[16];
                        tmem_ld16(t_s + 16 * h, v);
                        wait_ld16(v);
#pragma unroll
                        for (int j = 0; j < 16; j++) {
                            const int at = j0 + 16 * h + j;
                            if (at <= hi && at >= lo) top = fmaxf(top, fmaf(__uint_as_float(v[j]), fg, lg));
                        }
                    }
                    const bool up = top > m + 4.0f;         // a sum over 2^12 has a weight over 2^8
                    if (__any_sync(0xffffffffu, up)) {
                        const float fix = up ? ex2(m - top) : 1.0f;
                        if (up) m = top;
                        l *= fix;
                        if (k > k0) {
                            if (!wait_values(done - 1)) return false;
                            fence_after();
#pragma unroll 1
                            for (int d = 0; d < HD; d += 16) {
                                uint32_t v[16];
                                tmem_ld16(t_o + d, v);
                                wait_ld16(v);
#pragma unroll
                                for (int j = 0; j < 16; j++) v[j] = __float_as_uint(__uint_as_float(v[j]) * fix);
                                tmem_st16(t_o + d, v);
                            }
                        }
                        wait_st();
                        // in 32 bits: fix may be far below fp16's normal numbers, and
                        // the weights as far above 1 (up to 2^12).  8 columns at a time:
                        // 16 take the kernel from 122 registers to 128
#pragma unroll 1
                        for (int d = 0; d < 16 * c; d += 8) {
                            uint32_t v[8];
                            tmem_ld8(t_s + d, v);
#pragma unroll
                            for (int j = 0; j < 8; j++) {
                                const float2 y = __half22float2(*reinterpret_cast<const __half2 *>(&v[j]));
                                const __half2 z = __floats2half2_rn(y.x * fix, y.y * fix);
                                v[j] = *reinterpret_cast<const uint32_t *>(&z);
                            }
                            tmem_st8(t_s + d, v);
                        }
                    }
#pragma unroll 1
                    for (int h = 2 * c; h < 2 * c + 2; h++) {
                        const float fg = sc[h].x * mul, lg = sc[h].y;
                        uint32_t v[16], p[8];
                        tmem_ld16(t_s + 16 * h, v);
                        wait_ld16(v);
                        float sum = 0.0f;
#pragma unroll
                        for (int j = 0; j < 16; j += 2) {
                            const int at = j0 + 16 * h + j;
                            const float x = at > hi || at < lo ? 0.0f : ex2(fmaf(__uint_as_float(v[j]), fg, lg) - m);
                            const float y = at + 1 > hi || at + 1 < lo ? 0.0f : ex2(fmaf(__uint_as_float(v[j + 1]), fg, lg) - m);
                            sum += x + y;
                            const __half2 hw = __floats2half2_rn(x, y);
                            p[j / 2] = *reinterpret_cast<const uint32_t *>(&hw);
                        }
                        l = fmaf(sum, sc[h].z, l);
                        tmem_st8(t_s + 8 * h, p);            // over scores already read
                    }
                    return true;
                };
                if (all && k > k0) {
                    uint32_t u[2][32];
                    tmem_ld32(t_s, u[0]);
#pragma unroll
                    for (int c = 0; c < BN / 32; c++) {
                        uint32_t p[16];
                        float sum;
                        wait_ld32(u[c & 1]);
                        if (c + 1 < BN / 32) tmem_ld32(t_s + 32 * (c + 1), u[(c + 1) & 1]);
                        const bool over = weights(u[c & 1], c, p, sum);
                        if (__any_sync(0xffffffffu, over)) {
                            if (!careful(c)) goto out;
                        } else {
                            l += sum;
                            tmem_st16(t_s + 16 * c, p);
                        }
                    }
                } else {
                    // a unit's first tile in this run, and tiles with masked positions
#pragma unroll 1
                    for (int c = 0; c < BN / 32; c++) {
                        const int at = j0 + 32 * c;
                        uint32_t p[16];
                        if (__all_sync(0xffffffffu, !real || at > hi || at + 31 < lo)) {
#pragma unroll
                            for (int j = 0; j < 16; j++) p[j] = 0;
                            tmem_st16(t_s + 16 * c, p);
                            continue;
                        }
                        bool slow = !__all_sync(0xffffffffu, at + 31 <= hi && at >= lo && m > kNone);
                        if (!slow) {
                            uint32_t u[32];
                            float sum;
                            tmem_ld32(t_s + 32 * c, u);
                            wait_ld32(u);
                            slow = __any_sync(0xffffffffu, weights(u, c, p, sum));
                            if (!slow) {
                                l += sum;
                                tmem_st16(t_s + 16 * c, p);
                            }
                        }
                        if (slow && !careful(c)) goto out;
                    }
                }
                wait_st();
                fence_before();
                __syncwarp();
                if (lane == 0) arrive(spb::smem_u32(&sm.p_full[buf]));
            }
            // ---- the unit's result, or this run's part of it
            if (!wait_values(done - 1)) goto out;
            fence_after();
            const bool whole = k0 == 0 && k1 == w.r.tiles;
            if (whole) {
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;      // a sum that is NaN stays
                // through the warp's own part of the queries' place, so that a row's
                // bytes leave together: 16-byte pieces, exchanged within groups of
                // eight by the row to fall on different banks
#pragma unroll 1
                for (int c = 0; c < HD; c += 32) {
                    uint32_t v[32];
                    tmem_ld32(t_o + c, v);
                    wait_ld32(v);
#pragma unroll
                    for (int b = 0; b < 32; b += 8) {
                        T x[8];
#pragma unroll
                        for (int j = 0; j < 8; j++)
                            x[j] = T(__uint_as_float(v[b + j]) * inv);
                        *reinterpret_cast<uint4 *>(own + lane * HD * 2 + (((c + b) / 8) ^ (lane & 7)) * 16) = *reinterpret_cast<const uint4 *>(x);
                    }
                }
                __syncwarp();
                constexpr int kPieces = HD / 8, kRowsAt = 32 / kPieces ? 32 / kPieces : 1;     // of a row; rows at a time
                const int pc = lane % kPieces, r0 = lane / kPieces;
#pragma unroll 4
                for (int rr = r0; rr < 32; rr += kRowsAt) {
                    int t, h;
                    map.at(128 * i + 32 * (warp & 3) + rr, t, h);
                    if (128 * i + 32 * (warp & 3) + rr < w.r.rows) {
                        T *out = static_cast<T *>(a.out) + (w.e.q0 + t) * a.out_stride + (w.head * a.group + h) * HD;
                        reinterpret_cast<uint4 *>(out)[pc] = *reinterpret_cast<const uint4 *>(own + rr * HD * 2 + (pc ^ (rr & 7)) * 16);
                    }
                }
                __syncwarp();
                if (real && a.lse) a.lse[(long long)tok * a.n_q_heads + qh] = l == 0.0f ? -INFINITY : kLn2 * (m + lg2(l));
            } else {
                // rows side by side, so that a warp's stores are contiguous
                float *part = a.partials + (long long)(2 * blockIdx.x + (apart(w.unit_t, (unsigned)run_begin(runs, blockIdx.x)) >= 0)) * S::SlotFloats;
                const int prow = 128 * i + r;
#pragma unroll 1
                for (int c = 0; c < HD; c += 32) {
                    uint32_t v[32];
                    tmem_ld32(t_o + c, v);
                    wait_ld32(v);
                    if (real) {
#pragma unroll
                        for (int b = 0; b < 32; b += 4)
                            __stcg(reinterpret_cast<float4 *>(part) + (c + b) / 4 * S::ROWS + prow,
                                   make_float4(__uint_as_float(v[b]), __uint_as_float(v[b + 1]), __uint_as_float(v[b + 2]),
                                               __uint_as_float(v[b + 3])));
                    }
                }
                if (real) __stcg(reinterpret_cast<float2 *>(part + S::ROWS * HD) + prow, make_float2(m, l));
                if (tid == 0 && k0 == 0) {
                    const unsigned long long begin_t = run_begin(runs, blockIdx.x);
                    const unsigned long long last = begin_t + apart(w.unit_t, (unsigned)begin_t) + w.r.tiles - 1;
                    *splits = {1, w.e.q0, w.r.row0, w.r.rows, w.head, (unsigned)blockIdx.x, run_of_tile(runs, last)};
                }
            }
            fence_before();
        }
    } else if (warp < S::SoftWarps + S::ConvWarps) {
        // ================= codes to fp16 operands =================
        // 16 codes a lane at a time, 8 positions x 4 runs of 16 dimensions, four
        // lanes for a position
        const int cw = warp - S::SoftWarps;
        constexpr int kSpan = HD / 64;                           // 64-dimension spans of a row
        constexpr int kUnits = BN / 8 * kSpan;                   // (8 positions, 64 dimensions)
        constexpr int kLoads = (kUnits + S::ConvWarps - 1) / S::ConvWarps;
        unsigned done = 0;
        uint4 kx[kLoads], vx[kLoads];                            // each loaded a tile ahead
        auto load = [&](uint4(&x)[kLoads], const uint8_t *p) {
#pragma unroll
            for (int n = 0; n < kLoads; n++) {
                const int u = cw + S::ConvWarps * n;
                if (u < kUnits)
                    x[n] = *reinterpret_cast<const uint4 *>(p + (long long)(u / kSpan * 8 + (lane >> 2)) * HD + u % kSpan * 64 + (lane & 3) * 16);
            }
        };
        auto store = [&](const uint4(&x)[kLoads], unsigned char *dst, unsigned long long &full) {
#pragma unroll
            for (int n = 0; n < kLoads; n++) {
                const int u = cw + S::ConvWarps * n;
                if (u >= kUnits) break;
                unsigned char *d = dst + u / kSpan * S::Rows8 + (u % kSpan * 8 + (lane & 3) * 2) * S::Core + (lane >> 2) * 16;
                uint4 lo, hi;
                unpack4<FMT>(x[n].x, lo.x, lo.y);
                unpack4<FMT>(x[n].y, lo.z, lo.w);
                unpack4<FMT>(x[n].z, hi.x, hi.y);
                unpack4<FMT>(x[n].w, hi.z, hi.w);
                *reinterpret_cast<uint4 *>(d) = lo;
                *reinterpret_cast<uint4 *>(d + S::Core) = hi;
            }
            spb::fence_proxy_async();
            __syncwarp();
            if (lane == 0) arrive(spb::smem_u32(&full));
        };
        for (; w.more(); w.next(a)) {
            const long long slot = (long long)w.e.seq * a.l.heads + w.head;
            const uint8_t *kp = a.l.k + slot * a.l.max_seq * HD + (long long)w.r.start * HD;
            const uint8_t *vp = a.l.v + slot * a.l.max_seq * HD + (long long)w.r.start * HD;
            const int k0 = w.k0(), k1 = w.k1();
            load(kx, kp + (long long)k0 * BN * HD);
            load(vx, vp + (long long)k0 * BN * HD);
            // the first warp's lanes: the scales of 16 positions each, a tile ahead
            // (harmless ones past the end).  Four places: those of tile n are written
            // after tile n - 2's scores were taken, so after tile n - 3's weights.
            const float *ksp = a.l.k_scale + slot * (a.l.max_seq >> a.l.block_log2);
            const float *vsp = a.l.v_scale + slot * (a.l.max_seq >> a.l.block_log2);
            float ks = 0.0f, vs = 1.0f;
            auto load_scales = [&](int k) {
                const int at = w.r.start + k * BN + 16 * lane;
                const bool in = cw == 0 && lane < BN / 16 && at < w.e.kv_len;
                ks = in ? ksp[at >> a.l.block_log2] : 0.0f;
                vs = in ? vsp[at >> a.l.block_log2] : 1.0f;
            };
            load_scales(k0);
            // codes of V past the end may be NaN, which a weight of 0 does not undo
            auto no_nan = [&](int j0) {
                if (FMT == SP_Q8_E4M3 && j0 + BN > w.e.kv_len) {
#pragma unroll
                    for (int n = 0; n < kLoads; n++)
                        if (j0 + (cw + S::ConvWarps * n) / kSpan * 8 + (lane >> 2) >= w.e.kv_len) vx[n] = make_uint4(0u, 0u, 0u, 0u);
                }
            };
            for (int k = k0; k < k1; k++, done++) {
                const int st = done & 1;
                if (done >= 2 && !wait(sm.k_free[st], done / 2 - 1)) goto out;
                if (cw == 0 && lane < BN / 16) {
                    const float v = fmaxf(vs, kScaleMin);
                    sm.scales[done & 3][lane] = make_float4(ks, lg2(v), __frcp_rn(v), 0.0f);
                }
                store(kx, sm.k[st], sm.k_full[st]);
                if (done >= 2 && !wait(sm.v_free[st], done / 2 - 1)) goto out;
                no_nan(w.r.start + k * BN);
                store(vx, sm.v[st], sm.v_full[st]);
                // both after the last fence: a fence waits for loads in flight too
                if (k + 1 < k1) {
                    load(kx, kp + (long long)(k + 1) * BN * HD);
                    load(vx, vp + (long long)(k + 1) * BN * HD);
                    load_scales(k + 1);
                }
            }
        }
    } else if (warp == kMmaWarp) {
        // ================= the tensor cores' warp =================
        unsigned done = 0, units = 0;
        auto scores = [&](int i, unsigned n) {                   // tile n of the run, counted over all units
            const uint32_t q = spb::smem_u32(sm.q[i]), k = spb::smem_u32(sm.k[n & 1]);
            const uint32_t d = tmem + (NQ == 2 ? 128 * i : 64 * (n & 1));
#pragma unroll
            for (int s = 0; s < HD / 16; s++)
                mma_ss(d, operand(q + 2 * s * S::Core, S::Core, S::Rows8), operand(k + 2 * s * S::Core, S::Core, S::Rows8), instr(BN, false), s > 0);
            commit(spb::smem_u32(&sm.s_full[NQ == 2 ? i : n & 1]));
        };
        auto values = [&](int i, unsigned n, bool add) {
            const uint32_t v = spb::smem_u32(sm.v[n & 1]);
            const uint32_t p = tmem + (NQ == 2 ? 128 * i : 64 * (n & 1));
#pragma unroll
            for (int s = 0; s < BN / 16; s++)
                mma_ts(tmem + S::ColO + HD * i, p + 8 * s, operand(v + 2 * s * S::Rows8, S::Rows8, S::Core), instr(HD, true), add || s > 0);
            commit(spb::smem_u32(&sm.pv_done[NQ == 2 ? i : n & 1]));
        };
        for (; w.more(); w.next(a), units++) {
            const int n = w.k1() - w.k0();
            if (!wait(sm.k_full[done & 1], done / 2)) goto mma_out;
            for (int i = 0; i < NQ; i++) {
                if (!wait(sm.q_full[i], units)) goto mma_out;
                fence_after();
                scores(i, done);
            }
            commit(spb::smem_u32(&sm.k_free[done & 1]));
            for (int k = 0; k < n; k++, done++) {
                if (k + 1 < n && !wait(sm.k_full[(done + 1) & 1], (done + 1) / 2)) goto mma_out;
                if (NQ == 1 && k + 1 < n) {
                    fence_after();
                    scores(0, done + 1);
                    commit(spb::smem_u32(&sm.k_free[(done + 1) & 1]));
                }
                for (int i = 0; i < NQ; i++) {
                    if (i == 0 && !wait(sm.v_full[done & 1], done / 2)) goto mma_out;
                    if (!wait(sm.p_full[NQ == 2 ? i : done & 1], NQ == 2 ? done : done >> 1)) goto mma_out;
                    fence_after();
                    values(i, done, k > 0);
                    if (NQ == 2 && k + 1 < n) scores(i, done + 1);
                }
                commit(spb::smem_u32(&sm.v_free[done & 1]));
                if (NQ == 2 && k + 1 < n) commit(spb::smem_u32(&sm.k_free[(done + 1) & 1]));
            }
        }
    mma_out:
        // whatever was issued is over before tensor memory goes back
        commit(spb::smem_u32(&sm.end));
        if (lane == 0) spb::wait_stage(spb::smem_u32(&sm.end), 0, nullptr);
    }
out:
    __syncwarp();
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == kMmaWarp)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// Joins the parts of units that fell into several runs (a unit of 256 rows and
// 128 dimensions leaves 133 KB a run, too much for the tail of one CTA): block (i, y) the unit
// that began in run i, 16 of the head's dimensions, a thread for each row.
template <typename T, int FMT, int HD>
__global__ void __launch_bounds__(Shape<HD>::ROWS) k_q8_attn_join(const __grid_constant__ AttnArgs a)
{
    using S = Shape<HD>;
    begin();
    const Split sp = reinterpret_cast<const Split *>(a.counters + kMaxCtas)[blockIdx.x];
    const int row = threadIdx.x;
    if (!sp.valid || row >= sp.rows) return;
    float top = kNone, sum = 0.0f, acc[16];
#pragma unroll
    for (int j = 0; j < 16; j++) acc[j] = 0.0f;
    for (unsigned r = sp.run0; r <= sp.run1; r++) {
        const float *part = a.partials + (long long)(2 * r + (r == sp.run0)) * S::SlotFloats;
        const float2 ml = __ldcg(reinterpret_cast<const float2 *>(part + S::ROWS * HD) + row);
        float4 x[4];
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = __ldcg(reinterpret_cast<const float4 *>(part) + (4 * blockIdx.y + j) * S::ROWS + row);
        const float up = fmaxf(top, ml.x), f0 = ex2(top - up), f1 = ex2(ml.x - up);
        top = up;
        sum = fmaf(ml.y, f1, sum * f0);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            acc[4 * j] = fmaf(x[j].x, f1, acc[4 * j] * f0);
            acc[4 * j + 1] = fmaf(x[j].y, f1, acc[4 * j + 1] * f0);
            acc[4 * j + 2] = fmaf(x[j].z, f1, acc[4 * j + 2] * f0);
            acc[4 * j + 3] = fmaf(x[j].w, f1, acc[4 * j + 3] * f0);
        }
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;      // a sum that is NaN stays
    int tok, qh;
    RowMap(sp.row0, a.group).at(row, tok, qh);
    tok += sp.q0;
    qh += sp.head * a.group;
    T x[16];
#pragma unroll
    for (int j = 0; j < 16; j++) x[j] = T(acc[j] * inv);
    T *out = static_cast<T *>(a.out) + (long long)tok * a.out_stride + qh * HD + 16 * blockIdx.y;
    reinterpret_cast<uint4 *>(out)[0] = reinterpret_cast<const uint4 *>(x)[0];
    reinterpret_cast<uint4 *>(out)[1] = reinterpret_cast<const uint4 *>(x)[1];
    if (a.lse && blockIdx.y == 0) a.lse[(long long)tok * a.n_q_heads + qh] = sum == 0.0f ? -INFINITY : kLn2 * (top + lg2(sum));
}

template <typename T, int FMT, int HD>
int launch_hd(const AttnArgs &a, int sms, cudaStream_t s)
{
    using S = Shape<HD>;
    auto kernel = k_q8_attn_many<T, FMT, HD>;
    constexpr int smem = sizeof(ManySmem<HD>);
    static std::atomic<unsigned long long> ready{0};      // devices whose attribute is set
    int dev = 0;
    cudaGetDevice(&dev);
    if (!(ready.load(std::memory_order_acquire) >> (dev & 63) & 1)) {
        const int rc = sp_check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem),
                                     "q8_attn shared memory");
        if (rc) return rc;
        if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_release);
    }
    const int rc = q8::launch("q8_attn launch", kernel, sms, S::Threads, smem, s, a);
    if (rc) return rc;
    return q8::launch("q8_attn join launch", k_q8_attn_join<T, FMT, HD>, dim3(sms, HD / 16), S::ROWS, 0, s, a);
}

template <typename T, int FMT>
int launch_of(const AttnArgs &a, int hd, int sms, cudaStream_t s)
{
    if (hd == 64) return launch_hd<T, FMT, 64>(a, sms, s);
    if (hd == 128) return launch_hd<T, FMT, 128>(a, sms, s);
    return launch_hd<T, FMT, 256>(a, sms, s);
}

}  // namespace

namespace q8 {
size_t split_bytes(int sm_count) { return ((size_t)sm_count * sizeof(Split) + 255) / 256 * 256; }

int launch_many(const AttnArgs &a, int format, int dtype, int hd, int sms, cudaStream_t s)
{
    if (dtype == SP_DTYPE_F16)
        return format == SP_Q8_INT8 ? launch_of<__half, SP_Q8_INT8>(a, hd, sms, s) : launch_of<__half, SP_Q8_E4M3>(a, hd, sms, s);
    return format == SP_Q8_INT8 ? launch_of<__nv_bfloat16, SP_Q8_INT8>(a, hd, sms, s)
                                : launch_of<__nv_bfloat16, SP_Q8_E4M3>(a, hd, sms, s);
}
}  // namespace q8
