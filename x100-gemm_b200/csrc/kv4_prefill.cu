// kv4_prefill.cu -- attention of many query rows (prompt chunks) over the paged
// 4-bit KV cache on the 5th-generation tensor cores.
//
// Row tiles of 128 rows (token x head of the group, as in kv4_attn.cu) and key
// tiles of 128 positions.  Per key tile and row tile S = Q K^T and O += P V, both
// 128 x 128 x D tcgen05.mma with S, P (over S) and O in TMEM.  One CTA per SM:
//   warps 0-3, 4-7   softmax of step X = 0, 1: a thread owns a row; S from TMEM, running max
//                    (moved only when a score passes it by 2^kLag), P as fp16 back to TMEM
//   fp32 q: 4 warps  add up the products of the steps, a row each (below)
//   4 or 8 warps     raw codes in shared memory -> fp16 K and V tiles in the 128-byte-swizzled
//                    layouts the MMA reads; scale * (code - 8) is an fp16 value, so exact
//   a warp each      issues the MMAs; copies the raw tiles (bulk copies);
//                    walks the work list and hands every role its segments through shared memory
// fp16 q: the steps X are two row tiles over the same key tile (256 rows per item), so that
// a key tile is unpacked once for both; O stays in TMEM.  fp32 q: q and P are carried as hi + lo halves, two
// products each, the steps X are every other key tile of one row tile, and O of a step is added to fp32
// registers: summed in TMEM it was off by 3e-6 at 2600 positions and more at each further one, and is now by 5e-7, for
// some 22 us more (1024 tokens over 2600 positions, 32 heads: 124 us; tensor pipe 0.28 busy, issue slots 0.31, every role waits for others
// most of the time).  fp16 q: 4096 tokens over 8192 positions 405 us (tensor pipe 0.48, issue slots 0.44); p in hi + lo halves there too would
// take 644, so it is rounded to fp16, which with the output's own rounding makes 2.9e-4 instead of 2.1e-4 of the result.
// Either way one step's softmax runs beside the other's products.
//
// The work list is the one of kv4_attn.cu with units of 128 positions, each row
// tile counted with the units that its last row sees.
#include <algorithm>

#include "kv4_attn.cuh"

namespace x100 {
namespace kv4 {

constexpr int kRawStages = 3;
constexpr int kKeys = 128;                 // positions per key tile
constexpr int kPfCtas = 160;               // bound of the grid, which sizes the workspace
constexpr int kPfRows = 256;               // rows per slot of the workspace

// Warps: 8 of softmax, ACC that add up the sums (fp32 q), DQ that unpack, then one each.  SEGS: those that read segments.  Four
// unpacking warps feed two row tiles per key tile (fp16 q; eight only take issue slots from the softmax: 488 against 509 us
// for 2048 tokens over 16384 positions), eight a key tile per step (fp32 q; 135 against 168 us with four).
template <typename T>
struct Roles {
    static constexpr int ACC = sizeof(T) == 4 ? 4 : 0, DQ = sizeof(T) == 4 ? 8 : 4, kDq = 8 + ACC, kMma = kDq + DQ, THREADS = (kMma + 4) * 32, SEGS = kMma + 2;
};

template <int D>
struct Pf {
    static constexpr int QT = 128 * D * 2;                       // one Q tile, or half of fp32 q
    static constexpr int KT = kKeys * D * 2;                     // a K or V tile
    static constexpr int RAW = 4 * Lay<D>::BYTES;                // 64 positions
    static constexpr int K0 = 2 * QT, V0 = K0 + 2 * KT, RAW0 = V0 + 2 * KT, SMEM = RAW0 + kRawStages * RAW;
    static constexpr int SUB = 128 * 128;                        // 128 rows of 64 dims
};

// ---- tcgen05 pieces that ptx.cuh lacks --------------------------------------------
// Issued by the lane whose `lead` is not zero, from code that the whole warp runs: the descriptors then are
// warp-uniform values in uniform registers.  (With one lane in a branch of its own each of them is moved there
// for every instruction, and the products waited for their issue: 140 cycles per 128 x 128 x 16 instead of 64.)
__device__ __forceinline__ void umma_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t acc, uint32_t lead) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc), "r"(lead)
        : "memory");
}
// A from tensor memory
__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t acc, uint32_t lead) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(acc), "r"(lead)
        : "memory");
}
__device__ __forceinline__ void umma_commit_lead(uint64_t *bar, uint32_t lead) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
        "r"(lead)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t *r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void regs_more() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_less() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// ---- the work list ------------------------------------------------------------------
// Positions that row tile rt of a sequence sees, and its units.
template <int RT>
__device__ __forceinline__ int seen(const AttnArgs &a, const Seq &s, int rt) {
    const int rows = min(RT, s.nq * a.G - rt * RT);
    return max(0, min(s.len, s.len - s.nq + div_g(a, rt * RT + rows - 1) + 1));
}
// Units of a row tile in the list: its key tiles, and kLead more for what an item costs besides (q in, sums out),
// so that runs of many short items do not take longer than the others.
constexpr int kLead = 2;
template <int RT>
__device__ __forceinline__ int units_of(const AttnArgs &a, const Seq &s, int rt) { return kLead + max(1, (seen<RT>(a, s, rt) + kKeys - 1) / kKeys); }
// Units of one kv head of a sequence; by one whole warp.
template <int RT>
__device__ __forceinline__ uint32_t head_units(const AttnArgs &a, const Seq &s) {
    uint32_t n = 0;
    for (int rt = threadIdx.x & 31; rt < s.nrt; rt += 32) n += units_of<RT>(a, s, rt);
    return __reduce_add_sync(0xffffffffu, n);
}
// What units_of needs of sequence `j` of the 32 that the lanes have loaded.
__device__ __forceinline__ Seq seq_of_lane(const Seq &mine, int j) {
    Seq s;
    s.nq = __shfl_sync(0xffffffffu, mine.nq, j), s.len = __shfl_sync(0xffffffffu, mine.len, j);
    s.nrt = __shfl_sync(0xffffffffu, mine.nrt, j);
    return s;
}
// Where a run starts: unit u0 is unit `c` of (sequence b, kv head, row tile rt),
// whose first unit is `item`.
struct Start {
    uint32_t u0, u1, item;
    int b, kvh, rt;
};
template <int RT>
__device__ __forceinline__ Start my_start(const AttnArgs &a) {
    const int lane = threadIdx.x & 31;
    Start r = {0, 0, 0, 0, 0, 0};
    uint32_t U = 0;
    for (int b0 = 0; b0 < a.tab.n_seqs; b0 += 32) {
        Seq mine;
        mine.nrt = 0;
        if (b0 + lane < a.tab.n_seqs) mine = load_seq(a, b0 + lane, RT, blockIdx.x == 0);
        for (uint32_t has = __ballot_sync(0xffffffffu, mine.nrt > 0); has; has &= has - 1)
            U += a.pool.nkv * head_units<RT>(a, seq_of_lane(mine, __ffs(has) - 1));
    }
    const uint32_t per = (U + gridDim.x - 1) / gridDim.x;
    if (per * blockIdx.x >= U) return r;
    r.u0 = per * blockIdx.x, r.u1 = min(U, r.u0 + per);
    uint32_t base = 0, hu = 0;
    for (int b0 = 0; b0 < a.tab.n_seqs; b0 += 32) {
        Seq mine;
        mine.nrt = 0;
        if (b0 + lane < a.tab.n_seqs) mine = load_seq(a, b0 + lane, RT, false);
        uint32_t has = __ballot_sync(0xffffffffu, mine.nrt > 0);
        for (; has; has &= has - 1) {
            hu = head_units<RT>(a, seq_of_lane(mine, __ffs(has) - 1));
            if (r.u0 - base < hu * a.pool.nkv) break;
            base += hu * a.pool.nkv;
        }
        if (!has) continue;
        r.b = b0 + __ffs(has) - 1;
        const Seq s = seq_of_lane(mine, __ffs(has) - 1);
        r.kvh = (int)((r.u0 - base) / hu);
        base += r.kvh * hu;
        for (int r0 = 0;; r0 += 32) {
            const uint32_t mine = r0 + lane < s.nrt ? units_of<RT>(a, s, r0 + lane) : 0;
            uint32_t incl = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t up = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += up;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, base + incl > r.u0);
            if (hit) {
                const int l = __ffs(hit) - 1;
                r.item = base + __shfl_sync(0xffffffffu, incl - mine, l);
                r.rt = r0 + l;
                return r;
            }
            base += __shfl_sync(0xffffffffu, incl, 31);
        }
    }
    r.u0 = r.u1 = 0;                       // u0 < U: only if the lengths changed since they were added up
    return r;
}
// A segment: key tiles c0 .. c0 + n - 1 of an item (all cu of them, or a part).
struct Seg {
    int n;                                 // 0: the run is over
    int c0, cu, b, kvh, rt, q0, nq, len, row;
    uint32_t item;                         // the item's first unit
};
constexpr int kSegs = 4;                   // ring of segments

// Barriers that a step's MMAs signal come in pairs, the step's parity choosing one, so that the one for key tile k is
// also what frees that tile's stage (fp16 q, X = 1) and the issuing warp commits only twice a step.
struct PfBars {
    uint64_t raw_full[kRawStages], raw_empty[kRawStages], k_full[2], k_empty[2], v_full[2], v_empty[2];
    uint64_t s_full[2][2], p_ready[2], o_done[2][2], q_full, q_empty, drain, o_free[2], fin, ml_free, seg_full[kSegs], seg_empty[kSegs];
    uint32_t raw_ok[kRawStages];           // bit i: 16-position tile i of the raw stage was copied
    uint32_t tmem;
    int abort_flag;
    Seg seg[kSegs];
    float2 ml[2][128];                     // fp32 q: (m, l) of the two steps' rows at a segment's end
    float m_step[2][2][128];               // and the max that a step's products are relative to
};

// 8 codes of a word times their scale, as fp16 in the order 0, 4, 1, 5, 2, 6, 3, 7
__device__ __forceinline__ uint4 eight(uint32_t w, __half2 d, const Exponents &x) {
    const uint32_t w8 = w >> 8;
    return make_uint4(u32(__hmul2(low_codes(w, x), d)), u32(__hmul2(high_codes(w, x), d)), u32(__hmul2(low_codes(w8, x), d)),
                      u32(__hmul2(high_codes(w8, x), d)));
}

// The query order that goes with it: the halves of 8 dims (a.x = dims 0, 1 ..) as 0, 4, 1, 5, 2, 6, 3, 7
__device__ __forceinline__ uint4 as_eight(uint4 a) {
    return make_uint4(__byte_perm(a.x, a.z, 0x5410), __byte_perm(a.x, a.z, 0x7632), __byte_perm(a.y, a.w, 0x5410), __byte_perm(a.y, a.w, 0x7632));
}

// x * a + b for two floats at once
__device__ __forceinline__ void fma2(float &x, float &y, uint64_t a, uint64_t b) {
    asm("{\n\t.reg .b64 t;\n\tmov.b64 t, {%0, %1};\n\tfma.rn.f32x2 t, t, %2, %3;\n\tmov.b64 {%0, %1}, t;\n\t}" : "+f"(x), "+f"(y) : "l"(a), "l"(b));
}
__device__ __forceinline__ uint64_t both(float x) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %1};" : "=l"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t s, float x, float y) {
    asm("{\n\t.reg .b64 t;\n\tmov.b64 t, {%1, %2};\n\tadd.rn.f32x2 %0, %0, t;\n\t}" : "+l"(s) : "f"(x), "f"(y));
    return s;
}

// C columns of a row from `col` on: times inv to `op` (a live row of a whole item), or as they are to the slot of a part
template <typename T, int D, int C>
__device__ __forceinline__ void put_sums(const AttnArgs &a, const float (&o)[C], float inv, int col, bool whole, bool live, T *op, int slot, int prow) {
    if (!whole) {
        float4 *pp = reinterpret_cast<float4 *>(a.part) + ((long)slot * (D / 4) + col / 4) * kPfRows + prow;
#pragma unroll
        for (int k = 0; k < C / 4; ++k) pp[k * kPfRows] = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
    } else if (live) {
        // columns 0 .. 7 of a group of 8 are its dims 0, 4, 1, 5, 2, 6, 3, 7
#pragma unroll
        for (int h = 0; h < C; h += 8) {
            const float y[8] = {o[h] * inv, o[h + 2] * inv, o[h + 4] * inv, o[h + 6] * inv, o[h + 1] * inv, o[h + 3] * inv, o[h + 5] * inv, o[h + 7] * inv};
            if constexpr (sizeof(T) == 4) {
                *reinterpret_cast<float4 *>(op + col + h) = make_float4(y[0], y[1], y[2], y[3]);
                *reinterpret_cast<float4 *>(op + col + h + 4) = make_float4(y[4], y[5], y[6], y[7]);
            } else {
                *reinterpret_cast<uint4 *>(op + col + h) = make_uint4(u32(__floats2half2_rn(y[0], y[1])), u32(__floats2half2_rn(y[2], y[3])),
                                                                      u32(__floats2half2_rn(y[4], y[5])), u32(__floats2half2_rn(y[6], y[7])));
            }
        }
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(Roles<T>::THREADS, 1) prefill_kernel(const AttnArgs a) {
    using L = Lay<D>;
    using P = Pf<D>;
    constexpr bool HL = sizeof(T) == 4;
    constexpr int RT = HL ? 128 : 256;      // rows per item
    using W = Roles<T>;
    constexpr int KS = D / 16, VS = kKeys / 16, kDqWarps = W::DQ;
    extern __shared__ __align__(1024) uint8_t sm[];
    __shared__ PfBars bars;
    // broadcast, so that the compiler knows it for a warp-uniform value and the branches on it for uniform ones
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, wg = warp >> 2;
    if (threadIdx.x == 0) {
        bars.abort_flag = 0;
        for (int i = 0; i < kRawStages; ++i) mbar_init(&bars.raw_full[i], 1), mbar_init(&bars.raw_empty[i], kDqWarps);
        for (int i = 0; i < kSegs; ++i) mbar_init(&bars.seg_full[i], 1), mbar_init(&bars.seg_empty[i], W::SEGS);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars.k_full[i], kDqWarps), mbar_init(&bars.k_empty[i], 1);
            mbar_init(&bars.v_full[i], kDqWarps), mbar_init(&bars.v_empty[i], 1);
            mbar_init(&bars.p_ready[i], 4);
            for (int k = 0; k < 2; ++k) mbar_init(&bars.s_full[i][k], 1), mbar_init(&bars.o_done[i][k], 1);
        }
        mbar_init(&bars.q_full, 8), mbar_init(&bars.q_empty, 1), mbar_init(&bars.drain, 1);
        mbar_init(&bars.o_free[0], 4), mbar_init(&bars.o_free[1], 4), mbar_init(&bars.fin, 8), mbar_init(&bars.ml_free, 4);
        fence_barrier_init();
    }
    if (warp == W::kMma) {
        tmem_alloc(&bars.tmem, 512);
        tmem_relinquish();
    }
    pdl_launch_dependents();
    pdl_wait();
    if (threadIdx.x >= 32 && threadIdx.x < 34) a.meta[blockIdx.x * 2 + threadIdx.x - 32] = make_int4(-1, 0, 0, 0);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // S, O of step X: + 128 X columns.  All 512 columns are this CTA's, so they start at column 0.
    constexpr uint32_t tS = 0, tO = 256;
    const uint32_t tmem = bars.tmem;
    volatile int *abort_flag = &bars.abort_flag;
    auto wait = [&](uint64_t *bar, uint32_t parity) { return (bool)__all_sync(0xffffffffu, mbar_wait_quiet(bar, parity, abort_flag, a.status)); };
    // the i-th segment; a role reads what it needs of it before release(i)
    auto segment = [&](uint32_t i) { return wait(&bars.seg_full[i % kSegs], i / kSegs & 1); };
    auto release = [&](uint32_t i) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.seg_empty[i % kSegs]);
    };
    bool ok = __all_sync(0xffffffffu, tmem == 0 && (smem_u32(sm) & 1023) == 0);
    if (!ok && threadIdx.x == 0) atomicCAS(a.status, 0, X100_E_LAUNCH);
    if (wg < 2) {
        // ================================ softmax ================================
        // registers: the launch's 65536 (512 threads of 128) or 61440 (768 of 80) shared out anew; fp32 q's softmax keeps its 80
        regs_more<HL ? 80 : 192>();
        const int X = wg, row = threadIdx.x & 127;
        const uint32_t toff = (uint32_t)((warp & 3) * 32) << 16, sx = tS + 128 * X + toff, ox = tO + 128 * X + toff;
        uint32_t step = 0;                       // steps of this X
        // q of a segment into the swizzled K-major tiles.  fp16 q: a thread its own row.  fp32 q: a warp 16 of the 128 rows, with D / 8
        // neighbouring lanes a row (a thread half of its own row took 130 instead of 124 us for 1024 tokens over 2600 positions).
        auto q_row = [&](const Seg &v, int row) -> const T * {
            const int r = v.rt * RT + row, tok = div_g(a, r);
            return r < v.nq * a.G ? static_cast<const T *>(a.q) + (long)(v.q0 + tok) * a.qs + (long)(v.kvh * a.G + r - tok * a.G) * D : nullptr;
        };
        auto put_q = [&](const Seg &v) {
            if constexpr (HL) {
                constexpr int LR = D / 8, RW = 32 / LR;
                const int ch = lane % LR;                // 8 dims
#pragma unroll 2
                for (int i = 0; i < 16 / RW; ++i) {
                    const int r = warp * 16 + i * RW + lane / LR;
                    uint4 hi = make_uint4(0, 0, 0, 0), lo = hi;
                    if (const T *qp = q_row(v, r)) {
                        const float4 x = *reinterpret_cast<const float4 *>(qp + ch * 8), y = *reinterpret_cast<const float4 *>(qp + ch * 8 + 4);
                        const float u = a.q_up;
                        split2(x.x * u, x.y * u, hi.x, lo.x), split2(x.z * u, x.w * u, hi.y, lo.y);
                        split2(y.x * u, y.y * u, hi.z, lo.z), split2(y.z * u, y.w * u, hi.w, lo.w);
                    }
                    uint8_t *at = sm + r * 128 + (ch >> 3) * P::SUB + (((ch & 7) ^ (r & 7)) << 4);
                    *reinterpret_cast<uint4 *>(at) = as_eight(hi);
                    *reinterpret_cast<uint4 *>(at + P::QT) = as_eight(lo);
                }
            } else {
                const T *qp = q_row(v, 128 * X + row);
                uint8_t *qs = sm + X * P::QT + row * 128;
#pragma unroll
                for (int ch = 0; ch < D / 8; ++ch) {     // 8 dims
                    const uint4 x = qp ? *reinterpret_cast<const uint4 *>(qp + ch * 8) : make_uint4(0, 0, 0, 0);
                    *reinterpret_cast<uint4 *>(qs + (ch >> 3) * P::SUB + (((ch & 7) ^ (row & 7)) << 4)) = as_eight(x);
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.q_full);
        };
        uint32_t nseg = 0;
        ok = segment(0);
        if (ok && bars.seg[0].n) put_q(bars.seg[0]);
        for (; ok; ++nseg) {
            const Seg &w = bars.seg[nseg % kSegs];
            const int n = w.n;
            if (n == 0) break;
            const int *trow = a.tab.page + (long)w.row * a.tab.stride;
            const int c0 = w.c0, len = w.len;
            int lim;                             // positions the row sees
            {
                const int r = w.rt * RT + (HL ? 0 : 128 * X) + row;
                lim = r < w.nq * a.G ? min(len, len - w.nq + div_g(a, r) + 1) : 0;
            }
            bool hole = false;                   // pages out of range among the segment's
            {
                const int ps = a.pool.page_shift, e0 = (c0 * kKeys) >> ps, e1 = (min((c0 + n) * kKeys, len) + (1 << ps) - 1) >> ps;
                for (int i = e0 + lane; i < e1; i += 32) hole = hole || (unsigned)__ldg(trow + i) >= (unsigned)a.pool.n_pages;
                hole = __any_sync(0xffffffffu, hole);
                if (hole && lane == 0) atomicCAS(a.status, 0, X100_E_ARG);
            }
            float m = -INFINITY, nm = 0.f, l = 0.f;
            const uint64_t sl2 = both(a.sl);
            for (int c = HL ? X : 0; c < n; c += HL ? 2 : 1, ++step) {
                const int p0 = (c0 + c) * kKeys;
                ok = wait(&bars.s_full[X][step & 1], step >> 1 & 1);
                if (!ok) break;
                tc_fence_after();
                // fp16 q keeps all scores of the row; fp32 q, whose registers the sums need, loads them twice, 32 at a time
                float s[HL ? 32 : 128], mx[4];
                auto load = [&](float *v, int i) { tmem_ld32(sx + 32 * i, *reinterpret_cast<uint32_t(*)[32]>(v)); };
                bool mask = false;               // fp32 q: this tile has masked positions
                uint32_t gone = 0;               // 16-position tiles without a page
                auto find_gone = [&]() {
                    if (hole)
                        for (int i = 0; i < 8 && p0 + 16 * i < len; ++i)
                            if ((unsigned)__ldg(trow + ((p0 + 16 * i) >> a.pool.page_shift)) >= (unsigned)a.pool.n_pages) gone |= 1u << i;
                };
                auto cover = [&](float *v, int i) {
                    const int cut = lim - p0 - 32 * i;
#pragma unroll
                    for (int k = 0; k < 32; ++k)
                        if (k >= cut) v[k] = -INFINITY;
                    if (gone) {
#pragma unroll
                        for (int k = 0; k < 32; ++k)
                            if (gone >> (2 * i + k / 16) & 1) v[k] = -INFINITY;
                    }
                };
                if constexpr (HL) {
                    mask = __any_sync(0xffffffffu, p0 + kKeys > lim) || hole;
                    find_gone();
                    mx[0] = mx[1] = mx[2] = mx[3] = -INFINITY;
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        load(s, h);
                        tmem_wait_ld();
                        if (mask) cover(s, h);
#pragma unroll
                        for (int i = 0; i < 32; i += 8)
#pragma unroll
                            for (int k = 0; k < 4; ++k) mx[k] = fmaxf(fmaxf(mx[k], s[i + k]), s[i + 4 + k]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) load(s + 32 * i, i);
                    tmem_wait_ld();
                    if (__any_sync(0xffffffffu, p0 + kKeys > lim) || hole) {
                        const int cut = lim - p0;
#pragma unroll
                        for (int i = 0; i < 128; ++i)
                            if (i >= cut) s[i] = -INFINITY;
                        find_gone();
                        if (gone)
#pragma unroll
                            for (int i = 0; i < 128; ++i)
                                if (gone >> (i / 16) & 1) s[i] = -INFINITY;
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) mx[k] = s[k];
#pragma unroll
                    for (int i = 4; i < 124; i += 8)
#pragma unroll
                        for (int k = 0; k < 4; ++k) mx[k] = fmaxf(fmaxf(mx[k], s[i + k]), s[i + 4 + k]);
#pragma unroll
                    for (int k = 0; k < 4; ++k) mx[k] = fmaxf(mx[k], s[124 + k]);
                }
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.sl;
                if (__any_sync(0xffffffffu, top > m + kLag)) {
                    const float mn = fmaxf(m, top), f = mn == -INFINITY ? 1.f : ex2(m - mn);
                    m = mn;
                    nm = mn == -INFINITY ? 0.f : kUp - mn;
                    l *= f;
                    if (!HL && c >= 1) {         // O holds sums
                        ok = wait(&bars.o_done[X][(step - 1) & 1], (step - 1) >> 1 & 1);
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll
                        for (int i = 0; i < D / 16; ++i) {
                            uint32_t v[16];
                            tmem_ld16(ox + 16 * i, v);
                            tmem_wait_ld();
#pragma unroll
                            for (int k = 0; k < 16; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) * f);
                            tmem_st16(ox + 16 * i, v);
                        }
                    }
                }
                if constexpr (HL) bars.m_step[X][step & 1][row] = m;
                const uint64_t nm2 = both(nm);
                uint64_t sum[2] = {0ull, 0ull};   // two floats each
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float *v = s + (HL ? 0 : 32 * i);
                    if constexpr (HL) {
                        load(v, i);
                        tmem_wait_ld();
                        if (mask) cover(v, i);
                    }
                    uint32_t hi[16], lo[8];
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        float x = v[2 * k], y = v[2 * k + 1];
                        fma2(x, y, sl2, nm2);
                        x = ex2(x), y = ex2(y);
                        sum[k & 1] = add2(sum[k & 1], x, y);
                        if constexpr (HL) {              // 16 positions' hi and lo over the scores they came from
                            split2(x, y, hi[k & 7], lo[k & 7]);
                            if (k % 8 == 7) tmem_st8(sx + 32 * i + 2 * (k - 7), hi), tmem_st8(sx + 32 * i + 2 * (k - 7) + 8, lo);
                        } else {
                            hi[k] = u32(__floats2half2_rn(x, y));
                        }
                    }
                    if constexpr (!HL) tmem_st16(sx + 16 * i, hi);
                }
                {
                    float s0, s1, s2, s3;
                    asm("mov.b64 {%0, %1}, %2;" : "=f"(s0), "=f"(s1) : "l"(sum[0]));
                    asm("mov.b64 {%0, %1}, %2;" : "=f"(s2), "=f"(s3) : "l"(sum[1]));
                    l += (s0 + s1) + (s2 + s3);
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars.p_ready[X]);
            }
            if (!ok) break;
            // ---- the next segment's q, as soon as the products have read this one's: its first scores then come
            // while the sums go out ----
            ok = segment(nseg + 1);
            if (ok && bars.seg[(nseg + 1) % kSegs].n) {
                ok = wait(&bars.q_empty, nseg & 1);
                if (ok) put_q(bars.seg[(nseg + 1) % kSegs]);
            }
            if constexpr (HL) {
                if (ok) ok = wait(&bars.ml_free, (nseg & 1) ^ 1);
                bars.ml[X][row] = make_float2(m, l);
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars.fin);
                release(nseg);
                continue;
            }
            // ---- out ----
            if (ok) ok = wait(&bars.o_done[X][(step - 1) & 1], (step - 1) >> 1 & 1);
            if (!ok) break;
            tc_fence_after();
            const int r = w.rt * RT + 128 * X + row;
            const bool live = r < w.nq * a.G, whole = n == w.cu;
            const int tok = live ? div_g(a, r) : 0;
            const int slot = (int)blockIdx.x * 2 + (nseg ? 1 : 0);
            const float inv = whole ? (l > 0.f ? 1.f / l : 0.f) : 1.f;
            T *op = static_cast<T *>(a.out) + (long)(w.q0 + tok) * a.os + (long)(w.kvh * a.G + r - tok * a.G) * D;
#pragma unroll
            for (int col = 0; col < D; col += 64) {  // every round trip to tensor memory takes some hundred cycles
                float o[64];
#pragma unroll
                for (int k = 0; k < 64; k += 16) tmem_ld16(ox + col + k, *reinterpret_cast<uint32_t(*)[16]>(o + k));
                tmem_wait_ld();
                put_sums<T, D, 64>(a, o, inv, col, whole, live, op, slot, 128 * X + row);
            }
            if (!whole) {
                a.ml[(long)slot * kPfRows + 128 * X + row] = make_float2(m, l);
                if (X == 0 && row == 0) a.meta[slot] = make_int4((int)w.item, w.b, w.kvh, w.rt | (c0 ? kInside : 0));
            }
            tc_fence_before();                      // the next step's products overwrite the sums
            release(nseg);
        }
    } else if (HL && warp < W::kDq) {
        // ================================ sums (fp32 q) ================================
        // A tensor-core sum truncates, 1.9e-8 of what it holds at each product, 16 a step.  So each step's products start
        // from zero, and these warps add the steps up, each by its max; a thread has a row.
        regs_more<176>();
        const int row = threadIdx.x & 127;
        const uint32_t toff = (uint32_t)((warp & 3) * 32) << 16;
        uint32_t steps = 0;                      // X = 1's in the high half
        for (uint32_t nseg = 0; ok; ++nseg) {
            ok = segment(nseg);
            if (!ok) break;
            const Seg &w = bars.seg[nseg % kSegs];
            const int n = w.n;
            if (n == 0) break;
            float o[HL ? D : 64], M = -INFINITY;
#pragma unroll
            for (int i = 0; i < D; ++i) o[i] = 0.f;
            for (int c = 0; c < n; ++c) {
                const int X = c & 1;
                const uint32_t st = steps >> (16 * X);
                ok = wait(&bars.o_done[X][st & 1], st >> 1 & 1);
                if (!ok) break;
                tc_fence_after();
                const float mx = bars.m_step[X][st & 1][row], mn = fmaxf(M, mx);
                if (__any_sync(0xffffffffu, mx > M)) {
                    const float f = mn == -INFINITY ? 0.f : ex2(M - mn);
#pragma unroll
                    for (int i = 0; i < D; ++i) o[i] *= f;
                    M = mn;
                }
                const float f = mx == -INFINITY ? 0.f : ex2(mx - M);
#pragma unroll
                for (int i = 0; i < D; i += 32) {
                    float v[32];
                    tmem_ld32(tO + 128 * X + toff + i, *reinterpret_cast<uint32_t(*)[32]>(v));
                    tmem_wait_ld();
#pragma unroll
                    for (int k = 0; k < 32; ++k) o[i + k] = fmaf(v[k], f, o[i + k]);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars.o_free[X]);
                steps = X ? steps + 0x10000u : (steps & 0xffff0000u) | (steps + 1 & 0xffffu);
            }
            if (ok) ok = wait(&bars.fin, nseg & 1);
            if (!ok) break;
            const float2 s0 = bars.ml[0][row], s1 = bars.ml[1][row];
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.ml_free);
            // M is the larger max of the last step of either; a later, lower one cannot be
            const float l = M == -INFINITY ? 0.f : s0.y * ex2(s0.x - M) + s1.y * ex2(s1.x - M);
            const int r = w.rt * RT + row;
            const bool live = r < w.nq * a.G, whole = n == w.cu;
            const int tok = live ? div_g(a, r) : 0, slot = (int)blockIdx.x * 2 + (nseg ? 1 : 0);
            const float inv = whole ? (l > 0.f ? 1.f / l : 0.f) : 1.f;
            T *op = static_cast<T *>(a.out) + (long)(w.q0 + tok) * a.os + (long)(w.kvh * a.G + r - tok * a.G) * D;
            put_sums<T, D, HL ? D : 64>(a, o, inv, 0, whole, live, op, slot, row);
            if (!whole) {
                a.ml[(long)slot * kPfRows + row] = make_float2(M, l);
                if (row == 0) a.meta[slot] = make_int4((int)w.item, w.b, w.kvh, w.rt | (w.c0 ? kInside : 0));
            }
            release(nseg);
        }
    } else if (warp < W::kMma) {
        // ================================ codes -> fp16 tiles ================================
        regs_less<HL ? 48 : 72>();
        const Exponents expo;
        const int th = threadIdx.x - W::kDq * 32;
        uint32_t tile = 0, raw = 0;                // key tiles, raw stages so far
        for (uint32_t nseg = 0; ok; ++nseg) {
            ok = segment(nseg);
            if (!ok) break;
            const Seg &w = bars.seg[nseg % kSegs];
            const int n = w.n, c0 = w.c0, len = w.len;
            release(nseg);
            if (n == 0) break;
            for (int c = c0; c < c0 + n && ok; ++c, ++tile) {
                const uint32_t st = tile & 1, par = (tile >> 1 & 1) ^ 1;
                uint8_t *kt = sm + P::K0 + st * P::KT, *vt = sm + P::V0 + st * P::KT;
                // all of K first: its products come a step ahead of V's
                ok = wait(HL ? &bars.k_empty[st] : &bars.s_full[1][st], par);
                if (!ok) break;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t rs = (raw + half) % kRawStages;
                    ok = wait(&bars.raw_full[rs], (raw + half) / kRawStages & 1);
                    if (!ok) break;
                    const uint8_t *rp = sm + P::RAW0 + rs * P::RAW;
                    const uint32_t have = bars.raw_ok[rs];
                    // 4 lanes per position, a word of every block each
#pragma unroll
                    for (int u = 0; u < 8 / kDqWarps; ++u) {
                        const int key = u * (8 * kDqWarps) + (th >> 2), t = th & 3, in = key & 15, kk = half * 64 + key;
                        const uint8_t *tp = rp + (key >> 4) * L::BYTES;
                        const bool on = (have >> (key >> 4) & 1) && c * kKeys + kk < len;
                        uint32_t kw[L::NB];
                        __half kd[L::NB];
                        if constexpr (D == 128) {
                            *reinterpret_cast<uint4 *>(kw) = *reinterpret_cast<const uint4 *>(tp + L::k_word(in, 0, t));
                            *reinterpret_cast<uint2 *>(kd) = *reinterpret_cast<const uint2 *>(tp + L::k_scale(in, 0));
                        } else {
                            *reinterpret_cast<uint2 *>(kw) = *reinterpret_cast<const uint2 *>(tp + L::k_word(in, 0, t));
                            *reinterpret_cast<uint32_t *>(kd) = *reinterpret_cast<const uint32_t *>(tp + L::k_scale(in, 0));
                        }
#pragma unroll
                        for (int b = 0; b < L::NB; ++b) {
                            const __half2 d = __half2half2(on ? kd[b] : __ushort_as_half(0));
                            *reinterpret_cast<uint4 *>(kt + (b >> 1) * P::SUB + kk * 128 + ((((b & 1) * 4 + t) ^ (kk & 7)) << 4)) = eight(kw[b], d, expo);
                        }
                    }
                }
                if (!ok) break;
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars.k_full[st]);
                ok = wait(HL ? &bars.v_empty[st] : &bars.o_done[1][st], par);
                if (!ok) break;
#pragma unroll
                for (int u = 0; u < 8 / kDqWarps; ++u) {
                    // a warp has a 16-position tile; a lane the D / 8 dims from g * D / 8 of positions t + 4 m
                    const int tl = u * kDqWarps + warp - W::kDq, g = lane >> 2, t = lane & 3;
                    const uint32_t rs = (raw + (tl >> 2)) % kRawStages;
                    const uint8_t *tp = sm + P::RAW0 + rs * P::RAW + (tl & 3) * L::BYTES;
                    const int left = bars.raw_ok[rs] >> (tl & 3) & 1 ? len - c * kKeys : 0;   // positions of the sequence from the key tile on
                    __half vd[4];
                    *reinterpret_cast<uint2 *>(vd) = *reinterpret_cast<const uint2 *>(tp + L::v_scale(t, g * (D / 8) / 32));
#pragma unroll
                    for (int i = 0; i < (D == 128 ? 2 : 1); ++i) {
                        const uint4 x = *reinterpret_cast<const uint4 *>(tp + L::V0 + i * 512 + lane * 16);
                        const uint32_t vw[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            // D = 128: words 2 q, 2 q + 1 of position t + 4 (2 i + q); D = 64: word q of position t + 4 q
                            const int m = D == 128 ? 2 * i + (k >> 1) : k, kk = tl * 16 + 4 * m + t;
                            const int dim = g * (D / 8) + (D == 128 ? (k & 1) * 8 : 0);
                            const __half2 d = __half2half2(kk < left ? vd[m] : __ushort_as_half(0));
                            *reinterpret_cast<uint4 *>(vt + (dim >> 6) * P::SUB + kk * 128 + ((((dim & 63) >> 3) ^ (kk & 7)) << 4)) = eight(vw[k], d, expo);
                        }
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&bars.raw_empty[raw % kRawStages]);
                    mbar_arrive(&bars.raw_empty[(raw + 1) % kRawStages]);
                    mbar_arrive(&bars.v_full[st]);
                }
                raw += 2;
            }
        }
    } else {
        regs_less<HL ? 48 : 56>();
        if (warp == W::kMma) {
            // ================================ products ================================
            const uint32_t lead = lane == 0 ? 1u : 0u;
            constexpr uint32_t idS = idesc_make(1, 0, 0, 128, 128), idO = idesc_make(1, 0, 1, 128, D);
            // matrix descriptors; tiles and slices of them differ in the address field (16-byte steps) alone
            const uint64_t descQ = smem_desc_sw128(smem_u32(sm), 16, 1024), descK = smem_desc_sw128(smem_u32(sm + P::K0), 16, 1024);
            const uint64_t descV = smem_desc_sw128(smem_u32(sm + P::V0), P::SUB, 1024);
            uint32_t tile = 0, sdone = 0, pdone = 0;   // key tiles; bit X: scores and sums issued of step X so far, odd or even
            for (uint32_t nseg = 0; ok; ++nseg) {
                ok = segment(nseg);
                if (!ok) break;
                const int n = __shfl_sync(0xffffffffu, bars.seg[nseg % kSegs].n, 0);   // uniform for the compiler too
                release(nseg);
                if (n == 0) break;
                const int S = HL ? n : 2 * n;
                ok = wait(&bars.q_full, nseg & 1);
                if (!ok) break;
                auto scores = [&](int s) {
                    const int X = s & 1;
                    const uint32_t tl = tile + (HL ? s : s >> 1), st = tl & 1;
                    if (HL || X == 0) {
                        if (!wait(&bars.k_full[st], tl >> 1 & 1)) return false;
                    }
                    tc_fence_after();
                    const uint64_t qd = descQ + (HL ? 0 : X * (P::QT >> 4)), kd = descK + st * (P::KT >> 4);
#pragma unroll
                    for (int p = HL ? 1 : 0; p >= 0; --p)    // lo first: what is added to is small then, and with it what is cut off
#pragma unroll
                        for (int k = 0; k < KS; ++k) {
                            const uint32_t off = ((k >> 2) * P::SUB + (k & 3) * 32) >> 4;
                            umma_ss(tS + 128 * X, qd + p * (P::QT >> 4) + off, kd + off, idS, (p < (HL ? 1 : 0) || k) ? 1u : 0u, lead);
                        }
                    umma_commit_lead(&bars.s_full[X][sdone >> X & 1], lead);
                    sdone ^= 1u << X;
                    if (HL) umma_commit_lead(&bars.k_empty[st], lead);
                    if (s == S - 1) umma_commit_lead(&bars.q_empty, lead);
                    return true;
                };
                for (int s = 0; s < 2 && s < S && ok; ++s) ok = scores(s);
                for (int s = 0; s < S && ok; ++s) {
                    const int X = s & 1;
                    const uint32_t tl = tile + (HL ? s : s >> 1), st = tl & 1, odd = pdone >> X & 1;
                    ok = wait(&bars.p_ready[X], odd);
                    if (ok && (HL || X == 0)) ok = wait(&bars.v_full[st], tl >> 1 & 1);
                    if (HL && ok) ok = wait(&bars.o_free[X], odd ^ 1);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t vd = descV + st * (P::KT >> 4);
                    const uint32_t more = !HL && s >= 2 ? 1u : 0u;      // O of X holds sums of the segment
#pragma unroll
                    for (int p = HL ? 1 : 0; p >= 0; --p)
#pragma unroll
                        for (int k = 0; k < VS; ++k)
                            umma_ts(tO + 128 * X, tS + 128 * X + (HL ? 16 * k + 8 * p : 8 * k), vd + k * (2048 >> 4), idO, (p < (HL ? 1 : 0) || k) ? 1u : more, lead);
                    umma_commit_lead(&bars.o_done[X][odd], lead);
                    pdone ^= 1u << X;
                    if (HL) umma_commit_lead(&bars.v_empty[st], lead);
                    if (s + 2 < S) ok = scores(s + 2);
                }
                tile += n;
            }
            umma_commit_lead(&bars.drain, lead);    // every product issued has ended when this completes
            mbar_wait_drain(&bars.drain, 0, kWaitLimitNs);
        } else if (warp == W::kMma + 1) {
            // ================================ raw tiles ================================
            uint32_t raw = 0;
            const int ps = a.pool.page_shift;
            const long page_step = a.pool.page_bytes * a.pool.nkv;
            for (uint32_t nseg = 0; ok; ++nseg) {
                ok = segment(nseg);
                if (!ok) break;
                const Seg &w = bars.seg[nseg % kSegs];
                const int n = w.n, c0 = w.c0, len = w.len;
                const int *trow = a.tab.page + (long)w.row * a.tab.stride;
                const uint8_t *base = a.pool.pages + (long)w.kvh * a.pool.page_bytes;
                release(nseg);
                if (n == 0) break;
                for (int h = 2 * c0; h < 2 * (c0 + n) && ok; ++h, ++raw) {
                    const uint32_t rs = raw % kRawStages;
                    const int pos = h * 64 + lane * 16;
                    const int page = lane < 4 && pos < len ? __ldg(trow + (pos >> ps)) : -1;
                    const bool on = (unsigned)page < (unsigned)a.pool.n_pages;
                    const uint32_t have = __ballot_sync(0xffffffffu, on);
                    ok = wait(&bars.raw_empty[rs], (raw / kRawStages & 1) ^ 1);
                    if (!ok) break;
                    if (lane == 0) {
                        bars.raw_ok[rs] = have;
                        mbar_arrive_expect_tx(&bars.raw_full[rs], __popc(have) * L::BYTES);
                    }
                    __syncwarp();
                    if (on)
                        bulk_load(sm + P::RAW0 + rs * P::RAW + lane * L::BYTES, base + page * page_step + ((pos & ((1 << ps) - 1)) >> 4) * L::BYTES, L::BYTES,
                                  &bars.raw_full[rs]);
                }
            }
            if (!ok) {                              // let the copies in flight land before the CTA ends
                *abort_flag = 1;
                if (lane == 0)
                    for (uint32_t i = raw > kRawStages ? raw - kRawStages : 0; i < raw; ++i)
                        mbar_wait_drain(&bars.raw_full[i % kRawStages], i / kRawStages & 1, kWaitLimitNs);
            }
        } else if (warp == W::kMma + 2) {
            // ================================ work list ================================
            const Start at = my_start<RT>(a);
            uint32_t u = at.u0, item = at.item, nseg = 0;
            int b = at.b, kvh = at.kvh, rt = at.rt;
            Seq sq;
            if (u < at.u1) sq = load_seq(a, b, RT, false);
            for (bool more = true; more && ok;) {
                Seg g = {};
                more = u < at.u1;
                if (more) {
                    // a run that ends within an item's kLead units has none of its key tiles, and one that starts there has all
                    const int cu = units_of<RT>(a, sq, rt) - kLead, k0 = (int)(u - item), k1 = (int)min((uint32_t)(cu + kLead), k0 + (at.u1 - u));
                    g.c0 = max(0, k0 - kLead);
                    g.n = max(0, k1 - kLead) - g.c0;
                    g.cu = cu, g.b = b, g.kvh = kvh, g.rt = rt, g.q0 = sq.q0, g.nq = sq.nq, g.len = sq.len, g.row = sq.row, g.item = item;
                    item += cu + kLead;
                    u = item;
                    if (u < at.u1 && ++rt >= sq.nrt) {
                        rt = 0;
                        if (++kvh == a.pool.nkv) {
                            kvh = 0;
                            do {
                                if (++b < a.tab.n_seqs) sq = load_seq(a, b, RT, false);
                                else u = at.u1;
                            } while (!sq.nrt && u < at.u1);
                        }
                    }
                    if (g.n <= 0) continue;
                }
                ok = wait(&bars.seg_empty[nseg % kSegs], (nseg / kSegs & 1) ^ 1);
                if (!ok) break;
                if (lane == 0) {
                    bars.seg[nseg % kSegs] = g;
                    mbar_arrive(&bars.seg_full[nseg % kSegs]);
                }
                ++nseg;
            }
        }
    }
    if (!ok) *abort_flag = 1;
    tc_fence_before();
    __syncthreads();
    if (warp == W::kMma) tmem_dealloc(tmem, 512);
}

// Joins the parts of an item at the first cut inside it (as merge_kernel in kv4_attn.cu): a thread per row, 16 columns per CTA.
template <typename T, int D>
__global__ void __launch_bounds__(kPfRows) prefill_merge_kernel(const AttnArgs a, int grid) {
    constexpr int RT = sizeof(T) == 4 ? 128 : 256;
    pdl_launch_dependents();
    pdl_wait();
    const int c = blockIdx.x + 1, col = blockIdx.y * 16, row = threadIdx.x;
    const int4 here = __ldcg(a.meta + 2 * c), p0 = __ldcg(a.meta + 2 * c - 2), p1 = __ldcg(a.meta + 2 * c - 1);
    if (here.x == -1 || !(here.w & kInside)) return;
    int slot0 = 2 * c - 1;
    if (p1.x != here.x) {
        if (p0.x != here.x || (p0.w & kInside)) return;
        slot0 = 2 * c - 2;
    }
    const int b = here.y, rt = here.w & (kInside - 1), r = rt * RT + row;
    int q0, nq;
    load_rows(a, b, q0, nq);
    if (row >= RT || r >= nq * a.G) return;
    float m = -INFINITY, l = 0.f, o[16] = {};
    for (int i = c - 1; i < grid; ++i) {
        if (i > c) {
            const int4 x = __ldcg(a.meta + 2 * i);
            if (x.x != here.x || !(x.w & kInside)) break;
        }
        const long slot = i == c - 1 ? slot0 : 2 * i;
        const float2 ml = __ldcg(a.ml + slot * kPfRows + row);
        const float4 *pp = reinterpret_cast<const float4 *>(a.part) + (slot * (D / 4) + col / 4) * kPfRows + row;
        float4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = __ldcg(pp + k * kPfRows);
        const float mn = fmaxf(m, ml.x), f = mn == -INFINITY ? 0.f : ex2(m - mn), g = mn == -INFINITY ? 0.f : ex2(ml.x - mn);
        m = mn;
        l = l * f + ml.y * g;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            o[4 * k] = o[4 * k] * f + v[k].x * g, o[4 * k + 1] = o[4 * k + 1] * f + v[k].y * g;
            o[4 * k + 2] = o[4 * k + 2] * f + v[k].z * g, o[4 * k + 3] = o[4 * k + 3] * f + v[k].w * g;
        }
    }
    const int tok = div_g(a, r);
    const float inv = l > 0.f ? 1.f / l : 0.f;
    T *op = static_cast<T *>(a.out) + (long)(q0 + tok) * a.os + (long)(here.z * a.G + r - tok * a.G) * D + col;
#pragma unroll
    for (int h = 0; h < 16; h += 8) {
        const float y[8] = {o[h] * inv, o[h + 2] * inv, o[h + 4] * inv, o[h + 6] * inv, o[h + 1] * inv, o[h + 3] * inv, o[h + 5] * inv, o[h + 7] * inv};
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4 *>(op + h) = make_float4(y[0], y[1], y[2], y[3]);
            *reinterpret_cast<float4 *>(op + h + 4) = make_float4(y[4], y[5], y[6], y[7]);
        } else {
            *reinterpret_cast<uint4 *>(op + h) = make_uint4(u32(__floats2half2_rn(y[0], y[1])), u32(__floats2half2_rn(y[2], y[3])),
                                                            u32(__floats2half2_rn(y[4], y[5])), u32(__floats2half2_rn(y[6], y[7])));
        }
    }
}

size_t prefill_work(int head_dim) {
    return (size_t)kPfCtas * 2 * (kPfRows * (head_dim + 2) * sizeof(float) + sizeof(int4));
}

bool prefill_fits(const AttnArgs &a, int dtype) {
    const long RT = dtype == X100Q_F32 ? 128 : 256, cover = std::min(0x7fffffffl, (long)a.tab.stride << a.pool.page_shift);
    const long items = (long)a.tab.n_seqs * a.pool.nkv * (((long)a.max_q * a.G + RT - 1) / RT);
    return items <= 0xfffff000l / (cover / kKeys + 1 + kLead);
}

template <typename T, int D>
static int launch_pf(DevCtx *c, AttnArgs &a, cudaStream_t s) {
    constexpr int RT = sizeof(T) == 4 ? 128 : 256;
    static bool attr[64];
    if (!attr[c->device]) {
        set_qkernel_attrs(prefill_kernel<T, D>, Pf<D>::SMEM);
        attr[c->device] = true;
    }
    const long items = (long)a.tab.n_seqs * a.pool.nkv * (((long)a.max_q * a.G + RT - 1) / RT);
    const long cover = std::min(0x7fffffffl, (long)a.tab.stride << a.pool.page_shift);
    const long most = std::min<long>(items, kPfCtas) * (cover / kKeys + 1);
    const int grid = (int)std::min<long>(std::min(kPfCtas, c->sm_count), most);
    a.ml = reinterpret_cast<float2 *>(a.part + (size_t)kPfCtas * 2 * kPfRows * D);
    a.meta = reinterpret_cast<int4 *>(a.ml + kPfCtas * 2 * kPfRows);
    a.unit_shift = 7, a.lead = 0;
    int st = launch_pdl(prefill_kernel<T, D>, dim3(grid), dim3(Roles<T>::THREADS), Pf<D>::SMEM, s, a);
    if (st || grid == 1) return st;
    return launch_pdl(prefill_merge_kernel<T, D>, dim3(grid - 1, D / 16), dim3(kPfRows), 0, s, a, grid);
}

int launch_prefill(DevCtx *c, AttnArgs &a, int dtype, int head_dim, cudaStream_t s) {
    if (dtype == X100Q_F32) return head_dim == 128 ? launch_pf<float, 128>(c, a, s) : launch_pf<float, 64>(c, a, s);
    return head_dim == 128 ? launch_pf<__half, 128>(c, a, s) : launch_pf<__half, 64>(c, a, s);
}

}  // namespace kv4
}  // namespace x100
