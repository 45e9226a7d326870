// kv4_attn.cu -- attention over the paged 4-bit KV cache (x100q_kv4_attn_dev).
//
// A sequence's query rows of one kv head are its tokens x the group's heads,
// row r = (token r / G, head r % G), in row tiles of 8 NR.  The work list is every
// (sequence, kv head, row tile) cut into units of 128 positions; CTA i of
// the grid takes the i-th run of equally many units, so ragged lengths and a single long
// sequence both fill the card, whatever the lengths (which only the device
// knows).  Row tiles that a run cuts leave partial (o, m, l) sums in `work`;
// merge_kernel joins them in run order, so results do not depend on timing.  Few items of
// few positions take clusters instead, which join without it.
// Long contexts are not bound by bytes: 255 instructions for 16 positions of 8 fp16 rows, most of them unpacking, of which an SM issues one
// in two cycles (each waits 1.2 cycles for a fixed latency and 1.0 for the mma pipe; DRAM 0.33, tensor pipe 0.24), and some 8 us that
// do not depend on the length (the list, the first round trips, the joins): 16 tokens over 16384 positions each, 85 MB, in 34.4 us; one
// fp32 token over 131071, 76 MB, in 32.4 us.  Short ones by a chain of round trips: one token over 4096 positions 8.1 us.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "kv4_attn.cuh"

namespace x100 {
namespace kv4 {

constexpr int kWarps = 8;
constexpr int kLead = 3;                // units (of 128 positions) that starting an item costs: 2 and 5 measured alike, 0 5 % slower

// Few items over a table that cannot hold long sequences go to clusters: of the most CTAs of which all items' fit the card at
// once, if that makes at most cluster_units units a CTA.  One fp32 token over 1024, 4096, 8192 positions 9.6, 10.8,
// 12.7 us by runs and 7.5, 8.1, 11.3 by clusters of 16, over 12288 (6 units each) 13.3 and 14.3; 16 fp16 tokens over 4096 each (8 units)
// 16.5 and 14.6; with several row groups 2 units a CTA took as long either way.
constexpr int cluster_units(int row_groups, bool fp32) { return row_groups > 1 ? 1 : fp32 ? 4 : 8; }

// A run's share of the list, found by one whole warp: its units, and the
// sequence holding the first with the units before it.
struct Share {
    uint32_t u0, u1, before, per;        // per: units of every run but the last
    int b;
};
__device__ __forceinline__ Share my_share(const AttnArgs &a, int R) {
    const int lane = threadIdx.x & 31;
    uint32_t n = 0, mine = 0, incl = 0;
    for (int b0 = 0; b0 < a.tab.n_seqs; b0 += 32) {
        mine = b0 + lane < a.tab.n_seqs ? load_seq(a, b0 + lane, R, blockIdx.x == 0).units : 0;
        n += mine;
    }
    incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
    }
    const uint32_t U = __reduce_add_sync(0xffffffffu, n), per = (U + gridDim.x - 1) / gridDim.x;
    Share s = {0, 0, 0, per, 0};
    if (per * blockIdx.x >= U) return s;     // the longest run is as long as with more, shorter ones; fewer items are cut
    s.u0 = per * blockIdx.x, s.u1 = min(U, s.u0 + per);
    uint32_t base = 0;
    for (int b0 = 0; b0 < a.tab.n_seqs; b0 += 32) {
        if (a.tab.n_seqs > 32) {         // else the one chunk's sums are still here
            mine = b0 + lane < a.tab.n_seqs ? load_seq(a, b0 + lane, R, false).units : 0;
            incl = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t up = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += up;
            }
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, base + incl > s.u0);
        if (hit) {
            const int l = __ffs(hit) - 1;
            s.before = base + __shfl_sync(0xffffffffu, incl - mine, l);
            s.b = b0 + l;
            return s;
        }
        base += __shfl_sync(0xffffffffu, incl, 31);
    }
    s.u0 = s.u1 = 0;                     // u0 < U: only if the lengths changed since they were added up
    return s;
}
// Row tile of an item index: from both ends in turn, so that a run of neighbouring
// items of a causal prompt holds early (short) and late (long) ones alike.
__device__ __forceinline__ int row_tile(int j, int n) { return j & 1 ? n - 1 - (j >> 1) : j >> 1; }

// ---- fragments --------------------------------------------------------------------
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ int cluster_ctas() {
    uint32_t n;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
    return (int)n;
}
// 16 bytes of another CTA's shared memory
__device__ __forceinline__ float4 ld_cluster(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
// D = A B
__device__ __forceinline__ void mma_init(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
template <int D, int NR>
struct Cfg {
    static constexpr int ST = 3;                              // ring stages per warp, two tiles each
    static constexpr int RING = kWarps * ST * 2 * Lay<D>::BYTES;
    static constexpr int RED = kWarps * 8 * D * 4;            // one 8-row group of every warp, over the idle ring
    static constexpr int QF = NR * (D / 16) * 32 * 16;        // Q fragments: (hi b0, b1, lo b0, b1) per lane
    static constexpr int ML = kWarps * 8 * NR * 2 * 4;
    static constexpr int SMEM = RING + QF + ML;
    static_assert(RED <= RING, "");
};

// S^T = K Q^T and O^T = V^T P^T: positions (then dims) are the M side of
// m16n8k16, the 8 query rows the N side, so that a group of 8 heads wastes no
// tensor rows.  K codes go into the product as code - 8 and the block's scale multiplies its sum in fp32; V codes become
// scale * (code - 8), an exact fp16.  (K as 1024 + code, an instruction less each, with sums that start from -1032 sum q: what cancels
// there is 129 times what is left, which one large element of q makes an error of the score, and it took longer, 33.6 against
// 32.4 us for 16 fp16 tokens over 16384 positions each, for the registers that those starts need.)
// Position k of a tile's MMA rows r: r / 2 + 4 (r % 2) of each half, so that
// transposing the score fragment gives P^T's B fragment for the positions t,
// t + 4, t + 8, t + 12 that a lane's V codes hold.  p goes in as hi + lo halves: rounded to fp16 it was as far off as the output's own
// rounding, 2.8e-4 instead of 2.1e-4 of the result together (16 x 16384 positions 32.5 -> 34.4 us).  HL (fp32 q): q as hi + lo halves
// too, and each tile's
// P V in sums of its own that fp32 additions take up: the tensor core truncates what it adds to, 1.2e-8 of it a step.
// Every warp walks its own positions with its own ring of bulk copies (two tiles a
// stage), so the loop has no CTA barrier.  One row group at heads of 128 takes all of the 128 registers that two CTAs an SM leave it
// (32 to 40 bytes spilled).
// CLUSTER: an item is a cluster's, its positions shared out among the CTAs and their sums joined through shared memory,
// with no second kernel.
template <typename T, int D, int NR, bool CLUSTER>
__global__ void __launch_bounds__(kWarps * 32, NR == 1 ? 2 : 1) attn_kernel(const AttnArgs a) {
    using L = Lay<D>;
    using C = Cfg<D, NR>;
    constexpr int NB = L::NB, R = 8 * NR, MT = D / 16, TT = NR == 1 ? 2 : 1;   // TT tiles worked on at once
    constexpr bool HL = sizeof(T) == 4;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t *ring = smem;
    float4 *red = reinterpret_cast<float4 *>(smem);
    uint4 *qf = reinterpret_cast<uint4 *>(smem + C::RING);
    float *sm = reinterpret_cast<float *>(smem + C::RING + C::QF), *sl = sm + kWarps * R;
    __shared__ uint64_t bars[kWarps * C::ST];
    __shared__ Share s_share;
    __shared__ int abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    if (threadIdx.x == 0) abort_flag = 0;
    if (lane == 0)
        for (int s = 0; s < C::ST; ++s) mbar_init(&bars[warp * C::ST + s], 1);
    fence_barrier_init();
    pdl_launch_dependents();
    pdl_wait();
    uint32_t u = 0, u1 = 1, before = 0;
    int b, rank = 0, cl = 1, kvh = 0, rt = 0;
    Seq sq;
    if constexpr (CLUSTER) {
        rank = cluster_ctarank(), cl = cluster_ctas();
        const int id = blockIdx.x / cl, h = id / a.nrt_max;
        rt = id - h * a.nrt_max, b = h / a.pool.nkv, kvh = h - b * a.pool.nkv;
        sq = load_seq(a, b, R, rank + rt + kvh == 0);
        __syncthreads();
    } else {
        if (warp == 0) {
            const Share s = my_share(a, R);
            if (lane == 0) s_share = s;
        }
        if (threadIdx.x >= 32 && threadIdx.x < 34) a.meta[blockIdx.x * 2 + threadIdx.x - 32] = make_int4(-1, 0, 0, 0);
        __syncthreads();
        u1 = s_share.u1;
        u = s_share.u0, before = s_share.before;
        b = s_share.b;
        if (u >= u1) return;
        sq = load_seq(a, b, R, false);
    }
    const Exponents expo;
    int nseg = 0;                              // segments done
    uint32_t st = 0, phase = 0;                // this warp's ring: next stage to read, and its parity
    uint64_t *bar = bars + warp * C::ST;
    uint8_t *wring = ring + warp * C::ST * 2 * L::BYTES;
    while (u < u1) {
        uint32_t iu = 0, item = 0;
        int c0, c1;
        if constexpr (CLUSTER) {
            const int per = rt < sq.nrt ? (sq.cu + cl - 1) / cl : 0;   // a tile that the sequence does not have: no positions, no rows
            c0 = min(rank * per, sq.cu), c1 = min(c0 + per, sq.cu);
            u = u1;
        } else {
            while (u - before >= sq.units) {
                before += sq.units;
                if (++b >= a.tab.n_seqs) return;
                sq = load_seq(a, b, R, false);
            }
            // `lead` units stand for starting an item (queries, an empty ring, joining the warps): a run that ends among them
            // has none of the item's positions
            iu = sq.cu + a.lead;
            const uint32_t off = u - before;
            item = off / iu;
            const uint32_t k0u = off - item * iu, k1u = min(iu, k0u + (u1 - u));
            c0 = max(0, (int)k0u - a.lead), c1 = max(0, (int)k1u - a.lead);
            u += k1u - k0u;
            if (c1 == c0) continue;
            kvh = sq.nrt == 1 ? (int)item : (int)(item / (uint32_t)sq.nrt), rt = row_tile((int)(item - (uint32_t)kvh * sq.nrt), sq.nrt);
        }
        const int rows = min(R, sq.nq * a.G - rt * R);                   // live rows of the tile
        const int first = sq.len - sq.nq;                               // position of token 0
        const int nk = max(0, min(sq.len, first + div_g(a, rt * R + rows - 1) + 1));   // positions the last row sees
        const int t0 = c0 << (a.unit_shift - 4), t1 = min(c1 << (a.unit_shift - 4), (nk + kTile - 1) / kTile);
        // stage j of this warp: `tps` tiles from t0 + tps (warp + 8 j); one each where two would leave warps idle
        const int tps = t1 - t0 > kWarps ? 2 : 1, ts0 = t0 + tps * warp;
        const int n_mine = t1 > ts0 ? (t1 - ts0 + tps * kWarps - 1) / (tps * kWarps) : 0;
        // ---- start the ring (lane 0).  128 or 256 positions between a warp's stages are whole pages, so the place in
        // the page stays; a page out of range is read as page 0 here and masked below ----
        const int ps = a.pool.page_shift, tp = ps - 4;       // log2 tiles per page
        const int *row = a.tab.page + (long)sq.row * a.tab.stride;
        const int *nxt = row + (ts0 >> tp);                   // table entry of the stage to be issued next
        const int pstep = (tps * kWarps) >> tp;
        const bool two = ps == 4 && tps == 2;                 // a stage's tiles lie on two pages
        const uint8_t *const src0 = a.pool.pages + (long)kvh * a.pool.page_bytes + (ts0 & ((1 << tp) - 1)) * L::BYTES;
        const long page_step = a.pool.page_bytes * a.pool.nkv;
        int left = n_mine, id0 = 0, id1 = 0;                  // stages to issue, and the next one's pages
        auto fetch = [&](int tile) {
            id0 = __ldg(nxt);
            if (two && tile + 1 < t1) id1 = __ldg(nxt + 1);
            nxt += pstep;
        };
        auto issue = [&](uint32_t s, int tile) {              // a stage whose first tile is `tile`
            uint8_t *dst = wring + s * 2 * L::BYTES;
            const uint32_t bytes = tps == 2 && tile + 1 < t1 ? 2 * L::BYTES : L::BYTES;
            mbar_arrive_expect_tx(&bar[s], bytes);
            const uint8_t *src = src0 + ((unsigned)id0 < (unsigned)a.pool.n_pages ? id0 : 0) * page_step;
            if (!two) bulk_load(dst, src, bytes, &bar[s]);
            else {
                bulk_load(dst, src, L::BYTES, &bar[s]);
                if (bytes > L::BYTES)
                    bulk_load(dst + L::BYTES, src0 + ((unsigned)id1 < (unsigned)a.pool.n_pages ? id1 : 0) * page_step, L::BYTES, &bar[s]);
            }
            if (--left > 0) fetch(tile + tps * kWarps);
        };
        if (lane == 0 && n_mine) {
            fetch(ts0);
            uint32_t s = st;
            for (int j = 0; j < min(C::ST, n_mine); ++j) {
                issue(s, ts0 + j * tps * kWarps);
                s = s + 1 == C::ST ? 0 : s + 1;
            }
        }
        // ---- pages out of range, and query fragments: rows are the N side ----
        bool hole = false;
        for (int i = (t0 >> tp) + threadIdx.x; i << tp < t1; i += kWarps * 32) hole = hole || (unsigned)__ldg(row + i) >= (unsigned)a.pool.n_pages;
        if (hole) atomicCAS(a.status, 0, X100_E_ARG);
        for (int e = threadIdx.x; e < NR * NB * 32; e += kWarps * 32) {
            const int nr = e / (NB * 32), blk = e / 32 % NB, ln = e % 32, r = rt * R + nr * 8 + ln / 4;
            float x[8] = {};
            if (nr * 8 + ln / 4 < rows) {
                const int tok = div_g(a, r);
                const T *p = static_cast<const T *>(a.q) + (long)(sq.q0 + tok) * a.qs +
                             (long)(kvh * a.G + r - tok * a.G) * D + blk * 32 + (ln & 3) * 8;
                if constexpr (HL) {
                    const float4 v0 = *reinterpret_cast<const float4 *>(p), v1 = *reinterpret_cast<const float4 *>(p + 4);
                    x[0] = v0.x, x[1] = v0.y, x[2] = v0.z, x[3] = v0.w, x[4] = v1.x, x[5] = v1.y, x[6] = v1.z, x[7] = v1.w;
                } else {
                    const uint4 v = *reinterpret_cast<const uint4 *>(p);
                    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 f = __half22float2(h2(w[i]));
                        x[2 * i] = f.x, x[2 * i + 1] = f.y;
                    }
                }
            }
            if constexpr (HL)
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] *= a.q_up;
            // half2 number j of a block's K words holds codes j and j + 4
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint4 f;
                split2(x[2 * j], x[2 * j + 4], f.x, f.z);
                split2(x[2 * j + 1], x[2 * j + 5], f.y, f.w);
                qf[(nr * (D / 16) + 2 * blk + j) * 32 + ln] = f;
            }
        }
        const bool any_hole = __syncthreads_or(hole);
        float m[NR][2], nm[NR][2], l[NR][2], o[NR][MT][4];   // m in units of log2: score * sl; nm = kUp - m, or 0 at the start
        int lim[NR][2];                         // positions that rows 2 t, 2 t + 1 of a group see
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                m[nr][i] = -INFINITY, nm[nr][i] = 0.f, l[nr][i] = 0.f;
                const int r = nr * 8 + 2 * t + i;
                lim[nr][i] = r < rows ? min(sq.len, first + div_g(a, rt * R + r) + 1) : 0;
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) o[nr][i][0] = o[nr][i][1] = o[nr][i][2] = o[nr][i][3] = 0.f;
        }
        const int minlim = max(0, first + div_g(a, rt * R) + 1);
        const int k0 = (g >> 1) + 4 * (g & 1);              // this lane's two positions of a tile: k0, k0 + 8

        // n <= TT tiles at position p0; EDGE: fewer than TT, masked positions, or missing pages.
        auto stage = [&](const uint8_t *sp, int p0, int n, auto edge_c) {
            constexpr bool EDGE = decltype(edge_c)::value;
            bool gone[TT] = {};
            if (EDGE && any_hole)
                for (int tt = 0; tt < n; ++tt) gone[tt] = (unsigned)__ldg(row + ((p0 + tt * kTile) >> ps)) >= (unsigned)a.pool.n_pages;
            // ---- scores ----
            float sc[TT][NR][4];
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) {
                if (EDGE && tt >= n) {
#pragma unroll
                    for (int nr = 0; nr < NR; ++nr) sc[tt][nr][0] = sc[tt][nr][1] = sc[tt][nr][2] = sc[tt][nr][3] = -INFINITY;
                    continue;
                }
                uint32_t kw[2][NB];
                __half kd[2][NB];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint8_t *kp = sp + tt * L::BYTES + L::k_word(k0 + 8 * i, 0, t), *dp = sp + tt * L::BYTES + L::k_scale(k0 + 8 * i, 0);
                    if constexpr (NB == 4) {
                        *reinterpret_cast<uint4 *>(kw[i]) = *reinterpret_cast<const uint4 *>(kp);
                        *reinterpret_cast<uint2 *>(kd[i]) = *reinterpret_cast<const uint2 *>(dp);
                    } else {
                        *reinterpret_cast<uint2 *>(kw[i]) = *reinterpret_cast<const uint2 *>(kp);
                        *reinterpret_cast<uint32_t *>(kd[i]) = *reinterpret_cast<const uint32_t *>(dp);
                    }
                }
#pragma unroll
                for (int blk = 0; blk < NB; ++blk) {
                    uint32_t f[2][4];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t w = kw[i][blk];
                        f[i][0] = u32(low_codes(w, expo)), f[i][1] = u32(high_codes(w, expo));
                        f[i][2] = u32(low_codes(w >> 8, expo)), f[i][3] = u32(high_codes(w >> 8, expo));
                    }
                    const float d0 = __half2float(kd[0][blk]), d1 = __half2float(kd[1][blk]);
#pragma unroll
                    for (int nr = 0; nr < NR; ++nr) {
                        float acc[4];
                        const uint4 *qp = qf + (nr * (D / 16) + 2 * blk) * 32 + lane;
                        uint4 q[2];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if constexpr (HL) q[h] = qp[h * 32];
                            else *reinterpret_cast<uint2 *>(q + h) = *reinterpret_cast<const uint2 *>(qp + h * 32);
                        }
                        if constexpr (HL) {             // lo first: what is added to is small then, and with it what is cut off
                            mma_init(acc, f[0][0], f[1][0], f[0][1], f[1][1], q[0].z, q[0].w);
                            mma(acc, f[0][2], f[1][2], f[0][3], f[1][3], q[1].z, q[1].w);
                            mma(acc, f[0][0], f[1][0], f[0][1], f[1][1], q[0].x, q[0].y);
                        } else {
                            mma_init(acc, f[0][0], f[1][0], f[0][1], f[1][1], q[0].x, q[0].y);
                        }
                        mma(acc, f[0][2], f[1][2], f[0][3], f[1][3], q[1].x, q[1].y);
                        float(&x)[4] = sc[tt][nr];
                        if (blk == 0) x[0] = acc[0] * d0, x[1] = acc[1] * d0, x[2] = acc[2] * d1, x[3] = acc[3] * d1;
                        else {
                            x[0] = fmaf(acc[0], d0, x[0]), x[1] = fmaf(acc[1], d0, x[1]);
                            x[2] = fmaf(acc[2], d1, x[2]), x[3] = fmaf(acc[3], d1, x[3]);
                        }
                    }
                }
            }
            // ---- mask, running max ----
            if (EDGE) {
#pragma unroll
                for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (gone[tt] || p0 + tt * kTile + k0 + 8 * (i >> 1) >= lim[nr][i & 1]) sc[tt][nr][i] = -INFINITY;
            }
            bool grow = false;
            float top[NR][2];
#pragma unroll
            for (int nr = 0; nr < NR; ++nr)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    top[nr][i] = fmaxf(sc[0][nr][i], sc[0][nr][i + 2]);
                    if constexpr (TT == 2) top[nr][i] = fmaxf(top[nr][i], fmaxf(sc[1][nr][i], sc[1][nr][i + 2]));
                    grow = grow || top[nr][i] * a.sl > m[nr][i] + kLag;
                }
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int nr = 0; nr < NR; ++nr)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float x = top[nr][i];
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                        const float mn = fmaxf(m[nr][i], x * a.sl);
                        const float f = mn == -INFINITY ? 1.f : ex2(m[nr][i] - mn);
                        m[nr][i] = mn;
                        nm[nr][i] = mn == -INFINITY ? 0.f : kUp - mn;
                        l[nr][i] *= f;
#pragma unroll
                        for (int k = 0; k < MT; ++k) o[nr][k][i] *= f, o[nr][k][i + 2] *= f;
                    }
            }
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) {
                if (EDGE && tt >= n) break;
                uint32_t ph[NR][2], pl[NR][2];
#pragma unroll
                for (int nr = 0; nr < NR; ++nr) {
                    float p[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) p[i] = ex2(fmaf(sc[tt][nr][i], a.sl, nm[nr][i & 1]));
                    l[nr][0] += p[0] + p[2];
                    l[nr][1] += p[1] + p[3];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        split2(p[2 * i], p[2 * i + 1], ph[nr][i], pl[nr][i]);
                        ph[nr][i] = transpose8(ph[nr][i]), pl[nr][i] = transpose8(pl[nr][i]);
                    }
                }
                // ---- O += P V: this lane's positions t + 4 m, dims g * D / 8 .. ----
                const uint8_t *vp = sp + tt * L::BYTES;
                __half vd[4];
                *reinterpret_cast<uint2 *>(vd) = *reinterpret_cast<const uint2 *>(vp + L::v_scale(t, g * (D / 8) / 32));
                if (EDGE) {
                    // codes past the sequence's end are any bytes, their scales maybe NaN: 0 * NaN must not reach the sums
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (gone[tt] || p0 + tt * kTile + t + 4 * i >= sq.len) vd[i] = __ushort_as_half(0);
                }
                constexpr int W = D / 64;             // words per V piece
                uint32_t vw[4][W];
                {
                    const uint4 x = *reinterpret_cast<const uint4 *>(vp + L::V0 + lane * 16);
                    if constexpr (W == 2) {
                        const uint4 y = *reinterpret_cast<const uint4 *>(vp + L::V0 + 512 + lane * 16);
                        vw[0][0] = x.x, vw[0][1] = x.y, vw[1][0] = x.z, vw[1][1] = x.w;
                        vw[2][0] = y.x, vw[2][1] = y.y, vw[3][0] = y.z, vw[3][1] = y.w;
                    } else {
                        vw[0][0] = x.x, vw[1][0] = x.y, vw[2][0] = x.z, vw[3][0] = x.w;
                    }
                }
                const __half2 da = __halves2half2(vd[0], vd[1]), db = __halves2half2(vd[2], vd[3]);
#pragma unroll
                for (int w = 0; w < W; ++w)
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        // 16-bit halves of two positions side by side: 4 dims x 2 positions
                        const uint32_t x = __byte_perm(vw[0][w], vw[1][w], hf ? 0x7632 : 0x5410);
                        const uint32_t y = __byte_perm(vw[2][w], vw[3][w], hf ? 0x7632 : 0x5410);
#pragma unroll
                        for (int e = 0; e < 2; ++e) {   // dims 8 w + 4 hf + 2 e, + 1
                            const uint32_t xe = x >> (8 * e), ye = y >> (8 * e);
                            const uint32_t a0 = u32(__hmul2(low_codes(xe, expo), da)), a1 = u32(__hmul2(high_codes(xe, expo), da));
                            const uint32_t a2 = u32(__hmul2(low_codes(ye, expo), db)), a3 = u32(__hmul2(high_codes(ye, expo), db));
#pragma unroll
                            for (int nr = 0; nr < NR; ++nr) {
                                float(&sum)[4] = o[nr][4 * w + 2 * hf + e];
                                if constexpr (HL) {
                                    float x4[4];
                                    mma_init(x4, a0, a1, a2, a3, pl[nr][0], pl[nr][1]);
                                    mma(x4, a0, a1, a2, a3, ph[nr][0], ph[nr][1]);
#pragma unroll
                                    for (int i = 0; i < 4; ++i) sum[i] += x4[i];
                                } else {
                                    mma(sum, a0, a1, a2, a3, pl[nr][0], pl[nr][1]);
                                    mma(sum, a0, a1, a2, a3, ph[nr][0], ph[nr][1]);
                                }
                            }
                        }
                    }
            }
        };
        for (int j = 0, tile = ts0; j < n_mine; ++j, tile += tps * kWarps) {
            const bool ok = mbar_wait(&bar[st], phase, &abort_flag, a.status);
            if (!__all_sync(0xffffffffu, ok)) {     // gave up: let the copies in flight land, then leave with the CTA
                abort_flag = 1;
                for (int i = j; i < min(j + C::ST, n_mine); ++i) {
                    mbar_wait_drain(&bar[st], phase, kWaitLimitNs);
                    st = st + 1 == C::ST ? (phase ^= 1, 0) : st + 1;
                }
                break;
            }
            const uint8_t *sp = wring + st * 2 * L::BYTES;
            const int p0 = tile * kTile, n = min(tps, t1 - tile);
            if constexpr (TT == 2) {
                if (n == 2 && p0 + 2 * kTile <= minlim && !any_hole) stage(sp, p0, 2, std::false_type{});
                else stage(sp, p0, n, std::true_type{});
            } else {
                for (int tt = 0; tt < n; ++tt)
                    if (p0 + (tt + 1) * kTile <= minlim && !any_hole) stage(sp + tt * L::BYTES, p0 + tt * kTile, 1, std::false_type{});
                    else stage(sp + tt * L::BYTES, p0 + tt * kTile, 1, std::true_type{});
            }
            __syncwarp();                          // the stage is read: refill it
            if (lane == 0 && left > 0) issue(st, tile + C::ST * tps * kWarps);
            st = st + 1 == C::ST ? (phase ^= 1, 0) : st + 1;
        }
        // ---- join the warps ----
#pragma unroll
        for (int nr = 0; nr < NR; ++nr)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int sh = 4; sh < 32; sh <<= 1) l[nr][i] += __shfl_xor_sync(0xffffffffu, l[nr][i], sh);
                if (g == 0) {
                    sm[warp * R + nr * 8 + 2 * t + i] = m[nr][i];
                    sl[warp * R + nr * 8 + 2 * t + i] = l[nr][i];
                }
            }
        __syncthreads();
        if (!CLUSTER && abort_flag) return;        // uniform: set before the barrier by a warp that gave up
        float4 *const xo = reinterpret_cast<float4 *>(smem + C::RED), *const xm = xo + NR * MT * 32;   // sums and (m, l) for the cluster
        const bool whole = c0 == 0 && c1 == sq.cu;
        const int slot = (int)blockIdx.x * 2 + (nseg ? 1 : 0);
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
            float M[2], f[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                M[i] = -INFINITY;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) M[i] = fmaxf(M[i], sm[w * R + nr * 8 + 2 * t + i]);
                f[i] = M[i] == -INFINITY ? 0.f : ex2(m[nr][i] - M[i]);
            }
#pragma unroll
            for (int k = 0; k < MT; ++k)
                red[(warp * MT + k) * 32 + lane] = make_float4(o[nr][k][0] * f[0], o[nr][k][1] * f[1], o[nr][k][2] * f[0],
                                                               o[nr][k][3] * f[1]);
            __syncthreads();
            if (threadIdx.x < MT * 32) {           // one fragment place each
                const int k = threadIdx.x / 32;
                float4 x = red[threadIdx.x];
#pragma unroll
                for (int w = 1; w < kWarps; ++w) {
                    const float4 y = red[w * MT * 32 + threadIdx.x];
                    x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
                }
                float Ls[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    Ls[i] = 0.f;
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) {
                        const int e = w * R + nr * 8 + 2 * t + i;
                        if (M[i] != -INFINITY) Ls[i] += sl[e] * ex2(sm[e] - M[i]);
                    }
                }
                if constexpr (CLUSTER) {
                    xo[nr * MT * 32 + threadIdx.x] = x;
                    if (k == 0 && g == 0) xm[(nr * 8 + 2 * t) / 2] = make_float4(M[0], Ls[0], M[1], Ls[1]);
                } else if (whole) {
                    const int dim = g * (D / 8) + 2 * k;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int rr = nr * 8 + 2 * t + i;
                        if (rr < rows) {
                            const int r = rt * R + rr;
                            const float inv = Ls[i] > 0.f ? 1.f / Ls[i] : 0.f;
                            const float y0 = (i ? x.y : x.x) * inv, y1 = (i ? x.w : x.z) * inv;
                            const int tok = div_g(a, r);
                            T *p = static_cast<T *>(a.out) + (long)(sq.q0 + tok) * a.os +
                                   (long)(kvh * a.G + r - tok * a.G) * D + dim;
                            if constexpr (HL) *reinterpret_cast<float2 *>(p) = make_float2(y0, y1);
                            else *reinterpret_cast<__half2 *>(p) = __floats2half2_rn(y0, y1);
                        }
                    }
                } else {
                    reinterpret_cast<float4 *>(a.part)[((long)slot * NR + nr) * MT * 32 + threadIdx.x] = x;
                    if (k == 0 && g == 0)
#pragma unroll
                        for (int i = 0; i < 2; ++i) a.ml[(long)slot * R + nr * 8 + 2 * t + i] = make_float2(M[i], Ls[i]);
                    if (nr == 0 && threadIdx.x == 0) {
                        const uint32_t ua = before + item * iu;
                        a.meta[slot] = make_int4((int)ua, b, kvh | (int)((ua + iu - 1) / s_share.per) << 16, rt | (c0 ? kInside : 0));
                    }
                }
            }
            if (nr == NR - 1) fence_proxy_async_smem();   // the next copies into the ring come after these accesses
            __syncthreads();
        }
        ++nseg;
        if constexpr (CLUSTER) {
            // ---- join the CTAs: `cl` neighbouring lanes have a place of the fragments, each the sums of one CTA ----
            cluster_sync_all();
            constexpr int E = NR * MT * 32;
            const int p = lane & (cl - 1), per = E / cl;
            for (int j = threadIdx.x; j < E; j += kWarps * 32) {
                const int e = rank * per + j / cl, nr = e / (MT * 32), k = e / 32 % MT, gg = e % 32 >> 2, tt = e & 3;
                const float4 y = ld_cluster(mapa_shared(xo + e, p)), ml = ld_cluster(mapa_shared(xm + nr * 4 + tt, p));
                const float v[2][3] = {{ml.y, y.x, y.z}, {ml.w, y.y, y.w}}, mx[2] = {ml.x, ml.z};   // l and two dims of rows 2 t, 2 t + 1
                float out[2][3];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float M = mx[i];
                    for (int o = 1; o < cl; o <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
                    const float f = M == -INFINITY ? 0.f : ex2(mx[i] - M);
#pragma unroll
                    for (int n = 0; n < 3; ++n) {
                        float z = v[i][n] * f;
                        for (int o = 1; o < cl; o <<= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
                        out[i][n] = z;
                    }
                }
                if (p < 2) {
                    const int rr = nr * 8 + 2 * tt + p;
                    if (rr < rows) {
                        const float l_ = p ? out[1][0] : out[0][0], inv = l_ > 0.f ? 1.f / l_ : 0.f;
                        const float y0 = (p ? out[1][1] : out[0][1]) * inv, y1 = (p ? out[1][2] : out[0][2]) * inv;
                        const int r = rt * R + rr, tok = div_g(a, r);
                        T *q = static_cast<T *>(a.out) + (long)(sq.q0 + tok) * a.os + (long)(kvh * a.G + r - tok * a.G) * D + gg * (D / 8) + 2 * k;
                        if constexpr (HL) *reinterpret_cast<float2 *>(q) = make_float2(y0, y1);
                        else *reinterpret_cast<__half2 *>(q) = __floats2half2_rn(y0, y1);
                    }
                }
            }
            cluster_sync_all();                    // the others have read this CTA's
        }
    }
}

// Joins at the first cut inside an item the partials of all runs that share the
// item, in a fixed order.  What each run left, and the last run of its item, is in its meta
// entries, so that the many cuts with nothing to do leave after one round of loads.  PW warps share the runs of
// one 16-dim fragment, 8 / PW fragments per CTA: with few items each is cut into
// many parts and the loads of one warp would follow each other; with many items the CTAs would.
template <typename T, int D, int NR, int PW>
__global__ void __launch_bounds__(kWarps * 32) merge_kernel(const AttnArgs a) {
    constexpr int R = 8 * NR, MT = D / 16, KC = kWarps / PW, NY = (MT + KC - 1) / KC;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int nr = blockIdx.y / NY, k = blockIdx.y % NY * KC + warp / PW, w = warp % PW;
    __shared__ float4 s_o[kWarps][32], s_ml[kWarps][4];
    pdl_launch_dependents();
    pdl_wait();
    const int c = blockIdx.x + 1;                            // the cut before run c
    const int4 here = __ldcg(a.meta + 2 * c), p0 = __ldcg(a.meta + 2 * c - 2), p1 = __ldcg(a.meta + 2 * c - 1);
    if (here.x == -1 || !(here.w & kInside)) return;         // run c starts with an item of its own
    int slot0 = 2 * c - 1;                                   // the item's first part, where it lies in run c - 1
    if (p1.x != here.x) {
        if (p0.x != here.x || (p0.w & kInside)) return;      // an earlier cut joins this item
        slot0 = 2 * c - 2;
    }
    const int b = here.y, kvh = here.z & 0xffff, rt = here.w & (kInside - 1), np = min(here.z >> 16, (int)gridDim.x) - c + 2;
    int q0, nq;
    load_rows(a, b, q0, nq);
    const int rows = min(R, nq * a.G - rt * R);
    // each warp its parts, four loads under way at a time, with a running max of its own
    float M[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (k < MT) {
        for (int p = w; p < np; p += 4 * PW) {
            float4 y[4];
            float4 ml[4];                                    // (m, l) of rows 2 t, 2 t + 1
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int pj = p + j * PW;
                const int slot = pj == 0 ? slot0 : 2 * (c - 1 + pj);
                const bool on = pj < np;
                y[j] = on ? __ldcg(reinterpret_cast<const float4 *>(a.part) + ((long)slot * NR + nr) * MT * 32 + k * 32 + lane) : make_float4(0.f, 0.f, 0.f, 0.f);
                ml[j] = on ? __ldcg(reinterpret_cast<const float4 *>(a.ml + (long)slot * R + nr * 8 + 2 * t)) : make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
            }
            const float mn[2] = {fmaxf(fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)), M[0]),
                                 fmaxf(fmaxf(fmaxf(ml[0].z, ml[1].z), fmaxf(ml[2].z, ml[3].z)), M[1])};
            const float b0 = mn[0] == -INFINITY ? 0.f : mn[0], b1 = mn[1] == -INFINITY ? 0.f : mn[1];
            const float f0 = ex2(M[0] - b0), f1 = ex2(M[1] - b1);
            M[0] = mn[0], M[1] = mn[1];
            o.x *= f0, o.y *= f1, o.z *= f0, o.w *= f1, l[0] *= f0, l[1] *= f1;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float h0 = ex2(ml[j].x - b0), h1 = ex2(ml[j].z - b1);
                l[0] = fmaf(ml[j].y, h0, l[0]), l[1] = fmaf(ml[j].w, h1, l[1]);
                o.x = fmaf(y[j].x, h0, o.x), o.y = fmaf(y[j].y, h1, o.y), o.z = fmaf(y[j].z, h0, o.z), o.w = fmaf(y[j].w, h1, o.w);
            }
        }
    }
    if constexpr (PW > 1) {
        s_o[warp][lane] = o;
        if (g == 0) s_ml[warp][t] = make_float4(M[0], l[0], M[1], l[1]);
        __syncthreads();
        if (w) return;
        float4 ml[PW];
        float b0 = -INFINITY, b1 = -INFINITY;
#pragma unroll
        for (int i = 0; i < PW; ++i) {
            ml[i] = s_ml[warp + i][t];
            b0 = fmaxf(b0, ml[i].x), b1 = fmaxf(b1, ml[i].z);
        }
        b0 = b0 == -INFINITY ? 0.f : b0, b1 = b1 == -INFINITY ? 0.f : b1;
        o = make_float4(0.f, 0.f, 0.f, 0.f);
        l[0] = l[1] = 0.f;
#pragma unroll
        for (int i = 0; i < PW; ++i) {
            const float4 y = s_o[warp + i][lane];
            const float h0 = ex2(ml[i].x - b0), h1 = ex2(ml[i].z - b1);
            l[0] = fmaf(ml[i].y, h0, l[0]), l[1] = fmaf(ml[i].w, h1, l[1]);
            o.x = fmaf(y.x, h0, o.x), o.y = fmaf(y.y, h1, o.y), o.z = fmaf(y.z, h0, o.z), o.w = fmaf(y.w, h1, o.w);
        }
    }
    if (k >= MT || nr * 8 >= rows) return;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int rr = nr * 8 + 2 * t + i;
        if (rr >= rows) continue;
        const int r = rt * R + rr, tok = div_g(a, r);
        const float inv = l[i] > 0.f ? 1.f / l[i] : 0.f;
        const float y0 = (i ? o.y : o.x) * inv, y1 = (i ? o.w : o.z) * inv;
        T *p = static_cast<T *>(a.out) + (long)(q0 + tok) * a.os + (long)(kvh * a.G + r - tok * a.G) * D + g * (D / 8) + 2 * k;
        if constexpr (sizeof(T) == 4) *reinterpret_cast<float2 *>(p) = make_float2(y0, y1);
        else *reinterpret_cast<__half2 *>(p) = __floats2half2_rn(y0, y1);
    }
}

static int launch_cluster(void (*kernel)(const AttnArgs), int grid, int cl, int smem, cudaStream_t s, const AttnArgs &a) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid), cfg.blockDim = dim3(kWarps * 32), cfg.dynamicSmemBytes = smem, cfg.stream = s;
    cudaLaunchAttribute at[2] = {};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization, at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension, at[1].val.clusterDim = {(unsigned)cl, 1, 1};
    cfg.attrs = at, cfg.numAttrs = 2;
    return check_cuda(cudaLaunchKernelEx(&cfg, kernel, a), X100_E_LAUNCH);
}

template <typename T, int D, int NR>
static int launch(DevCtx *c, AttnArgs &a, cudaStream_t s) {
    constexpr int R = 8 * NR;
    static bool attr[64];
    static int fit[64][3];                 // clusters of 16, 8, 4 CTAs on the card at once
    if (!attr[c->device]) {
        set_qkernel_attrs(attn_kernel<T, D, NR, false>, Cfg<D, NR>::SMEM);
        set_qkernel_attrs(attn_kernel<T, D, NR, true>, Cfg<D, NR>::SMEM);
        cudaFuncSetAttribute(attn_kernel<T, D, NR, true>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        for (int i = 0; i < 3; ++i) {
            cudaLaunchAttribute at = {};
            at.id = cudaLaunchAttributeClusterDimension, at.val.clusterDim = {16u >> i, 1, 1};
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(16 >> i), cfg.blockDim = dim3(kWarps * 32), cfg.dynamicSmemBytes = Cfg<D, NR>::SMEM, cfg.attrs = &at, cfg.numAttrs = 1;
            if (cudaOccupancyMaxActiveClusters(&fit[c->device][i], attn_kernel<T, D, NR, true>, &cfg) != cudaSuccess) {
                cudaGetLastError();
                fit[c->device][i] = 0;
            }
        }
        attr[c->device] = true;
    }
    const long nrt = ((long)a.max_q * a.G + R - 1) / R, cover = std::min(0x7fffffffl, (long)a.tab.stride << a.pool.page_shift);
    const long items = (long)a.tab.n_seqs * a.pool.nkv * nrt;
    a.unit_shift = 7;
    int cl = 16;
    for (const int *f = fit[c->device]; cl > 2 && (items > *f || (cl > 4 && cover <= 64 * cl)); ++f) cl >>= 1;
    if (cl > 2 && cover > 128 && cover <= 128l * cluster_units(NR, sizeof(T) == 4) * cl) {   // one unit needs no joining either way
        a.lead = 0;
        a.nrt_max = (int)nrt;
        return launch_cluster(attn_kernel<T, D, NR, true>, (int)items * cl, cl, Cfg<D, NR>::SMEM, s, a);
    }
    a.lead = kLead;
    while (items * ((cover >> a.unit_shift) + 1 + a.lead) > 0x7fffffffl) ++a.unit_shift;   // items <= 2^24: ends by 25
    const long most = std::min<long>(items, kMaxCtas) * ((cover >> a.unit_shift) + 1 + a.lead);
    const int grid = (int)std::min<long>(std::min(kMaxCtas, c->sm_count * (NR == 1 ? 2 : 1)), most);
    a.ml = reinterpret_cast<float2 *>(a.part + (size_t)kMaxCtas * 2 * R * D);
    a.meta = reinterpret_cast<int4 *>(a.ml + kMaxCtas * 2 * R);
    int st = launch_pdl(attn_kernel<T, D, NR, false>, dim3(grid), dim3(kWarps * 32), Cfg<D, NR>::SMEM, s, a);
    if (st || grid == 1 || cover <= 1l << a.unit_shift) return st;   // items of one unit are never cut
    if (items * 8 >= grid) return launch_pdl(merge_kernel<T, D, NR, 1>, dim3(grid - 1, NR), dim3(kWarps * 32), 0, s, a);
    return launch_pdl(merge_kernel<T, D, NR, 8>, dim3(grid - 1, NR * (D / 16)), dim3(kWarps * 32), 0, s, a);
}

template <typename T, int D>
static int launch_rows(DevCtx *c, AttnArgs &a, cudaStream_t s) {
    // row tiles of up to 4 groups of 8 rows, as few as there can be and as even: 35 rows go as 24 + 11 (3 groups each), not 32 + 3
    // (7 x 5 tokens of 14 heads over 2 kv heads of 64, 8192 positions: 17.8 us against 20.4; 3 fp32 tokens over 4096, 24 rows, 15.2 against 18.1)
    const int groups = (int)(((long)a.max_q * a.G + 7) / 8), nrt = (groups + 3) / 4, nr = (groups + nrt - 1) / nrt;
    if (nr == 1) return launch<T, D, 1>(c, a, s);
    if (nr == 2) return launch<T, D, 2>(c, a, s);
    if (nr == 3) return launch<T, D, 3>(c, a, s);
    return launch<T, D, 4>(c, a, s);
}

int launch_attention(DevCtx *c, AttnArgs &p, int dtype, int head_dim, cudaStream_t s) {
    if ((long)p.max_q * p.G >= kPrefillRows) return launch_prefill(c, p, dtype, head_dim, s);
    if (dtype == X100Q_F32) return head_dim == 128 ? launch_rows<float, 128>(c, p, s) : launch_rows<float, 64>(c, p, s);
    return head_dim == 128 ? launch_rows<__half, 128>(c, p, s) : launch_rows<__half, 64>(c, p, s);
}

void attn_shape(AttnArgs &p, int n_heads, float scale, int dtype, int head_dim) {
    p.nh = n_heads, p.G = n_heads / p.pool.nkv;
    p.g_mul = (uint32_t)(((1ull << 32) + p.G - 1) / p.G);
    // fp32 q: by the power of two next to scale * sqrt(head_dim), 1 for the usual scale.  (A power of two for each row from its largest
    // element, whose inverse every score then takes from a register, cost prompts 10 % and single tokens 2 %.)
    const int k = dtype == X100Q_F32 ? (int)std::lrint(std::log2((double)scale) + 0.5 * std::log2((double)head_dim)) : 0;
    p.q_up = std::ldexp(1.f, std::max(-100, std::min(k, 100)));
    p.sl = scale / p.q_up * 1.4426950408889634f;
}

}  // namespace kv4
}  // namespace x100

using namespace x100;
using namespace x100::kv4;

static int refuse(int code) {
    set_error(code);
    return code;
}

extern "C" {

size_t x100q_kv4_attn_work(const x100q_kv4 *kv, int n_tokens, int n_heads, int n_seqs) {
    if (!shape_ok(kv) || n_tokens < 0 || n_seqs < 1 || n_heads < 1 || n_heads % kv->n_kv_heads) return 0;
    const size_t few = (size_t)kMaxCtas * 2 * (32 * (kv->head_dim + 2) * sizeof(float) + sizeof(int4));
    // no sequence can have more rows than the call
    return (long)n_tokens * (n_heads / kv->n_kv_heads) < kPrefillRows ? few : std::max(few, prefill_work(kv->head_dim));
}

int x100q_kv4_attn_dev(const x100q_kv4 *kv, const x100q_kv4_attn_args *a, void *stream) {
    set_error(X100_OK);
    if (!shape_ok(kv) || !a || a->n_tokens < 0) return refuse(X100_E_ARG);
    if (a->n_tokens == 0) return X100_OK;
    if (a->dtype != X100Q_F32 && a->dtype != X100Q_F16) return refuse(X100_E_UNSUPPORTED);
    const int es = a->dtype == X100Q_F32 ? 4 : 2;
    if (!kv->pages || !aligned16(kv->pages) || a->n_heads < 1 || a->n_heads > 4096 || a->n_heads % kv->n_kv_heads || !a->q ||
        !a->out || !aligned16(a->q) || !aligned16(a->out) || !a->kv_len || !a->page_table || a->table_stride < 1 ||
        a->n_seqs < 1 || a->max_q < 1 || (!a->q_start && a->n_tokens != a->n_seqs) ||
        !pitch_ok(a->q_stride, a->n_heads * kv->head_dim, es) || !pitch_ok(a->out_stride, a->n_heads * kv->head_dim, es) ||
        !in_place_ok(a->q, a->q_stride, a->out, a->out_stride, a->n_tokens) ||
        !(a->scale > 0.f) || !(a->scale < INFINITY) || !a->work || !aligned16(a->work))
        return refuse(X100_E_ARG);
    if (a->work_bytes < x100q_kv4_attn_work(kv, a->n_tokens, a->n_heads, a->n_seqs)) return refuse(X100_E_TOO_LARGE);
    if (a->n_seqs > 65536) return refuse(X100_E_TOO_LARGE);
    AttnArgs p = {};
    p.pool = make_pool(kv);
    p.tab = {a->page_table, a->table_stride, a->n_seqs};
    p.q = a->q, p.out = a->out, p.qs = a->q_stride, p.os = a->out_stride;
    p.q_start = a->q_start, p.kv_len = a->kv_len;
    p.n_tokens = a->n_tokens, p.max_q = a->q_start ? std::min(a->max_q, a->n_tokens) : 1;
    attn_shape(p, a->n_heads, a->scale, a->dtype, kv->head_dim);
    const long rows = (long)p.max_q * p.G, items = (long)a->n_seqs * kv->n_kv_heads * ((rows + 7) / 8);
    if (items > (1l << 24) || rows > (1l << 20) || (rows >= kPrefillRows && !prefill_fits(p, a->dtype))) return refuse(X100_E_TOO_LARGE);
    DevCtx *c = ctx();
    if (!c) return get_error();
    p.part = static_cast<float *>(a->work);
    p.status = c->d_status;
    return launch_attention(c, p, a->dtype, kv->head_dim, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
