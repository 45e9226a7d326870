// kv4_attn.cu -- attention over the paged 4-bit KV cache (x100q_kv4_attn_dev).
//
// A sequence's query rows of one kv head are its tokens x the group's heads,
// row r = (token r / G, head r % G), in row tiles of 8 NR.  The work list is every
// (sequence, kv head, row tile) cut into units of 128 positions; CTA i of
// the grid takes the i-th equal run of units, so ragged lengths and a single long
// sequence both fill the card, whatever the lengths (which only the device
// knows).  Row tiles that a run cuts leave partial (o, m, l) sums in `work`;
// merge_kernel joins them in run order, so results do not depend on timing.
#include <algorithm>
#include <cmath>

#include "kv4.cuh"
#include "ptx.cuh"
#include "qformats.cuh"
#include "qgemv.h"

namespace x100 {
namespace kv4 {

using q::pdl_launch_dependents;
using q::pdl_wait;

constexpr int kWarps = 8;
constexpr int kUnit = kWarps * kTile;   // positions per unit: a tile for each warp
constexpr int kMaxCtas = 320;           // bound of the grid, which sizes the workspace

struct AttnArgs {
    Pool pool;
    Table tab;
    const void *q;
    void *out;
    long qs, os;
    const int *q_start, *kv_len;
    int n_tokens, max_q, nh, G;
    float sl;                            // scale * log2(e)
    float *part;                         // [grid][2][8 NR * D] fragment-ordered o, then [grid][2][8 NR][2] m, l
    float *ml;
    int *status;
};

// ---- the work list -------------------------------------------------------------
// Sequence b: first row of q, tokens, positions; `cu` units of every (kv head, row
// tile) item, at least one so that rows without positions are written.
struct Seq {
    int q0, nq, len, nrt, cu;
    __device__ long units(int nkv) const { return (long)nkv * nrt * cu; }
};
__device__ __forceinline__ Seq load_seq(const AttnArgs &a, int b, int R, bool report) {
    Seq s;
    s.q0 = a.q_start ? a.q_start[b] : b;
    s.nq = a.q_start ? a.q_start[b + 1] - s.q0 : 1;
    s.len = a.kv_len[b];
    const int cover = a.tab.stride > (0x7fffffff >> a.pool.page_shift) ? 0x7fffffff : a.tab.stride << a.pool.page_shift;
    const bool bad_q = s.q0 < 0 || s.nq < 0 || s.nq > a.max_q || s.q0 > a.n_tokens - s.nq;
    if (bad_q) s.nq = 0;
    if (bad_q || s.len < 0 || s.len > cover) {
        if (report) atomicCAS(a.status, 0, X100_E_ARG);
        s.len = s.len < 0 ? 0 : min(s.len, cover);
    }
    s.nrt = (s.nq * a.G + R - 1) / R;
    s.cu = max(1, (s.len + kUnit - 1) / kUnit);
    return s;
}
// Units of all sequences, and the sequence holding unit u with the units before
// it.  Called by one whole warp.
__device__ __forceinline__ long total_units(const AttnArgs &a, int R, bool report) {
    long n = 0;
    for (int b0 = 0; b0 < a.tab.n_seqs; b0 += 32) {
        const int b = b0 + (threadIdx.x & 31);
        if (b < a.tab.n_seqs) n += load_seq(a, b, R, report).units(a.pool.nkv);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    return n;
}
__device__ __forceinline__ int find_unit(const AttnArgs &a, int R, long u, long &before) {
    long base = 0;
    for (int b0 = 0; b0 < a.tab.n_seqs; b0 += 32) {
        const int lane = threadIdx.x & 31, b = b0 + lane;
        const long mine = b < a.tab.n_seqs ? load_seq(a, b, R, false).units(a.pool.nkv) : 0;
        long incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, base + incl > u);
        if (hit) {
            const int l = __ffs(hit) - 1;
            before = base + __shfl_sync(0xffffffffu, incl - mine, l);
            return b0 + l;
        }
        base += __shfl_sync(0xffffffffu, incl, 31);
    }
    before = base;
    return a.tab.n_seqs;
}
// Row tile of an item index: from both ends in turn, so that a run of neighbouring
// items of a causal prompt holds early (short) and late (long) ones alike.
__device__ __forceinline__ int row_tile(int j, int n) { return j & 1 ? n - 1 - (j >> 1) : j >> 1; }
__device__ __forceinline__ int item_of_row_tile(int rt, int n) { return 2 * rt < n ? 2 * rt : 2 * (n - 1 - rt) + 1; }

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
__device__ __forceinline__ uint32_t u32(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ __half2 h2(uint32_t u) { return *reinterpret_cast<__half2 *>(&u); }
// Bits 0-3 (or 4-7) of both halves of w as fp16 code - 8, exactly: the bits under
// the exponent of 1024 read as 1024 + code (or 1024 + 16 code).
__device__ __forceinline__ __half2 low_codes(uint32_t w) {
    return __hsub2(h2((w & 0x000f000fu) | 0x64006400u), __float2half2_rn(1032.f));
}
__device__ __forceinline__ __half2 high_codes(uint32_t w) {
    return __hfma2(h2((w & 0x00f000f0u) | 0x64006400u), __float2half2_rn(0.0625f), __float2half2_rn(-72.f));
}
__device__ __forceinline__ float ex2(float x) { return exp2f(x); }
// x = hi + lo to 22 bits
__device__ __forceinline__ void split2(float x, float y, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    hi = u32(h);
    lo = u32(__floats2half2_rn(x - f.x, y - f.y));
}

template <int D, int NR>
struct Cfg {
    static constexpr int ST = 4;                              // ring stages per warp
    static constexpr int RING = kWarps * ST * Lay<D>::BYTES;
    static constexpr int QF = NR * (D / 16) * 32 * 16;        // Q fragments: (hi b0, b1, lo b0, b1) per lane
    static constexpr int RED = kWarps * 8 * D * 4;            // one 8-row group of every warp
    static constexpr int ML = kWarps * 8 * NR * 2 * 4;
    static constexpr int SMEM = RING + QF + RED + ML;
};

// S^T = K Q^T and O^T = V^T P^T: positions (then dims) are the M side of
// m16n8k16, the 8 query rows the N side, so that a group of 8 heads wastes no
// tensor rows.  The codes become fp16 in registers (K: code - 8, the block's scale
// applied to the fp32 score sums; V: scale * (code - 8), an exact fp16).
// Position k of a tile's MMA rows r: r / 2 + 4 (r % 2) of each half, so that
// transposing the score fragment gives P^T's B fragment for the positions t,
// t + 4, t + 8, t + 12 that a lane's V codes hold.  HL: q as hi + lo halves.
template <typename T, int D, int NR>
__global__ void __launch_bounds__(kWarps * 32, NR == 1 ? 2 : 1) attn_kernel(const AttnArgs a) {
    using L = Lay<D>;
    using C = Cfg<D, NR>;
    constexpr int NB = L::NB, R = 8 * NR, MT = D / 16;
    constexpr bool HL = sizeof(T) == 4;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t *ring = smem;
    uint4 *qf = reinterpret_cast<uint4 *>(smem + C::RING);
    float4 *red = reinterpret_cast<float4 *>(smem + C::RING + C::QF);
    float *sm = reinterpret_cast<float *>(smem + C::RING + C::QF + C::RED), *sl = sm + kWarps * R;
    __shared__ uint64_t bars[kWarps * C::ST];
    __shared__ long s_u0, s_u1, s_before;
    __shared__ int s_b, abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    if (threadIdx.x == 0) abort_flag = 0;
    if (lane == 0)
        for (int s = 0; s < C::ST; ++s) mbar_init(&bars[warp * C::ST + s], 1);
    fence_barrier_init();
    pdl_launch_dependents();
    pdl_wait();
    if (warp == 0) {
        const long U = total_units(a, R, blockIdx.x == 0);
        const long nc = min((long)gridDim.x, U);   // runs: none is empty
        const long u0 = blockIdx.x < nc ? U * blockIdx.x / nc : 0, u1 = blockIdx.x < nc ? U * (blockIdx.x + 1) / nc : 0;
        long before = 0;
        const int b = u0 < u1 ? find_unit(a, R, u0, before) : a.tab.n_seqs;
        if (lane == 0) s_u0 = u0, s_u1 = u1, s_before = before, s_b = b;
    }
    __syncthreads();
    const long u1 = s_u1;
    long u = s_u0, before = s_before;
    int b = s_b;
    if (u >= u1) return;
    Seq sq = load_seq(a, b, R, false);
    int nseg = 0;                              // segments done
    uint32_t cnt = 0;                          // tiles this warp has consumed
    uint64_t *bar = bars + warp * C::ST;
    uint8_t *wring = ring + warp * C::ST * L::BYTES;
    while (u < u1) {
        while (u - before >= sq.units(a.pool.nkv)) {
            before += sq.units(a.pool.nkv);
            sq = load_seq(a, ++b, R, false);
        }
        const long off = u - before;
        const long item = off / sq.cu;
        const int c0 = (int)(off % sq.cu), c1 = (int)min((long)sq.cu, c0 + (u1 - u));
        const int kvh = (int)(item / sq.nrt), rt = row_tile((int)(item % sq.nrt), sq.nrt);
        const int rows = min(R, sq.nq * a.G - rt * R);                   // live rows of the tile
        const int first = sq.len - sq.nq;                               // position of token 0
        const int nk = max(0, min(sq.len, first + (rt * R + rows - 1) / a.G + 1));   // positions the last row sees
        const int t0 = c0 * kWarps, t1 = min(c1 * kWarps, (nk + kTile - 1) / kTile);
        const int n_mine = t1 > t0 + warp ? (t1 - t0 - warp + kWarps - 1) / kWarps : 0;
        // ---- start the ring: tile j of this warp is t0 + warp + 8 j ----
        const uint32_t base = cnt;
        uint32_t bad = 0;                       // bit s: stage s holds a position without a page
        auto issue = [&](int j) {
            const uint8_t *src = tile_of(a.pool, a.tab, b, (t0 + warp + kWarps * j) * kTile, kvh);
            const int s = (base + j) % C::ST;
            bad = (bad & ~(1u << s)) | (src ? 0u : 1u << s);
            if (!src) src = a.pool.pages;       // some page: it is masked
            if (lane == 0) {
                if (bad >> s & 1) atomicCAS(a.status, 0, X100_E_ARG);
                mbar_arrive_expect_tx(&bar[s], L::BYTES);
                bulk_load(wring + s * L::BYTES, src, L::BYTES, &bar[s]);
            }
        };
        for (int j = 0; j < min(C::ST, n_mine); ++j) issue(j);
        // ---- query fragments: rows are the N side ----
        __syncthreads();                        // the previous segment's readers of qf are done
        for (int e = threadIdx.x; e < NR * NB * 32; e += kWarps * 32) {
            const int nr = e / (NB * 32), blk = e / 32 % NB, ln = e % 32, r = rt * R + nr * 8 + ln / 4;
            float x[8] = {};
            if (nr * 8 + ln / 4 < rows) {
                const T *p = static_cast<const T *>(a.q) + (long)(sq.q0 + r / a.G) * a.qs +
                             (long)(kvh * a.G + r % a.G) * D + blk * 32 + (ln & 3) * 8;
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
            // half2 number j of a block's K words holds codes j and j + 4
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint4 f;
                split2(x[2 * j], x[2 * j + 4], f.x, f.z);
                split2(x[2 * j + 1], x[2 * j + 5], f.y, f.w);
                qf[(nr * (D / 16) + 2 * blk + j) * 32 + ln] = f;
            }
        }
        __syncthreads();
        float m[NR][2], l[NR][2], o[NR][MT][4];
        int lim[NR][2], minlim = 0x7fffffff;    // positions that rows 2 t, 2 t + 1 of a group see
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                m[nr][i] = -INFINITY, l[nr][i] = 0.f;
                const int r = nr * 8 + 2 * t + i;
                lim[nr][i] = r < rows ? min(sq.len, first + (rt * R + r) / a.G + 1) : 0;
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) o[nr][i][0] = o[nr][i][1] = o[nr][i][2] = o[nr][i][3] = 0.f;
        }
        minlim = max(0, first + rt * R / a.G + 1);
        for (int j = 0; j < n_mine; ++j) {
            const int s = cnt % C::ST, p0 = (t0 + warp + kWarps * j) * kTile;
            const bool ok = mbar_wait(&bar[s], cnt / C::ST & 1, &abort_flag, a.status);
            if (!__all_sync(0xffffffffu, ok)) {     // gave up: let the copies in flight land, then leave with the CTA
                abort_flag = 1;
                for (int i = j; i < min(j + C::ST, n_mine); ++i)
                    mbar_wait_drain(&bar[(base + i) % C::ST], (base + i) / C::ST & 1, kWaitLimitNs);
                break;
            }
            const uint8_t *sp = wring + s * L::BYTES;
            const int k0 = (g >> 1) + 4 * (g & 1);          // this lane's two positions of the tile: k0, k0 + 8
            // ---- scores ----
            float sc[NR][4];
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) sc[nr][0] = sc[nr][1] = sc[nr][2] = sc[nr][3] = 0.f;
            uint32_t kw[2][NB];
            __half kd[2][NB];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint8_t *kp = sp + L::k_word(k0 + 8 * i, 0, t), *dp = sp + L::k_scale(k0 + 8 * i, 0);
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
                    const uint32_t w = kw[i][blk], w8 = w >> 8;
                    f[i][0] = u32(low_codes(w)), f[i][1] = u32(high_codes(w));
                    f[i][2] = u32(low_codes(w8)), f[i][3] = u32(high_codes(w8));
                }
                const float d0 = __half2float(kd[0][blk]), d1 = __half2float(kd[1][blk]);
#pragma unroll
                for (int nr = 0; nr < NR; ++nr) {
                    float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint4 q = qf[(nr * (D / 16) + 2 * blk + h) * 32 + lane];
                        mma(acc, f[0][2 * h], f[1][2 * h], f[0][2 * h + 1], f[1][2 * h + 1], q.x, q.y);
                        if (HL) mma(acc, f[0][2 * h], f[1][2 * h], f[0][2 * h + 1], f[1][2 * h + 1], q.z, q.w);
                    }
                    sc[nr][0] = fmaf(acc[0], d0, sc[nr][0]);
                    sc[nr][1] = fmaf(acc[1], d0, sc[nr][1]);
                    sc[nr][2] = fmaf(acc[2], d1, sc[nr][2]);
                    sc[nr][3] = fmaf(acc[3], d1, sc[nr][3]);
                }
            }
            // ---- mask, running max ----
            const bool missing = bad >> s & 1;
            const bool edge = missing || p0 + kTile > minlim;
            bool grow = false;
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) {
                if (edge) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (missing || p0 + k0 + 8 * (i >> 1) >= lim[nr][i & 1]) sc[nr][i] = -INFINITY;
                }
                // the running max follows only when a score passes it by 2^8: until then
                // exp2 of the difference stays within fp16 and the sums need no rescaling
#pragma unroll
                for (int i = 0; i < 4; ++i) grow = grow || (sc[nr][i] - m[nr][i & 1]) * a.sl > 8.f;
            }
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int nr = 0; nr < NR; ++nr)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float x = fmaxf(sc[nr][i], sc[nr][i + 2]);
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                        const float mn = fmaxf(m[nr][i], x);
                        const float f = mn == -INFINITY ? 1.f : ex2((m[nr][i] - mn) * a.sl);
                        m[nr][i] = mn;
                        l[nr][i] *= f;
#pragma unroll
                        for (int k = 0; k < MT; ++k) o[nr][k][i] *= f, o[nr][k][i + 2] *= f;
                    }
            }
            uint32_t ph[NR][2], pl[NR][2];
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) {
                float p[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float mm = m[nr][i & 1];
                    p[i] = ex2((sc[nr][i] - (mm == -INFINITY ? 0.f : mm)) * a.sl);
                }
                l[nr][0] += p[0] + p[2];
                l[nr][1] += p[1] + p[3];
                split2(p[0], p[1], ph[nr][0], pl[nr][0]);
                split2(p[2], p[3], ph[nr][1], pl[nr][1]);
#pragma unroll
                for (int i = 0; i < 2; ++i) ph[nr][i] = transpose8(ph[nr][i]), pl[nr][i] = transpose8(pl[nr][i]);
            }
            // ---- O += P V: this lane's positions t + 4 m, dims g * D / 8 .. ----
            __half vd[4];
            *reinterpret_cast<uint2 *>(vd) = *reinterpret_cast<const uint2 *>(sp + L::v_scale(t, g * (D / 8) / 32));
            if (p0 + kTile > sq.len || missing) {
                // codes past the sequence's end are any bytes, their scales maybe NaN: 0 * NaN must not reach the sums
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (missing || p0 + t + 4 * i >= sq.len) vd[i] = __ushort_as_half(0);
            }
            constexpr int W = D / 64;             // words per V piece
            uint32_t vw[4][W];
            {
                const uint4 x = *reinterpret_cast<const uint4 *>(sp + L::V0 + lane * 16);
                if constexpr (W == 2) {
                    const uint4 y = *reinterpret_cast<const uint4 *>(sp + L::V0 + 512 + lane * 16);
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
                        const uint32_t a0 = u32(__hmul2(low_codes(xe), da)), a1 = u32(__hmul2(high_codes(xe), da));
                        const uint32_t a2 = u32(__hmul2(low_codes(ye), db)), a3 = u32(__hmul2(high_codes(ye), db));
#pragma unroll
                        for (int nr = 0; nr < NR; ++nr) {
                            mma(o[nr][4 * w + 2 * hf + e], a0, a1, a2, a3, ph[nr][0], ph[nr][1]);
                            mma(o[nr][4 * w + 2 * hf + e], a0, a1, a2, a3, pl[nr][0], pl[nr][1]);
                        }
                    }
                }
            __syncwarp();                          // the stage is read: refill it
            if (j + C::ST < n_mine) issue(j + C::ST);
            ++cnt;
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
        if (abort_flag) return;                    // uniform: set before the barrier by a warp that gave up
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
                f[i] = M[i] == -INFINITY ? 0.f : ex2((m[nr][i] - M[i]) * a.sl);
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
                        if (M[i] != -INFINITY) Ls[i] += sl[e] * ex2((sm[e] - M[i]) * a.sl);
                    }
                }
                if (whole) {
                    const int dim = g * (D / 8) + 2 * k;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int rr = nr * 8 + 2 * t + i;
                        if (rr < rows) {
                            const int r = rt * R + rr;
                            const float inv = Ls[i] > 0.f ? 1.f / Ls[i] : 0.f;
                            const float y0 = (i ? x.y : x.x) * inv, y1 = (i ? x.w : x.z) * inv;
                            T *p = static_cast<T *>(a.out) + (long)(sq.q0 + r / a.G) * a.os +
                                   (long)(kvh * a.G + r % a.G) * D + dim;
                            if constexpr (HL) *reinterpret_cast<float2 *>(p) = make_float2(y0, y1);
                            else *reinterpret_cast<__half2 *>(p) = __floats2half2_rn(y0, y1);
                        }
                    }
                } else {
                    reinterpret_cast<float4 *>(a.part)[((long)slot * NR + nr) * MT * 32 + threadIdx.x] = x;
                    if (k == 0 && g == 0)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            float *p = a.ml + ((long)slot * R + nr * 8 + 2 * t + i) * 2;
                            p[0] = M[i], p[1] = Ls[i];
                        }
                }
            }
            __syncthreads();
        }
        u += c1 - c0;
        ++nseg;
    }
}

// One warp per (item, 8-row group, 16-dim fragment): joins the partials of an item
// that several runs share, in run order.  Items that lie in one run are done.
template <typename T, int D, int NR>
__global__ void __launch_bounds__(32) merge_kernel(const AttnArgs a, int grid, int nrt_max) {
    constexpr int R = 8 * NR, MT = D / 16;
    const int lane = threadIdx.x, g = lane >> 2, t = lane & 3;
    const int b = blockIdx.x / (a.pool.nkv * nrt_max), kvh = blockIdx.x / nrt_max % a.pool.nkv, rt = blockIdx.x % nrt_max;
    const int nr = blockIdx.y / MT, k = blockIdx.y % MT;
    pdl_launch_dependents();
    pdl_wait();
    const Seq sq = load_seq(a, b, R, false);
    if (rt >= sq.nrt) return;
    const int rows = min(R, sq.nq * a.G - rt * R);
    if (nr * 8 >= rows) return;
    long U = 0, before = 0;
    for (int b0 = 0; b0 < a.tab.n_seqs; b0 += 32) {
        const int bb = b0 + lane;
        const long n = bb < a.tab.n_seqs ? load_seq(a, bb, R, false).units(a.pool.nkv) : 0;
        U += n;
        before += bb < b ? n : 0;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        U += __shfl_xor_sync(0xffffffffu, U, o);
        before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    const long ua = before + ((long)kvh * sq.nrt + item_of_row_tile(rt, sq.nrt)) * sq.cu, ub = ua + sq.cu;
    const long nc = min((long)grid, U);
    const int c_first = (int)(((ua + 1) * nc - 1) / U), c_last = (int)((ub * nc - 1) / U);
    if (c_first == c_last) return;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = c_first; c <= c_last; ++c) {
        const int slot = 2 * c + (c == c_first && U * c / nc != ua ? 1 : 0);
        const float4 y = __ldcg(reinterpret_cast<const float4 *>(a.part) + ((long)slot * NR + nr) * MT * 32 + k * 32 + lane);
        float f[2], h[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float2 p = __ldcg(reinterpret_cast<const float2 *>(a.ml) + (long)slot * R + nr * 8 + 2 * t + i);
            const float mn = fmaxf(m[i], p.x);
            f[i] = mn == -INFINITY ? 0.f : ex2((m[i] - mn) * a.sl);
            h[i] = mn == -INFINITY ? 0.f : ex2((p.x - mn) * a.sl);
            m[i] = mn;
            l[i] = l[i] * f[i] + p.y * h[i];
        }
        x.x = x.x * f[0] + y.x * h[0], x.y = x.y * f[1] + y.y * h[1];
        x.z = x.z * f[0] + y.z * h[0], x.w = x.w * f[1] + y.w * h[1];
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int rr = nr * 8 + 2 * t + i;
        if (rr >= rows) continue;
        const int r = rt * R + rr;
        const float inv = l[i] > 0.f ? 1.f / l[i] : 0.f;
        const float y0 = (i ? x.y : x.x) * inv, y1 = (i ? x.w : x.z) * inv;
        T *p = static_cast<T *>(a.out) + (long)(sq.q0 + r / a.G) * a.os + (long)(kvh * a.G + r % a.G) * D + g * (D / 8) + 2 * k;
        if constexpr (sizeof(T) == 4) *reinterpret_cast<float2 *>(p) = make_float2(y0, y1);
        else *reinterpret_cast<__half2 *>(p) = __floats2half2_rn(y0, y1);
    }
}

template <typename T, int D, int NR>
static int launch(DevCtx *c, AttnArgs &a, cudaStream_t s) {
    constexpr int R = 8 * NR;
    static bool attr[64];
    if (!attr[c->device]) {
        set_qkernel_attrs(attn_kernel<T, D, NR>, Cfg<D, NR>::SMEM);
        attr[c->device] = true;
    }
    const long nrt = ((long)a.max_q * a.G + R - 1) / R, cover = (long)a.tab.stride << a.pool.page_shift;
    const long most = std::min<long>((long)a.tab.n_seqs * a.pool.nkv * nrt, kMaxCtas) * std::max<long>(1, (cover + kUnit - 1) / kUnit);
    const int grid = (int)std::min<long>(std::min(kMaxCtas, c->sm_count * (NR == 1 ? 2 : 1)), most);
    a.ml = a.part + (size_t)kMaxCtas * 2 * R * D;
    int st = launch_pdl(attn_kernel<T, D, NR>, dim3(grid), dim3(kWarps * 32), Cfg<D, NR>::SMEM, s, a);
    if (st) return st;
    const long items = (long)a.tab.n_seqs * a.pool.nkv * nrt;
    return launch_pdl(merge_kernel<T, D, NR>, dim3((unsigned)items, NR * (D / 16)), dim3(32), 0, s, a, grid, (int)nrt);
}

template <typename T, int D>
static int launch_rows(DevCtx *c, AttnArgs &a, cudaStream_t s) {
    const long rows = (long)a.max_q * a.G;
    if (rows <= 8) return launch<T, D, 1>(c, a, s);
    if (rows <= 16) return launch<T, D, 2>(c, a, s);
    return launch<T, D, 4>(c, a, s);
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
    return (size_t)kMaxCtas * 2 * 32 * (kv->head_dim + 2) * sizeof(float);
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
        !(a->scale > 0.f) || !(a->scale < INFINITY) || !a->work || !aligned16(a->work))
        return refuse(X100_E_ARG);
    if (a->work_bytes < x100q_kv4_attn_work(kv, a->n_tokens, a->n_heads, a->n_seqs)) return refuse(X100_E_TOO_LARGE);
    if (a->n_seqs > 65536) return refuse(X100_E_TOO_LARGE);
    DevCtx *c = ctx();
    if (!c) return get_error();
    AttnArgs p;
    p.pool = make_pool(kv);
    p.tab = {a->page_table, a->table_stride, a->n_seqs};
    p.q = a->q, p.out = a->out, p.qs = a->q_stride, p.os = a->out_stride;
    p.q_start = a->q_start, p.kv_len = a->kv_len;
    p.n_tokens = a->n_tokens, p.max_q = a->q_start ? std::min(a->max_q, a->n_tokens) : 1;
    p.nh = a->n_heads, p.G = a->n_heads / kv->n_kv_heads;
    p.sl = a->scale * 1.4426950408889634f;
    p.part = static_cast<float *>(a->work);
    p.status = c->d_status;
    const long items = (long)a->n_seqs * kv->n_kv_heads * (((long)p.max_q * p.G + 7) / 8);
    if (items > 0x7fffffffl || (long)p.max_q * p.G > (1l << 30)) return refuse(X100_E_TOO_LARGE);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a->dtype == X100Q_F32)
        return kv->head_dim == 128 ? launch_rows<float, 128>(c, p, s) : launch_rows<float, 64>(c, p, s);
    return kv->head_dim == 128 ? launch_rows<__half, 128>(c, p, s) : launch_rows<__half, 64>(c, p, s);
}

}  // extern "C"
