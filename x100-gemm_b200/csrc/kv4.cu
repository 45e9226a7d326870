// kv4.cu -- the paged 4-bit KV cache: appending (head norm, rotation and
// quantisation on the way), reading back, and the rotation table.
#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>

#include "kv4.cuh"
#include "qformats.cuh"
#include "qgemv.h"

namespace x100 {
namespace kv4 {

using q::pdl_launch_dependents;
using q::pdl_wait;

struct AppendArgs {
    Pool pool;
    Table tab;
    const void *q, *k, *v;
    void *qo;
    long qs, ks, vs, qos;
    const float *qn, *kn;
    float eps;
    const float2 *rope;
    int rope_len, n_tokens, nh, slices;
    const int *pos, *seq;
    int *status;
};

// 8 elements of a head, as loaded and in fp32.
template <typename T>
struct Eight {
    uint4 v[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = *(reinterpret_cast<const uint4 *>(p) + i);
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
        const uint32_t *w = reinterpret_cast<const uint32_t *>(v);
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(w + i));
                x[2 * i] = f.x, x[2 * i + 1] = f.y;
            }
        }
    }
    static __device__ __forceinline__ void store(T *p, const float (&x)[8]) {
        if constexpr (sizeof(T) == 4) {
            reinterpret_cast<float4 *>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
            reinterpret_cast<float4 *>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
        } else {
            __half2 h[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
            *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(h);
        }
    }
};

// A lane holds 8 elements of a head (a K word's codes), so LH = D / 8 lanes have a head and a warp HW = 32 / LH
// heads side by side.  An element's rotation partner (j + D / 2) is the same element of lane ^ LH / 2, and a block
// of 32 is 4 neighbouring lanes.  A warp takes the groups of HW heads of one token that are its slice's
// (slice, slice + slices, ..), the next group's bytes on their way while one is worked on; the rotation's row is
// loaded once.  Every product, sum and quotient up to the code is rounded by itself (no contraction), which
// makes the codes the same on any machine that follows the formula.  Codes are taken before the factor
// 1 / rms, which a block's scale carries: rounding of the sum of squares cannot move a value over a code's
// border.
// Bound by instructions when there are many tokens (issue slots 0.72 busy for fp16, DRAM 0.28; 8 shuffles a lane and group are the
// partners' elements, which this layout has in another lane), by the launch when there are
// few.  1024 tokens of 32 + 2 x 4 heads of 128, fp32: 38 MB in 10.8 us; 8 x 2047 of 16 + 2 x 8 heads of 64, fp16: 112 MB in
// 33.5 us.  A warp per head with 4 elements a lane took 195 us there (with the read-back), a loop per kind of head 4 us more than
// one over all, two groups on their way or k's and v's heads as one list the same.
template <typename T, int D>
__global__ void __launch_bounds__(256, sizeof(T) == 4 ? 3 : 4) append_kernel(const AppendArgs a) {
    using L = Lay<D>;
    constexpr int LH = D / 8, HW = 32 / LH;
    const int lane = threadIdx.x & 31, in = lane % LH, hl = lane / LH;          // place in the head, head of the group
    const int nkv = a.pool.nkv, gq = (a.nh + HW - 1) / HW, gk = (nkv + HW - 1) / HW, groups = gq + 2 * gk;
    const uint32_t item = blockIdx.x * 8 + (threadIdx.x >> 5);   // slices are several only for few tokens
    pdl_launch_dependents();
    pdl_wait();
    if (item >= (uint32_t)a.n_tokens * a.slices) return;
    const int i = a.slices == 1 ? item : item / a.slices, slice = (int)item - i * a.slices;
    const int pos = a.pos[i];
    if (pos < 0) return;                                  // padding
    const int seq = a.seq ? a.seq[i] : i;
    // this lane's elements of group g; past the last head, the last one's
    const T *const qb = static_cast<const T *>(a.q) + i * a.qs + in * 8, *const kb = static_cast<const T *>(a.k) + i * a.ks + in * 8,
                  *const vb = static_cast<const T *>(a.v) + i * a.vs + in * 8;
    auto at_group = [&](int g) {
        const bool is_q = g < gq, is_k = g < gq + gk;
        const int h = min((g - (is_q ? 0 : is_k ? gq : gq + gk)) * HW + hl, (is_q ? a.nh : nkv) - 1);
        return (is_q ? qb : is_k ? kb : vb) + h * D;
    };
    int g = slice;
    if (g >= groups) return;
    Eight<T> next;
    next.load(at_group(g));
    // the rotation's row and the token's page: a bad position or page is left out and reported
    const bool turn = a.rope != nullptr, far = turn && pos >= a.rope_len;
    float cs[8], sn[8];                                   // the sine with the sign that the lane's half takes it with
#pragma unroll
    for (int e = 0; e < 8; ++e) cs[e] = 1.f, sn[e] = 0.f;
    if (turn && !far) {
        const float4 *row = reinterpret_cast<const float4 *>(a.rope + (long)pos * (D / 2) + (in * 8 & (D / 2 - 1)));
        const float sign = in < LH / 2 ? -1.f : 1.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float4 r = __ldg(row + e);
            cs[2 * e] = r.x, sn[2 * e] = sign * r.y, cs[2 * e + 1] = r.z, sn[2 * e + 1] = sign * r.w;
        }
    }
    uint8_t *tile = nullptr;                              // of kv head 0
    if (g + (groups - 1 - g) / a.slices * a.slices >= gq) tile = tile_of(a.pool, a.tab, seq, pos, 0);   // the slice has k or v
    float wq[sizeof(T) == 4 ? 8 : 1];                      // q has most of the groups; fp16's registers are better spent on warps
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int e = 0; e < 8; ++e) wq[e] = a.qn && g < gq ? __ldg(a.qn + in * 8 + e) : 1.f;
    }
    bool bad = far;
    if (far) g = groups;
    for (; g < groups; g += a.slices) {
        float t[8];
        next.get(t);
        if (g + a.slices < groups) next.load(at_group(g + a.slices));
        const bool is_q = g < gq, is_k = !is_q && g < gq + gk;
        float s = 1.f;
        const float *w = is_q ? a.qn : is_k ? a.kn : nullptr;
        if (w) {
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = fmaf(t[e], t[e], ss);
#pragma unroll
            for (int o = LH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            s = ss < INFINITY ? __frsqrt_rn(ss * (1.f / D) + a.eps) : NAN;   // past fp32's range: not a head of zeros
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] = __fmul_rn(t[e], sizeof(T) == 4 && is_q ? wq[sizeof(T) == 4 ? e : 0] : __ldg(w + in * 8 + e));
        }
        if (turn && (is_q || is_k)) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {                 // x c - o s or x c + o s, each step rounded
                const float o = __shfl_xor_sync(0xffffffffu, t[e], LH / 2);
                t[e] = __fadd_rn(__fmul_rn(t[e], cs[e]), __fmul_rn(o, sn[e]));
            }
        }
        if (is_q) {
            const int h = g * HW + hl;
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] *= s;
            if (h < a.nh) Eight<T>::store(static_cast<T *>(a.qo) + i * a.qos + (long)h * D + in * 8, t);
            continue;
        }
        if (!tile) {
            bad = true;
            continue;
        }
        float top = t[0], low = t[0], z = 0.f;            // z: 0, or NaN where a value is not finite
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            top = fmaxf(top, t[e]);
            low = fminf(low, t[e]);
            z = fmaf(t[e], 0.f, z);
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
        }
        const float m = top >= -low ? top : low;
        float inv = fabsf(m) < kTinyBlock ? 0.f : __fdiv_rn(-8.f, m);
        float d = __fmul_rn(__fmul_rn(m, -0.125f), s);
        const uint32_t fine = __ballot_sync(0xffffffffu, z == 0.f && fabsf(d) < INFINITY), mine = 15u << (lane & 28);
        if ((fine & mine) != mine) {                      // a NaN or an infinity in the block
            inv = 0.f, d = 0.f;
            bad = true;
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] = 0.f;
        }
        // x * inv + 8.5 lies in (0, 17): added to 2^23 rounding down, its floor is the low bits (8 where inv is 0).
        // The codes are summed up with the exponent's bits still on, whose sum is known.
        uint32_t codes = 0u - 0x4b000000u;                // of the 8 shifted exponents only the first reaches the word
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t c = __float_as_uint(__fadd_rd(__fadd_rn(__fmul_rn(t[e], inv), 8.5f), 8388608.f));
            codes += min(c, 0x4b00000fu) << (4 * e);
            if (e == 1) codes -= 0xb0000000u;             // 0x4b000000 << 4; the further ones leave the word
        }
        const __half dh = __float2half_rn(__bfloat162float(__float2bfloat16_rn(fminf(fmaxf(d, -kMostScale), kMostScale))));
        const int h = (g - (is_k ? gq : gq + gk)) * HW + hl, sp = pos & 15, b = in / 4;
        if (h >= nkv) continue;
        uint8_t *th = tile + h * a.pool.page_bytes;
        *reinterpret_cast<uint32_t *>(is_k ? th + L::k_word(sp, b, in & 3) : th + L::v_piece(sp, in * 8 / (D / 8)) + in * 8 % (D / 8) / 2) = codes;
        if ((lane & 3) == 0) *reinterpret_cast<__half *>(th + (is_k ? L::k_scale(sp, b) : L::v_scale(sp, b))) = dh;
    }
    if (bad) atomicCAS(a.status, 0, X100_E_ARG);
}

struct ReadArgs {
    Pool pool;
    Table tab;
    const int *pos, *seq;
    int n_tokens, slices;
    __half *k, *v;
    int *status;
};

// The inverse: a lane has 8 dims of a head (a word of codes, 16 bytes out), d * (code - 8) in fp16 (exact); warps and
// slices as in append_kernel, over k's and v's heads as one list.  Bound by the chain position -> page -> codes, so
// 32 registers: 3.0 us for the 1024 tokens and 10.5 us for the 8 x 2047 (5 and 15 with lists apart and 48 registers).
template <int D>
__global__ void __launch_bounds__(256, 8) read_kernel(const ReadArgs a) {
    using L = Lay<D>;
    constexpr int LH = D / 8, HW = 32 / LH;
    const int lane = threadIdx.x & 31, in = lane % LH, hl = lane / LH, nkv = a.pool.nkv;
    const int nk = a.k ? nkv : 0, heads = nk + (a.v ? nkv : 0), groups = (heads + HW - 1) / HW;
    const uint32_t item = blockIdx.x * 8 + (threadIdx.x >> 5);
    pdl_launch_dependents();
    pdl_wait();
    if (item >= (uint32_t)a.n_tokens * a.slices) return;
    const int i = a.slices == 1 ? item : item / a.slices, slice = (int)item - i * a.slices;
    const int pos = a.pos[i];
    if (pos < 0) return;
    const uint8_t *tile = tile_of(a.pool, a.tab, a.seq ? a.seq[i] : i, pos, 0);
    if (!tile) {
        if (lane == 0) atomicCAS(a.status, 0, X100_E_ARG);
        return;
    }
    const int sp = pos & 15, b = in / 4;
#pragma unroll 2
    for (int g = slice; g < groups; g += a.slices) {
        const int at = g * HW + hl, h = at < nk ? at : at - nk;
        if (at >= heads) break;
        const uint8_t *th = tile + h * a.pool.page_bytes;
        const uint32_t codes = *reinterpret_cast<const uint32_t *>(at < nk ? th + L::k_word(sp, b, in & 3) : th + L::v_piece(sp, in * 8 / (D / 8)) + in * 8 % (D / 8) / 2);
        const float d = __half2float(*reinterpret_cast<const __half *>(th + (at < nk ? L::k_scale(sp, b) : L::v_scale(sp, b))));
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = d * ((int)(codes >> (4 * e) & 15) - 8);
        Eight<__half>::store((at < nk ? a.k : a.v) + ((long)i * nkv + h) * D + in * 8, x);
    }
}

// Warps per token: enough to fill the card when there are few tokens, one when there are many.
inline int slices_for(const DevCtx *c, int n_tokens, int groups) {
    const long want = ((long)c->sm_count * 32 + n_tokens - 1) / n_tokens;
    return (int)std::max<long>(1, std::min<long>(want, groups));
}

__global__ void rope64_kernel(float2 *rope, long n, int half, double step) {
    for (long j = blockIdx.x * (long)blockDim.x + threadIdx.x; j < n; j += (long)gridDim.x * blockDim.x) {
        double s, c;
        sincos((double)(j / half) * exp(step * (double)(j % half)), &s, &c);
        rope[j] = make_float2((float)c, (float)s);
    }
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

size_t x100q_kv4_bytes(const x100q_kv4 *kv) {
    if (!shape_ok(kv)) return 0;
    return (size_t)kv->n_pages * kv->n_kv_heads * (size_t)make_pool(kv).page_bytes;
}

int x100q_kv4_append_dev(const x100q_kv4 *kv, const x100q_kv4_append_args *a, void *stream) {
    set_error(X100_OK);
    if (!shape_ok(kv) || !a || a->n_tokens < 0) return refuse(X100_E_ARG);
    if (a->n_tokens == 0) return X100_OK;
    if (a->dtype != X100Q_F32 && a->dtype != X100Q_F16) return refuse(X100_E_UNSUPPORTED);
    const int es = a->dtype == X100Q_F32 ? 4 : 2, kw = kv->n_kv_heads * kv->head_dim;
    if (!kv->pages || !aligned16(kv->pages) || !a->k || !a->v || !a->pos || !a->page_table || a->table_stride < 1 ||
        a->n_seqs < 1 || (!a->seq && a->n_tokens > a->n_seqs) || !aligned16(a->k) || !aligned16(a->v) ||
        !pitch_ok(a->k_stride, kw, es) || !pitch_ok(a->v_stride, kw, es) || (a->rope && a->rope_len < 1) ||
        !aligned16(a->rope) || ((a->q_norm || a->k_norm) && !(a->eps >= 0.f)))
        return refuse(X100_E_ARG);
    if (a->q && (a->n_heads < 1 || a->n_heads > 4096 || !a->q_out || !aligned16(a->q) || !aligned16(a->q_out) ||
                 !pitch_ok(a->q_stride, a->n_heads * kv->head_dim, es) ||
                 !pitch_ok(a->q_out_stride, a->n_heads * kv->head_dim, es) ||
                 !in_place_ok(a->q, a->q_stride, a->q_out, a->q_out_stride, a->n_tokens)))
        return refuse(X100_E_ARG);
    DevCtx *c = ctx();
    if (!c) return get_error();
    AppendArgs p;
    p.pool = make_pool(kv);
    p.tab = {a->page_table, a->table_stride, a->n_seqs};
    p.q = a->q, p.k = a->k, p.v = a->v, p.qo = a->q_out;
    p.qs = a->q_stride, p.ks = a->k_stride, p.vs = a->v_stride, p.qos = a->q_out_stride;
    p.qn = a->q_norm, p.kn = a->k_norm, p.eps = a->eps;
    p.rope = reinterpret_cast<const float2 *>(a->rope), p.rope_len = a->rope_len;
    p.n_tokens = a->n_tokens, p.nh = a->q ? a->n_heads : 0;
    p.pos = a->pos, p.seq = a->seq, p.status = c->d_status;
    const int hw = 256 / kv->head_dim, kvg = (p.pool.nkv + hw - 1) / hw;   // heads per warp, groups of k or v
    p.slices = slices_for(c, p.n_tokens, (p.nh + hw - 1) / hw + 2 * kvg);
    const long ctas = ((long)p.n_tokens * p.slices + 7) / 8;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const dim3 grid((unsigned)ctas), blk(256);
    int st;
    if (a->dtype == X100Q_F32)
        st = kv->head_dim == 128 ? launch_pdl(append_kernel<float, 128>, grid, blk, 0, s, p)
                                 : launch_pdl(append_kernel<float, 64>, grid, blk, 0, s, p);
    else
        st = kv->head_dim == 128 ? launch_pdl(append_kernel<__half, 128>, grid, blk, 0, s, p)
                                 : launch_pdl(append_kernel<__half, 64>, grid, blk, 0, s, p);
    return st;
}

int x100q_kv4_read_dev(const x100q_kv4 *kv, const int *pos, const int *seq, int n_tokens, const int *page_table,
                       int table_stride, int n_seqs, void *k_out, void *v_out, void *stream) {
    set_error(X100_OK);
    if (!shape_ok(kv) || n_tokens < 0) return refuse(X100_E_ARG);
    if (n_tokens == 0 || (!k_out && !v_out)) return X100_OK;
    if (!kv->pages || !aligned16(kv->pages) || !pos || !page_table || table_stride < 1 || n_seqs < 1 ||
        (!seq && n_tokens > n_seqs) || !aligned16(k_out) || !aligned16(v_out))
        return refuse(X100_E_ARG);
    DevCtx *c = ctx();
    if (!c) return get_error();
    const int hw = 256 / kv->head_dim, groups = (kv->n_kv_heads * ((k_out ? 1 : 0) + (v_out ? 1 : 0)) + hw - 1) / hw;
    ReadArgs p = {make_pool(kv), {page_table, table_stride, n_seqs}, pos, seq, n_tokens, slices_for(c, n_tokens, groups), static_cast<__half *>(k_out),
                  static_cast<__half *>(v_out), c->d_status};
    const long ctas = ((long)n_tokens * p.slices + 7) / 8;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return kv->head_dim == 128 ? launch_pdl(read_kernel<128>, dim3((unsigned)ctas), dim3(256), 0, s, p)
                               : launch_pdl(read_kernel<64>, dim3((unsigned)ctas), dim3(256), 0, s, p);
}

int x100q_rope_table_dev(float *rope, int n_pos, int head_dim, float base, void *stream) {
    set_error(X100_OK);
    if (!rope || (reinterpret_cast<uintptr_t>(rope) & 7) || n_pos < 0 || head_dim < 2 || head_dim % 2 || !(base > 0.f) ||
        !(base < INFINITY))
        return refuse(X100_E_ARG);
    if (n_pos == 0) return X100_OK;
    DevCtx *c = ctx();
    if (!c) return get_error();
    const long n = (long)n_pos * (head_dim / 2);
    const int grid = (int)std::min<long>((n + 255) / 256, (long)c->sm_count * 16);
    return launch_k(rope64_kernel, dim3(grid), dim3(256), 0, static_cast<cudaStream_t>(stream), false,
                    reinterpret_cast<float2 *>(rope), n, head_dim / 2, -2.0 * std::log((double)base) / head_dim);
}

}  // extern "C"
