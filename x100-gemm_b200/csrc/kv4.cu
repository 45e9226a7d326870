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
    int rope_len, n_tokens, nh;
    const int *pos, *seq;
    int *status;
};

// The E consecutive elements of a lane (E = D / 32: lane l holds E l ..), in fp32.
template <typename T, int E>
__device__ __forceinline__ void load_lane(const T *p, int lane, float (&x)[E]) {
    if constexpr (sizeof(T) == 4) {
        if constexpr (E == 4) {
            const float4 v = *(reinterpret_cast<const float4 *>(p) + lane);
            x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
        } else {
            const float2 v = *(reinterpret_cast<const float2 *>(p) + lane);
            x[0] = v.x, x[1] = v.y;
        }
    } else {
        __half2 h[E / 2];
        if constexpr (E == 4) *reinterpret_cast<uint2 *>(h) = *(reinterpret_cast<const uint2 *>(p) + lane);
        else *reinterpret_cast<uint32_t *>(h) = *(reinterpret_cast<const uint32_t *>(p) + lane);
#pragma unroll
        for (int i = 0; i < E / 2; ++i) {
            const float2 f = __half22float2(h[i]);
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
    }
}
template <typename T, int E>
__device__ __forceinline__ void store_lane(T *p, int lane, const float (&x)[E]) {
    if constexpr (sizeof(T) == 4) {
        if constexpr (E == 4) *(reinterpret_cast<float4 *>(p) + lane) = make_float4(x[0], x[1], x[2], x[3]);
        else *(reinterpret_cast<float2 *>(p) + lane) = make_float2(x[0], x[1]);
    } else {
        __half2 h[E / 2];
#pragma unroll
        for (int i = 0; i < E / 2; ++i) h[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        if constexpr (E == 4) *(reinterpret_cast<uint2 *>(p) + lane) = *reinterpret_cast<uint2 *>(h);
        else *(reinterpret_cast<uint32_t *>(p) + lane) = *reinterpret_cast<uint32_t *>(h);
    }
}

// One head of q, k or v of one token per warp; a lane holds E = D / 32
// consecutive elements, so an element's rotation partner (j + D / 2) is lane ^ 16's
// same element and a block of 32 is 32 / E neighbouring lanes.  Every product, sum and
// quotient up to the code is rounded by itself (no contraction), which makes the codes
// the same on any machine that follows the formula.  Codes are taken before
// the factor 1 / rms, which a block's scale carries: rounding of the sum of squares
// cannot move a value over a code's border.
template <typename T, int D>
__global__ void __launch_bounds__(256) append_kernel(const AppendArgs a) {
    using L = Lay<D>;
    constexpr int E = D / 32, LB = 32 / E;   // LB lanes per block
    const int lane = threadIdx.x & 31;
    const int heads = a.nh + 2 * a.pool.nkv;
    const long item = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
    pdl_launch_dependents();
    pdl_wait();
    if (item >= (long)a.n_tokens * heads) return;
    const int i = (int)(item / heads), h = (int)(item % heads);
    const int pos = a.pos[i];
    if (pos < 0) return;                                  // padding
    const bool is_q = h < a.nh, is_k = !is_q && h < a.nh + a.pool.nkv;
    const int seq = a.seq ? a.seq[i] : i;
    const bool rotate = a.rope && (is_q || is_k);
    uint8_t *tile = nullptr;
    bool bad = rotate && pos >= a.rope_len;
    if (!is_q && !bad) {
        tile = tile_of(a.pool, a.tab, seq, pos, is_k ? h - a.nh : h - a.nh - a.pool.nkv);
        bad = tile == nullptr;
    }
    if (bad) {
        if (lane == 0) atomicCAS(a.status, 0, X100_E_ARG);
        return;
    }
    float x[E], t[E];
    const T *src = is_q ? static_cast<const T *>(a.q) + i * a.qs + (long)h * D
                        : is_k ? static_cast<const T *>(a.k) + i * a.ks + (long)(h - a.nh) * D
                               : static_cast<const T *>(a.v) + i * a.vs + (long)(h - a.nh - a.pool.nkv) * D;
    load_lane<T, E>(src, lane, x);
    float s = 1.f;
    const float *w = is_q ? a.qn : is_k ? a.kn : nullptr;
    if (w) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) ss += x[e] * x[e];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        s = 1.f / sqrtf(ss / (float)D + a.eps);
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = __fmul_rn(x[e], __ldg(w + E * lane + e));
    }
    if (rotate) {
        const float2 *row = a.rope + (long)pos * (D / 2) + ((E * lane) & (D / 2 - 1));
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float2 cs = __ldg(row + e);
            const float o = __shfl_xor_sync(0xffffffffu, x[e], 16);
            t[e] = lane < 16 ? __fsub_rn(__fmul_rn(x[e], cs.x), __fmul_rn(o, cs.y))
                             : __fadd_rn(__fmul_rn(x[e], cs.x), __fmul_rn(o, cs.y));
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) t[e] = x[e];
    }
    if (is_q) {
#pragma unroll
        for (int e = 0; e < E; ++e) t[e] *= s;
        store_lane<T, E>(static_cast<T *>(a.qo) + i * a.qos + (long)h * D, lane, t);
        return;
    }
    float top = t[0], low = t[0];
    bool fin = true;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        top = fmaxf(top, t[e]);
        low = fminf(low, t[e]);
        fin = fin && fabsf(t[e]) < INFINITY;
    }
#pragma unroll
    for (int o = 1; o < LB; o <<= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
    }
    const float m = top >= -low ? top : low;
    float inv = fabsf(m) < kTinyBlock ? 0.f : __fdiv_rn(-8.f, m);
    float d = __fmul_rn(__fmul_rn(m, -0.125f), s);
    const uint32_t mask = __ballot_sync(0xffffffffu, fin && fabsf(d) < INFINITY) | 0u;
    const uint32_t mine = (LB == 32 ? 0xffffffffu : ((1u << LB) - 1u)) << (lane & ~(LB - 1));
    if ((mask & mine) != mine) {                          // a NaN or an infinity in the block
        inv = 0.f, d = 0.f;
        if (lane % LB == 0) atomicCAS(a.status, 0, X100_E_ARG);
    }
    uint32_t codes = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float c = inv == 0.f ? 8.f : floorf(__fadd_rn(__fmul_rn(t[e], inv), 8.5f));
        codes |= (uint32_t)fminf(fmaxf(c, 0.f), 15.f) << (4 * e);
    }
    const __half dh = __float2half_rn(__bfloat162float(__float2bfloat16_rn(fminf(fmaxf(d, -kMostScale), kMostScale))));
    const int sp = pos & 15, b = E * lane / 32;
    if (is_k) {
        const int in = E * lane & 31;                     // first dim of the lane in its block
        uint8_t *at = tile + L::k_word(sp, b, in >> 3) + (in & 7) / 2;
        if constexpr (E == 4) *reinterpret_cast<uint16_t *>(at) = (uint16_t)codes;
        else *at = (uint8_t)codes;
        if (lane % LB == 0) *reinterpret_cast<__half *>(tile + L::k_scale(sp, b)) = dh;
    } else {
        const int g = E * lane / (D / 8);
        uint8_t *at = tile + L::v_piece(sp, g) + (E * lane % (D / 8)) / 2;
        if constexpr (E == 4) *reinterpret_cast<uint16_t *>(at) = (uint16_t)codes;
        else *at = (uint8_t)codes;
        if (lane % LB == 0) *reinterpret_cast<__half *>(tile + L::v_scale(sp, b)) = dh;
    }
}

struct ReadArgs {
    Pool pool;
    Table tab;
    const int *pos, *seq;
    int n_tokens;
    __half *k, *v;
    int *status;
};

// The inverse: one head of k or v of one token per warp, d * (code - 8) in fp16 (exact).
template <int D>
__global__ void __launch_bounds__(256) read_kernel(const ReadArgs a) {
    using L = Lay<D>;
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31;
    const int kinds = (a.k ? 1 : 0) + (a.v ? 1 : 0), heads = kinds * a.pool.nkv;
    const long item = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
    pdl_launch_dependents();
    pdl_wait();
    if (item >= (long)a.n_tokens * heads) return;
    const int i = (int)(item / heads), r = (int)(item % heads), h = r % a.pool.nkv;
    const bool is_k = a.k && r < a.pool.nkv;
    const int pos = a.pos[i];
    if (pos < 0) return;
    const uint8_t *tile = tile_of(a.pool, a.tab, a.seq ? a.seq[i] : i, pos, h);
    if (!tile) {
        if (lane == 0) atomicCAS(a.status, 0, X100_E_ARG);
        return;
    }
    const int sp = pos & 15, b = E * lane / 32, in = E * lane & 31, g = E * lane / (D / 8);
    const uint8_t *at = is_k ? tile + L::k_word(sp, b, in >> 3) + (in & 7) / 2
                             : tile + L::v_piece(sp, g) + (E * lane % (D / 8)) / 2;
    const float d = __half2float(*reinterpret_cast<const __half *>(tile + (is_k ? L::k_scale(sp, b) : L::v_scale(sp, b))));
    uint32_t codes;
    if constexpr (E == 4) codes = *reinterpret_cast<const uint16_t *>(at);
    else codes = *at;
    float x[E];
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = d * ((int)(codes >> (4 * e) & 15) - 8);
    store_lane<__half, E>((is_k ? a.k : a.v) + ((long)i * a.pool.nkv + h) * D, lane, x);
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
        (reinterpret_cast<uintptr_t>(a->rope) & 7) || ((a->q_norm || a->k_norm) && !(a->eps >= 0.f)))
        return refuse(X100_E_ARG);
    if (a->q && (a->n_heads < 1 || a->n_heads > 4096 || !a->q_out || !aligned16(a->q) || !aligned16(a->q_out) ||
                 !pitch_ok(a->q_stride, a->n_heads * kv->head_dim, es) ||
                 !pitch_ok(a->q_out_stride, a->n_heads * kv->head_dim, es)))
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
    const long warps = (long)p.n_tokens * (p.nh + 2 * p.pool.nkv), ctas = (warps + 7) / 8;
    if (ctas > 0x7fffffffl) return refuse(X100_E_TOO_LARGE);
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
    ReadArgs p = {make_pool(kv), {page_table, table_stride, n_seqs}, pos, seq, n_tokens, static_cast<__half *>(k_out),
                  static_cast<__half *>(v_out), c->d_status};
    const long warps = (long)n_tokens * kv->n_kv_heads * ((k_out ? 1 : 0) + (v_out ? 1 : 0)), ctas = (warps + 7) / 8;
    if (ctas > 0x7fffffffl) return refuse(X100_E_TOO_LARGE);
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
