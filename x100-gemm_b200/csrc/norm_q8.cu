// norm_q8.cu -- residual addition, RMS norm and int8 quantisation of activation
// rows in one pass (x100q_add_rmsnorm_q8_dev).
//
// The code of an element needs only its group: with t = h * w,
//   y / scale = (t / rms) / (max|t| / 127 / rms) = t * 127 / max|t|,
// so 1 / rms enters the scale alone and its rounding cannot move a code.
#include <algorithm>
#include <cmath>
#include <cuda_fp16.h>

#include "../../include/x100q.h"
#include "qformats.cuh"
#include "qgemv.h"
#include "runtime.h"

namespace x100 {
namespace normq8 {

using q::pdl_launch_dependents;
using q::pdl_wait;

constexpr float kTiny = 7.7037197775489434e-34f;   // 2^-110

struct Args {
    const void *x, *res;
    void *out;
    long ldx, ldr, ldo, ldq;
    const float *w;
    float eps;
    int rows, d, group;
    int8_t *q;
    float *scales;
};

template <typename T>
__device__ __forceinline__ float to_f(T v) {
    if constexpr (sizeof(T) == 4) return v;
    else return __half2float(v);
}
// h of one element: the sum rounded to T, as it is stored
template <typename T>
__device__ __forceinline__ T add_t(T x, T r) {
    if constexpr (sizeof(T) == 4) return x + r;
    else return __float2half_rn(__half2float(x) + __half2float(r));
}
// |t|, with a NaN counted as an infinity (fmaxf would drop it)
__device__ __forceinline__ float mag(float t) {
    const float a = fabsf(t);
    return a < INFINITY ? a : INFINITY;
}
__device__ __forceinline__ float inv_of(float top) { return top < kTiny || top == INFINITY ? 0.f : __fdiv_rn(127.f, top); }
__device__ __forceinline__ float scale_of(float top, float rstd) {
    return top == INFINITY || rstd == 0.f ? NAN : top < kTiny ? 0.f : top * (1.f / 127.f) * rstd;   // rstd 0: the sum of squares is infinite
}
__device__ __forceinline__ int code_of(float t, float inv) {
    return inv == 0.f ? 0 : __float2int_rn(fminf(fmaxf(__fmul_rn(t, inv), -127.f), 127.f));
}

// Rows of 16-byte units: unit u of a row belongs to thread u % NT of the NT that
// share the row, NV units each, kept in registers between the sum and the codes, so
// every byte is read once.  256 / NT rows per CTA and step (NT <= 256), rows in
// grid strides so that the weights stay in registers.  Bound by HBM: 16384 rows of 4096, fp16, 470 MB in 83 us
// (5.6 TB/s); 1024 of 2048, fp32, 28 MB in 7.2 us (inputs from L2 in part); a row alone 1.9 us.
template <typename T, int NV, int NT>
__global__ void __launch_bounds__(NT > 256 ? NT : 256) row_kernel(const Args a) {
    constexpr int UE = 16 / sizeof(T), CT = NT > 256 ? NT : 256, RPC = CT / NT, WPR = NT / 32;
    __shared__ float s_sum[2][CT / 32], s_top[2][CT / 32];
    const int tid = threadIdx.x % NT, lane = threadIdx.x & 31, warp = threadIdx.x / 32, units = a.d / UE;
    pdl_launch_dependents();
    pdl_wait();
    float w[NV][UE];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int u = tid + v * NT;
#pragma unroll
        for (int e = 0; e < UE; e += 4) {
            const float4 f = u < units ? __ldg(reinterpret_cast<const float4 *>(a.w + (long)u * UE + e)) : make_float4(0.f, 0.f, 0.f, 0.f);
            w[v][e] = f.x, w[v][e + 1] = f.y, w[v][e + 2] = f.z, w[v][e + 3] = f.w;
        }
    }
    int buf = 0;
    for (long r0 = (long)blockIdx.x * RPC; r0 < a.rows; r0 += (long)gridDim.x * RPC, buf ^= 1) {
        const long r = r0 + threadIdx.x / NT;
        const bool live = r < a.rows;
        uint4 xv[NV], rv[NV];
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int u = tid + v * NT;
            const bool on = live && u < units;
            xv[v] = on ? *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.x) + r * a.ldx + (long)u * UE) : make_uint4(0, 0, 0, 0);
            if (a.res) rv[v] = on ? *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.res) + r * a.ldr + (long)u * UE) : make_uint4(0, 0, 0, 0);
        }
        float t[NV][UE], ss = 0.f, top = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            T *h = reinterpret_cast<T *>(&xv[v]);
            const T *o = reinterpret_cast<const T *>(&rv[v]);
            const int u = tid + v * NT;
            if (a.res) {
#pragma unroll
                for (int e = 0; e < UE; ++e) h[e] = add_t(h[e], o[e]);
                if (a.out && live && u < units)
                    *reinterpret_cast<uint4 *>(static_cast<T *>(a.out) + r * a.ldo + (long)u * UE) = xv[v];
            }
#pragma unroll
            for (int e = 0; e < UE; ++e) {
                const float f = to_f(h[e]);
                ss = fmaf(f, f, ss);
                t[v][e] = __fmul_rn(f, w[v][e]);
                if (a.group == 0) top = fmaxf(top, mag(t[v][e]));
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            ss += __shfl_xor_sync(0xffffffffu, ss, o);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        }
        if constexpr (WPR > 1) {
            if (lane == 0) s_sum[buf][warp] = ss, s_top[buf][warp] = top;
            __syncthreads();      // the other buffer is written next, so one barrier a row is enough
            const int w0 = warp / WPR * WPR;
            ss = 0.f, top = 0.f;
#pragma unroll
            for (int i = 0; i < WPR; ++i) ss += s_sum[buf][w0 + i], top = fmaxf(top, s_top[buf][w0 + i]);
        }
        const float rstd = 1.f / sqrtf(ss / (float)a.d + a.eps);
        if (a.group == 0 && live && tid == 0) a.scales[r] = scale_of(top, rstd);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int u = tid + v * NT;
            float gt = top;
            if (a.group) {        // group / UE neighbouring lanes
                gt = 0.f;
#pragma unroll
                for (int e = 0; e < UE; ++e) gt = fmaxf(gt, mag(t[v][e]));
                const int lg = a.group / UE;
                for (int o = 1; o < lg; o <<= 1) gt = fmaxf(gt, __shfl_xor_sync(0xffffffffu, gt, o));
                if (live && u < units && lane % lg == 0) a.scales[r * (a.d / a.group) + (long)u * UE / a.group] = scale_of(gt, rstd);
            }
            const float inv = inv_of(gt);
            uint32_t c[UE / 4];
#pragma unroll
            for (int e = 0; e < UE; e += 4) {
                c[e / 4] = (uint32_t)(code_of(t[v][e], inv) & 255) | (uint32_t)(code_of(t[v][e + 1], inv) & 255) << 8 |
                           (uint32_t)(code_of(t[v][e + 2], inv) & 255) << 16 | (uint32_t)(code_of(t[v][e + 3], inv) & 255) << 24;
            }
            if (live && u < units) {
                int8_t *p = a.q + r * a.ldq + (long)u * UE;
                if constexpr (UE == 4) *reinterpret_cast<uint32_t *>(p) = c[0];
                else *reinterpret_cast<uint2 *>(p) = make_uint2(c[0], c[1]);
            }
        }
    }
}

// Any width, alignment and pitch: one CTA per row, element by element, three
// walks over the row (the later ones from cache).  A warp takes 128 neighbouring
// elements at a time, lane + 32 j, so groups lie within one.  Two to four times row_kernel's time (a row of 2048 4.1 us,
// 16384 rows of 4096 300 us), and only for rows that it cannot take: other alignments and pitches, and rows past its registers (fp32
// from 8192 elements, fp16 from 16384).
template <typename T>
__global__ void __launch_bounds__(256) any_kernel(const Args a) {
    __shared__ float s_sum[8], s_top[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    pdl_launch_dependents();
    pdl_wait();
    for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + r * a.ldx;
        const T *res = a.res ? static_cast<const T *>(a.res) + r * a.ldr : nullptr;
        T *out = a.res && a.out ? static_cast<T *>(a.out) + r * a.ldo : nullptr;
        float ss = 0.f, top = 0.f;
        for (int e = warp * 32 + lane; e < a.d; e += 256) {
            const T h = res ? add_t(x[e], res[e]) : x[e];
            const float f = to_f(h);
            ss = fmaf(f, f, ss);
            top = fmaxf(top, mag(__fmul_rn(f, a.w[e])));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            ss += __shfl_xor_sync(0xffffffffu, ss, o);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        }
        __syncthreads();          // the previous row's readers are done
        if (lane == 0) s_sum[warp] = ss, s_top[warp] = top;
        __syncthreads();
        ss = 0.f, top = 0.f;
        for (int i = 0; i < 8; ++i) ss += s_sum[i], top = fmaxf(top, s_top[i]);
        const float rstd = 1.f / sqrtf(ss / (float)a.d + a.eps);
        if (a.group == 0 && threadIdx.x == 0) a.scales[r] = scale_of(top, rstd);
        for (int e0 = warp * 128; e0 < a.d; e0 += 8 * 128) {
            float t[4], gt[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int e = e0 + 32 * j + lane;
                t[j] = 0.f;
                if (e < a.d) {
                    const T h = res ? add_t(x[e], res[e]) : x[e];
                    if (out) out[e] = h;     // last use of x[e] and res[e], which out may be
                    t[j] = __fmul_rn(to_f(h), a.w[e]);
                }
                gt[j] = mag(t[j]);
            }
            if (a.group) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) gt[j] = fmaxf(gt[j], __shfl_xor_sync(0xffffffffu, gt[j], o));
                if (a.group >= 64) gt[0] = gt[1] = fmaxf(gt[0], gt[1]), gt[2] = gt[3] = fmaxf(gt[2], gt[3]);
                if (a.group == 128) gt[0] = gt[1] = gt[2] = gt[3] = fmaxf(gt[0], gt[2]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int e = e0 + 32 * j + lane;
                if (e >= a.d) continue;
                const float m = a.group ? gt[j] : top;
                a.q[r * a.ldq + e] = (int8_t)code_of(t[j], inv_of(m));
                if (a.group && e % a.group == 0) a.scales[r * (a.d / a.group) + e / a.group] = scale_of(m, rstd);
            }
        }
    }
}

template <typename T, int NV, int NT>
static int launch_row(DevCtx *c, const Args &a, cudaStream_t s) {
    constexpr int CT = NT > 256 ? NT : 256, RPC = CT / NT;
    const long need = (a.rows + RPC - 1) / RPC;
    const int grid = (int)std::min<long>(need, (long)c->sm_count * (2048 / CT));
    return launch_pdl(row_kernel<T, NV, NT>, dim3(grid), dim3(CT), 0, s, a);
}

template <typename T>
static int launch(DevCtx *c, const Args &a, cudaStream_t s) {
    constexpr int UE = 16 / sizeof(T), QA = UE == 4 ? 4 : 8;
    const auto al = [](const void *p, int n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
    const int units = a.d / UE;
    const bool vec = a.d % UE == 0 && units <= 2048 && al(a.x, 16) && a.ldx % UE == 0 && al(a.w, 16) && al(a.q, QA) && a.ldq % QA == 0 &&
                     (!a.res || (al(a.res, 16) && a.ldr % UE == 0)) && (!a.res || !a.out || (al(a.out, 16) && a.ldo % UE == 0));
    if (!vec) {
        const int grid = (int)std::min<long>(a.rows, (long)c->sm_count * 8);
        return launch_pdl(any_kernel<T>, dim3(grid), dim3(256), 0, s, a);
    }
    // two units per thread while that fills a CTA of up to 512 threads, then four
    if (units <= 64) return launch_row<T, 2, 32>(c, a, s);
    if (units <= 128) return launch_row<T, 2, 64>(c, a, s);
    if (units <= 256) return launch_row<T, 2, 128>(c, a, s);
    if (units <= 512) return launch_row<T, 2, 256>(c, a, s);
    if (units <= 1024) return launch_row<T, 2, 512>(c, a, s);
    return launch_row<T, 4, 512>(c, a, s);
}

}  // namespace normq8
}  // namespace x100

using namespace x100;

extern "C" int x100q_add_rmsnorm_q8_dev(const x100q_norm_q8_args *a, void *stream) {
    auto refuse = [](int code) {
        set_error(code);
        return code;
    };
    set_error(X100_OK);
    if (!a || a->rows < 0 || a->d < 1) return refuse(X100_E_ARG);
    if (a->rows == 0) return X100_OK;
    if (a->dtype != X100Q_F32 && a->dtype != X100Q_F16) return refuse(X100_E_UNSUPPORTED);
    const int es = a->dtype == X100Q_F32 ? 4 : 2;
    const auto al = [es](const void *p) { return reinterpret_cast<uintptr_t>(p) % es == 0; };
    if (!a->x || !a->w || !a->q || !a->scales || !(a->eps > 0.f) || a->ldx < a->d || a->ldq < a->d || !al(a->x) || !al(a->residual) ||
        !al(a->residual_out) || (a->residual && a->ldr < a->d) || (a->residual && a->residual_out && a->ldo < a->d) ||
        (!a->residual && a->residual_out) || reinterpret_cast<uintptr_t>(a->w) % 4 || reinterpret_cast<uintptr_t>(a->scales) % 4)
        return refuse(X100_E_ARG);
    // in place row for row: with another pitch one row's sum would be another row's input
    if (a->rows > 1 && a->residual_out && ((a->residual_out == a->x && a->ldo != a->ldx) || (a->residual_out == a->residual && a->ldo != a->ldr)))
        return refuse(X100_E_ARG);
    if (a->group != 0 && ((a->group != 32 && a->group != 64 && a->group != 128) || a->d % a->group)) return refuse(X100_E_ARG);
    DevCtx *c = ctx();
    if (!c) return get_error();
    normq8::Args p = {a->x, a->residual, a->residual_out, a->ldx, a->ldr, a->ldo, a->ldq, a->w, a->eps, a->rows, a->d, a->group, a->q, a->scales};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return a->dtype == X100Q_F32 ? normq8::launch<float>(c, p, s) : normq8::launch<__half>(c, p, s);
}
