// kv4_attn.cuh -- what the attention kernels over the 4-bit KV cache share: the
// call's arguments, the work list and the exact fp16 forms of the codes.
#pragma once
#include "kv4.cuh"
#include "ptx.cuh"
#include "qformats.cuh"
#include "qgemv.h"

namespace x100 {
namespace kv4 {

using q::pdl_launch_dependents;
using q::pdl_wait;

constexpr int kMaxCtas = 320;           // bound of the grid, which sizes the workspace

struct AttnArgs {
    Pool pool;
    Table tab;
    const void *q;
    void *out;
    long qs, os;
    const int *q_start, *kv_len;
    // the model's calls: sequence b reads row row_of[b] < n_rows of the page table (null: row b) and has
    // kv_len[b] + len_add positions, none where kv_len[b] is negative
    const int *row_of = nullptr;
    int n_rows = 0, len_add = 0;
    int nrt_max;                         // row tiles of a sequence of max_q tokens (clusters)
    int n_tokens, max_q, nh, G;
    uint32_t g_mul;                      // ceil(2^32 / G): n / G = umulhi(n, g_mul) for n < 2^32 / G
    int unit_shift;                      // positions per unit, a power of two (128 unless the list would pass 2^31 units)
    int lead;                            // units that an item counts for besides its positions' (see kv4_attn.cu)
    float sl;                            // scale * log2(e) / q_up
    float q_up;                          // power of two that fp32 q is multiplied with before it is split (attn_shape)
    // work: of the first (slot 0) and last (slot 1) item that a run has a part of only
    float *part;                         // [kMaxCtas][2][8 NR * D] o in fragment order
    float2 *ml;                          // [kMaxCtas][2][8 NR] running max (log2 units) and sum
    int4 *meta;                          // [kMaxCtas][2] the item: first unit, sequence, kv head (kv4_attn.cu: | its last run << 16), row tile | kInside; or -1
    int *status;
};

constexpr int kInside = 1 << 30;         // the run starts inside the item

// Row number over the group's heads: rows of a sequence are at most 2^20 and G 4096 (the host checks), and the rounding of
// g_mul, under 1 in 2^32 / G, reaches a quotient only from 2^32 / G on.
__device__ __forceinline__ int div_g(const AttnArgs &a, int n) { return a.G == 1 ? n : (int)__umulhi((uint32_t)n, a.g_mul); }

// ---- the work list -------------------------------------------------------------
// Sequence b: first row of q, tokens, positions; `cu` units of positions in every (kv head, row
// tile) item, at least one so that rows without positions are written.
constexpr int kMostPositions = 0x7fffff00;      // a tile past it still is an int
struct Seq {
    int q0, nq, len, nrt, cu, row;       // row: of the page table
    uint32_t units;                      // of all its items, each cu + lead
};
// Rows q0 .. q0 + nq - 1 of sequence b; false (and none) where they are not the call's.
__device__ __forceinline__ bool load_rows(const AttnArgs &a, int b, int &q0, int &nq) {
    q0 = a.q_start ? a.q_start[b] : b;
    nq = a.q_start ? a.q_start[b + 1] - q0 : 1;
    const bool bad = q0 < 0 || nq < 0 || nq > a.max_q || q0 > a.n_tokens - nq;
    if (bad) nq = 0;
    return !bad;
}
// The arrays are read more than once in a call.  Should they change meanwhile (a caller's mistake) results mean nothing, but
// the walks end with the list, and what is read and written stays in the call's tensors.
__device__ __forceinline__ Seq load_seq(const AttnArgs &a, int b, int R, bool report) {
    Seq s;
    const bool bad_q = !load_rows(a, b, s.q0, s.nq);
    s.len = a.kv_len[b];
    if (a.len_add) s.len = s.len < 0 ? 0 : (int)((unsigned)s.len + a.len_add);   // a position; any below 0 is padding
    s.row = a.row_of ? a.row_of[b] : b;
    if (a.row_of && (unsigned)s.row >= (unsigned)a.n_rows) s.row = 0, s.len = s.len ? -1 : 0;
    const int cover = min(a.tab.stride, kMostPositions >> a.pool.page_shift) << a.pool.page_shift;
    if (bad_q || s.len < 0 || s.len > cover) {
        if (report) atomicCAS(a.status, 0, X100_E_ARG);
        s.len = s.len < 0 ? 0 : min(s.len, cover);
    }
    s.nrt = (int)((unsigned)(s.nq * a.G + R - 1) / (unsigned)R);
    s.cu = max(1, (s.len >> a.unit_shift) + ((s.len & ((1 << a.unit_shift) - 1)) != 0));
    s.units = (uint32_t)a.pool.nkv * s.nrt * (s.cu + a.lead);
    return s;
}
// ---- values ---------------------------------------------------------------------
__device__ __forceinline__ uint32_t u32(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ __half2 h2(uint32_t u) { return *reinterpret_cast<__half2 *>(&u); }
// Codes of both halves of a word as fp16 by placing them under an exponent:
// bits 0-3 under 1024's read as 1024 + code, bits 4-7 as 1024 + 16 code (the int4 to fp16 conversion of Kim et al., "Who Says
// Elephants Can't Run: Bringing Large Scale MoE Models into Cloud Scale Production", 2022).  The exponent comes in a register that the
// compiler cannot see through: with it as an immediate each (w & mask) | exponent
// would be two instructions instead of one.
struct Exponents {
    uint32_t e1024;
    __device__ Exponents() { asm volatile("mov.b32 %0, 0x64006400;" : "=r"(e1024)); }
};
__device__ __forceinline__ uint32_t field(uint32_t w, uint32_t mask, uint32_t expo) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(expo));
    return r;
}
constexpr uint32_t kLow = 0x000f000fu, kHigh = 0x00f000f0u;
// code - 8, exactly
__device__ __forceinline__ __half2 low_codes(uint32_t w, const Exponents &x) {
    return __hsub2(h2(field(w, kLow, x.e1024)), __float2half2_rn(1032.f));
}
__device__ __forceinline__ __half2 high_codes(uint32_t w, const Exponents &x) {
    return __hfma2(h2(field(w, kHigh, x.e1024)), __float2half2_rn(0.0625f), __float2half2_rn(-72.f));
}
// 2^x: x <= 8 here; results under 2^-126 are zeros
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The running maximum m of a row follows only when a score passes it by 2^kLag, so that its sums are rarely rescaled, and a
// probability is held as 2^(score - m + kUp), at most 2^15.  fp16 then has 11 bits of those down to 2^-25 of the row's largest and
// hi + lo halves 22 bits down to 2^-14 of it; smaller ones are known to 2^-36 of it (without the factor 2^kUp, to 2^-25: a long
// flat tail 17 nats under one position lost up to 3 % of itself).  A lag of 8 with kUp = 7 is 2 % faster for fp16 prompts (397
// against 405 us for 4096 tokens over 8192 positions) and the same elsewhere; 2 and 1 cost them 9 and 15 %.
constexpr float kLag = 4.f, kUp = 11.f;

// x = hi + lo: 22 bits from 2^-3 up, and to 2^-25 below.  q is brought near the size that it has with a scale of head_dim^-0.5 first
// (attn_shape), so that 2^-25 of it is as little of a score whatever the scale.
__device__ __forceinline__ void split2(float x, float y, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    hi = u32(h);
    lo = u32(__floats2half2_rn(x - f.x, y - f.y));
}

// Prompt chunks on the 5th-generation tensor cores (kv4_prefill.cu): taken when a
// sequence may have this many query rows.
constexpr long kPrefillRows = 256;
size_t prefill_work(int head_dim);
bool prefill_fits(const AttnArgs &a, int dtype);   // its units can be counted in 32 bits, whatever q_start and kv_len hold
int launch_prefill(DevCtx *c, AttnArgs &a, int dtype, int head_dim, cudaStream_t s);

// n_heads, G and the scale; then the call, its arguments checked (kv4_attn.cu).
void attn_shape(AttnArgs &p, int n_heads, float scale, int dtype, int head_dim);
int launch_attention(DevCtx *c, AttnArgs &p, int dtype, int head_dim, cudaStream_t s);

}  // namespace kv4
}  // namespace x100
