// kv4.cuh -- the paged 4-bit KV cache: tile layout, host-side argument checks
// and the launchers shared by the x100q_kv4_* entry points and the model.
//
// Layout of a tile (16 positions of one kv head, D = head_dim, NB = D / 32;
// include/x100q.h): K codes, V codes, K scales, V scales.  The places are the
// lanes' own: in the attention kernels lane 4 g + t of a warp reads the K
// words of one position (blocks 0 .. NB - 1, its 8 dims of each) with one load, and
// the V codes of 4 positions x D / 8 dims with 16-byte loads at lane * 16, all without
// shared-memory bank conflicts and already in mma.sync fragment order.
#pragma once
#include <cuda_fp16.h>

#include "../../include/x100q.h"
#include "runtime.h"

namespace x100 {
namespace kv4 {

constexpr int kTile = 16;          // positions per tile
constexpr float kTinyBlock = 7.8886090522101181e-31f;   // 2^-100
constexpr float kMostScale = 8160.f;                    // 255 * 32: 8 * scale is the largest fp16 value of 8 bits

template <int D>
struct Lay {
    static constexpr int NB = D / 32;            // blocks of 32 per head
    static constexpr int R = D == 128 ? 2 : 4;   // V pieces of one lane that share 16 bytes
    static constexpr int PB = D / 16;            // bytes of a V piece (D / 8 codes)
    static constexpr int KROW = D / 2;           // bytes of a K row
    static constexpr int V0 = 8 * D, KS0 = 16 * D, VS0 = 17 * D, BYTES = 18 * D;
    // byte of the V piece of dims g * D / 8 .. at position s of the tile
    static __host__ __device__ constexpr int v_piece(int s, int g) {
        return V0 + (((s >> 2) / R * 8 + g) * 4 + (s & 3)) * 16 + (s >> 2) % R * PB;
    }
    // byte of the K word of block b, dims 8 t .. 8 t + 7 of it, at position s
    static __host__ __device__ constexpr int k_word(int s, int b, int t) { return s * KROW + (t * NB + b) * 4; }
    static __host__ __device__ constexpr int k_scale(int s, int b) { return KS0 + (s * NB + b) * 2; }
    static __host__ __device__ constexpr int v_scale(int s, int b) { return VS0 + ((b * 4 + (s & 3)) * 4 + (s >> 2)) * 2; }
};

// Page pool and table as the kernels take them.
struct Pool {
    uint8_t *pages;
    long page_bytes;               // bytes of one kv head of a page
    int n_pages, page_shift, nkv;  // page_size = 1 << page_shift
};
struct Table {
    const int *page;               // [n_seqs][stride]
    int stride, n_seqs;
};

inline bool shape_ok(const x100q_kv4 *kv) {
    return kv && kv->n_pages > 0 && kv->n_kv_heads > 0 && kv->n_kv_heads <= 256 &&
           (kv->head_dim == 64 || kv->head_dim == 128) &&
           (kv->page_size == 16 || kv->page_size == 32 || kv->page_size == 64 || kv->page_size == 128);
}
inline Pool make_pool(const x100q_kv4 *kv) {
    Pool p;
    p.pages = static_cast<uint8_t *>(kv->pages);
    p.page_bytes = (long)kv->page_size / kTile * 18 * kv->head_dim;
    p.n_pages = kv->n_pages;
    p.page_shift = kv->page_size == 16 ? 4 : kv->page_size == 32 ? 5 : kv->page_size == 64 ? 6 : 7;
    p.nkv = kv->n_kv_heads;
    return p;
}
inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// a row pitch in elements: whole 16 bytes, and rows do not overlap
inline bool pitch_ok(long stride, int width, int esize) { return stride >= width && stride * esize % 16 == 0; }
// an output may be its input itself, row for row: with another pitch one row's output would be another row's input
inline bool in_place_ok(const void *in, long stride, const void *out, long out_stride, int rows) {
    return in != out || stride == out_stride || rows < 2;
}

// Tile of position `pos` of sequence `seq` for kv head `h`, or nullptr when
// the table or the pool does not cover it.
__device__ __forceinline__ uint8_t *tile_of(const Pool &p, const Table &t, int seq, int pos, int h) {
    const int i = pos >> p.page_shift;
    if (seq < 0 || seq >= t.n_seqs || i >= t.stride) return nullptr;
    const int page = __ldg(t.page + (long)seq * t.stride + i);
    if (page < 0 || page >= p.n_pages) return nullptr;
    const int in = (pos & ((1 << p.page_shift) - 1)) >> 4, tiles = 1 << (p.page_shift - 4);
    return p.pages + ((long)page * p.nkv + h) * p.page_bytes + (p.page_bytes / tiles) * in;
}

}  // namespace kv4
}  // namespace x100
