// The paged 4-bit cache: where a token lives and how a tile is laid out.
//
// Of a sequence of L tokens the first w_sink and the last w_recent ..
// w_recent + 31 are held in the dtype in the sequence's slot, the ones between
// in 4-bit tiles of 32 tokens (symmetric codes, groups of 32: keys over
// channels, values over tokens).  Everything follows from L alone, so the
// kernels need no state but the lengths:
//   n_packed(L) = max(0, L - w_sink - w_recent) / 32 * 32
//   t < w_sink                       row t of the slot
//   t - w_sink < n_packed(L)         tile (t - w_sink) / 32 of the pages
//   else                             row w_sink + (t - w_sink) % (w_recent + 32)
//
// One tile of one head is one block of 4608 contiguous bytes (codes and scales
// of both sides), so a consumer fetches it, and the tiles after it in the same
// page, with a single bulk copy:
//   0     K codes   32-bit words [j 4][i 8][l 4][g 4]; nibble n: token 8j + i,
//                   channel 32g + 8l + n
//   2048  K scales  [i 8][j 4][g 4]
//   2304  V codes   32-bit words [p 4][i 8][l 4][m 2][h 2]; nibble n: channel
//                   16i + 4p + 2m + h, token 8 (n & 3) + 2l + (n >> 2)
//   4352  V scales  [channel 128]
// A lane (i = lane / 4, l = lane % 4) of the attention finds its words in four
// 16-byte pieces per side, piece-major, so that a warp's 128-bit loads of a
// piece cover 512 contiguous bytes.  Codes are stored offset-binary (c + 8).
#pragma once
#include "../../include/innerq_b200.h"
#include "common.cuh"

namespace innerq {

constexpr int kBlockBytes = 4608;
constexpr int kKScale = 2048, kVCodes = 2304, kVScale = 4352;

struct PagedDev {
  uint8_t* pages;
  uint16_t* dk;
  uint16_t* dv;
  const int32_t* table;
  const int32_t* slots;
  const int32_t* lens;
  int64_t table_stride;
  int B, Hkv, page_tiles, n_pages, n_slots, w_sink, w_recent, max_pages;

  __device__ __forceinline__ int n_packed(int len) const {
    return max(0, len - w_sink - w_recent) & ~31;
  }
  __device__ __forceinline__ int ring() const { return w_recent + 32; }
  __device__ __forceinline__ int dense_rows() const { return w_sink + w_recent + 32; }
  __device__ __forceinline__ int row_of(int t) const {
    return t < w_sink ? t : w_sink + (t - w_sink) % ring();
  }
  // first row of (slot of sequence b, head h), in elements; -1: no such slot
  __device__ __forceinline__ int64_t dense_base(int b, int h) const {
    const int s = slots[b];
    if ((unsigned)s >= (unsigned)n_slots) return -1;
    return ((int64_t)s * Hkv + h) * dense_rows() * kD;
  }
  // block of packed tile `tile` of sequence b, head h; null where the page
  // table has no such page (the caller answers NaN or drops the write)
  __device__ __forceinline__ uint8_t* tile(int b, int h, int tile) const {
    const int pg = tile / page_tiles;
    if (pg >= max_pages) return nullptr;
    const int id = table[b * table_stride + pg];
    if ((unsigned)id >= (unsigned)n_pages) return nullptr;
    return pages + (((int64_t)id * Hkv + h) * page_tiles + (tile - pg * page_tiles)) * (int64_t)kBlockBytes;
  }
};

// Checks the cache description and fills the kernels' form of it.
int paged_dev(const innerq_paged* c, PagedDev& d);

}  // namespace innerq
