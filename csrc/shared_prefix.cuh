// Attention of many continuations of one prompt: how the work over the prompts' keys is laid out.  Both kernels go by it.
//
// A unit is (prompt b, key head, row tile): up to 128 query rows, wt continuations times the query heads of the key head.  Its keys come in
// tiles of 128.  The tiles of all units, one after the other, are dealt out to the CTAs in equal ranges, so that every SM has the same
// share whatever the lengths of the prompts; a CTA leaves one partial result for every unit that its range meets.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace kf {
namespace shared_prefix {

constexpr int TILE_KEYS = 128, TILE_ROWS = 128;

struct Layout {
  const int* lens;     // keys of each prompt, or null: P for all
  int B, W, P;
  int per_prompt;      // units of a prompt: key heads x row tiles
  int row_tiles, wt;   // row tiles of a key head, continuations per row tile
  int ctas;
};

__host__ __device__ __forceinline__ int tiles_of(int len) { return (len + TILE_KEYS - 1) / TILE_KEYS; }
__device__ __forceinline__ int length(const Layout& l, int b) { return l.lens ? min(max(l.lens[b], 0), l.P) : l.P; }

// CTAs that have work: with fewer tiles than CTAs one tile each, so that no CTA between two others has none.
__device__ __forceinline__ int working(const Layout& l, long long total) { return total < l.ctas ? int(total) : l.ctas; }
// First tile of the range of one of `ctas` CTAs that all have work; the ranges follow one another.
__device__ __forceinline__ long long range_begin(long long total, int cta, int ctas) { return total * cta / ctas; }
// The CTA whose range holds tile t: the last one with range_begin <= t.
__device__ __forceinline__ int cta_of(long long total, long long t, int ctas) { return int(((t + 1) * ctas - 1) / total); }

// Tiles of the prompts before b (all: b = B), by one warp; every lane has the result.
__device__ __forceinline__ long long tiles_before(const Layout& l, int b) {
  if (!l.lens) return (long long)tiles_of(l.P) * l.per_prompt * b;
  long long n = 0;
  for (int i = threadIdx.x & 31; i < b; i += 32) n += tiles_of(length(l, i));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  return n * l.per_prompt;
}

// A partial result of unit u by CTA c lies in slot u + c: along the tiles every step raises one of the two, so no two share one.
__host__ __device__ __forceinline__ long long slots(const Layout& l) { return (long long)l.B * l.per_prompt + l.ctas; }

}  // namespace shared_prefix
}  // namespace kf
