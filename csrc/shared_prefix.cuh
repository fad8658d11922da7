// Attention of many continuations of one prompt: how the work over the prompts' keys is laid out.  Both kernels go by it.
//
// A unit is (prompt b, key head, one or two row tiles): a row tile is up to 128 query rows, wt continuations times the query heads of the
// key head, and with more rows than that two of them may share the keys.  Keys come in tiles of 128.  The tiles of all units, one after the
// other, are dealt out to the CTAs in equal ranges, so that every SM has the same share whatever the lengths of the prompts; a CTA leaves
// one partial result for every unit that its range meets.
//
// Without lens, and where that makes the ranges no more than SPARE tiles longer, a unit counts for a whole number of ranges: a CTA that ends a
// unit and begins another one has two results to write, 5800 cycles each, and waits for first keys twice.  Equal ranges / whole numbers, us:
// 2 x 30 x 8254 (32 heads on 8) 27.5 / 24.1, 6 x 16 x 1568 (16 on 4) 15.6 / 13.1, 4 x 3 x 6522 (40 on 8) 29.3 / 26.6, 2 x 64 x 8000 32.3 / 28.4.
//
// Which form a call takes, in this order (kf_shared_prefix_attn_bf16, launch_own, launch_hd):
//   prompts      the second kernel alone (is_direct): up to 4 MB times continuations, prompts of one tile up to 64;
//                else the first kernel, two row tiles a unit (make_layout) where a key head has over 128 rows and the prompts 168 MB or more;
//                else one row tile, LEAN up to three tiles a CTA, or with heads of 128, one row tile a key head and at most 128 own keys;
//                else one row tile with all scores in registers.
//   own keys     (launch_own; tiles of 16, the prompts' among them where this kernel is alone) rings of one, then of two tiles, with 1, 2 or 4
//                warps a unit, where these hold all tiles and no more warps come to an SM than fit at once;
//                else 1 to 32 warps a unit that stream, as many as fit, through 16 KB each where 8 to 12 come to an SM, else through 24.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace kf {
namespace shared_prefix {

constexpr int TILE_KEYS = 128, TILE_ROWS = 128;
constexpr int SPARE = 3;

struct Layout {
  const int* lens;     // keys of each prompt, or null: P for all
  int B, W, P;
  int per_prompt;      // units of a prompt: key heads x row_units
  int row_units;       // units of a key head
  int pair, wt;        // row tiles of a unit, 1 or 2; continuations per row tile
  int ctas, most;      // how many are launched; how many might be, whatever the lengths
  int span;            // without lens: tiles that a unit counts for
  int k_step, v_step;  // 0: all prompts have the first one's keys, or values
};

__host__ __device__ __forceinline__ int tiles_of(int len) { return (len + TILE_KEYS - 1) / TILE_KEYS; }
__device__ __forceinline__ int length(const Layout& l, int b) { return l.lens ? min(max(l.lens[b], 0), l.P) : l.P; }

// Tiles of a CTA's range: as few as cover all with the CTAs there are.  Counts of tiles have 32 bits (kf_shared_prefix_scratch), and
// CTAs without work are the last ones, so that none lies between two parts of a unit.
__device__ __forceinline__ uint32_t range(uint32_t total, int ctas) { return (total + ctas - 1) / ctas; }

// Tiles of the prompts before b (all: b = B), by one warp; every lane has the result.
__device__ __forceinline__ uint32_t tiles_before(const Layout& l, int b) {
  if (!l.lens) return uint32_t(l.span) * l.per_prompt * b;
  uint32_t n = 0;
  for (int i = threadIdx.x & 31; i < b; i += 32) n += tiles_of(length(l, i));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  return n * l.per_prompt;
}

// A partial result of unit u by CTA c lies in slot u + c: along the tiles every step raises one of the two, so no two share one.
__host__ __device__ __forceinline__ long long slots(const Layout& l) { return (long long)l.B * l.per_prompt + l.most; }

}  // namespace shared_prefix
}  // namespace kf
