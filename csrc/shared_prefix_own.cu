// Attention of the new tokens of many continuations over their own tokens, joined with what the prompt gave (second of two kernels).
//
// What a continuation has written itself is its own, so these keys are read by its group of query heads only: a stream as in the generation
// step of single sequences.  In a beam search the cache of a continuation does not move when beams are exchanged; own_rows says in whose
// cache each position lies.  Beams share most of their ancestors, so most of these keys come out of L2 for all beams but the first.
//   * a unit is a continuation's key head; its query heads are the 16 rows of an m16n8k16 MMA, its keys are dealt out to 1 to 32 warps:
//     few units need many warps for one, many (a batch of short continuations) one each;
//   * every warp streams tiles of 16 keys through a cp.async ring of its own, without a barrier; 16-byte chunks are
//     XOR-swizzled, so that ldmatrix is free of bank conflicts; a warp of one or two tiles has them all under way at once;
//   * the (max, sum, output) triples of the warps, of the CTAs of a cluster and of the prompt are joined in a fixed order.
// All of it up to that last step runs without the prompt's kernel, and starts on the SMs that it leaves (programmatic launch).
//
// Where the prompts are short, this kernel alone reads them too, for every continuation again (out of L2), as the tiles before those of its
// own: `direct`.  What that costs is traffic, what it saves a launch, the partial results and the wait between the kernels.
#include "decode_common.cuh"
#include "shared_prefix.cuh"

#include <type_traits>

namespace kf {
namespace shared_prefix {

using namespace kf::decode;

constexpr int OWN_WARPS = 4, OWN_THREADS = OWN_WARPS * 32;
constexpr int OWN_TILE = 16;       // keys per ring stage of a warp
constexpr int OWN_ROWS = 16;       // query heads per unit (MMA rows)

// RING_TILES: tiles in a warp's ring, up to which it has them all under way at once.  WIDE, NARROW: it streams through 24 KB (two CTAs an SM,
// 192 KB under way; refilled before a tile is worked on, with a stage less under way, it was 1 to 4 % slower) or 16 KB (three CTAs).
constexpr int WIDE = 0, NARROW = -1;
template <int HD, int RING_TILES>
struct OwnCfg {
  static constexpr int TILE_BYTES = OWN_TILE * HD * 2;
  static constexpr bool STREAM = RING_TILES <= 0;
  static constexpr int STAGES = STREAM ? ((RING_TILES == WIDE ? 24 : 16) << 10) / (2 * TILE_BYTES) : RING_TILES;   // of 128: 3 or 2
  static constexpr int RING = STAGES * 2 * TILE_BYTES;
  static constexpr int PART = OWN_ROWS * HD * 4;                     // a warp's partial output, over its ring
  static constexpr int STATS = OWN_ROWS * 2 * 4;                     // (max, sum) of its rows, behind it
  static constexpr int SEEN = STREAM ? OWN_WARPS * 8 * 4 : 0;        // per stage: which of its keys are visible
  static constexpr int WARP = RING > PART + STATS ? RING : PART + STATS;
  static constexpr size_t SMEM = size_t(OWN_WARPS) * WARP + SEEN;
};

struct Own {
  const __nv_bfloat16 *q, *k, *v;
  __nv_bfloat16* o;
  const uint8_t* rows;                                       // [B][W][S] or null
  int S, Hkv, group;
  const __nv_bfloat16 *pk, *pv;                              // the prompts, where they are read here
  int direct;
  long long pk_b, pk_s, pk_h, pv_b, pv_s, pv_h;
  long long q_b, q_w, q_h, k_b, k_w, k_s, k_h, v_b, v_w, v_s, v_h;   // elements
  long long r_b, r_w;
  float scale_log2;
};

// WPU: warps of a CTA that share a unit.  Clusters of more than one CTA (WPU = 4) share one too.
// Four CTAs an SM where all tiles are under way at once, which is 128 registers: heads of 128 with rings of two spill 172 to 212 bytes.  With three
// and 12, us: 1 x 8 x 4000 of 96 own 11.8 / 11.3, 8 x 5 x 1777 of 65 23.5 / 22.5, 24 x 8 x 512 of 200 24.8 / 24.9.
template <int HD, int WPU, int RING_TILES>
__global__ void __launch_bounds__(OWN_THREADS, RING_TILES <= 0 ? 3 : 4)
kf_shared_prefix_own(const Own a, const Layout lay, const float* part_o, const float2* part_ml, const uint32_t units) {
  using C = OwnCfg<HD, RING_TILES>;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  // Behind the prompt's kernel everything but its results is there at the start, because it has waited itself; alone nothing is.
  if (part_o == nullptr) {
    grid_dep_wait();
    grid_dep_launch();
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int splits = WPU == OWN_WARPS ? int(cluster_nctaid()) : 1, rank = WPU == OWN_WARPS ? int(cluster_ctarank()) : 0;
  const int way = rank * WPU + warp % WPU, ways = splits * WPU;     // which share of the unit's keys
  const uint32_t ring = smem_u32(smem_raw) + warp * C::WARP;
  volatile uint32_t* seen = reinterpret_cast<uint32_t*>(smem_raw + OWN_WARPS * C::WARP) + warp * 8;

  const uint32_t unit0 = blockIdx.x / uint32_t(splits) * (OWN_WARPS / WPU) + warp / WPU;
  const bool there = unit0 < units;
  uint32_t unit = there ? unit0 : 0u;
  uint32_t next = unit / lay.W;
  const int w = int(unit - next * lay.W);   // continuations of a prompt side by side: their common keys are in L2, some in L1
  unit = next;
  const uint32_t blocks_per_kv = (a.group + OWN_ROWS - 1) / OWN_ROWS;
  next = blocks_per_kv > 1 ? unit / blocks_per_kv : unit;
  const int hb = int(unit - next * blocks_per_kv);
  const int b = int(next / a.Hkv), hk = int(next - uint32_t(b) * a.Hkv);
  const int n_heads = there ? min(OWN_ROWS, a.group - hb * OWN_ROWS) : 0;     // query heads of this unit
  const int h0 = hk * a.group + hb * OWN_ROWS;

  const int plen = a.direct ? length(lay, b) : 0, prompt_tiles = (plen + OWN_TILE - 1) / OWN_TILE;
  const int n_tiles = there ? prompt_tiles + (a.S + OWN_TILE - 1) / OWN_TILE : 0;
  const int each = (n_tiles + ways - 1) / ways, t0 = min(n_tiles, each * way), t1 = min(n_tiles, t0 + each);
  const __nv_bfloat16* kb = a.k + b * a.k_b + hk * a.k_h;
  const __nv_bfloat16* vb = a.v + b * a.v_b + hk * a.v_h;
  const __nv_bfloat16 *pkb = a.pk + b * a.pk_b + hk * a.pk_h, *pvb = a.pv + b * a.pv_b + hk * a.pv_h;
  const uint8_t* table = a.rows ? a.rows + b * a.r_b + w * a.r_w : nullptr;

  // whose cache holds the lane's key of the two tiles from t on (-1: the prompt's, lay.W: nobody's)
  auto slots_of = [&](int t) {
    const int tile = t + (lane >> 4), pos = t * OWN_TILE + lane, own = pos - prompt_tiles * OWN_TILE;
    if (tile >= t1) return lay.W;
    if (tile < prompt_tiles) return pos < plen ? -1 : lay.W;
    return own >= a.S ? lay.W : table ? int(table[own]) : w;
  };
  int slots = slots_of(t0), ahead = t0 + 2 < t1 ? slots_of(t0 + 2) : lay.W;   // of the tiles issued next and the two after them
  // Four lanes a key: 64 bytes side by side at a time, of keys lane / 4 and that + 8.  The 16-byte chunk c of row r lies at c ^ (r & 7).
  const int row0 = lane >> 2;
  const uint32_t dst0 = uint32_t(row0 * HD * 2 + (((lane & 3) ^ row0) << 4));   // bit 6 of it turned over by row0's bit 2
  uint32_t masks[C::STREAM ? 1 : C::STAGES];
  auto issue = [&](int t) {
    const int st = (t - t0) % C::STAGES, half = ((t - t0) & 1) * 16;
    const uint32_t ks = ring + uint32_t(st) * 2u * C::TILE_BYTES, vs = ks + C::TILE_BYTES;
    const uint32_t mask = __ballot_sync(0xffffffffu, slots < lay.W) >> half;
    if (!C::STREAM) masks[st % (C::STREAM ? 1 : C::STAGES)] = mask;
    else if (lane == 0) seen[st] = mask;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = row0 + h * 8, sl = __shfl_sync(0xffffffffu, slots, half + r);
      const bool in = (mask >> r) & 1u;
      const bool prompt = t < prompt_tiles;   // of the whole tile, so that a hidden key's address is in the same tensor
      const long long of = in ? sl : 0, pos = in ? (t - (prompt ? 0 : prompt_tiles)) * OWN_TILE + r : 0;
      const __nv_bfloat16* kp = (prompt ? pkb + pos * a.pk_s : kb + of * a.k_w + pos * a.k_s) + (lane & 3) * 8;
      const __nv_bfloat16* vp = (prompt ? pvb + pos * a.pv_s : vb + of * a.v_w + pos * a.v_s) + (lane & 3) * 8;
#pragma unroll
      for (int c = 0; c < HD / 32; ++c) {
        const uint32_t dst = (dst0 ^ uint32_t(c * 64)) + uint32_t(h * 8 * HD * 2);
        cp_async16(ks + dst, kp + c * 32, in);
        cp_async16(vs + dst, vp + c * 32, in);
      }
    }
    if (half) {
      slots = ahead;
      ahead = t + 3 < t1 ? slots_of(t + 3) : lay.W;
    }
  };
  // query rows as MMA A fragments (rows past the group are zero)
  uint32_t qa[HD / 16][4];
  {
    const int g = lane >> 2, c = (lane & 3) * 2;
    const __nv_bfloat16* q0 = a.q + b * a.q_b + w * a.q_w + (h0 + g) * a.q_h;
    const __nv_bfloat16* q1 = q0 + 8 * a.q_h;
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk) {
      qa[kk][0] = g < n_heads ? *reinterpret_cast<const uint32_t*>(q0 + kk * 16 + c) : 0u;
      qa[kk][1] = g + 8 < n_heads ? *reinterpret_cast<const uint32_t*>(q1 + kk * 16 + c) : 0u;
      qa[kk][2] = g < n_heads ? *reinterpret_cast<const uint32_t*>(q0 + kk * 16 + 8 + c) : 0u;
      qa[kk][3] = g + 8 < n_heads ? *reinterpret_cast<const uint32_t*>(q1 + kk * 16 + 8 + c) : 0u;
    }
  }
#pragma unroll
  for (int i = 0; i < C::STAGES; ++i) {
    if (t0 + i < t1) issue(t0 + i);
    cp_commit();
  }

  float o[HD / 8][4];
#pragma unroll
  for (int i = 0; i < HD / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

#pragma unroll(C::STREAM ? 1 : C::STAGES)
  for (int i = 0; i < (C::STREAM ? t1 - t0 : C::STAGES); ++i) {
    const int t = t0 + i;
    if (t >= t1) break;
    cp_wait<C::STREAM ? C::STAGES - 1 : 0>();
    __syncwarp();   // tile t has landed for every lane
    const int st = C::STREAM ? i % C::STAGES : i;
    const uint32_t ks = ring + uint32_t(st) * 2u * C::TILE_BYTES, vs = ks + C::TILE_BYTES;
    const int mi = lane >> 3, lr = lane & 7;
    float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    {
      const uint32_t row = ks + uint32_t((lr + (mi >> 1) * 8) * HD * 2);
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk) {
        uint32_t f[4];
        ldsm4(row + uint32_t(((kk * 2 + (mi & 1)) ^ lr) << 4), f);
        mma16816(s[0], qa[kk], f[0], f[1]);
        mma16816(s[1], qa[kk], f[2], f[3]);
      }
    }
    // Rounded by itself, so that the largest is its own maximum: fused with the difference below, a product of over 2^31 would be off from the
    // maximum by its rounding, more than an exponent holds.
    const uint32_t sees = (C::STREAM ? seen[st] : masks[st % (C::STREAM ? 1 : C::STAGES)]) >> ((lane & 3) * 2);
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = (sees >> (n * 8 + (e & 1))) & 1u ? __fmul_rn(s[n][e], a.scale_log2) : -INFINITY;
    uint32_t pa[4];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      float mx = fmaxf(fmaxf(s[0][2 * hf], s[0][2 * hf + 1]), fmaxf(s[1][2 * hf], s[1][2 * hf + 1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float mn = fmaxf(m[hf], mx);
      const float base = mn == -INFINITY ? 0.f : mn;
      const float alpha = weight(m[hf], base);
      m[hf] = mn;
      float p[2][2], sum = 0.f;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          p[n][e] = fast_exp2(s[n][2 * hf + e] - base);
          sum += p[n][e];
        }
      l[hf] = l[hf] * alpha + sum;  // this thread's four keys; the quad is summed at the end
      // Weights are rounded to bf16 for the second product, the only form in which the tensor cores take them beside values in bf16; their sum is
      // of the unrounded ones.  At most 2^-8 of a weight, up or down, where the result is rounded by as much once.
      pa[hf] = pack_bf16(p[0][0], p[0][1]);
      pa[2 + hf] = pack_bf16(p[1][0], p[1][1]);
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) {
        o[i][2 * hf] *= alpha;
        o[i][2 * hf + 1] *= alpha;
      }
    }
    {
      const uint32_t row = vs + uint32_t((lr + (mi & 1) * 8) * HD * 2);
#pragma unroll
      for (int d = 0; d < HD / 16; ++d) {
        uint32_t f[4];
        ldsm4_t(row + uint32_t(((d * 2 + (mi >> 1)) ^ lr) << 4), f);
        mma16816(o[2 * d], pa, f[0], f[1]);
        mma16816(o[2 * d + 1], pa, f[2], f[3]);
      }
    }
    if (C::STREAM) {
      __syncwarp();   // every lane has read the stage
      if (t + C::STAGES < t1) issue(t + C::STAGES);
      cp_commit();
    }
  }
  cp_wait<0>();
  __syncwarp();  // the ring is idle: the warp's partial result takes its place
  float *part = reinterpret_cast<float*>(smem_raw + warp * C::WARP), *stats = part + C::PART / 4;
#pragma unroll
  for (int hf = 0; hf < 2; ++hf) {
    l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 1);
    l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 2);
    const int r = (lane >> 2) + hf * 8;
    if (r < n_heads) {
      if ((lane & 3) == 0) {
        stats[r * 2] = m[hf];
        stats[r * 2 + 1] = l[hf];
      }
      float* dst = part + r * HD + (lane & 3) * 2;
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) *reinterpret_cast<float2*>(dst + i * 8) = make_float2(o[i][2 * hf], o[i][2 * hf + 1]);
    }
  }
  // ---- the prompt's partial results: which there are
  int c0 = 0, parts = 0;
  const int u = hk * lay.row_units + w / (lay.wt * lay.pair), slot_rows = TILE_ROWS * lay.pair;
  if (part_o != nullptr) {
    const uint32_t first = tiles_before(lay, b), chunk = range(tiles_before(lay, lay.B), lay.ctas);
    const int nt = there ? tiles_of(length(lay, b)) : 0;
    if (nt > 0) {
      const uint32_t begin = first + uint32_t(u) * (lay.lens ? nt : lay.span);
      c0 = int(begin / chunk);
      parts = int((begin + nt - 1) / chunk) - c0 + 1;
    }
  }
  if (WPU == 1) __syncwarp();
  else if (splits == 1) __syncthreads();
  else cluster_sync_all();
  if (part_o != nullptr) {
    grid_dep_wait();
    grid_dep_launch();
  }
  const long long slot0 =
      ((long long)b * lay.per_prompt + u + c0) * slot_rows + (w / lay.wt % lay.pair) * TILE_ROWS + (w % lay.wt) * a.group + hb * OWN_ROWS;
  const int warp0 = warp / WPU * WPU;
  const uint32_t part_a = smem_u32(smem_raw) + warp0 * C::WARP, stats_a = part_a + C::PART;
  auto own_at = [&](uint32_t base, int s) {   // of the unit's s-th warp
    const uint32_t at = base + (s % WPU) * C::WARP;
    return splits > 1 ? mapa_shared(at, s / WPU) : at;
  };
  // ---- each warp of the unit its share of the output: a lane four values of a row, over the prompt's parts and the unit's warps; several
  // rows at once where a warp has several, with eight loads of parts under way
  constexpr int ITEMS = WPU == 1 ? 4 : WPU == 2 ? 2 : 1, AT_ONCE = 8 / ITEMS;
  const int n_items = n_heads * (HD / 4);
  for (int i0 = way * 32 + lane; i0 < n_items; i0 += ways * 32 * ITEMS) {
    float4 acc[ITEMS];
    float top[ITEMS], sum[ITEMS];
    float2 x[ITEMS][AT_ONCE];
    float4 v[ITEMS][AT_ONCE];
    int r[ITEMS], d[ITEMS];
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      const int i = min(i0 + j * ways * 32, n_items - 1);   // one too many is worked on with the others, and not written
      r[j] = i / (HD / 4), d[j] = (i % (HD / 4)) * 4;
      acc[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      top[j] = -INFINITY, sum[j] = 0.f;
    }
    auto join = [&](int n) {   // the first n of them
#pragma unroll
      for (int j = 0; j < ITEMS; ++j) {
        float higher = top[j];
#pragma unroll
        for (int e = 0; e < AT_ONCE; ++e)
          if (e < n) higher = fmaxf(higher, x[j][e].x);
        const float f = weight(top[j], higher);
        acc[j].x *= f; acc[j].y *= f; acc[j].z *= f; acc[j].w *= f;
        sum[j] *= f;
        top[j] = higher;
#pragma unroll
        for (int e = 0; e < AT_ONCE; ++e)
          if (e < n) {
            const float g = weight(x[j][e].x, higher);
            acc[j].x += g * v[j][e].x; acc[j].y += g * v[j][e].y; acc[j].z += g * v[j][e].z; acc[j].w += g * v[j][e].w;
            sum[j] += g * x[j][e].y;
          }
      }
    };
    for (int c = 0; c < parts; c += AT_ONCE) {
#pragma unroll
      for (int e = 0; e < AT_ONCE; ++e)
#pragma unroll
        for (int j = 0; j < ITEMS; ++j)
          if (c + e < parts) {
            const long long at = slot0 + r[j] + (long long)(c + e) * slot_rows;
            x[j][e] = ld_after_wait(part_ml + at);
            v[j][e] = ld_after_wait(reinterpret_cast<const float4*>(part_o + at * HD + d[j]));
          }
      join(parts - c);
    }
    for (int s = 0; s < ways; s += AT_ONCE) {
#pragma unroll
      for (int e = 0; e < AT_ONCE; ++e)
#pragma unroll
        for (int j = 0; j < ITEMS; ++j)
          if (s + e < ways) {
            const uint32_t at = own_at(stats_a + r[j] * 8, s + e);
            x[j][e] = make_float2(ld_cluster_f1(at), ld_cluster_f1(at + 4));
            v[j][e] = ld_cluster_f4(own_at(part_a + uint32_t(r[j] * HD + d[j]) * 4u, s + e));
          }
      join(ways - s);
    }
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      if (i0 + j * ways * 32 >= n_items) break;
      const float inv = sum[j] == 0.f ? 0.f : 1.f / sum[j];   // nothing visible: zeros
      uint2 out;
      out.x = pack_bf16(acc[j].x * inv, acc[j].y * inv);
      out.y = pack_bf16(acc[j].z * inv, acc[j].w * inv);
      *reinterpret_cast<uint2*>(a.o + (((long long)b * lay.W + w) * a.Hkv * a.group + h0 + r[j]) * HD + d[j]) = out;
    }
  }
  if (splits > 1) cluster_sync_all();   // no CTA leaves while another reads its shared memory
}

template <int HD, int WPU, int RING_TILES>
static int launch_ways(const Own& a, const Layout& l, const float* part_o, const float2* part_ml, long long units, int splits, cudaStream_t stream) {
  using C = OwnCfg<HD, RING_TILES>;
  auto kern = kf_shared_prefix_own<HD, WPU, RING_TILES>;
  static bool attr_set[16] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 16 || !attr_set[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM);
    // all of the SM's memory as shared memory: CTAs of both kernels side by side
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e != cudaSuccess) return 300 + (int)e;
    if (dev < 16) attr_set[dev] = true;
  }
  const int per_cta = OWN_WARPS / WPU;
  const long long ctas = (units + per_cta - 1) / per_cta * splits;
  if (ctas > 0x7fffffffLL) return 6;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(OWN_THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  cfg.numAttrs = 0;
  if (splits > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = (unsigned)splits;
    attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
  ++cfg.numAttrs;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a, l, part_o, part_ml, (uint32_t)units);
  return e == cudaSuccess ? 0 : 500 + (int)e;
}

template <int HD>
static int launch_own(const Own& a, const Layout& l, const float* part_o, const float2* part_ml, int num_sms, cudaStream_t stream) {
  const long long units = (long long)l.B * l.W * a.Hkv * ((a.group + OWN_ROWS - 1) / OWN_ROWS);
  const int tiles = (a.S + OWN_TILE - 1) / OWN_TILE + (a.direct ? (l.P + OWN_TILE - 1) / OWN_TILE : 0);
  auto go = [&](auto ring, int ways) {
    constexpr int R = decltype(ring)::value;
    if (ways == 1) return launch_ways<HD, 1, R>(a, l, part_o, part_ml, units, 1, stream);
    if (ways == 2) return launch_ways<HD, 2, R>(a, l, part_o, part_ml, units, 1, stream);
    return launch_ways<HD, 4, R>(a, l, part_o, part_ml, units, ways / 4, stream);
  };
  // One or two tiles a warp, where that takes a CTA a unit at most and no more than 16 or 12 warps on an SM, which is what registers or
  // memory hold: everything is under way at once, and nothing crosses CTAs (8 x 5 continuations of 65 keys: 27.2 -> 23 us, 1 x 8 of 96
  // 15.6 -> 13; but 8 x 8 of 65, 14 warps an SM, 17.8, and streaming 12.9).  Units of one tile so however many they are (64 x 8 of 16 keys:
  // streaming 18.6, so 11.6; two tiles, of 30, 20.9 and 24.9).  Else as many warps a unit as fit on the SMs at once, each with a
  // tile at least: up to eight an SM with wide rings, or twelve with narrow ones (3 x 32 of 240 keys, 5.2 warps an SM / 10.4, 20.9 / 15.2;
  // 8 x 16 of 128, 12 heads of 64, 10.4 warps with wide / narrow rings 15.6 / 10.2).
  for (int ring = 1; ring <= 2; ++ring) {
    int ways = 1;
    while (ways < 4 && ways * ring < tiles) ways *= 2;
    if (ways * ring >= tiles && (units * ways <= (ring == 1 ? 16LL : 12LL) * num_sms || ring * ways == 1))
      return ring == 1 ? go(std::integral_constant<int, 1>(), ways) : go(std::integral_constant<int, 2>(), ways);
  }
  int ways = 1;
  while (ways < 32 && units * ways * 2 <= 12LL * num_sms && tiles >= ways * 2) ways *= 2;
  const bool narrow = units * ways > 8LL * num_sms && units * ways <= 12LL * num_sms;
  return narrow ? go(std::integral_constant<int, NARROW>(), ways) : go(std::integral_constant<int, WIDE>(), ways);
}

int launch_prefix(const void* q, const void* k, const void* v, const Layout& l, int H, int Hkv, int hd, bool few, const long long* qs,
                  const long long* ks, const long long* vs, float scale, float* part_o, float2* part_ml, int* status, cudaStream_t stream);

// Prompts of this many bytes outlast L2 (126 MB): two row tiles share a key.  Otherwise the second finds it there, and units of one tile
// deal out more evenly and join both groups.  Alone / shared, us: 8 x 64 x 4000 (131 MB) 64.2 / 68.8, 1 x 32 x 32 768 (134 MB) 46.2 / 50.7,
// 1 x 32 x 40 000 (164 MB) 55.0 / 56.6, 10 x 64 x 4000 (164 MB) 108.8 / 109.0, 12 x 64 x 4000 (197 MB) 133.9 / 127.4, 2 x 32 x 24 000
// (197 MB) 76.3 / 61.4, 2 x 32 x 32 768 (268 MB) 98 / 76, 4 x 32 x 32 768 (537 MB) 184 / 142.
constexpr long long PAIR_BYTES = 168LL << 20;

static bool make_layout(Layout& l, const void* lens, int B, int W, int P, int group, int Hkv, int hd, int num_sms) {
  if (group > TILE_ROWS) return false;
  const int wt = TILE_ROWS / group < W ? TILE_ROWS / group : W;
  const int pair = wt < W && 4LL * B * P * Hkv * hd > PAIR_BYTES ? 2 : 1, row_units = (W + wt * pair - 1) / (wt * pair);
  const long long tiles = (long long)tiles_of(P) * Hkv * row_units * B;
  const int most = (int)(tiles < num_sms ? tiles : num_sms);
  l = Layout{(const int*)lens, B, W, P, Hkv * row_units, row_units, pair, wt, most, most, tiles_of(P), 1, 1};
  const long long units = (long long)B * l.per_prompt;
  if (!lens && P > 0 && units <= num_sms) {
    const int ways = num_sms / (int)units, each = (l.span + ways - 1) / ways, whole = (l.span + each - 1) / each;
    if (each <= (tiles + most - 1) / most + SPARE) l.ctas = (int)units * whole, l.span = whole * each;
  }
  return tiles < 0x7fff0000LL && (long long)B * W * Hkv * group < 1LL << 27;   // counts of tiles and units in 32 bits
}

// Whether one kernel reads the prompts for every continuation again.  Up to 4 MB of them that is a launch and an allocation less for the host
// (1 x 4 x 300, 12 heads of 64: eager 10.9 -> 7.7 us); beyond, a warp's chain of tiles is longer than what two kernels take.  Prompts of one
// tile of 128 keys have no chain: up to 12 MB, and up to 64 where the other kernel's tiles are for few keys or continuations.  One kernel / two,
// in a graph, us: 6 MB (1 x 4 x 375) 7.8 / 7.0, 8 MB (1 x 4 x 500) 11.5 / 7.2; one tile, 8 MB (1 x 32 x 64) 7.1 / 8.8, 20 MB in 24 tiles
// (3 x 32 x 52) 25.6 / 22.9, 34 in 128 (16 x 8 x 64) 11.0 / 11.7, 67 in 512 (64 x 8 x 32) 29.4 / 37.3, 134 in 256 (32 x 8 x 128) 28.8 / 21.2.
constexpr long long DIRECT_BYTES = 4LL << 20, DIRECT_SHORT = 12LL << 20, DIRECT_MOST = 64LL << 20, DIRECT_OF_A_TILE = 256LL << 10;
static bool is_direct(int direct, const Layout& l, int Hkv, int hd) {
  const long long bytes = 4LL * l.B * l.W * l.P * Hkv * hd, tiles = (long long)l.per_prompt * l.B;
  if (l.P == 0 || direct >= 0) return l.P > 0 && direct != 0;
  if (l.P > TILE_KEYS) return bytes <= DIRECT_BYTES;
  return bytes <= DIRECT_SHORT || (bytes <= DIRECT_MOST && bytes <= tiles * DIRECT_OF_A_TILE);
}

}  // namespace shared_prefix
}  // namespace kf

extern "C" void* kf_status_device_ptr();

extern "C" {

// Bytes of scratch that kf_shared_prefix_attn_bf16 needs for these sizes (0: none, and one launch), negative where it does not take them.
// direct: whether the prompts are read for every continuation again; below 0: where that is the faster way.
long long kf_shared_prefix_scratch(int B, int W, int P, int H, int Hkv, int hd, int direct, int num_sms) {
  using namespace kf::shared_prefix;
  Layout l;
  if (B < 1 || W < 1 || P < 0 || Hkv < 1 || H % Hkv || (hd != 64 && hd != 128)) return -1;
  if (!make_layout(l, nullptr, B, W, P, H / Hkv, Hkv, hd, num_sms)) return -1;
  return P == 0 || is_direct(direct, l, Hkv, hd) ? 0 : slots(l) * l.pair * TILE_ROWS * (hd * 4 + 8);
}

// o (B, W, H, hd), dense = attention of q (B, W, H, hd) over k, v (B, P, Hkv, hd), of which lens[b] positions count (null: all), and over
// own_k, own_v (B, W, S, Hkv, hd), where position s of continuation w lies in the cache of continuation rows[b][w][s] (null: w).
// steps: in elements, of q (prompt, continuation, head), k and v (prompt, position, head), own_k and own_v (prompt, continuation, position,
// head) and rows (prompt, continuation): 19 numbers.  Head dim 64 or 128, dense; steps multiples of 8 and bases on 16 bytes (rows: any).  Of k and v
// the step from prompt to prompt may be 0; other steps are of dimensions of one entry where they are.
int kf_shared_prefix_attn_bf16(const void* q, const void* k, const void* v, const void* own_k, const void* own_v, const void* lens,
                               const void* rows, void* o, void* scratch, int B, int W, int P, int S, int H, int Hkv, int hd,
                               const long long* steps, float scale, int direct, int num_sms, void* stream) {
  using namespace kf::shared_prefix;
  Layout l;
  if (kf_shared_prefix_scratch(B, W, P, H, Hkv, hd, direct, num_sms) < 0 || S < 0 || !(scale > 0.f)) return 3;
  make_layout(l, lens, B, W, P, H / Hkv, Hkv, hd, num_sms);
  l.k_step = steps[3] != 0;
  l.v_step = steps[6] != 0;
  const long long *qs = steps, *ks = steps + 3, *vs = steps + 6, *oks = steps + 9, *ovs = steps + 13, *rs = steps + 17;
  for (int i = 0; i < 17; ++i)
    if (steps[i] & 7) return 5;
  cudaStream_t st = (cudaStream_t)stream;
  const bool alone = P == 0 || is_direct(direct, l, Hkv, hd);
  float* part_o = alone ? nullptr : (float*)scratch;
  float2* part_ml = alone ? nullptr : (float2*)(part_o + slots(l) * l.pair * TILE_ROWS * hd);
  if (!alone) {
    const bool few = S <= 2 * OWN_WARPS * OWN_TILE;   // rings of one or two tiles
    const int rc = launch_prefix(q, k, v, l, H, Hkv, hd, few, qs, ks, vs, scale, part_o, part_ml, (int*)kf_status_device_ptr(), st);
    if (rc) return rc;
  }
  const Own a{(const __nv_bfloat16*)q, (const __nv_bfloat16*)own_k, (const __nv_bfloat16*)own_v, (__nv_bfloat16*)o, (const uint8_t*)rows,
              S, Hkv, H / Hkv, (const __nv_bfloat16*)k, (const __nv_bfloat16*)v, alone && P > 0, ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
              qs[0], qs[1], qs[2], oks[0], oks[1], oks[2], oks[3], ovs[0], ovs[1], ovs[2], ovs[3], rs[0], rs[1],
              scale * 1.4426950408889634f};
  return hd == 128 ? launch_own<128>(a, l, part_o, part_ml, num_sms, st) : launch_own<64>(a, l, part_o, part_ml, num_sms, st);
}

}  // extern "C"
