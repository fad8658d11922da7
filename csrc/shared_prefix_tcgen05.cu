// Attention of the new tokens of many continuations over the prompt that they share: partial results (first of two kernels).
//
// The W continuations of a prompt and the query heads of a key head are the rows of one tile, up to 128 of them, so that a key is read
// once for all and S = Q K^T and O += P V are 128-row products on the tensor cores; one kernel per continuation reads it W times.
// What bounds it: the keys and values, 4 hd bytes per position and head.  A tile of 128 keys of 128 values is 64 KB, which is 2700 cycles
// of an SM's share of HBM; its two products take 1040, its 16 384 exponentials 1024.  So rows that are not there (a tile is always 128)
// cost nothing, and all that counts is to keep the copies in flight: two stages each of K and V (128 KB) run ahead of the products.  Three
// were slower (4 x 32 768 keys, 64 heads of 128, with the second kernel: 102 and 98 us).  With more rows (64 continuations of 8000 keys:
// two row tiles of each key head) the chain scores - weights - products of a row tile, 3000 cycles with two of them under way, is what takes
// the time; first keys (6000 cycles) and a unit's partial result (5800) come on top.
// Where the softmax does not take the time it is LEAN: 96 registers a thread, with scores taken from tensor memory twice, 32 at a time, for
// the maximum and for the weights, and at most 162 KB, so that the second kernel does its own part meanwhile, beside it on the same SM.  That
// is up to three tiles a CTA, and with heads of 128 (of 64 there are twice the scores per byte) wherever one row tile reads the keys and the
// second kernel's rings are small.  Not LEAN / LEAN, us: 1 x 8 x 4000 (two tiles) 14.2 / 11.3, 1 x 8 x 16 000 of 96 own (seven) 23.6 / 21.5,
// 4 x 8 x 32 768 of 20 own (56) 94.8 / 93.0; of 200 own 106.9 / 109.8, 8 x 8 x 4000, 12 heads of 64, 29.5 / 32.9, 2 x 64 x 8000 (two row
// tiles) 31.3 / 32.9.
#include "attention_common.cuh"
#include "shared_prefix.cuh"
#include "skinny_common.cuh"

namespace kf {
namespace shared_prefix {

using namespace kf::attn;

constexpr int THREADS = 384;
constexpr int REGS_ISSUE = 72, REGS_SOFTMAX = 216;  // per thread; 72 + 2 * 216 = 3 * 168, what the launch gets (68 bytes are spilled)
constexpr int LEAN_BOUND = 608;                     // threads that a block might have: 96 registers each
constexpr int LEAN_TILES = 3;
constexpr int TMEM_COLS = 512;
constexpr float RESCALE_THRESHOLD = 8.0f;           // P up to 2^8 before the accumulator is scaled again
constexpr float FAR = 0x1p30f;

template <int HD>
struct Cfg {
  static constexpr int BLOCKS = HD / 64;
  static constexpr int TILE_BYTES = TILE_KEYS * HD * 2;
  static constexpr int BLOCK_BYTES = TILE_KEYS * 128;
  static constexpr int STAGES = HD == 128 ? 2 : 3;  // of K and of V at most; a CTA with fewer tiles takes less memory
  static constexpr int STATS = 3 * TILE_ROWS * 4;   // each group's maxima, the odd one's sums
  // Q, K ring, V ring, STATS, barriers: with one row tile up to 162 KB, which leaves 64 KB for a CTA of the second kernel
  static constexpr size_t smem(int stages, int q_tiles) { return (q_tiles + 2 * size_t(stages)) * TILE_BYTES + STATS + 256; }
};

// Where a CTA is in its range.
struct Walk {
  int b, u, j, nt;      // prompt, unit of the prompt, tile of the unit, tiles of a unit of this prompt
  int left;             // tiles of the range that are still to come
};

__device__ __forceinline__ void advance(const Layout& l, Walk& w, int n) {
  w.left -= n;
  w.j = 0;
  if (++w.u == l.per_prompt) {
    w.u = 0;
    if (w.left > 0) {
      do {
        w.nt = tiles_of(length(l, ++w.b));
      } while (w.nt == 0);
    }
  }
}

__device__ __forceinline__ int segment(const Walk& w) { return min(w.left, w.nt - w.j); }

// Start of this CTA's range, by one warp.
__device__ Walk locate(const Layout& l) {
  Walk w;
  const uint32_t total = tiles_before(l, l.B), chunk = range(total, l.ctas);
  const uint32_t t0 = chunk * blockIdx.x;
  w.left = t0 < total ? int(min(chunk, total - t0)) : 0;
  w.b = w.u = w.j = 0;
  w.nt = 1;
  if (w.left <= 0) return w;
  uint32_t before = 0;
  if (!l.lens) {
    const uint32_t each = uint32_t(l.span) * l.per_prompt;
    w.b = int(t0 / each);
    before = each * w.b;
  } else {
    const int lane = threadIdx.x & 31;
    for (int base = 0; base < l.B; base += 32) {
      const uint32_t own = base + lane < l.B ? uint32_t(tiles_of(length(l, base + lane))) * l.per_prompt : 0u;
      uint32_t upto = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, before + upto > t0);
      if (past) {
        const int at = __ffs(past) - 1;
        w.b = base + at;
        before += __shfl_sync(0xffffffffu, upto - own, at);
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  w.nt = tiles_of(length(l, w.b));
  const int span = l.lens ? w.nt : l.span;
  w.u = int((t0 - before) / span);
  w.j = int((t0 - before) % span);
  if (span > w.nt) w.left = min(w.left, w.nt - w.j);   // one unit, whose last range may be shorter
  return w;
}

// Stage and phase of a ring's next use.
struct Turn {
  int st = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int stages) {
    if (++st == stages) st = 0, phase ^= 1u;
  }
};

template <int N>
__device__ __forceinline__ void regs_give() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_take() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

__device__ __forceinline__ void st_global_v8(float* p, const float (&v)[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]),
               "f"(v[6]), "f"(v[7])
               : "memory");
}

template <int HD, bool LEAN, bool PAIR>
__global__ void __launch_bounds__(LEAN ? LEAN_BOUND : THREADS, 1)
kf_shared_prefix_tcgen05(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                         const __grid_constant__ CUtensorMap map_v, const Layout lay, int group, int stages, float scale_log2,
                         float* __restrict__ part_o, float2* __restrict__ part_ml, int* status) {
  using C = Cfg<HD>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t smem_base = smem_u32(smem_raw);
  uint8_t* smem = smem_raw;
  if (smem_base & 1023u) {   // not as declared: nothing is touched
    if (threadIdx.x == 0) atomicCAS(status, 0, int(KF_ERR_WAIT_DRAIN));
    return;
  }
  constexpr int Q_TILES = PAIR ? 2 : 1;
  const uint32_t q_smem = smem_base, k_smem = q_smem + Q_TILES * C::TILE_BYTES, v_smem = k_smem + stages * C::TILE_BYTES;
  float* stats = reinterpret_cast<float*>(smem + (Q_TILES + 2 * stages) * C::TILE_BYTES);
  uint8_t* bar_generic = reinterpret_cast<uint8_t*>(stats) + C::STATS;
  const uint32_t bar_base = smem_u32(bar_generic);
  auto k_full = [&](int st) { return bar_base + 8u * st; };
  auto k_empty = [&](int st) { return bar_base + 8u * (3 + st); };
  auto v_full = [&](int st) { return bar_base + 8u * (6 + st); };
  auto v_empty = [&](int st) { return bar_base + 8u * (9 + st); };
  auto s_full = [&](int g) { return bar_base + 8u * (12 + g); };
  auto p_half = [&](int g) { return bar_base + 8u * (14 + g); };   // weights of the first 64 keys are in tensor memory
  auto p_full = [&](int g) { return bar_base + 8u * (16 + g); };
  auto pv_done = [&](int g) { return bar_base + 8u * (18 + g); };
  const uint32_t q_full = bar_base + 8u * 20, q_empty = bar_base + 8u * 21;
  const uint32_t o_final = bar_base + 8u * 22, o_free = bar_base + 8u * 23, drain_bar = bar_base + 8u * 24;
  const uint32_t v_begun = bar_base + 8u * 25;   // V's producer has seen the first K
  volatile uint32_t* tmem_slot_ptr = reinterpret_cast<volatile uint32_t*>(bar_generic + 8 * 26);
  Walk* start = reinterpret_cast<Walk*>(bar_generic + 8 * 27);
  static_assert(8 * 27 + sizeof(Walk) <= 256, "what Cfg::smem has for barriers");

  const int warp = warp_index();
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 3; ++i) {
      mbar_init(k_full(i), 1);
      mbar_init(k_empty(i), 1);
      mbar_init(v_full(i), 1);
      mbar_init(v_empty(i), 1);
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(s_full(g), 1);
      mbar_init(p_half(g), 4);
      mbar_init(p_full(g), 4);
      mbar_init(pv_done(g), 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    mbar_init(o_final, 1);
    mbar_init(o_free, 8);
    mbar_init(drain_bar, 1);
    mbar_init(v_begun, 1);
    mbar_fence_init();
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot_ptr)), TMEM_COLS);
    tmem_relinquish();
  }
  grid_dep_wait();
  if (warp == 2) {
    const Walk w = locate(lay);
    if (lane == 0) *start = w;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_dep_launch();
  const uint32_t tmem_base = *tmem_slot_ptr;
  Walk wk = *start;
  auto s_col = [&](int g) { return tmem_base + uint32_t(g * 128); };
  // query rows of a unit's tile g (none: not there)
  auto rows_of = [&](const Walk& w, int g) { return min(lay.wt, lay.W - (w.u % lay.row_units * Q_TILES + g) * lay.wt) * group; };
  auto o_col = [&](int g) { return tmem_base + uint32_t(256 + g * 128); };

  if (warp < 4) {
    if (!LEAN) regs_give<REGS_ISSUE>();
    if (warp == 0) {
      // ------------------------------------------------------------ TMA producer of Q and K
      if (elect_one()) {
        bool ok = true;
        int seg = 0, issued = 0, q_issued = 0;   // units and tiles so far
        Turn turn;
        while (wk.left > 0 && ok) {
          const int n = segment(wk), hk = wk.u / lay.row_units, tiles = PAIR && rows_of(wk, 1) > 0 ? 2 : 1;
          if (seg > 0 && !mbar_wait(q_empty, (seg - 1) & 1, status, KF_ERR_WAIT_EMPTY)) { ok = false; break; }
          mbar_expect_tx(q_full, uint32_t(tiles * group * lay.wt * HD * 2));
          for (int g = 0; g < tiles; ++g)
#pragma unroll
            for (int c = 0; c < C::BLOCKS; ++c)
              tma_load_4d(q_smem + g * C::TILE_BYTES + c * C::BLOCK_BYTES, &map_q, q_full, 64 * c, hk * group,
                          (wk.u % lay.row_units * Q_TILES + g) * lay.wt, wk.b);
          ++q_issued;
          for (int j = wk.j; j < wk.j + n; ++j, turn.next(stages)) {
            // A wait knows a phase by its parity alone.  Nothing else that comes before a second K in the first stage waits for V, and after it V's
            // producer would not see the first any more.
            if (issued == stages && !mbar_wait(v_begun, 0, status, KF_ERR_WAIT_EMPTY)) { ok = false; break; }
            if (issued >= stages && !mbar_wait(k_empty(turn.st), turn.phase ^ 1u, status, KF_ERR_WAIT_EMPTY)) { ok = false; break; }
            mbar_expect_tx(k_full(turn.st), C::TILE_BYTES);
#pragma unroll
            for (int c = 0; c < C::BLOCKS; ++c)
              tma_load_4d(k_smem + turn.st * C::TILE_BYTES + c * C::BLOCK_BYTES, &map_k, k_full(turn.st), 64 * c, hk, j * TILE_KEYS,
                          wk.b * lay.k_step);
            ++issued;
          }
          advance(lay, wk, n);
          ++seg;
        }
        if (!ok) {
          if (q_issued > 0) mbar_wait(q_full, (q_issued - 1) & 1, status, KF_ERR_WAIT_DRAIN);
          for (int j = max(0, issued - stages); j < issued; ++j) mbar_wait(k_full(j % stages), (j / stages) & 1, status, KF_ERR_WAIT_DRAIN);
        }
      }
    } else if (warp == 2) {
      // ------------------------------------------------------------ TMA producer of V
      if (elect_one()) {
        bool ok = true;
        int issued = 0;
        Turn turn;
        // the first K before the first V: the scores can begin
        if (wk.left > 0) ok = mbar_wait(k_full(0), 0, status, KF_ERR_WAIT_FULL);
        mbar_arrive(v_begun);
        while (wk.left > 0 && ok) {
          const int n = segment(wk), hk = wk.u / lay.row_units;
          for (int j = wk.j; j < wk.j + n; ++j, turn.next(stages)) {
            if (issued >= stages && !mbar_wait(v_empty(turn.st), turn.phase ^ 1u, status, KF_ERR_WAIT_EMPTY)) { ok = false; break; }
            mbar_expect_tx(v_full(turn.st), C::TILE_BYTES);
#pragma unroll
            for (int c = 0; c < C::BLOCKS; ++c)
              tma_load_4d(v_smem + turn.st * C::TILE_BYTES + c * C::BLOCK_BYTES, &map_v, v_full(turn.st), 64 * c, hk, j * TILE_KEYS,
                          wk.b * lay.v_step);
            ++issued;
          }
          advance(lay, wk, n);
        }
        if (!ok)
          for (int j = max(0, issued - stages); j < issued; ++j) mbar_wait(v_full(j % stages), (j / stages) & 1, status, KF_ERR_WAIT_DRAIN);
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------ MMA issuer
      if (elect_one()) {
        constexpr uint32_t idesc_s = umma_idesc_bf16(TILE_ROWS, TILE_KEYS, false, false);
        constexpr uint32_t idesc_o = umma_idesc_bf16(TILE_ROWS, HD, false, true);
        bool ok = true;
        int seg = 0;                   // units so far
        int done[2] = {0, 0};          // tiles of each group whose P has been read
        Turn kt, vt;
        // S_g = Q K^T with the tile of keys whose turn it is
        auto issue_s = [&](int g) {
          const int st = kt.st;
          if (!mbar_wait(k_full(st), kt.phase, status, KF_ERR_WAIT_FULL)) return false;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            const uint32_t off = (kk / 4) * C::BLOCK_BYTES + (kk % 4) * 32;
            tc_mma_f16(s_col(g), umma_desc_sw128(q_smem + (PAIR ? g * C::TILE_BYTES : 0) + off, 16, 1024),
                       umma_desc_sw128(k_smem + st * C::TILE_BYTES + off, 16, 1024), idesc_s, kk != 0);
          }
          tc_commit(s_full(g));
          return true;
        };
        auto k_read = [&]() {   // every S that wants the tile has been issued
          tc_commit(k_empty(kt.st));
          kt.next(stages);
        };
        // O_g += P_g V: A = P from tensor memory, B = V with the head dim contiguous, in two halves of the keys
        auto issue_o = [&](int g, bool start) {
          const int st = vt.st;
          if (!mbar_wait(v_full(st), vt.phase, status, KF_ERR_WAIT_FULL)) return false;
          if (!mbar_wait(p_half(g), done[g] & 1, status, KF_ERR_WAIT_TMEM_EMPTY)) return false;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < TILE_KEYS / 32; ++kk)
            tc_mma_f16_ts(o_col(g), s_col(g) + kk * 8, umma_desc_sw128(v_smem + st * C::TILE_BYTES + kk * 2048, C::BLOCK_BYTES, 1024), idesc_o,
                          !start || kk != 0);
          if (!mbar_wait(p_full(g), done[g] & 1, status, KF_ERR_WAIT_TMEM_EMPTY)) return false;
          tc_fence_after();
#pragma unroll
          for (int kk = TILE_KEYS / 32; kk < TILE_KEYS / 16; ++kk)
            tc_mma_f16_ts(o_col(g), s_col(g) + kk * 8, umma_desc_sw128(v_smem + st * C::TILE_BYTES + kk * 2048, C::BLOCK_BYTES, 1024), idesc_o, 1u);
          tc_commit(pv_done(g));
          ++done[g];
          return true;
        };
        while (wk.left > 0 && ok) {
          const int n = segment(wk), groups = !PAIR || rows_of(wk, 1) > 0 ? 2 : 1;
          ok = mbar_wait(q_full, seg & 1, status, KF_ERR_WAIT_FULL);
          if (ok) tc_fence_after();
          // the first scores of both groups: of the unit's first two tiles, or (PAIR) of its first tile with both row tiles
          const int ahead = PAIR ? 1 : 2;
          for (int g = 0; g < (PAIR ? groups : min(n, 2)) && ok; ++g) {
            ok = issue_s(g);
            if (ok && (!PAIR || g + 1 == groups)) k_read();
          }
          if (ok && n <= ahead) tc_commit(q_empty);
          // the accumulators of the unit before have been read
          if (ok && seg > 0) ok = mbar_wait(o_free, (seg - 1) & 1, status, KF_ERR_WAIT_TMEM_EMPTY);
          for (int i = 0; i < n && ok; ++i, vt.next(stages)) {
            for (int g = PAIR ? 0 : i & 1; g < (PAIR ? groups : (i & 1) + 1) && ok; ++g) {
              const bool last = !PAIR || g + 1 == groups;
              ok = issue_o(g, i < ahead);
              if (ok && last) tc_commit(v_empty(vt.st));
              if (ok && last && i + 1 == n) tc_commit(o_final);
              // the group's next scores follow at once: the products just issued have read its P before they are written
              if (ok && i + ahead < n) {
                ok = issue_s(g);
                if (ok && last) {
                  k_read();
                  if (i + ahead + 1 == n) tc_commit(q_empty);
                }
              }
            }
          }
          ++seg;
          advance(lay, wk, n);
        }
        if (!ok) {
          tc_commit(drain_bar);
          mbar_wait(drain_bar, 0, status, KF_ERR_WAIT_DRAIN);
        }
      }
    }
  } else {
    // ------------------------------------------------------------ softmax: warps 4-7 even tiles, 8-11 odd tiles
    if (!LEAN) regs_take<REGS_SOFTMAX>();
    const int g = (warp >> 2) - 1;
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lane_off = uint32_t(quarter * 32) << 16;
    const uint32_t t_s = s_col(g) + lane_off, t_o = o_col(g) + lane_off;
    const float NEG_INF = -INFINITY;
    // Weights are 2^(x scale - m), fused, so the largest score's is 2 to the rounding of m.  All of a row share that factor, but beyond 2^31 it is
    // more than an exponent holds.  From 2^30 on a power of two serves as the scale: its products are exact, and scores that differ at all
    // differ by 32 or more in the exponent, so that with either scale nothing counts but the largest.
    const float rough_scale = __uint_as_float(__float_as_uint(scale_log2) & 0xff800000u);
    bool ok = true;
    int first = 0, seg = 0, mine = 0;   // tiles before this unit, units, tiles of this group
    while (wk.left > 0) {
      const int n = segment(wk), rows = rows_of(wk, PAIR ? g : 0);
      const bool active = quarter * 32 < rows;   // the warp has rows at all
      const int len = length(lay, wk.b);
      float m_run = NEG_INF, l_run = 0.f, factor = scale_log2, less = 0.f;
      for (int i = PAIR ? (rows > 0 ? 0 : n) : g; i < n; i += PAIR ? 1 : 2, ++mine) {
        const int n0 = (wk.j + i) * TILE_KEYS;
        if (ok && !mbar_wait(s_full(g), mine & 1, status, KF_ERR_WAIT_TMEM_FULL)) ok = false;
        tc_fence_after();
        if (n0 + TILE_KEYS > len && len < lay.P && (!PAIR || g == 0)) {   // PAIR: the products of group 0 come first
          // positions behind the prompt hold anything, and 0 times that need not be 0: their values become zeros
          const int st = (first + i) % stages;
          if (ok && !mbar_wait(v_full(st), ((first + i) / stages) & 1, status, KF_ERR_WAIT_FULL)) ok = false;
          if (ok && n0 + row >= len) {
#pragma unroll
            for (int c = 0; c < C::BLOCKS; ++c)
#pragma unroll
              for (int e = 0; e < 8; ++e)
                *reinterpret_cast<uint4*>(smem + (Q_TILES + stages + st) * C::TILE_BYTES + c * C::BLOCK_BYTES + row * 128 + e * 16) =
                    make_uint4(0, 0, 0, 0);
          }
          fence_async_smem();
        }
        if (!active) {
          // rows that are not there: whatever their P is, nobody reads what comes of it
          __syncwarp();
          tc_fence_before();
          if (lane == 0) {
            mbar_arrive(p_half(g));
            mbar_arrive(p_full(g));
          }
          continue;
        }
        // the scores: all at once, or (LEAN) in pieces, twice; what lies behind the prompt is hidden
        constexpr int PIECE = LEAN ? 32 : TILE_KEYS;
        const int visible = len - n0;
        auto scores = [&](uint32_t* x, int k0, int n) {
#pragma unroll
          for (int c = 0; c < n; c += 32) tmem_ld_32x32_at(t_s + k0 + c, x + c);
          tmem_ld_wait();
          if (visible < k0 + n) {
#pragma unroll
            for (int k = 0; k < n; ++k) x[k] = k0 + k < visible ? x[k] : __float_as_uint(NEG_INF);
          }
        };
        uint32_t sv[PIECE];
        float mx = NEG_INF;
#pragma unroll(LEAN ? 1 : TILE_KEYS / PIECE)
        for (int k0 = 0; k0 < TILE_KEYS; k0 += PIECE) {
          scores(sv, k0, PIECE);
          float mx4[4] = {mx, NEG_INF, NEG_INF, NEG_INF};
#pragma unroll
          for (int k = 0; k < PIECE; k += 8)
#pragma unroll
            for (int q = 0; q < 4; ++q) mx4[q] = fmax3(mx4[q], __uint_as_float(sv[k + 2 * q]), __uint_as_float(sv[k + 2 * q + 1]));
          mx = fmax3(fmaxf(mx4[0], mx4[1]), mx4[2], mx4[3]);
        }
        const float m_new = fmaxf(m_run, mx * scale_log2);
        const bool grow = m_new > m_run + RESCALE_THRESHOLD;
        if (__any_sync(0xffffffffu, grow)) {
          const float alpha = grow ? (m_run == NEG_INF ? 0.f : fast_exp2(m_run - m_new)) : 1.f;
          if (i >= (PAIR ? 1 : 2)) {
            if (ok && !mbar_wait(pv_done(g), (mine - 1) & 1, status, KF_ERR_WAIT_TMEM_FULL)) ok = false;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < HD / 32; ++c) {
              uint32_t o[32];
              tmem_ld_32x32_at(t_o + c * 32, o);
              tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
              tmem_st_32x32(t_o + c * 32, o);
            }
          }
          if (grow) {
            l_run *= alpha;
            m_run = m_new;
            const bool far = fabsf(m_new) >= FAR;
            factor = far ? rough_scale : scale_log2;
            less = far ? -(mx * rough_scale) : -m_new;
          }
        }
        const uint64_t scale2 = pack2(factor, factor), neg_m2 = pack2(less, less);
        uint64_t lsum[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll(LEAN ? 1 : TILE_KEYS / 32)
        for (int c = 0; c < TILE_KEYS / 32; ++c) {
          uint32_t again[LEAN ? 32 : 1], pk[16];
          if (LEAN) scores(again, c * 32, LEAN ? 32 : 0);   // the weights go over scores that have been taken
          const uint32_t* x = LEAN ? again : sv + c * 32;
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const uint64_t x2 = ffma2(pack2(__uint_as_float(x[2 * k]), __uint_as_float(x[2 * k + 1])), scale2, neg_m2);
            float x0, x1;
            unpack2(x2, x0, x1);
            const float e0 = fast_exp2(x0), e1 = fast_exp2(x1);
            lsum[k & 3] = fadd2(lsum[k & 3], pack2(e0, e1));
            pk[k] = pack_bf16(e0, e1);   // as V is, which the product asks for; the sum is of the unrounded weights
          }
          tmem_st_32x16(t_s + c * 16, pk);
          if (c & 1) {   // half of the keys are in place
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(c == 1 ? p_half(g) : p_full(g));
          }
        }
        float a0, a1;
        unpack2(fadd2(fadd2(lsum[0], lsum[1]), fadd2(lsum[2], lsum[3])), a0, a1);
        l_run += a0 + a1;
      }
      const long long slot = ((long long)wk.b * lay.per_prompt + wk.u + blockIdx.x) * Q_TILES + (PAIR ? g : 0);
      float* dst = part_o + (slot * TILE_ROWS + row) * HD;
      if (PAIR) {
        // ---- the row tile's partial result
        if (ok && !mbar_wait(o_final, seg & 1, status, KF_ERR_WAIT_TMEM_FULL)) ok = false;
        tc_fence_after();
        if (ok && active) {
#pragma unroll 1
          for (int c = 0; c < HD; c += 32) {
            uint32_t o[32];
            tmem_ld_32x32_at(t_o + c, o);
            tmem_ld_wait();
            if (row < rows) {
#pragma unroll
              for (int k = 0; k < 32; k += 8) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(o[k + e]);
                st_global_v8(dst + c + k, v);   // whole sectors: every lane writes a row of its own
              }
            }
          }
          if (row < rows) part_ml[slot * TILE_ROWS + row] = make_float2(m_run, l_run);
        }
        tc_fence_before();
        __syncwarp();
      } else {
        // ---- the unit's partial result: both groups' rows joined, each group writes half of the columns
        stats[g * TILE_ROWS + row] = m_run;
        if (g == 1) stats[2 * TILE_ROWS + row] = l_run;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        const float m_other = stats[(1 - g) * TILE_ROWS + row];
        const float top = fmaxf(m_run, m_other);
        const float f_mine = m_run == NEG_INF ? 0.f : fast_exp2(m_run - top), f_other = m_other == NEG_INF ? 0.f : fast_exp2(m_other - top);
        const float f0 = g == 0 ? f_mine : f_other, f1 = g == 0 ? f_other : f_mine;
        if (ok && !mbar_wait(o_final, seg & 1, status, KF_ERR_WAIT_TMEM_FULL)) ok = false;
        tc_fence_after();
        if (ok && active) {
#pragma unroll 1
          for (int c = 0; c < HD / 64; ++c) {
            const int col = g * (HD / 2) + c * 32;
            uint32_t o0[32], o1[32];
            tmem_ld_32x32_at(o_col(0) + lane_off + col, o0);
            if (n > 1) tmem_ld_32x32_at(o_col(1) + lane_off + col, o1);
            tmem_ld_wait();
            if (row < rows) {
#pragma unroll
              for (int k = 0; k < 32; k += 8) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                  v[e] = f0 * __uint_as_float(o0[k + e]);
                  if (n > 1) v[e] = __fmaf_rn(f1, __uint_as_float(o1[k + e]), v[e]);
                }
                st_global_v8(dst + col + k, v);   // whole sectors: every lane writes a row of its own
              }
            }
          }
          if (g == 0 && row < rows) part_ml[slot * TILE_ROWS + row] = make_float2(top, f0 * l_run + f1 * stats[2 * TILE_ROWS + row]);
        }
        tc_fence_before();
        // the accumulators may be written again, and stats by the next unit
        asm volatile("bar.sync 1, 256;" ::: "memory");
      }
      if (lane == 0) mbar_arrive(o_free);
      first += n;
      ++seg;
      advance(lay, wk, n);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// bf16 tensor of four dimensions, the last one dense; steps in elements.  A box that reaches over an end is filled with zeros.
static int make_map_4d(CUtensorMap* map, const void* base, const uint64_t (&size)[4], const long long (&step)[3], const uint32_t (&box_)[4]) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return -1;
  cuuint64_t dims[4], strides[3];
  cuuint32_t box[4], estr[4] = {1, 1, 1, 1};
  for (int i = 0; i < 4; ++i) dims[i] = size[i], box[i] = box_[i];
  for (int i = 0; i < 3; ++i) strides[i] = cuuint64_t(size[i + 1] > 1 ? step[i] * 2 : 16);   // of a single entry nothing is stepped over
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : (int)r;
}

template <int HD, bool LEAN, bool PAIR>
static int launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const Layout& l, int group, int stages, float scale,
                  float* part_o, float2* part_ml, int* status, cudaStream_t stream) {
  auto kern = kf_shared_prefix_tcgen05<HD, LEAN, PAIR>;
  static bool attr_set[16] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 16 || !attr_set[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Cfg<HD>::smem(Cfg<HD>::STAGES, PAIR ? 2 : 1));
    // all of the SM's memory as shared memory: CTAs of both kernels side by side
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e != cudaSuccess) return 300 + (int)e;
    if (dev < 16) attr_set[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)l.ctas);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = Cfg<HD>::smem(stages, PAIR ? 2 : 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, mq, mk, mv, l, group, stages, scale * 1.4426950408889634f, part_o, part_ml, status);
  return e == cudaSuccess ? 0 : 400 + (int)e;
}

template <int HD>
static int launch_hd(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const Layout& l, int group, bool few, float scale,
                     float* part_o, float2* part_ml, int* status, cudaStream_t stream) {
  const long long tiles = (long long)tiles_of(l.P) * l.per_prompt * l.B, each = (tiles + l.ctas - 1) / l.ctas;   // most tiles of a CTA
  const int stages = each < Cfg<HD>::STAGES ? (int)each : Cfg<HD>::STAGES;
  if (l.pair == 2) return launch<HD, false, true>(mq, mk, mv, l, group, stages, scale, part_o, part_ml, status, stream);
  const bool lean = each <= LEAN_TILES || (HD == 128 && l.row_units == 1 && few);
  return lean ? launch<HD, true, false>(mq, mk, mv, l, group, stages, scale, part_o, part_ml, status, stream)
              : launch<HD, false, false>(mq, mk, mv, l, group, stages, scale, part_o, part_ml, status, stream);
}

// Steps in elements: q prompt, continuation, head; k and v prompt, position, head.  few: the second kernel's own keys are.
int launch_prefix(const void* q, const void* k, const void* v, const Layout& l, int H, int Hkv, int hd, bool few, const long long* qs,
                  const long long* ks, const long long* vs, float scale, float* part_o, float2* part_ml, int* status, cudaStream_t stream) {
  const int group = H / Hkv;
  CUtensorMap mq, mk, mv;
  int rc = make_map_4d(&mq, q, {(uint64_t)hd, (uint64_t)H, (uint64_t)l.W, (uint64_t)l.B}, {qs[2], qs[1], qs[0]},
                       {64u, (uint32_t)group, (uint32_t)l.wt, 1u});
  if (rc) return 1000 + rc;
  rc = make_map_4d(&mk, k, {(uint64_t)hd, (uint64_t)Hkv, (uint64_t)l.P, (uint64_t)(l.k_step ? l.B : 1)}, {ks[2], ks[1], ks[0]},
                   {64u, 1u, (uint32_t)TILE_KEYS, 1u});
  if (rc) return 2000 + rc;
  rc = make_map_4d(&mv, v, {(uint64_t)hd, (uint64_t)Hkv, (uint64_t)l.P, (uint64_t)(l.v_step ? l.B : 1)}, {vs[2], vs[1], vs[0]},
                   {64u, 1u, (uint32_t)TILE_KEYS, 1u});
  if (rc) return 3000 + rc;
  return hd == 128 ? launch_hd<128>(mq, mk, mv, l, group, few, scale, part_o, part_ml, status, stream)
                   : launch_hd<64>(mq, mk, mv, l, group, few, scale, part_o, part_ml, status, stream);
}

}  // namespace shared_prefix
}  // namespace kf
