// Product of two matrices in the 8-bit form with a scale for each block of 128 (fp8_blocks.cuh) on the 5th-generation tensor cores:
//
//   C[m, n] (+)= sum over blocks b of 2^(sa[b, m] + sb[b, n] - 254) * sum over k in b of qa[m, k] qb[n, k]
//
// tcgen05.mma kind::mxf8f6f4 takes a scale byte for every row of A, row of B and 32 values of k from tensor memory and multiplies it into
// the products, in the same time as the instruction without scales.  A stage of the ring is one block of 128: its four instructions
// read the same bytes.  The scales so cost no pass over the accumulators, which would have to be read back, scaled and added outside the
// tensor cores once per block.
//
// Roles of a CTA: warp 0 loads the operands by TMA and warp 10 the scale bytes, warps 2 .. 5 move the bytes from shared to tensor memory (row r of
// A's 128 to lane r % 32 of column r / 32, the same in each quarter of the lanes, as the instruction wants them; B's rows likewise), warp 1
// issues the instructions, warps 6 .. 9 store the tile before.  Scales travel four blocks at a time, as the four bytes of a word of tensor
// memory of which an instruction names one: a hand-over for every block, with its wait for the stores and the arrival at the other CTA,
// took 1600 clocks where the block's instructions take 450 (8192 x 28 672 from 4096, us: 1569, in fours 808, ahead of the operands' ring and
// on signals that are no fences 653).
#include "fp8_blocks.cuh"
#include "gemm_epilogue.cuh"
#include "pair_common.cuh"
#include "tile_math.h"

#include <type_traits>
#include <utility>

namespace kf {
namespace f8b {

using namespace kf::pairops;

constexpr int CTA_M = 128;    // rows of A per CTA
constexpr int TILE_M = 256;   // rows per CTA pair
constexpr int MAX_N = 224;    // columns of the widest tile: two accumulators and the scales share 512 columns of tensor memory
constexpr int BK = BLOCK;     // bytes per row of a stage
constexpr int UMMA_K = 32;
constexpr int STAGES = 7;
constexpr int A_BYTES = CTA_M * BK;
constexpr int B_BYTES = (MAX_N / 2) * BK;
constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
constexpr int GROUP = 4;                            // blocks whose scale bytes travel together
constexpr int SLOTS = 3;                            // groups under way
constexpr int SFA_BYTES = GROUP * CTA_M;            // [block][row]
constexpr int SF_BYTES = SFA_BYTES + GROUP * 256;
constexpr int SF_COLS = 12;                         // their columns of tensor memory: 4 and 8
constexpr int SF_BASE = 2 * MAX_N;
constexpr int TMEM_COLS = 512;
static_assert(SF_BASE + SLOTS * SF_COLS <= TMEM_COLS && STAGE_BYTES % 1024 == 0, "tensor memory; swizzled tiles start on 1024 bytes");
constexpr int GROUP_M = 8;
constexpr int BOX_BYTES = 2048;  // one staged 32 x 32 box per epilogue warp
constexpr int THREADS = 352;
constexpr size_t SMEM = size_t(STAGES) * STAGE_BYTES + SLOTS * SF_BYTES + 4 * BOX_BYTES + 1024 + 256;

__device__ __forceinline__ void mma_pair_blocks(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                                uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
// Arrival and wait that hand over tensor memory only: what orders tcgen05.st before another CTA's tcgen05.mma is tcgen05.wait::st, the
// tcgen05 fences on both sides and this signal.  With release and acquire at cluster scope in their stead a hand-over of four blocks'
// scales took 2000 ns, whatever the width of the tile (74 x 256 rows, 128 to 224 columns, K 4096, us: 132 to 137, so 109 to 116).
__device__ __forceinline__ void arrive_relaxed_on_cta(uint32_t bar, uint32_t cta) {
  asm volatile(
      "{\n\t.reg .b32 ra;\n\t"
      "mapa.shared::cluster.u32 ra, %0, %1;\n\t"
      "mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [ra];\n\t}" ::"r"(bar),
      "r"(cta)
      : "memory");
}
// Arrival on the barrier at the same place in the CTAs of the mask once all instructions issued by this thread have retired.
__device__ __forceinline__ void commit_to(uint32_t bar, uint16_t mask) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"(mask)
      : "memory");
}
__device__ __forceinline__ void st_cluster_f4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// All CTAs of the cluster have come here; orders nothing in memory, and so waits for no store that is under way (0.7 us at the end of a tile).
__device__ __forceinline__ void cluster_meet() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_nctaid() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t mapa_shared(uint32_t addr, uint32_t cta) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(cta));
  return r;
}
__device__ __forceinline__ bool mbar_wait_relaxed(uint32_t bar, uint32_t parity, int* status, int code) {
  const long long t0 = clock64();
  uint32_t spins = 0;
  while (true) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred P;\n\t"
        "mbarrier.try_wait.parity.relaxed.cluster.shared::cta.b64 P, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, P;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    if (ok) return true;
    if ((++spins & 0x3ff) == 0) {
      if (*reinterpret_cast<volatile int*>(status) != 0) return false;
      if (clock64() - t0 > KF_WAIT_CYCLES) {
        atomicCAS(status, 0, code);
        return false;
      }
    }
  }
}
// bytes at p, p + step, .. as a word
__device__ __forceinline__ uint32_t four_bytes(const uint8_t* p, int step) {
  const uint32_t a = p[0], b = p[step], c = p[2 * step], d = p[3 * step];
  return a | b << 8 | c << 16 | d << 24;
}
__device__ __forceinline__ void sts32(uint32_t addr, uint32_t v) { asm volatile("st.shared.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ unsigned short lds_u16(uint32_t addr) {
  unsigned short v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr) : "memory");
  return v;
}

// Where a product goes: C[row * ld + column], or with `turned` (A's rows are C's columns) C[column * ld + row].
// One of the four kinds (bf16 or fp32, set or added to) to a kernel: with all of them in one, the registers and the instructions of the others
// cost bf16 outputs up to a fifth (us, 14 336 x 4096 from 2048: 96 -> 108).
template <typename T, bool ADD>
struct Output {
  T* C;
  long long ld;
  int turned;
  bool wide;  // rows of C start on 16 bytes and hold a multiple of eight values

  // 32 x 32 values of a warp at (row0, col0), a row per lane, of which rows x cols exist; box: 2 KB of the warp's own
  __device__ __forceinline__ void put(uint32_t box, int lane, const uint32_t (&v)[32], int row0, int col0, int rows, int cols) const {
    constexpr bool BF16 = sizeof(T) == 2;
    T* dst = C + (turned ? (long long)col0 * ld + row0 : (long long)row0 * ld + col0);
    if (turned) {
      if constexpr (BF16 && !ADD) {
        if (wide) {
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 32; ++i) sts_bf16(box_row_chunk(box, i, lane >> 3) + (lane & 7) * 2, __uint_as_float(v[i]));
          copy_box(box, lane, dst, cols, rows);
          return;
        }
      }
      if constexpr (!(BF16 && !ADD)) {
        if (wide) return put_words<true>(box, lane, dst, v, cols, rows);
      }
      if (lane < rows) put_each(dst + lane, v, cols);
      return;
    }
    if constexpr (BF16 && !ADD) {
      const Rows32 own = pack_row32(v);
      __syncwarp();
#pragma unroll
      for (int q = 0; q < 4; ++q) sts128(box_row_chunk(box, lane, q), own.q[q]);
      if (wide) {
        copy_box(box, lane, dst, rows, cols);
      } else {  // 64 contiguous bytes of one row per instruction
        __syncwarp();
        for (int r = 0; r < rows; ++r)
          if (lane < cols) reinterpret_cast<unsigned short*>(dst)[r * ld + lane] = lds_u16(box_row_chunk(box, r, lane >> 3) + (lane & 7) * 2);
      }
    } else if (!wide) {
      put_rows(box, lane, dst, v, rows, cols);
    } else {
      put_words<false>(box, lane, dst, v, rows, cols);
    }
  }

 private:
  static __device__ __forceinline__ float sum(float old, uint32_t v) { return ADD ? old + __uint_as_float(v) : __uint_as_float(v); }
  static __device__ __forceinline__ float read(const T* p) {
    if constexpr (sizeof(T) == 2) return __bfloat162float(*p);
    else return *p;
  }
  static __device__ __forceinline__ void write(T* p, float v) {
    if constexpr (sizeof(T) == 2) *p = __float2bfloat16(v);
    else *p = v;
  }
  // What is added to is read ahead of the stores: behind a store that might be to the same place each read would wait for the one before (us,
  // added to 1001 x 4097 from 1024 in bf16 110 -> 28, 777 x 1001 from 999 in fp32 31 -> 9.4).
  //
  // Rows of the output, 32 neighbours from the warp's lanes
  __device__ __forceinline__ void put_each(T* dst, const uint32_t (&v)[32], int cols) const {
#pragma unroll
    for (int h = 0; h < 32; h += 16) {
      float old[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) old[i] = ADD && h + i < cols ? read(dst + (h + i) * ld) : 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (h + i < cols) write(dst + (h + i) * ld, sum(old[i], v[h + i]));
    }
  }
  // A row of the output from a lane: 16 columns at a time go through the warp's box, so that an instruction writes 16 neighbours of two rows.
  // The word of a row is permuted by its number, which keeps both ways through the box free of bank conflicts.  (A row per lane with the reads
  // ahead: 332 us for those 28.)
  __device__ __forceinline__ void put_rows(uint32_t box, int lane, T* dst, const uint32_t (&v)[32], int rows, int cols) const {
    const int half = lane >> 4, c = lane & 15;
#pragma unroll
    for (int h = 0; h < 32; h += 16) {
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 16; ++i) sts32(box + lane * 64 + ((i ^ (lane >> 1)) << 2), v[h + i]);
      __syncwarp();
#pragma unroll 1
      for (int r0 = half; r0 < rows; r0 += 16) {
        float old[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) old[j] = ADD && r0 + 2 * j < rows && h + c < cols ? read(dst + (r0 + 2 * j) * ld + h + c) : 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int r = r0 + 2 * j;
          if (r < rows && h + c < cols) write(dst + r * ld + h + c, sum(old[j], lds32(box + r * 64 + ((c ^ (r >> 1)) << 2))));
        }
      }
    }
  }
  // rows x cols of the output in words of 16 bytes, each row's by neighbouring lanes; with TURNED v holds columns of it.  Half of the values go
  // through the box at a time, as 32 rows of 16 or 16 rows of 32, with 16-byte words permuted so that no way through it has bank conflicts.
  // A word per lane's own row fills half a sector at a time, single values are many instructions (us, 4096 x 4096 from 6144 in fp32 92 -> 83; from
  // 4096 64 -> 55, added to 222 -> 65, in bf16 70 -> 57), and with all that is added to read first its way is waited for once (added to 14 336 x 4096
  // from 2048, bf16, 1492 -> 134, in fp32 1499 -> 154).
  template <bool TURNED>
  __device__ __forceinline__ void put_words(uint32_t box, int lane, T* dst, const uint32_t (&v)[32], int rows, int cols) const {
    constexpr int PER = 16 / sizeof(T), W = TURNED ? 32 : 16, LANES = W / PER, STEP = 32 / LANES, N = 16 / PER;
    const int r0 = lane / LANES, c = lane % LANES * PER;
    auto at = [&](int row, int word) { return box + row * (4 * W) + ((word ^ (TURNED ? row & 1 : (row >> 1) & 3)) << 4); };
    const long long step = STEP * ld, half = TURNED ? 16 * ld : 16;
    T* const to = dst + r0 * ld + c;
    // row i and half h of this lane's words exist
    auto exists = [&](int i, int h) { return r0 + (TURNED ? h : 0) + i * STEP < rows && (TURNED ? 0 : h) + c < cols; };
    uint4 old[2][N];
    if constexpr (ADD) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (exists(i, 16 * h)) old[h][i] = *reinterpret_cast<const uint4*>(to + h * half + i * step);
    }
#pragma unroll
    for (int h = 0; h < 32; h += 16) {
      __syncwarp();
      if constexpr (TURNED) {
#pragma unroll
        for (int i = 0; i < 16; ++i) sts32(at(i, lane >> 2) + (lane & 3) * 4, v[h + i]);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) sts128(at(lane, q), make_uint4(v[h + 4 * q], v[h + 4 * q + 1], v[h + 4 * q + 2], v[h + 4 * q + 3]));
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int r = r0 + i * STEP;
        const uint4 a = lds128(at(r, c >> 2));
        const uint4 o = old[h >> 4][i];
        uint4 w;
        if constexpr (PER == 4) {
          w = make_uint4(plus(o.x, a.x), plus(o.y, a.y), plus(o.z, a.z), plus(o.w, a.w));
        } else {
          const uint4 b = lds128(at(r, (c >> 2) + 1));
          w = make_uint4(plus2(o.x, a.x, a.y), plus2(o.y, a.z, a.w), plus2(o.z, b.x, b.y), plus2(o.w, b.z, b.w));
        }
        if (exists(i, h)) *reinterpret_cast<uint4*>(to + (h >> 4) * half + i * step) = w;
      }
    }
  }
  static __device__ __forceinline__ uint32_t plus(uint32_t old, uint32_t v) { return __float_as_uint(sum(__uint_as_float(old), v)); }
  static __device__ __forceinline__ uint32_t plus2(uint32_t old, uint32_t v, uint32_t w) {
    const float2 o = unpack_bf16(old);
    return pack_bf16(sum(o.x, v), sum(o.y, w));
  }
  static __device__ __forceinline__ void sts_bf16(uint32_t addr, float v) {
    asm volatile("st.shared.u16 [%0], %1;" ::"r"(addr), "h"(__bfloat16_as_ushort(__float2bfloat16(v))) : "memory");
  }
  __device__ __forceinline__ void copy_box(uint32_t box, int lane, __nv_bfloat16* dst, int rows, int cols) const {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = i * 8 + (lane >> 2), ch = lane & 3;
      if (row < rows && ch * 8 < cols) *reinterpret_cast<uint4*>(dst + row * ld + ch * 8) = lds128(box_row_chunk(box, row, ch));
    }
  }
};

template <typename T, bool ADD>
__global__ void __launch_bounds__(THREADS, 1)
kf_gemm_fp8_blocks_2cta(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                        const __grid_constant__ CUtensorMap map_sa, const __grid_constant__ CUtensorMap map_sb,
                        const Output<T, ADD> out, int M, int N, int K, int a_fmt, int b_fmt, int tile_n, int* status) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t sf_smem = smem_base + STAGES * STAGE_BYTES;
  const uint32_t box_smem = sf_smem + SLOTS * SF_BYTES;
  const uint32_t bar_base = box_smem + 4 * BOX_BYTES;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };                  // the leader's: both CTAs' operands
  auto empty_bar = [&](int s) { return bar_base + 8u * (STAGES + s); };
  auto tfull_bar = [&](int a) { return bar_base + 8u * (2 * STAGES + a); };
  auto tempty_bar = [&](int a) { return bar_base + 8u * (2 * STAGES + 2 + a); };
  const uint32_t sf_bars = bar_base + 8u * (2 * STAGES + 4);
  auto sf_full_bar = [&](int g) { return sf_bars + 8u * g; };                 // this CTA's scale bytes are in shared memory
  auto sf_ready_bar = [&](int g) { return sf_bars + 8u * (SLOTS + g); };      // the leader's: both CTAs' are in tensor memory
  auto sf_empty_bar = [&](int g) { return sf_bars + 8u * (2 * SLOTS + g); };  // shared bytes and columns may be overwritten
  const uint32_t drain_bar = sf_bars + 8u * (3 * SLOTS);
  const uint32_t tmem_slot = drain_bar + 8u;
  static_assert(8 * (2 * STAGES + 4 + 3 * SLOTS + 1) + 4 <= 256, "barriers");
  volatile uint32_t* tmem_slot_ptr = reinterpret_cast<volatile uint32_t*>(smem_raw + (tmem_slot - smem_u32(smem_raw)));

  const int warp = warp_index();
  const int lane = threadIdx.x & 31;
  // A cluster is `splits` pairs that divide the reduction of a tile; with one pair it walks over its share of the tiles.
  const uint32_t cta = cluster_ctarank(), rank = cta & 1, lead = cta & ~1u;
  const uint16_t pair_mask = uint16_t(3u << lead);
  const bool leader = rank == 0;
  const int splits = int(cluster_nctaid()) >> 1, split = int(cta) >> 1;
  const int pair = int(blockIdx.x) / (2 * splits), num_pairs = int(gridDim.x) / (2 * splits);
  const int half_n = tile_n >> 1;
  const int m_blocks = (M + TILE_M - 1) / TILE_M;
  const int n_blocks = (N + tile_n - 1) / tile_n;
  const int num_tiles = m_blocks * n_blocks;
  const int all_blocks = (K + BK - 1) / BK;
  const int kb0 = all_blocks * split / splits, k_blocks = all_blocks * (split + 1) / splits - kb0;  // this pair's
  const int groups = (k_blocks + GROUP - 1) / GROUP;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int g = 0; g < SLOTS; ++g) {
      mbar_init(sf_full_bar(g), 1);
      mbar_init(sf_ready_bar(g), 8);  // four warps of both CTAs
      mbar_init(sf_empty_bar(g), 5);  // the instructions, and four warps that have read the shared bytes
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(tempty_bar(a), 8);  // the epilogue warps of both CTAs
    }
    mbar_init(drain_bar, 1);
    mbar_fence_init();
    tma_prefetch_desc(&map_a);
    tma_prefetch_desc(&map_b);
    tma_prefetch_desc(&map_sa);
    tma_prefetch_desc(&map_sb);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_meet();  // both CTAs' barriers exist (fence.mbarrier_init released them) before anyone signals across the pair
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot_ptr;
  wait_for_previous();
  let_next_in();

  const int quarter = warp & 3;
  const uint32_t box = box_smem + uint32_t((warp - 6) & 3) * BOX_BYTES, t_row = tmem_base + (uint32_t(quarter * 32) << 16);

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (one per CTA)
    if (elect_one()) {
      int it = 0;
      bool ok = true;
      for (int t = pair; t < num_tiles && ok; t += num_pairs) {
        int tm, tn;
        tilemath::raster(t, m_blocks, n_blocks, GROUP_M, tm, tn);
        const int m0 = tm * TILE_M + int(rank) * CTA_M, n0 = tn * tile_n + int(rank) * half_n;
        for (int kb = 0; kb < k_blocks; ++kb, ++it) {
          const int s = it % STAGES;
          const uint32_t ph = (it / STAGES) & 1;
          if (!mbar_wait(empty_bar(s), ph ^ 1, status, KF_ERR_WAIT_EMPTY)) { ok = false; break; }
          const uint32_t a_dst = smem_base + s * STAGE_BYTES;
          const uint32_t lead_full = full_bar(s) & PEER_BIT_MASK;
          if (leader) mbar_expect_tx(full_bar(s), 2 * (A_BYTES + half_n * BK));
          tma_load_2d_pair(a_dst, &map_a, lead_full, (kb0 + kb) * BK, m0);
          tma_load_2d_pair(a_dst + A_BYTES, &map_b, lead_full, (kb0 + kb) * BK, n0);
        }
      }
      // copies into this CTA's shared memory are complete once their stages were consumed or, on the error path, once
      // the leader's full barrier flipped
      if (leader)
        for (int j = max(0, it - STAGES); j < it; ++j)
          mbar_wait(full_bar(j % STAGES), (j / STAGES) & 1, status, KF_ERR_WAIT_DRAIN);
    }
  } else if (warp == 10) {
    // ------------------------------------------------------------ TMA producer of the scale bytes, ahead of the operands' ring
    if (elect_one()) {
      int gi = 0;
      bool ok = true;
      for (int t = pair; t < num_tiles && ok; t += num_pairs) {
        int tm, tn;
        tilemath::raster(t, m_blocks, n_blocks, GROUP_M, tm, tn);
        const int m0 = tm * TILE_M + int(rank) * CTA_M, n0 = tn * tile_n;
        for (int i = 0; i < groups; ++i, ++gi) {
          const int g = gi % SLOTS;
          if (!mbar_wait(sf_empty_bar(g), ((gi / SLOTS) & 1) ^ 1, status, KF_ERR_WAIT_EMPTY)) { ok = false; break; }
          mbar_expect_tx(sf_full_bar(g), GROUP * (CTA_M + tile_n));
          tma_load_2d(sf_smem + g * SF_BYTES, &map_sa, sf_full_bar(g), m0, kb0 + i * GROUP);
          tma_load_2d(sf_smem + g * SF_BYTES + SFA_BYTES, &map_sb, sf_full_bar(g), n0, kb0 + i * GROUP);
        }
      }
      for (int j = max(0, gi - SLOTS); j < gi; ++j)
        mbar_wait(sf_full_bar(j % SLOTS), (j / SLOTS) & 1, status, KF_ERR_WAIT_DRAIN);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader CTA only)
    if (leader && elect_one()) {
      const uint32_t idesc = idesc_blocks(TILE_M, tile_n, a_fmt, b_fmt);
      int it = 0, gi = 0, tile_iter = 0;
      bool ok = true;
      for (int t = pair; t < num_tiles && ok; t += num_pairs, ++tile_iter) {
        const int acc = tile_iter & 1;
        const uint32_t acc_ph = (tile_iter >> 1) & 1;
        if (!mbar_wait(tempty_bar(acc), acc_ph ^ 1, status, KF_ERR_WAIT_TMEM_EMPTY)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * MAX_N;
        for (int kb = 0; kb < k_blocks; ++kb, ++it) {
          const int s = it % STAGES;
          const uint32_t ph = (it / STAGES) & 1;
          const int b = kb % GROUP, g = gi % SLOTS;
          if (b == 0 && !mbar_wait_relaxed(sf_ready_bar(g), (gi / SLOTS) & 1, status, KF_ERR_WAIT_FULL)) { ok = false; break; }
          if (!mbar_wait(full_bar(s), ph, status, KF_ERR_WAIT_FULL)) { ok = false; break; }
          tc_fence_after();
          const uint32_t a_src = smem_base + s * STAGE_BYTES;
          const uint32_t b_src = a_src + A_BYTES;
          const uint32_t sfa = tmem_base + SF_BASE + g * SF_COLS, sfb = sfa + 4;
#pragma unroll
          for (int k = 0; k < BK / UMMA_K; ++k)
            mma_pair_blocks(d_tmem, umma_desc_sw128(a_src + k * UMMA_K, 16, 1024), umma_desc_sw128(b_src + k * UMMA_K, 16, 1024),
                            idesc + b * IDESC_NEXT_BYTE, sfa, sfb, (kb | k) != 0);
          commit_to(empty_bar(s), pair_mask);
          if (b == GROUP - 1 || kb == k_blocks - 1) {
            commit_to(sf_empty_bar(g), pair_mask);
            ++gi;
          }
        }
        if (ok) commit_to(tfull_bar(acc), pair_mask);
      }
      // every MMA must have retired before either CTA gives up its shared or tensor memory
      asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(drain_bar)
                   : "memory");
      mbar_wait(drain_bar, 0, status, KF_ERR_WAIT_DRAIN);
    }
  } else if (warp < 6) {
    // ------------------------------------------------------------ scale bytes: shared -> tensor memory
    // A slot's bytes land only after the instructions that read its columns before have retired (sf_empty_bar).
    const uint32_t t_lane = tmem_base + (uint32_t((warp & 3) * 32) << 16) + SF_BASE;
    int gi = 0;
    bool ok = true;
    for (int t = pair; t < num_tiles && ok; t += num_pairs) {
      for (int i = 0; i < groups; ++i, ++gi) {
        const int g = gi % SLOTS;
        if (!mbar_wait(sf_full_bar(g), (gi / SLOTS) & 1, status, KF_ERR_WAIT_FULL)) { ok = false; break; }
        tc_fence_after();
        const uint8_t* a_src = smem_raw + (sf_smem - smem_u32(smem_raw)) + g * SF_BYTES + lane;
        const uint8_t* b_src = a_src + SFA_BYTES;
        uint32_t a[4], b[8];
#pragma unroll
        for (int c = 0; c < 4; ++c) a[c] = four_bytes(a_src + c * 32, CTA_M);
#pragma unroll
        for (int c = 0; c < 8; ++c) b[c] = c * 32 < tile_n ? four_bytes(b_src + c * 32, tile_n) : 0u;
        tmem_st_x4(t_lane + g * SF_COLS, a);
        tmem_st_x8(t_lane + g * SF_COLS + 4, b);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(sf_empty_bar(g));
          arrive_relaxed_on_cta(sf_ready_bar(g), lead);
        }
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue (warps 6 .. 9 of both CTAs)
    int tile_iter = 0;
    bool ok = true;
    for (int t = pair; t < num_tiles && ok; t += num_pairs, ++tile_iter) {
      const int acc = tile_iter & 1;
      if (!mbar_wait(tfull_bar(acc), (tile_iter >> 1) & 1, status, KF_ERR_WAIT_TMEM_FULL)) { ok = false; break; }
      tc_fence_after();
      if (splits > 1) break;  // the only tile: below, together with the other pairs
      int tm, tn;
      tilemath::raster(t, m_blocks, n_blocks, GROUP_M, tm, tn);
      const int row0 = tm * TILE_M + int(rank) * CTA_M + quarter * 32;  // this warp's rows, and how many exist
      const int rows = max(0, min(32, M - row0));
      const int col0 = tn * tile_n, width = min(tile_n, N - col0);
      // the next 32 columns are under way while these are stored; where the output is read too, its values need the registers
      const uint32_t from = t_row + acc * MAX_N;
      uint32_t v[32], w[32];
      if constexpr (ADD) {
#pragma unroll 1
        for (int c = 0; c < width; c += 32) {
          tmem_ld_32x32(from + c, v);
          tmem_ld_wait();
          out.put(box, lane, v, row0, col0 + c, rows, min(32, width - c));
        }
      } else {
        tmem_ld_32x32(from, v);
      }
#pragma unroll 1
      for (int c = ADD ? width : 0; c < width; c += 64) {
        tmem_ld_wait();
        if (c + 32 < width) tmem_ld_32x32(from + c + 32, w);
        out.put(box, lane, v, row0, col0 + c, rows, min(32, width - c));
        if (c + 32 >= width) break;
        tmem_ld_wait();
        if (c + 64 < width) tmem_ld_32x32(from + c + 64, v);
        out.put(box, lane, w, row0, col0 + c + 32, rows, min(32, width - c - 32));
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_on_cta(tempty_bar(acc), lead);
    }
  }

  if (splits > 1) {
    // ------------------------------------------------------------ sum over the pairs of the cluster
    // Chunk c of 32 columns belongs to pair c % splits.  Every pair hands the other chunks of its accumulator to their owners' shared memory
    // (16 bytes of a lane's row after 16 of its neighbour's), where the rings are idle once all instructions have retired, and the owner adds
    // them in the order of the pairs, in 32 bits.
    constexpr uint32_t CHUNK_BYTES = CTA_M * 32 * 4, WARP_BYTES = 32 * 32 * 4;
    int tm, tn;
    tilemath::raster(pair, m_blocks, n_blocks, GROUP_M, tm, tn);
    const int row0 = tm * TILE_M + int(rank) * CTA_M + quarter * 32, rows = max(0, min(32, M - row0));
    const int col0 = tn * tile_n, width = min(tile_n, N - col0);
    const uint32_t mine = smem_base + uint32_t(quarter) * WARP_BYTES + uint32_t(lane) * 16;
    __syncwarp();
    cluster_meet();
    tc_fence_after();
    // warps 2 .. 5, which have no scales to move any more, take every other chunk; their boxes lie behind what arrives
    const bool works = warp >= 2 && warp < 10;
    const int half = warp < 6;
    const uint32_t my_box = half ? smem_base + 6 * CHUNK_BYTES + uint32_t(warp - 2) * BOX_BYTES : box;
    static_assert(6 * CHUNK_BYTES + 4 * BOX_BYTES <= STAGES * STAGE_BYTES, "at most two chunks of three pairs, three of two, or four of one, then the boxes");
    if (works) {
      int turn = 0;
#pragma unroll 1
      for (int c = 0; c * 32 < width; ++c) {
        const int owner = c % splits;
        if (owner == split || (turn++ & 1) != half) continue;
        uint32_t v[32];
        tmem_ld_32x32(t_row + c * 32, v);
        tmem_ld_wait();
        const uint32_t at = mapa_shared(mine + uint32_t((c / splits) * (splits - 1) + (split < owner ? split : split - 1)) * CHUNK_BYTES, 2 * owner + rank);
#pragma unroll
        for (int q = 0; q < 8; ++q) st_cluster_f4(at + q * 512, v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
      }
    }
    __syncwarp();
    cluster_sync_all();
    if (works) {
#pragma unroll 1
      for (int c = split + half * splits; c * 32 < width; c += 2 * splits) {
        uint32_t own[32], v[32];
        tmem_ld_32x32(t_row + c * 32, own);
        tmem_ld_wait();
        const uint32_t at = mine + uint32_t((c / splits) * (splits - 1)) * CHUNK_BYTES;
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = 0u;
#pragma unroll 1
        for (int j = 0; j < splits; ++j) {
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            uint4 u = make_uint4(own[4 * q], own[4 * q + 1], own[4 * q + 2], own[4 * q + 3]);
            if (j != split) u = lds128(at + uint32_t(j < split ? j : j - 1) * CHUNK_BYTES + q * 512);
            v[4 * q] = __float_as_uint(__uint_as_float(v[4 * q]) + __uint_as_float(u.x));
            v[4 * q + 1] = __float_as_uint(__uint_as_float(v[4 * q + 1]) + __uint_as_float(u.y));
            v[4 * q + 2] = __float_as_uint(__uint_as_float(v[4 * q + 2]) + __uint_as_float(u.z));
            v[4 * q + 3] = __float_as_uint(__uint_as_float(v[4 * q + 3]) + __uint_as_float(u.w));
          }
        }
        out.put(my_box, lane, v, row0, col0 + c * 32, rows, min(32, width - c * 32));
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_meet();  // neither CTA's tensor memory is in use
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

// How a product is cut: which matrix gives the rows of 256, the columns of a tile, the pairs that divide its reduction.
struct Cut {
  int turned, tile_n, splits;
};
// The cheapest by what was measured, in ns: a block of 128 takes 0.66 (columns + 250) on a pair while all of them ask for operands (64 columns
// 207, 128 250, 192 300, 224 313), the last tile's way out 4.5 a column, and the sum over a cluster its barriers and its copies.  Of 74 pairs
// 33 clusters of two fit, 22 of three and 15 of four; some are left free, since the last of a launch right behind another had to wait (13.3 us for
// 339 x 576 from 8064 in 33 clusters of two, in 12 of four 9.9; 24 of three where 22 fit take 15.0 for 9.0).  us, graph of launches on weights in
// turn, cut by columns only -> so: 200 x 4096 from 14 336 36.5 -> 18.0, 64 x 4096 from 4096 12.5 -> 8.4, 1554 x 7168 from 5120 50.9 -> 43.2, 2000 x
// 2048 from 2048 14.9 -> 12.3, 120 x 1304 from 952 6.6 -> 6.0; by powers of two only -> by three, too: 1 x 4096 from 14 336 16.6 -> 14.5.
static Cut cut_of(int M, int N, int K, int num_sms) {
  const int pairs = num_sms / 2, k_blocks = (K + BK - 1) / BK;
  Cut best{0, MAX_N, 1};
  float best_cost = 3.4e38f;
  for (int turned = 0; turned < 2; ++turned) {
    const int m = turned ? N : M, n = turned ? M : N, m_blocks = (m + TILE_M - 1) / TILE_M;
    for (int tn = MAX_N; tn >= 32; tn -= 32) {
      if (tn - 32 >= n) continue;
      const long long tiles = (long long)m_blocks * ((n + tn - 1) / tn);
      for (int splits = 1; splits <= 4; ++splits) {
        const int left = splits == 2 ? 14 : splits == 3 ? 8 : 18;  // pairs that such clusters leave idle
        if (splits > 1 && (tiles * splits > pairs - left || k_blocks < splits)) break;
        const long long rounds = splits > 1 ? 1 : (tiles + pairs - 1) / pairs;
        const float cost = float(rounds * ((k_blocks + splits - 1) / splits)) * 0.66f * float(tn + 250) + 4.5f * float(tn) +
                           (splits == 1 ? 0.f : splits == 2 ? 600.f + 9.f * float(tn) : splits == 3 ? 900.f + 12.f * float(tn) : 1200.f + 16.f * float(tn));
        if (cost < best_cost) {
          best = {turned, tn, splits};
          best_cost = cost;
        }
      }
    }
  }
  return best;
}

template <typename T, bool ADD>
static int launch_blocks(const Output<T, ADD>& out, int clusters, int splits, cudaStream_t stream, const CUtensorMap& ma, const CUtensorMap& mb,
                         const CUtensorMap& msa, const CUtensorMap& msb, int M, int N, int K, int a_fmt, int b_fmt, int tile_n, int* status) {
  static bool attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !attr_set[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kf_gemm_fp8_blocks_2cta<T, ADD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM);
    if (e != cudaSuccess) return 300 + (int)e;
    if (dev < 64) attr_set[dev] = true;
  }
  return launch_programmatic(kf_gemm_fp8_blocks_2cta<T, ADD>, dim3(unsigned(clusters * 2 * splits)), THREADS, SMEM, 2 * splits, stream, ma, mb, msa,
                             msb, out, M, N, K, a_fmt, b_fmt, tile_n, status);
}

// gemm_fp8_blocks_few.cu
bool few_serves(int M, int N, int K);
int gemm_blocks_few(const void* A, const void* sa, const void* B, const void* sb, void* C, int M, int N, int K, long long lda, long long ldsa,
                    long long ldb, long long ldsb, long long ldc, int f32, int a_fmt, int b_fmt, int accumulate, int num_sms, void* stream);

}  // namespace f8b
}  // namespace kf

extern "C" void* kf_status_device_ptr();

extern "C" {

// C[M,N] (+)= A8[M,K] B8[N,K]^T with the scales of blocks of 128 along K: sa (ceil(K / 128), M), sb (ceil(K / 128), N) bytes.  Pitches
// lda, ldb, ldsa, ldsb in bytes, multiples of 16 (bases too), ldc in elements.  C is bf16, or fp32 with f32.  a_fmt / b_fmt: 0 = e4m3, 1 = e5m2.
int kf_gemm_fp8_blocks(const void* A, const void* sa, const void* B, const void* sb, void* C, int M, int N, int K, long long lda,
                       long long ldsa, long long ldb, long long ldsb, long long ldc, int f32, int a_fmt, int b_fmt, int accumulate,
                       int num_sms, void* stream) {
  using namespace kf::f8b;
  if (((lda | ldb | ldsa | ldsb) & 15) || M <= 0 || N <= 0 || K <= 0 || num_sms < 2) return 5;
  int* status = reinterpret_cast<int*>(kf_status_device_ptr());
  if (few_serves(M, N, K)) return gemm_blocks_few(A, sa, B, sb, C, M, N, K, lda, ldsa, ldb, ldsb, ldc, f32, a_fmt, b_fmt, accumulate, num_sms, stream);
  const Cut cut = cut_of(M, N, K, num_sms);
  const bool wide = ((ldc | N) & 7) == 0 && (reinterpret_cast<uintptr_t>(C) & 15) == 0;
  if (cut.turned) {
    std::swap(A, B);
    std::swap(sa, sb);
    std::swap(lda, ldb);
    std::swap(ldsa, ldsb);
    std::swap(M, N);
    std::swap(a_fmt, b_fmt);
  }
  const int tile_n = cut.tile_n, k_blocks = (K + BK - 1) / BK;
  const long long tiles = (long long)((M + TILE_M - 1) / TILE_M) * ((N + tile_n - 1) / tile_n);
  if (tiles > 0x7fffffffLL) return 5;
  CUtensorMap ma, mb, msa, msb;
  int rc;
  if ((rc = make_map_u8(&ma, A, M, K, lda, BK, CTA_M, true))) return 100 + rc;
  if ((rc = make_map_u8(&mb, B, N, K, ldb, BK, tile_n / 2, true))) return 200 + rc;
  if ((rc = make_map_u8(&msa, sa, k_blocks, M, ldsa, CTA_M, GROUP, false))) return 100 + rc;
  if ((rc = make_map_u8(&msb, sb, k_blocks, N, ldsb, tile_n, GROUP, false))) return 200 + rc;
  const int clusters = cut.splits > 1 ? (int)tiles : (int)(tiles < num_sms / 2 ? tiles : num_sms / 2);
  auto launch = [&](auto* c, auto add) {
    using Out = Output<std::remove_pointer_t<decltype(c)>, decltype(add)::value>;
    return launch_blocks(Out{c, ldc, cut.turned, wide}, clusters, cut.splits, (cudaStream_t)stream, ma, mb, msa, msb, M, N, K, a_fmt, b_fmt, tile_n, status);
  };
  if (f32) return accumulate ? launch((float*)C, std::true_type{}) : launch((float*)C, std::false_type{});
  return accumulate ? launch((__nv_bfloat16*)C, std::true_type{}) : launch((__nv_bfloat16*)C, std::false_type{});
}

}  // extern "C"
