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
__device__ __forceinline__ void arrive_relaxed_on_leader(uint32_t bar) {
  asm volatile(
      "{\n\t.reg .b32 ra;\n\t"
      "mapa.shared::cluster.u32 ra, %0, 0;\n\t"
      "mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [ra];\n\t}" ::"r"(bar)
      : "memory");
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
__device__ __forceinline__ unsigned short lds_u16(uint32_t addr) {
  unsigned short v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr) : "memory");
  return v;
}

// 32 x 32 values of a warp (a row per lane) into a matrix whose rows do not start on 16 bytes: through the box, 64 contiguous bytes of one
// row per instruction.
__device__ __forceinline__ void store_rows32_any(uint32_t box, int lane, const Rows32& own, __nv_bfloat16* dst, size_t ld, int rows, int cols) {
  __syncwarp();
#pragma unroll
  for (int q = 0; q < 4; ++q) sts128(box_row_chunk(box, lane, q), own.q[q]);
  __syncwarp();
  for (int r = 0; r < rows; ++r)
    if (lane < cols) reinterpret_cast<unsigned short*>(dst)[r * ld + lane] = lds_u16(box_row_chunk(box, r, lane >> 3) + (lane & 7) * 2);
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
kf_gemm_fp8_blocks_2cta(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                        const __grid_constant__ CUtensorMap map_sa, const __grid_constant__ CUtensorMap map_sb,
                        __nv_bfloat16* __restrict__ C, int M, int N, int K, long long ldc, int accumulate, int a_fmt, int b_fmt, int tile_n,
                        int* status) {
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
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
  const int half_n = tile_n >> 1;
  const int m_blocks = (M + TILE_M - 1) / TILE_M;
  const int n_blocks = (N + tile_n - 1) / tile_n;
  const int num_tiles = m_blocks * n_blocks;
  const int k_blocks = (K + BK - 1) / BK, groups = (k_blocks + GROUP - 1) / GROUP;

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
  cluster_sync_all();  // both CTAs' barriers exist before anyone signals across the pair
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot_ptr;

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
          tma_load_2d_pair(a_dst, &map_a, lead_full, kb * BK, m0);
          tma_load_2d_pair(a_dst + A_BYTES, &map_b, lead_full, kb * BK, n0);
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
          tma_load_2d(sf_smem + g * SF_BYTES, &map_sa, sf_full_bar(g), m0, i * GROUP);
          tma_load_2d(sf_smem + g * SF_BYTES + SFA_BYTES, &map_sb, sf_full_bar(g), n0, i * GROUP);
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
          commit_pair(empty_bar(s));
          if (b == GROUP - 1 || kb == k_blocks - 1) {
            commit_pair(sf_empty_bar(g));
            ++gi;
          }
        }
        if (ok) commit_pair(tfull_bar(acc));
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
          arrive_relaxed_on_leader(sf_ready_bar(g));
        }
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue (warps 6 .. 9 of both CTAs)
    const int quarter = warp & 3;
    const uint32_t box = box_smem + uint32_t(warp - 6) * BOX_BYTES;
    const bool wide = ((ldc | N) & 7) == 0 && (reinterpret_cast<uintptr_t>(C) & 15) == 0;
    int tile_iter = 0;
    bool ok = true;
    for (int t = pair; t < num_tiles && ok; t += num_pairs, ++tile_iter) {
      int tm, tn;
      tilemath::raster(t, m_blocks, n_blocks, GROUP_M, tm, tn);
      const int acc = tile_iter & 1;
      const uint32_t acc_ph = (tile_iter >> 1) & 1;
      if (!mbar_wait(tfull_bar(acc), acc_ph, status, KF_ERR_WAIT_TMEM_FULL)) { ok = false; break; }
      tc_fence_after();
      const int row0 = tm * TILE_M + int(rank) * CTA_M + quarter * 32;  // this warp's rows, and how many exist
      const int rows = max(0, min(32, M - row0));
      const int col0 = tn * tile_n, width = min(tile_n, N - col0);
      const uint32_t t_row = tmem_base + (uint32_t(quarter * 32) << 16) + acc * MAX_N;
      __nv_bfloat16* c0 = C + size_t(row0) * ldc + col0;
#pragma unroll 1
      for (int c = 0; c * 32 < width; ++c) {
        uint32_t v[32];
        tmem_ld_32x32(t_row + c * 32, v);
        tmem_ld_wait();
        const int valid = min(32, width - c * 32);
        __nv_bfloat16* dst = c0 + c * 32;
        if (!accumulate) {
          if (wide) store_rows32(box, lane, pack_row32(v), dst, ldc, rows, valid);
          else store_rows32_any(box, lane, pack_row32(v), dst, ldc, rows, valid);
        } else if (lane < rows) {
          dst += size_t(lane) * ldc;
          if (wide) {
            store_chunk<__nv_bfloat16>(dst, v, valid, true, nullptr);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i < valid) dst[i] = __float2bfloat16(__bfloat162float(dst[i]) + __uint_as_float(v[i]));
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_on_cta(tempty_bar(acc), 0);
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

// Tile width of a launch: rounds of tiles over the pairs times the columns of a tile, narrow ones at a surcharge for the operand bytes
// that they need per clock (pair_tile_width has the figures).
static int tile_width(int M, int N, int pairs) {
  const int m_blocks = (M + TILE_M - 1) / TILE_M;
  int best = MAX_N;
  float best_cost = 3.4e38f;
  for (int tn = MAX_N; tn >= 128; tn -= 32) {
    const long long tiles = (long long)m_blocks * ((N + tn - 1) / tn);
    const long long rounds = (tiles + pairs - 1) / pairs;
    const float bytes_per_clk = (128.f + 0.5f * tn) * 64.f / tn;
    const float cost = float(rounds) * tn * (1.f + 0.1f * (bytes_per_clk - 64.f) / 32.f);
    if (cost < best_cost) {
      best = tn;
      best_cost = cost;
    }
  }
  return best;
}

// gemm_fp8_blocks_skinny.cu
int gemm_blocks_skinny(const void* A, const void* sa, const void* B, const void* sb, void* C, int M, int N, int K, long long lda,
                       long long ldsa, long long ldb, long long ldsb, long long ldc, int a_fmt, int b_fmt, int accumulate, int num_sms,
                       int* status, void* stream);

}  // namespace f8b
}  // namespace kf

extern "C" void* kf_status_device_ptr();

extern "C" {

// C[M,N] (+)= A8[M,K] B8[N,K]^T with the scales of blocks of 128 along K: sa (ceil(K / 128), M), sb (ceil(K / 128), N) bytes.  Pitches
// lda, ldb, ldsa, ldsb in bytes, multiples of 16 (bases too), ldc in elements.  a_fmt / b_fmt: 0 = e4m3, 1 = e5m2.
int kf_gemm_fp8_blocks(const void* A, const void* sa, const void* B, const void* sb, void* C, int M, int N, int K, long long lda,
                       long long ldsa, long long ldb, long long ldsb, long long ldc, int a_fmt, int b_fmt, int accumulate, int num_sms,
                       void* stream) {
  using namespace kf::f8b;
  if (((lda | ldb | ldsa | ldsb) & 15) || M <= 0 || N <= 0 || K <= 0 || num_sms < 2) return 5;
  int* status = reinterpret_cast<int*>(kf_status_device_ptr());
  if (M <= 256)
    return gemm_blocks_skinny(A, sa, B, sb, C, M, N, K, lda, ldsa, ldb, ldsb, ldc, a_fmt, b_fmt, accumulate, num_sms, status, stream);
  int pairs = num_sms / 2;
  const int tile_n = tile_width(M, N, pairs);
  const int k_blocks = (K + BK - 1) / BK;
  CUtensorMap ma, mb, msa, msb;
  int rc;
  if ((rc = make_map_u8(&ma, A, M, K, lda, BK, CTA_M, true))) return 100 + rc;
  if ((rc = make_map_u8(&mb, B, N, K, ldb, BK, tile_n / 2, true))) return 200 + rc;
  if ((rc = make_map_u8(&msa, sa, k_blocks, M, ldsa, CTA_M, GROUP, false))) return 100 + rc;
  if ((rc = make_map_u8(&msb, sb, k_blocks, N, ldsb, tile_n, GROUP, false))) return 200 + rc;
  static bool attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !attr_set[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kf_gemm_fp8_blocks_2cta, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM);
    if (e != cudaSuccess) return 300 + (int)e;
    if (dev < 64) attr_set[dev] = true;
  }
  const long long tiles = (long long)((M + TILE_M - 1) / TILE_M) * ((N + tile_n - 1) / tile_n);
  if (tiles > 0x7fffffffLL) return 5;
  if (tiles < pairs) pairs = (int)tiles;
  kf_gemm_fp8_blocks_2cta<<<pairs * 2, THREADS, SMEM, (cudaStream_t)stream>>>(ma, mb, msa, msb, reinterpret_cast<__nv_bfloat16*>(C), M, N, K,
                                                                             ldc, accumulate, a_fmt, b_fmt, tile_n, status);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 400 + (int)e;
}

}  // extern "C"
