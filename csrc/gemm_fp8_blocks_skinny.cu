// Product of two matrices in the 8-bit form with a scale for each block of 128 where one of them has few rows (decoding, short prompts):
//
//   out[m, n] (+)= x[m, :] . W[n, :],  1 <= M <= 256
//
// What bounds it: the stream of W, read once and used for M rows.  As in gemm_skinny_tcgen05.cu 128 rows of W are the M side of the
// instruction and the tokens (padded to NT = 16 .. 256) its N side, and K is split over a cluster of up to 8 CTAs whose partial tiles meet in
// distributed shared memory and are added in a fixed order, in 32 bits.
//
// Roles: warp 0 loads the operands by TMA, warp 1 issues the instructions, warps 2 .. 5 bring the scale bytes from global to tensor memory
// (four blocks at a time, those of the next four under way meanwhile) and then the accumulator out.
#include "fp8_blocks.cuh"
#include "skinny_common.cuh"

namespace kf {
namespace f8b {
namespace skinny {

constexpr int WROWS = 128;
constexpr int BK = BLOCK;
constexpr int THREADS = 192;
constexpr int W_BYTES = WROWS * BK;
constexpr int GROUP = 4;  // blocks whose scale bytes travel together
constexpr int SLOTS = 4;  // groups under way

template <int NT>
struct Cfg {
  static constexpr int X_BYTES = NT * BK;
  static constexpr int STAGE = W_BYTES + X_BYTES;
  // two CTAs per SM up to 64 tokens (about 100 KB of ring each), one above
  static constexpr int STAGES = NT <= 16 ? 5 : NT <= 64 ? 4 : NT <= 128 ? 6 : 4;
  static constexpr int RED_BYTES = NT * WROWS * 4;  // reduction buffer, aliases the ring
  static constexpr int BODY = STAGES * STAGE > RED_BYTES ? STAGES * STAGE : RED_BYTES;
  static constexpr size_t SMEM = size_t(BODY) + 1024 + 256;
  static constexpr int SFX_COLS = NT <= 128 ? 4 : 8;
  static constexpr int SF_COLS = 4 + SFX_COLS;
  static constexpr int COLS = NT + SLOTS * SF_COLS;
  static constexpr int TMEM_COLS = COLS <= 64 ? 64 : COLS <= 128 ? 128 : COLS <= 256 ? 256 : 512;
};

__device__ __forceinline__ void mma_blocks(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ uint32_t mapa_shared(uint32_t addr, uint32_t cta) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(cta));
  return r;
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

// The scale bytes of COLS x 32 rows and four blocks, in the lane's words: row c * 32 + lane in word c.  All loads leave before the first is
// waited for (one after another, as behind a test of each row, they took 7 us); in the place of rows and blocks that do not exist the
// last one's are read, for accumulators that nobody reads.
template <int COLS>
__device__ __forceinline__ void load_scales(const uint8_t* __restrict__ s, long long ld, int row0, int rows, int kb0, int kb1, int lane,
                                            uint32_t (&w)[COLS]) {
  uint8_t v[COLS][GROUP];
#pragma unroll
  for (int c = 0; c < COLS; ++c)
#pragma unroll
    for (int b = 0; b < GROUP; ++b) v[c][b] = __ldg(s + (long long)min(kb0 + b, kb1 - 1) * ld + min(row0 + c * 32 + lane, rows - 1));
#pragma unroll
  for (int c = 0; c < COLS; ++c) w[c] = uint32_t(v[c][0]) | uint32_t(v[c][1]) << 8 | uint32_t(v[c][2]) << 16 | uint32_t(v[c][3]) << 24;
}

struct Args {
  const uint8_t *sx, *sw;
  long long ldsx, ldsw;
  __nv_bfloat16* out;
  long long ldo;       // elements between rows of out
  int M, N, K, accumulate, x_fmt, w_fmt;
};

// This CTA's share of the tile: the sum of the SPLITS partial tiles at `red_addr` of each CTA, eight columns of a token per thread and step,
// their loads all at once.
template <int SPLITS>
__device__ __forceinline__ void add_and_store(const Args& a, uint32_t red_addr, int row0, int rank, bool wide) {
  const int valid = min(WROWS, a.N - row0);
  for (int i = rank * THREADS + threadIdx.x; i < a.M * (WROWS / 8); i += SPLITS * THREADS) {
    const int t = i / (WROWS / 8), n = (i % (WROWS / 8)) * 8;
    if (n >= valid) continue;
    const uint32_t off = red_addr + uint32_t(t * WROWS + n) * 4u;
    float4 u[SPLITS], v[SPLITS];
#pragma unroll
    for (int r = 0; r < SPLITS; ++r) {
      const uint32_t src = mapa_shared(off, r);
      u[r] = ld_cluster_f4(src);
      v[r] = ld_cluster_f4(src + 16);
    }
    float f[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int r = 0; r < SPLITS; ++r) {
      f[0] += u[r].x; f[1] += u[r].y; f[2] += u[r].z; f[3] += u[r].w;
      f[4] += v[r].x; f[5] += v[r].y; f[6] += v[r].z; f[7] += v[r].w;
    }
    __nv_bfloat16* p = a.out + (long long)t * a.ldo + row0 + n;
    if (wide) {
      uint4 o = make_uint4(0, 0, 0, 0);
      if (a.accumulate) o = *reinterpret_cast<const uint4*>(p);
      const uint32_t w[4] = {o.x, o.y, o.z, o.w};
      uint32_t q[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 old = a.accumulate ? unpack_bf16(w[j]) : make_float2(0.f, 0.f);
        q[j] = pack_bf16(f[2 * j] + old.x, f[2 * j + 1] + old.y);
      }
      *reinterpret_cast<uint4*>(p) = make_uint4(q[0], q[1], q[2], q[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (n + e < valid) p[e] = __float2bfloat16(a.accumulate ? f[e] + __bfloat162float(p[e]) : f[e]);
    }
  }
}

template <int NT>
__global__ void __launch_bounds__(THREADS)
kf_gemm_fp8_blocks_skinny(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ Args a,
                          int* status) {
  using C = Cfg<NT>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t bar_base = smem_base + C::BODY;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (C::STAGES + s); };
  const uint32_t acc_bar = bar_base + 8u * (2 * C::STAGES);
  auto sf_ready_bar = [&](int g) { return acc_bar + 8u * (1 + g); };
  auto sf_empty_bar = [&](int g) { return acc_bar + 8u * (1 + SLOTS + g); };
  const uint32_t tmem_slot = acc_bar + 8u * (1 + 2 * SLOTS);
  static_assert(8 * (2 * C::STAGES + 1 + 2 * SLOTS) + 4 <= 256, "barriers");
  volatile uint32_t* tmem_slot_ptr = reinterpret_cast<volatile uint32_t*>(smem_raw + (tmem_slot - smem_u32(smem_raw)));
  float* red = reinterpret_cast<float*>(smem_raw + (smem_base - smem_u32(smem_raw)));

  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int splits = int(cluster_nctaid()), rank = int(cluster_ctarank());
  const int row0 = int(blockIdx.x) / splits * WROWS;
  const int k_blocks = (a.K + BK - 1) / BK;
  const int kb0 = k_blocks * rank / splits, kb1 = k_blocks * (rank + 1) / splits;
  const int n_kb = kb1 - kb0;

  // the first scale bytes are asked for before the ring's first fill (up to 100 KB per CTA) stands in line at the memory
  uint32_t sw[4], sx[C::SFX_COLS];
  if (warp >= 2) {
    load_scales<4>(a.sw, a.ldsw, row0, a.N, kb0, kb1, lane, sw);
    load_scales<C::SFX_COLS>(a.sx, a.ldsx, 0, a.M, kb0, kb1, lane, sx);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    mbar_init(acc_bar, 1);
    for (int g = 0; g < SLOTS; ++g) {
      mbar_init(sf_ready_bar(g), 4);
      mbar_init(sf_empty_bar(g), 1);
    }
    mbar_fence_init();
    tma_prefetch_desc(&map_x);
    tma_prefetch_desc(&map_w);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot_ptr;
  const bool wide = ((a.ldo | a.N) & 7) == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;

  bool ok = true;
  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (elect_one()) {
      int i = 0;
      for (; i < n_kb; ++i) {
        const int s = i % C::STAGES;
        if (!mbar_wait(empty_bar(s), ((i / C::STAGES) & 1) ^ 1, status, KF_ERR_WAIT_EMPTY)) { ok = false; break; }
        const uint32_t dst = smem_base + s * C::STAGE;
        mbar_expect_tx(full_bar(s), C::STAGE);
        tma_load_2d(dst, &map_w, full_bar(s), (kb0 + i) * BK, row0);
        tma_load_2d(dst + W_BYTES, &map_x, full_bar(s), (kb0 + i) * BK, 0);
      }
      // on the error path nobody consumes the stages: wait for the copies still landing in this CTA's shared memory
      if (!ok)
        for (int j = max(0, i - C::STAGES); j < i; ++j)
          mbar_wait(full_bar(j % C::STAGES), (j / C::STAGES) & 1, status, KF_ERR_WAIT_DRAIN);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (elect_one()) {
      const uint32_t idesc = idesc_blocks(WROWS, NT, a.w_fmt, a.x_fmt);
      for (int i = 0; i < n_kb; ++i) {
        const int s = i % C::STAGES, b = i % GROUP, gi = i / GROUP, g = gi % SLOTS;
        if (b == 0 && !mbar_wait(sf_ready_bar(g), (gi / SLOTS) & 1, status, KF_ERR_WAIT_FULL)) { ok = false; break; }
        if (!mbar_wait(full_bar(s), (i / C::STAGES) & 1, status, KF_ERR_WAIT_FULL)) { ok = false; break; }
        tc_fence_after();
        const uint32_t w_src = smem_base + s * C::STAGE, x_src = w_src + W_BYTES;
        const uint32_t sfw = tmem_base + NT + g * C::SF_COLS, sfx = sfw + 4;
#pragma unroll
        for (int k = 0; k < BK / 32; ++k)
          mma_blocks(tmem_base, umma_desc_sw128(w_src + k * 32, 16, 1024), umma_desc_sw128(x_src + k * 32, 16, 1024),
                     idesc + b * IDESC_NEXT_BYTE, sfw, sfx, (i | k) != 0);
        tc_commit(empty_bar(s));
        if (b == GROUP - 1) tc_commit(sf_empty_bar(g));
      }
      tc_commit(acc_bar);  // every MMA has retired: the accumulator is final, the ring is free
      if (!ok) mbar_wait(acc_bar, 0, status, KF_ERR_WAIT_DRAIN);
    }
  } else {
    const int quarter = warp & 3;
    const uint32_t t_lane = tmem_base + (uint32_t(quarter * 32) << 16);
    // ------------------------------------------------------------ scale bytes: global -> tensor memory
    for (int gi = 0; gi * GROUP < n_kb; ++gi) {
      const int g = gi % SLOTS;
      if (!mbar_wait(sf_empty_bar(g), ((gi / SLOTS) & 1) ^ 1, status, KF_ERR_WAIT_EMPTY)) { ok = false; break; }
      tc_fence_after();
      const uint32_t col = t_lane + NT + g * C::SF_COLS;
      tmem_st_x4(col, sw);
      if constexpr (C::SFX_COLS == 4) tmem_st_x4(col + 4, sx);
      else tmem_st_x8(col + 4, sx);
      const int next = kb0 + (gi + 1) * GROUP;
      load_scales<4>(a.sw, a.ldsw, row0, a.N, next, kb1, lane, sw);
      load_scales<C::SFX_COLS>(a.sx, a.ldsx, 0, a.M, next, kb1, lane, sx);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(sf_ready_bar(g));
    }
    // ------------------------------------------------------------ accumulator -> reduction buffer [token][W row]
    ok = mbar_wait(acc_bar, 0, status, KF_ERR_WAIT_TMEM_FULL) && ok;
    tc_fence_after();
    float* dst = red + quarter * 32 + lane;
#pragma unroll 1
    for (int c = 0; c < (NT + 31) / 32; ++c) {
      if (c * 32 >= a.M) break;
      if constexpr (NT == 16) {
        uint32_t v[16];
        tmem_ld_32x16(t_lane, v);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (i < a.M) dst[i * WROWS] = __uint_as_float(v[i]);
      } else {
        uint32_t v[32];
        tmem_ld_32x32(t_lane + c * 32, v);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (c * 32 + i < a.M) dst[(c * 32 + i) * WROWS] = __uint_as_float(v[i]);
      }
    }
  }
  tc_fence_before();
  __syncthreads();     // threads of one CTA at any cluster size
  cluster_sync_all();  // partial tiles of every split are in shared memory
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::TMEM_COLS);
  }

  // ------------------------------------------------------------ sum over the splits (fixed order), store
  switch (splits) {
    case 1: add_and_store<1>(a, smem_base, row0, rank, wide); break;
    case 2: add_and_store<2>(a, smem_base, row0, rank, wide); break;
    case 4: add_and_store<4>(a, smem_base, row0, rank, wide); break;
    default: add_and_store<8>(a, smem_base, row0, rank, wide); break;
  }
  cluster_sync_all();  // the buffers stay valid until every CTA of the cluster has read them
}

// Number of CTAs a K range is split over: enough of them to fill the SMs (twice up to 16 tokens, whose rings are small), at least MIN_KB
// ring steps each.  More only add partial tiles: 64 x 4096 from 4096 over 4 / 8 CTAs 16.4 / 18.4 us, 128 x 4096 18.4 / 36.9.
static int pick_splits(int tiles, int k_blocks, int num_sms, int per_sm) {
  constexpr int MIN_KB = 4;
  int s = 1;
  while (s < 8 && tiles * s * 2 <= num_sms * per_sm && k_blocks >= 2 * s * MIN_KB) s *= 2;
  return s;
}

template <int NT>
static int launch(const CUtensorMap& mx, const CUtensorMap& mw, const Args& a, int num_sms, int* status, cudaStream_t stream) {
  using C = Cfg<NT>;
  auto kern = kf_gemm_fp8_blocks_skinny<NT>;
  static bool attr_set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !attr_set[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM);
    if (e != cudaSuccess) return 300 + (int)e;
    if (dev < 64) attr_set[dev] = true;
  }
  const int tiles = (a.N + WROWS - 1) / WROWS;
  const int splits = pick_splits(tiles, (a.K + BK - 1) / BK, num_sms, NT <= 16 ? 2 : 1);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * splits));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, mx, mw, a, status);
  return e == cudaSuccess ? 0 : 400 + (int)e;
}

}  // namespace skinny

// The call of kf_gemm_fp8_blocks for up to 256 rows of A.
int gemm_blocks_skinny(const void* A, const void* sa, const void* B, const void* sb, void* C, int M, int N, int K, long long lda,
                       long long ldsa, long long ldb, long long ldsb, long long ldc, int a_fmt, int b_fmt, int accumulate, int num_sms,
                       int* status, void* stream) {
  const int nt = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : M <= 128 ? 128 : 256;
  skinny::Args a{(const uint8_t*)sa, (const uint8_t*)sb, ldsa, ldsb, (__nv_bfloat16*)C, ldc, M, N, K, accumulate, a_fmt, b_fmt};
  CUtensorMap mx, mw;
  int rc;
  if ((rc = make_map_u8(&mx, A, M, K, lda, BLOCK, nt, true))) return 100 + rc;
  if ((rc = make_map_u8(&mw, B, N, K, ldb, BLOCK, skinny::WROWS, true))) return 200 + rc;
  cudaStream_t st = (cudaStream_t)stream;
  switch (nt) {
    case 16: return skinny::launch<16>(mx, mw, a, num_sms, status, st);
    case 32: return skinny::launch<32>(mx, mw, a, num_sms, status, st);
    case 64: return skinny::launch<64>(mx, mw, a, num_sms, status, st);
    case 128: return skinny::launch<128>(mx, mw, a, num_sms, status, st);
    default: return skinny::launch<256>(mx, mw, a, num_sms, status, st);
  }
}

}  // namespace f8b
}  // namespace kf
