// Product of two matrices in the 8-bit form with a scale for each block of 128 (fp8_blocks.cuh) for a token or a few:
//
//   out[m, n] (+)= sum over blocks b of 2^(sx[b, m] + sw[b, n] - 254) * sum over k in b of x[m, k] W[n, k],  1 <= M <= 16
//
// What bounds it: the stream of W, and with a few megabytes of it the chain from launch to result.  Nothing is set up here (no barriers, no
// tensor memory, no copies through shared memory): a warp reads rows of W in 16-byte pieces straight into fragments, multiplies a block's
// sum by its two factors and adds that up in 32 bits.  The warps of a block divide K and add up in a fixed order.
//
// The products are those of 16-bit halves (mma.sync.m16n8k16), which have every e4m3 and e5m2 value.  The order of k within a fragment is free as
// long as both operands have the same: lane (g, t) takes bytes 16 t .. 16 t + 15 of rows g and g + 8 of each 64, and a word's four bytes make a pair
// of each of a fragment's two.
//
// One token, graph of launches on weights in turn, us (at the copy rate): 1024 x 1024 2.2 (0.2), 2048 x 2048 3.7 (0.6); the tensor-memory kernel 5.2
// and 6.0.  Two to four blocks of K under way per warp instead of the next one change little (2048 x 2048 3.8 - 4.5, 4096 x 4096 8.1 - 9.6 for 8.2): per
// block of 2 KB a warp has 300 instructions to issue, and that and the wait for the next take turns.
#include "fp8_blocks.cuh"

#include <type_traits>

namespace kf {
namespace f8b {
namespace few {

constexpr int ROWS = 16;  // of W per block of threads
constexpr int MAX_WARPS = 16;
constexpr int MAX_TOKENS = 16;

struct Args {
  const uint8_t *x, *w, *sx, *sw;
  long long ldx, ldw, ldsx, ldsw;
  void* out;
  long long ldo;
  int M, N, K, f32, accumulate;
};

// v 2^(a + b - 254), NaN where a scale byte is 255: by two factors of half the exponent, since one of 2^(a - 127) could send beyond the range
// what the other brings back.  (A sum below -252, whose factors have no normal number, leaves nothing of a block's sum of at most 2^39.)
__device__ __forceinline__ float scaled(float v, uint32_t a, uint32_t b) {
  const int e = int(a + b) - 254, h = e >> 1;
  const float lo = __uint_as_float(uint32_t(max(h + 127, 0)) << 23), hi = __uint_as_float(uint32_t(max(e - h + 127, 0)) << 23);
  return a == 255 || b == 255 ? __uint_as_float(0x7fffffffu) : mul_full(mul_full(v, lo), hi);
}

__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// bytes 0 and 1, bytes 2 and 3 of a word as halves
template <bool E5M2>
__device__ __forceinline__ void halves(uint32_t w, uint32_t& low, uint32_t& high) {
  const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), E5M2 ? __NV_E5M2 : __NV_E4M3);
  const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), E5M2 ? __NV_E5M2 : __NV_E4M3);
  low = uint32_t(a.x) | uint32_t(a.y) << 16;
  high = uint32_t(b.x) | uint32_t(b.y) << 16;
}
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// 16 bytes of a row at column k; LAST: zeros past K
template <bool LAST>
__device__ __forceinline__ uint4 piece(const uint8_t* row, int k, int K) {
  if (!LAST) return *reinterpret_cast<const uint4*>(row + k);
  if (k >= K) return make_uint4(0, 0, 0, 0);
  const uint4 v = *reinterpret_cast<const uint4*>(row + k);
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = K - k - 4 * i;  // bytes of this word that exist
    w[i] = n >= 4 ? w[i] : n <= 0 ? 0u : w[i] & ((1u << (8 * n)) - 1u);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// TILES x 8 tokens, ROWS rows of W per block of threads
template <int TILES, bool W5, bool X5>
__global__ void __launch_bounds__(32 * MAX_WARPS)
kf_gemm_fp8_blocks_few(const Args a) {
  __shared__ float red[MAX_WARPS][ROWS * 8 * TILES];
  const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * ROWS, k_blocks = (a.K + BLOCK - 1) / BLOCK;
  // rows and tokens that do not exist stand for the last one: nobody reads what comes of them
  wait_for_previous();
  let_next_in();
  const int row[2] = {min(n0 + g, a.N - 1), min(n0 + 8 + g, a.N - 1)};
  float total[TILES][4] = {};
  struct Loaded {
    uint4 w[2][2], x[TILES][2];  // [row g or g + 8][half of the block]
    uint32_t sw[2], sx[TILES][2];
  };
  // all loads of a block leave before the first is used: none stands behind a test
  auto load = [&](Loaded& v, int kb, auto last) {
    constexpr bool LAST = decltype(last)::value;
    const int k = kb * BLOCK + t * 16;
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) v.w[r][h] = piece<LAST>(a.w + row[r] * a.ldw, k + 64 * h, a.K);
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
      const int m = min(8 * i + g, a.M - 1), c = 8 * i + 2 * t;
#pragma unroll
      for (int h = 0; h < 2; ++h) v.x[i][h] = piece<LAST>(a.x + m * a.ldx, k + 64 * h, a.K);
#pragma unroll
      for (int e = 0; e < 2; ++e) v.sx[i][e] = a.sx[kb * a.ldsx + min(c + e, a.M - 1)];
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) v.sw[r] = a.sw[kb * a.ldsw + row[r]];
  };
  auto add = [&](const Loaded& v) {
    float d[TILES][4] = {};
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t a0, a1, a2, a3;
        halves<W5>(word(v.w[0][h], q), a0, a2);
        halves<W5>(word(v.w[1][h], q), a1, a3);
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
          uint32_t b0, b1;
          halves<X5>(word(v.x[i][h], q), b0, b1);
          mma16(d[i], a0, a1, a2, a3, b0, b1);
        }
      }
#pragma unroll
    for (int i = 0; i < TILES; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) total[i][e] = add_full(total[i][e], scaled(d[i][e], v.sw[e >> 1], v.sx[i][e & 1]));
  };
  const int whole = a.K / BLOCK;
  int kb = warp;
  Loaded v;
  if (kb < whole) load(v, kb, std::false_type{});
  while (kb < whole) {
    add(v);
    kb += warps;
    if (kb < whole) load(v, kb, std::false_type{});
  }
  if (kb < k_blocks) {
    load(v, kb, std::true_type{});
    add(v);
  }
#pragma unroll
  for (int i = 0; i < TILES; ++i) {
    float* p = &red[warp][(8 * i + 2 * t) * ROWS + g];  // [token][row]
    p[0] = total[i][0];
    p[ROWS] = total[i][1];
    p[8] = total[i][2];
    p[ROWS + 8] = total[i][3];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < ROWS * 8 * TILES; i += blockDim.x) {
    const int m = i / ROWS, n = n0 + i % ROWS;
    if (m >= a.M || n >= a.N) continue;
    float v = 0.f;
    for (int w = 0; w < warps; ++w) v += red[w][i];
    if (a.f32) {
      float* p = static_cast<float*>(a.out) + m * a.ldo + n;
      *p = a.accumulate ? v + *p : v;
    } else {
      __nv_bfloat16* p = static_cast<__nv_bfloat16*>(a.out) + m * a.ldo + n;
      *p = __float2bfloat16(a.accumulate ? v + __bfloat162float(*p) : v);
    }
  }
}

template <int TILES>
static int launch(const Args& a, int a_fmt, int b_fmt, int warps, cudaStream_t stream) {
  auto kern = b_fmt ? (a_fmt ? kf_gemm_fp8_blocks_few<TILES, true, true> : kf_gemm_fp8_blocks_few<TILES, true, false>)
                    : (a_fmt ? kf_gemm_fp8_blocks_few<TILES, false, true> : kf_gemm_fp8_blocks_few<TILES, false, false>);
  return launch_programmatic(kern, dim3((a.N + ROWS - 1) / ROWS), 32 * warps, 0, 1, stream, a);
}

}  // namespace few

// Whether this kernel is the quicker one.  us, this / the tensor-memory kernel, graphs of launches on weights in turn: one token 256 x 256 1.9 /
// 3.1, 1024 x 1024 2.2 / 5.2, 2048 x 2048 3.7 / 6.0, 4096 x 4096 8.2 / 8.3, 6144 x 4096 12.6 / 9.0; 16 tokens 1304 x 952 3.4 / 4.6, 4096 x 2048
// 6.3 / 6.3.  In fours of eight tokens it gains little (32 x 1304 from 952 6.5 / 6.0): not built.
bool few_serves(int M, int N, int K) { return M <= few::MAX_TOKENS && (long long)N * K * ((M + 7) / 8) <= 12LL << 20; }

// The call of kf_gemm_fp8_blocks that few_serves.
int gemm_blocks_few(const void* A, const void* sa, const void* B, const void* sb, void* C, int M, int N, int K, long long lda, long long ldsa,
                    long long ldb, long long ldsb, long long ldc, int f32, int a_fmt, int b_fmt, int accumulate, int num_sms, void* stream) {
  const few::Args a{(const uint8_t*)A, (const uint8_t*)B, (const uint8_t*)sa, (const uint8_t*)sb, lda, ldb, ldsa, ldsb, C, ldc, M, N, K,
                    f32, accumulate};
  if (((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(B)) & 15) != 0) return 5;
  const int k_blocks = (K + BLOCK - 1) / BLOCK;
  int warps = (N + few::ROWS - 1) / few::ROWS <= num_sms ? 16 : 8;  // us with 16 / 8: 2048 x 2048, 8 tokens 3.7 / 4.3; 4096 x 2048, 16 tokens 8.2 / 6.3
  if (warps > k_blocks) warps = k_blocks;
  cudaStream_t st = (cudaStream_t)stream;
  return M <= 8 ? few::launch<1>(a, a_fmt, b_fmt, warps, st) : few::launch<2>(a, a_fmt, b_fmt, warps, st);
}

}  // namespace f8b
}  // namespace kf
