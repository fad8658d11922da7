// Product of two matrices in the 8-bit form with a scale for each block of 128 (fp8_blocks.cuh) for a token or a few:
//
//   out[m, n] (+)= sum over blocks b of 2^(sx[b, m] + sw[b, n] - 254) * sum over k in b of x[m, k] W[n, k],  1 <= M <= 16
//
// What bounds it: the stream of W, and with a few megabytes of it the chain from launch to result.  Nothing is set up here (no barriers, no
// tensor memory, no copies through shared memory): a warp reads rows of W in 16-byte pieces straight into fragments, multiplies a block's
// sum by its two factors and adds that up in 32 bits.  The warps of a block divide K and add up in a fixed order.
//
// The products are those of 16-bit halves (mma.sync.m16n8k16): an e4m3 byte moved to the exponent and fraction bits of a half is its value
// times 2^-8, an e5m2 byte is the upper byte of one, and four bytes become two pairs with seven shifts and masks.  NaN has no place in that
// move, so e4m3 operands are looked through for it.  The order of k within a fragment is free as long as both operands have the same: lane (g, t) takes bytes 16 t .. 16 t + 15 of
// rows g and g + 8 of each 64, and of a word the bytes 0 and 2, then 1 and 3.
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

// v 2^(a + b - 254 + UP), NaN where a scale byte is 255: by two factors of half the exponent, since one of 2^(a - 127) could send beyond the range
// what the other brings back.  (A sum below -252, whose factors have no normal number, leaves nothing of a block's sum of at most 2^33.)
template <int UP>
__device__ __forceinline__ float scaled(float v, uint32_t a, uint32_t b) {
  const int e = int(a + b) - 254 + UP, h = e >> 1;
  const float lo = __uint_as_float(uint32_t(max(h + 127, 0)) << 23), hi = __uint_as_float(uint32_t(max(e - h + 127, 0)) << 23);
  return a == 255 || b == 255 ? __uint_as_float(0x7fffffffu) : mul_full(mul_full(v, lo), hi);
}

__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// bytes 0 and 2, bytes 1 and 3 of a word as halves; e4m3 values times 2^-8, and NaN as something else: nan_in tells of it
template <bool E5M2>
__device__ __forceinline__ void halves(uint32_t w, uint32_t& even, uint32_t& odd) {
  if (E5M2) {
    even = (w << 8) & 0xff00ff00u;
    odd = w & 0xff00ff00u;
  } else {
    even = ((w << 8) & 0x80008000u) | ((w << 7) & 0x3f803f80u);
    odd = (w & 0x80008000u) | ((w >> 1) & 0x3f803f80u);
  }
}
template <bool E5M2>
__device__ __forceinline__ uint32_t nan_in(const uint4& v) {
  if (E5M2) return 0;  // a half has it
  auto in = [](uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; };
  return in(v.x) | in(v.y) | in(v.z) | in(v.w);
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
  uint32_t nan_w[2] = {}, nan_x[TILES] = {};
  // all loads of a block leave before the first is used: none stands behind a test
  auto block = [&](int kb, auto last) {
    constexpr bool LAST = decltype(last)::value;
    const int k = kb * BLOCK + t * 16;
    uint4 wv[2][2], xv[TILES][2];  // [row g or g + 8][half of the block]
    uint32_t sw[2], sx[TILES][2];
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) wv[r][h] = piece<LAST>(a.w + row[r] * a.ldw, k + 64 * h, a.K);
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
      const int m = min(8 * i + g, a.M - 1), c = 8 * i + 2 * t;
#pragma unroll
      for (int h = 0; h < 2; ++h) xv[i][h] = piece<LAST>(a.x + m * a.ldx, k + 64 * h, a.K);
#pragma unroll
      for (int e = 0; e < 2; ++e) sx[i][e] = a.sx[kb * a.ldsx + min(c + e, a.M - 1)];
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) sw[r] = a.sw[kb * a.ldsw + row[r]];
    float d[TILES][4] = {};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < TILES; ++i) nan_x[i] |= nan_in<X5>(xv[i][h]);
#pragma unroll
      for (int r = 0; r < 2; ++r) nan_w[r] |= nan_in<W5>(wv[r][h]);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t a0, a1, a2, a3;
        halves<W5>(word(wv[0][h], q), a0, a2);
        halves<W5>(word(wv[1][h], q), a1, a3);
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
          uint32_t b0, b1;
          halves<X5>(word(xv[i][h], q), b0, b1);
          mma16(d[i], a0, a1, a2, a3, b0, b1);
        }
      }
    }
    constexpr int UP = (W5 ? 0 : 8) + (X5 ? 0 : 8);  // what moving the bytes took away
#pragma unroll
    for (int i = 0; i < TILES; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) total[i][e] = add_full(total[i][e], scaled<UP>(d[i][e], sw[e >> 1], sx[i][e & 1]));
  };
  const int whole = a.K / BLOCK;
  int kb = warp;
#pragma unroll 2
  for (; kb < whole; kb += warps) block(kb, std::false_type{});
  if (kb < k_blocks) block(kb, std::true_type{});
  // a NaN among a row's or a token's values: in all that they take part in
  uint32_t any = nan_w[0] | nan_w[1];
#pragma unroll
  for (int i = 0; i < TILES; ++i) any |= nan_x[i];
  if (__any_sync(0xffffffffu, any != 0)) {
    const float nan = __uint_as_float(0x7fffffffu);
    auto over_t = [](uint32_t v) {
      v |= __shfl_xor_sync(0xffffffffu, v, 1);
      return v | __shfl_xor_sync(0xffffffffu, v, 2);
    };
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
      const uint32_t token = over_t(nan_x[i]);  // of token g, in its four lanes
      const uint32_t tok[2] = {__shfl_sync(0xffffffffu, token, 8 * t), __shfl_sync(0xffffffffu, token, 8 * t + 4)};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (over_t(nan_w[e >> 1]) | tok[e & 1]) total[i][e] = nan;
    }
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
// 4.0, 1024 x 1024 2.4 / 4.6, 2048 x 2048 3.9 / 6.3, 4096 x 2048 5.8 / 6.6, 4096 x 4096 9.3 / 8.5, 1024 x 14 336 14.1 / 11.1; 16 tokens 1304 x 952
// 3.5 / 4.5, 2048 x 2048 4.5 / 6.3, 4096 x 2048 6.7 / 6.7.  In fours of eight tokens it gains little (32 x 1304 from 952 6.5 / 6.0): not built.
bool few_serves(int M, int N, int K) { return M <= few::MAX_TOKENS && (long long)N * K * ((M + 7) / 8) <= 12LL << 20; }

// The call of kf_gemm_fp8_blocks that few_serves.
int gemm_blocks_few(const void* A, const void* sa, const void* B, const void* sb, void* C, int M, int N, int K, long long lda, long long ldsa,
                    long long ldb, long long ldsb, long long ldc, int f32, int a_fmt, int b_fmt, int accumulate, int num_sms, void* stream) {
  const few::Args a{(const uint8_t*)A, (const uint8_t*)B, (const uint8_t*)sa, (const uint8_t*)sb, lda, ldb, ldsa, ldsb, C, ldc, M, N, K,
                    f32, accumulate};
  if (((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(B)) & 15) != 0) return 5;
  const int k_blocks = (K + BLOCK - 1) / BLOCK;
  int warps = (N + few::ROWS - 1) / few::ROWS <= num_sms ? 16 : 8;  // 2048 x 2048, 8 tokens 4.4 / 4.9 us with 16 / 8; 4096 x 4096, one token 10.6 / 9.1
  if (warps > k_blocks) warps = k_blocks;
  cudaStream_t st = (cudaStream_t)stream;
  return M <= 8 ? few::launch<1>(a, a_fmt, b_fmt, warps, st) : few::launch<2>(a, a_fmt, b_fmt, warps, st);
}

}  // namespace f8b
}  // namespace kf
