// bf16 -> the 8-bit form with a scale for each block of 128 (fp8_blocks.cuh): the cast of a matrix, row-major and transposed, the
// residual's addition and RMSNorm that end in it, and the way back.
//
//   cast    q = round8(x 2^-e), e from the largest magnitude of a block: 1 x 128 (activations, gradients) or 128 x 128 (weights, whose two
//           copies then hold the same values).  A transposed copy of 1 x 128 blocks has blocks of 128 along the rows of x.
//   norm    t = bf16(x + residual), rstd = 1 / sqrt(mean(t^2) + eps), h = cast(t gain rstd), rounded once (in the transposed copy that a
//           backward pass makes of t and rstd twice: to 32 bits, then to 8)
//   norm's gradients  dx = dt + rstd (dh gain - t rstd^2 mean(dh gain t)), dgain = sum over rows of dh t rstd, of dh in 32 bits
//
// The kernels are programmatic launches, so no pointer is promised to be the only one to its memory: a load under that promise may be moved
// before the wait for the kernel that writes it.
//
// An infinity or a NaN is stored as NaN, and the other values of its block are scaled as if it were not there.
#include "fp8_blocks.cuh"

#include <type_traits>

namespace kf {
namespace f8b {

enum Source { PLAIN = 0, NORMED = 1 };  // the matrix itself, or x * rstd[row] * gain[column]

__device__ __forceinline__ float2 pair_at(const uint4& v, int j) { return unpack_bf16(j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w); }

// largest magnitude over the 16 lanes of a half warp
__device__ __forceinline__ float half_warp_max(float m) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) m = max_abs(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}
// of pairs of bf16 (a NaN counts for nothing)
__device__ __forceinline__ uint32_t max_abs2(uint32_t m, uint32_t v) {
  const __nv_bfloat162 r = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&m), __habs2(*reinterpret_cast<const __nv_bfloat162*>(&v)));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// One 128 x 128 tile per block of 512 threads: 16 threads x 8 columns, rows ty, ty + 32, ty + 64 and ty + 96 of a thread.
//
// Bound by memory: 2 bytes in, 1 or 2 out per element, and all of them pass through registers, so what counts is how many blocks an SM
// holds while others wait (registers: two to four) and how little is done per value: maxima of bf16 values are taken in pairs as they
// are, and infinities have a path of their own.  16 384 x 4096, us (at the copy rate): row-major 34 (31), transposed 40 (31), both 56 (41),
// squares both 48 (41), normed 51 (31); with 256 threads, two blocks on an SM and a look at each value for infinities 60, 68, 84, 59 and 128.
template <bool E5M2, int SRC, bool SQUARE, bool ROW, bool T>
__global__ void __launch_bounds__(512, ROW && !T ? 4 : SRC == NORMED ? 2 : 3)
kf_cast_blocks(const __nv_bfloat16* x, int rows, int cols, long long ldx, const float* rstd,
               const __nv_bfloat16* gain, uint8_t* out, long long ld_out, uint8_t* scales,
               long long ld_scales, uint8_t* out_t, long long ld_t, uint8_t* scales_t, long long ld_scales_t) {
  constexpr int PER = 4;  // rows of a thread
  __shared__ uint32_t tile[T ? 128 : 1][32];               // bytes of the tile on their way to the transposed copy
  __shared__ float part[T && !SQUARE ? 16 : 1][128];       // column maxima of each warp
  __shared__ float col_inv[128];
  __shared__ uint8_t row_byte[128], col_byte[128];
  __shared__ float red[16];
  const int r0 = blockIdx.y * 128, c0 = blockIdx.x * 128;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int c = c0 + tx * 8;
  const bool wide_in = c + 7 < cols && (ldx & 7) == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  wait_for_previous();
  let_next_in();
  uint4 v[PER];
  float s[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int r = r0 + ty + 32 * i;
    v[i] = make_uint4(0, 0, 0, 0);
    if (r < rows) {
      const __nv_bfloat16* p = x + size_t(r) * ldx + c;
      if (wide_in) {
        v[i] = *reinterpret_cast<const uint4*>(p);
      } else {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c + e < cols) w[e >> 1] |= uint32_t(*reinterpret_cast<const unsigned short*>(p + e)) << (16 * (e & 1));
        v[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    if (SRC == NORMED) s[i] = rstd[min(r, rows - 1)];
  }
  float g[8];
  if (SRC == NORMED) {
#pragma unroll
    for (int e = 0; e < 8; ++e) g[e] = __bfloat162float(gain[min(c + e, cols - 1)]);
  }
  // Two neighbouring values.  Of normed ones the first product is exact, the second is rounded to 32 bits and taken with the 32 bits of rstd that
  // are kept, where the norm kernel, which has the row's sum, keeps what is cut off: next to a border of two 8-bit numbers, 17 of 25
  // million values, the transposed copy has the neighbour of the byte that the formula and the forward pass give.
  auto value2 = [&](int i, int j) {
    float2 p = pair_at(v[i], j);
    if (SRC == NORMED) p = make_float2(mul_full(mul_full(p.x, g[2 * j]), s[i]), mul_full(mul_full(p.y, g[2 * j + 1]), s[i]));
    return p;
  };
  // maxima of the thread's part of each row, and of its columns
  float row_max[PER], col_max[8];
  if (SRC == PLAIN) {
    uint32_t rm[PER], cm[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      rm[i] = 0;
      const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (ROW || SQUARE) rm[i] = max_abs2(rm[i], w[j]);
        if (T && !SQUARE) cm[j] = max_abs2(cm[j], w[j]);
      }
    }
    if (ROW || SQUARE) {  // two rows to a word
#pragma unroll
      for (int i = 0; i < PER; i += 2) {
        uint32_t m = max_abs2(__byte_perm(rm[i], rm[i + 1], 0x5410), __byte_perm(rm[i], rm[i + 1], 0x7632));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = max_abs2(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float2 f = unpack_bf16(m);
        row_max[i] = f.x;
        row_max[i + 1] = f.y;
      }
    }
    if (T && !SQUARE) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = unpack_bf16(max_abs2(cm[j], __shfl_xor_sync(0xffffffffu, cm[j], 16)));
        col_max[2 * j] = f.x;
        col_max[2 * j + 1] = f.y;
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) col_max[e] = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = value2(i, j);
        col_max[2 * j] = max_abs(col_max[2 * j], f.x);
        col_max[2 * j + 1] = max_abs(col_max[2 * j + 1], f.y);
      }
#pragma unroll
    for (int e = 0; e < 8; ++e) col_max[e] = max_abs(col_max[e], __shfl_xor_sync(0xffffffffu, col_max[e], 16));
  }
  bool any_inf = false;
  if (ROW || SQUARE) {
#pragma unroll
    for (int i = 0; i < PER; ++i) any_inf |= is_inf(row_max[i]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) any_inf |= is_inf(col_max[e]);
  }
  any_inf = __syncthreads_or(any_inf);
  if (any_inf) {  // rare: once more, over the finite values
#pragma unroll
    for (int e = 0; e < 8; ++e) col_max[e] = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      float m = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float2 f = value2(i, j);
        f = make_float2(nan_if_inf(f.x), nan_if_inf(f.y));
        m = max_abs(max_abs(m, f.x), f.y);
        col_max[2 * j] = max_abs(col_max[2 * j], f.x);
        col_max[2 * j + 1] = max_abs(col_max[2 * j + 1], f.y);
      }
      row_max[i] = half_warp_max(m);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) col_max[e] = max_abs(col_max[e], __shfl_xor_sync(0xffffffffu, col_max[e], 16));
  }
  float block_inv = 0.f;
  uint32_t block_byte = 0;
  if (SQUARE) {
    float m = max_abs(max_abs(row_max[0], row_max[1]), max_abs(row_max[2], row_max[3]));
    m = max_abs(m, __shfl_xor_sync(0xffffffffu, m, 16));
    if (lane == 0) red[warp] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 16; ++w) m = max_abs(m, red[w]);
    block_byte = scale_byte<E5M2>(m);
    block_inv = inverse_of(block_byte);
  } else if (T) {
    if (lane < 16) {
      *reinterpret_cast<float4*>(&part[warp][tx * 8]) = make_float4(col_max[0], col_max[1], col_max[2], col_max[3]);
      *reinterpret_cast<float4*>(&part[warp][tx * 8 + 4]) = make_float4(col_max[4], col_max[5], col_max[6], col_max[7]);
    }
    __syncthreads();
    if (threadIdx.x < 128) {
      float m = 0.f;
#pragma unroll
      for (int k = 0; k < 16; ++k) m = max_abs(m, part[k][threadIdx.x]);
      const uint32_t b = scale_byte<E5M2>(m);
      col_byte[threadIdx.x] = uint8_t(b);
      col_inv[threadIdx.x] = inverse_of(b);
    }
    __syncthreads();
  }
  float ci[8];
  if (T && !SQUARE) {
    const float4 lo = *reinterpret_cast<const float4*>(&col_inv[tx * 8]), hi = *reinterpret_cast<const float4*>(&col_inv[tx * 8 + 4]);
    ci[0] = lo.x; ci[1] = lo.y; ci[2] = lo.z; ci[3] = lo.w;
    ci[4] = hi.x; ci[5] = hi.y; ci[6] = hi.z; ci[7] = hi.w;
  }
  const bool wide_out = c + 7 < cols && (ld_out & 7) == 0 && (reinterpret_cast<uintptr_t>(out) & 7) == 0;
  // with_inf: infinities are looked for, which costs as much again as all that is done otherwise
  auto give = [&](auto with_inf) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int rl = ty + 32 * i, r = r0 + rl;
      uint32_t q[2] = {0, 0}, qt[2] = {0, 0};
      float inv = block_inv;
      if (ROW && !SQUARE) {
        const uint32_t b = scale_byte<E5M2>(row_max[i]);
        inv = inverse_of(b);
        if (tx == 0) row_byte[rl] = uint8_t(b);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float2 f = value2(i, j);
        if (decltype(with_inf)::value) f = make_float2(nan_if_inf(f.x), nan_if_inf(f.y));
        if (ROW || SQUARE) q[j >> 1] |= to_bytes<E5M2>(mul_full(f.x, inv), mul_full(f.y, inv)) << (16 * (j & 1));
        if (T && !SQUARE) qt[j >> 1] |= to_bytes<E5M2>(mul_full(f.x, ci[2 * j]), mul_full(f.y, ci[2 * j + 1])) << (16 * (j & 1));
      }
      if (ROW && r < rows) {
        uint8_t* o = out + size_t(r) * ld_out + c;
        if (wide_out) {
          *reinterpret_cast<uint2*>(o) = make_uint2(q[0], q[1]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (c + e < cols) o[e] = uint8_t(q[e >> 2] >> (8 * (e & 3)));
        }
      }
      // word w of row r at w ^ 2 * (r / 8 % 16): the 32 lanes of a transposed read hit 32 different banks
      if (T) *reinterpret_cast<uint2*>(&tile[rl][(tx * 2) ^ (((rl >> 3) & 15) << 1)]) = SQUARE ? make_uint2(q[0], q[1]) : make_uint2(qt[0], qt[1]);
    }
  };
  if (any_inf) give(std::true_type{});
  else give(std::false_type{});
  __syncthreads();
  if (ROW && threadIdx.x < 128) {
    const int r = r0 + threadIdx.x;
    if (r < rows) scales[blockIdx.x * ld_scales + r] = SQUARE ? uint8_t(block_byte) : row_byte[threadIdx.x];
  } else if (T && threadIdx.x >= 128 && threadIdx.x < 256) {
    const int k = threadIdx.x - 128;
    if (c0 + k < cols) scales_t[blockIdx.y * ld_scales_t + c0 + k] = SQUARE ? uint8_t(block_byte) : col_byte[k];
  }
  if (!T) return;
  const int rg = lane & 15, cg = warp * 2 + (lane >> 4);  // 8 source rows x 4 source columns per thread
  uint32_t t[4][2];                                       // [column][word of four rows]
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t a[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = tile[rg * 8 + i * 4 + j][cg ^ (rg << 1)];
    const uint32_t p0 = __byte_perm(a[0], a[1], 0x5140), p1 = __byte_perm(a[0], a[1], 0x7362);
    const uint32_t p2 = __byte_perm(a[2], a[3], 0x5140), p3 = __byte_perm(a[2], a[3], 0x7362);
    t[0][i] = __byte_perm(p0, p2, 0x5410);
    t[1][i] = __byte_perm(p0, p2, 0x7632);
    t[2][i] = __byte_perm(p1, p3, 0x5410);
    t[3][i] = __byte_perm(p1, p3, 0x7632);
  }
  const int r = r0 + rg * 8;
  const bool wide_t = r + 7 < rows && (ld_t & 7) == 0 && (reinterpret_cast<uintptr_t>(out_t) & 7) == 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int oc = c0 + cg * 4 + j;
    if (oc >= cols) continue;
    uint8_t* o = out_t + size_t(oc) * ld_t + r;
    if (wide_t) {
      *reinterpret_cast<uint2*>(o) = make_uint2(t[j][0], t[j][1]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (r + e < rows) o[e] = uint8_t(t[j][e >> 2] >> (8 * (e & 3)));
    }
  }
}

// Sum over the threads of a block, in T; `red` is free again for the block after the next barrier.
template <int THREADS, class T>
__device__ __forceinline__ T block_sum(T v, T* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (THREADS <= 32) return v;
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) v += red[w];
  return v;
}

// the square of a bf16's magnitude (the low 16 bits of w, or the high ones) in 64 bits; subnormal numbers and zeros count as 2^-127 or a little
// more, whose squares are nothing in the 32 bits that a sum ends in, infinities and NaN as 2^128
__device__ __forceinline__ double square64(uint32_t w, bool high) {
  const uint32_t u = high ? (w >> 3) & 0x0fffe000u : (w & 0x7fffu) << 13;
  const double a = __hiloint2double(int(u + (uint32_t(1023 - 127) << 20)), 0);
  return a * a;
}
// p (hi + lo) on its way to 8 bits: towards zero, and odd where anything was cut off, which tells any shorter rounding on which side of a border
// the product is.  p has 16 bits, hi + lo 48, so only a hi of up to 8 bits without a lo can be exact (cut = 0).
__device__ __forceinline__ float times_odd(float p, float hi, float lo, uint32_t cut) {
  float r;
  asm("fma.rz.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(p), "f"(hi), "f"(mul_full(p, lo)));
  return __uint_as_float(__float_as_uint(r) | cut);
}

// One row per block of THREADS threads, VPT vectors of eight columns per thread held in registers; 16 neighbouring threads have a block
// of 128 columns between them.  Vector c of a thread is c * THREADS + thread.
//
// Bound by memory, 4 bytes an element in and 3 out, and by the instructions (82 % of the issue slots); few rows by the chain load - sum - store.
// EARLY reads the gain with the row instead of after the sum, for 20 more registers: us, with / without, 1 x 4096 2.5 / 3.2, 777 x 5120 8.3 / 8.9,
// 2048 x 2048 7.6 / 8.8, 4096 x 4096 22.6 / 22.9, 777 x 6144 9.3 / 9.2, 8192 x 5120 53 / 50, 16 384 x 4096 77 / 73 (at the copy rate 0.01, 4.3, 4.5, 18,
// 5, 45, 72).  A row has as many warps as hold it: with 256 threads for 5120 columns 777 rows are 9.2, with 128 for 2048 columns 2048 rows 9.7, for
// 2560 8192 rows 33 (29 so).  The sum and rstd in 64 bits and the products that keep what they cut off cost 2 to 7 % (16 384 x 4096 72.6, 777 x
// 5120 8.6 in 32 bits, where one byte in two million was the neighbour of the right one).
constexpr long long EARLY_THREADS = 1 << 18;  // rows x threads that the SMs hold at once
template <int THREADS, int VPT, bool EARLY>
__global__ void __launch_bounds__(THREADS)
kf_add_rmsnorm_blocks(const __nv_bfloat16* x, const __nv_bfloat16* residual, const __nv_bfloat16* gain,
                      __nv_bfloat16* t_out, float* rstd_out, uint8_t* out, long long ld_out,
                      uint8_t* scales, long long ld_scales, int D, double per_D, double eps) {
  __shared__ double red[32];
  const size_t row = blockIdx.x;
  const int nvec = D >> 3;
  const __nv_bfloat16* xr = x + row * D;
  wait_for_previous();
  let_next_in();
  uint4 v[VPT], rv[VPT], gv[VPT];
#pragma unroll
  for (int c = 0; c < VPT; ++c) {
    const int i = threadIdx.x + c * THREADS;
    v[c] = rv[c] = gv[c] = make_uint4(0, 0, 0, 0);
    if (i < nvec) {
      v[c] = *reinterpret_cast<const uint4*>(xr + i * 8);
      if (residual) rv[c] = *reinterpret_cast<const uint4*>(residual + row * D + i * 8);
    }
  }
#pragma unroll
  for (int c = 0; c < VPT; ++c)
    if (const int i = threadIdx.x + c * THREADS; EARLY && i < nvec) gv[c] = *reinterpret_cast<const uint4*>(gain + i * 8);
  double sum = 0.;
#pragma unroll
  for (int c = 0; c < VPT; ++c) {
    const int i = threadIdx.x + c * THREADS;
    if (residual) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 a = pair_at(v[c], j), b = pair_at(rv[c], j);
        w[j] = pack_bf16(add_full(a.x, b.x), add_full(a.y, b.y));
      }
      v[c] = make_uint4(w[0], w[1], w[2], w[3]);
      if (i < nvec) *reinterpret_cast<uint4*>(t_out + row * D + i * 8) = v[c];
    }
    if (i < nvec) {
      const uint32_t w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
      double even = 0., odd = 0.;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        even += square64(w[j], false);
        odd += square64(w[j], true);
      }
      sum += even + odd;
    }
  }
  // rstd = r + lo: its 24th bit says, for values next to a border, which of two 8-bit neighbours they go to, and with it they go where the
  // formula says.  One step of Newton's iteration for 1 / sqrt from the nearest 32-bit number.
  double mean = block_sum<THREADS>(sum, red) * per_D + eps;
  if (mean > 3.4e38) {  // infinities, NaN and sums that 32 bits do not hold: as they are there
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < VPT; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 a = pair_at(v[c], j);
        ss += a.x * a.x + a.y * a.y;
      }
    __syncthreads();
    mean = block_sum<THREADS>(double(ss), red) * per_D + eps;
  }
  const float first = __frsqrt_rn(float(mean));
  float r = first, lo = 0.f;
  if (first > 0.f && first <= 3.4e38f) {
    const double y = first;
    lo = first * (0.5f * float(1. - mean * (y * y)));
    r = add_full(first, lo);
    lo = add_full(lo, add_full(first, -r));
  }
  const uint32_t cut = lo == 0.f && (__float_as_uint(r) & 0xffffu) == 0 ? 0u : 1u;
  if (threadIdx.x == 0 && rstd_out) rstd_out[row] = r;
  const float largest = __uint_as_float(0x7f7fffffu);
#pragma unroll
  for (int c = 0; c < VPT; ++c) {
    const int i = threadIdx.x + c * THREADS;
    if (!EARLY && i < nvec) gv[c] = *reinterpret_cast<const uint4*>(gain + i * 8);
    float f[8], m = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 a = pair_at(v[c], j), g = pair_at(gv[c], j);
      f[2 * j] = times_odd(mul_full(a.x, g.x), r, lo, cut);  // the first product is exact: 16 bits
      f[2 * j + 1] = times_odd(mul_full(a.y, g.y), r, lo, cut);
      m = max_abs(max_abs(m, f[2 * j]), f[2 * j + 1]);
    }
    m = half_warp_max(m);
    // rare: towards zero, what 32 bits do not hold ends on their largest number.  (A half warp without one gets the same maximum again.)
    if (__any_sync(0xffffffffu, m >= largest)) {
      m = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (fabsf(f[e]) >= largest) f[e] = __uint_as_float(0x7fffffffu);
        m = max_abs(m, f[e]);
      }
      m = half_warp_max(m);
    }
    if (__float_as_uint(m) <= 1u) m = 0.f;  // zeros with their last bit set
    const uint32_t b = scale_byte<false>(m);
    const float inv = inverse_of(b);
    if (i < nvec) {
      uint32_t q[2] = {0, 0};
#pragma unroll
      for (int j = 0; j < 4; ++j) q[j >> 1] |= to_bytes<false>(mul_full(f[2 * j], inv), mul_full(f[2 * j + 1], inv)) << (16 * (j & 1));
      *reinterpret_cast<uint2*>(out + row * ld_out + i * 8) = make_uint2(q[0], q[1]);
      if ((i & 15) == 0) scales[(i >> 4) * ld_scales + row] = uint8_t(b);
    }
  }
}

// Gradients of RMSNorm from dh in 32 bits, one pass: a block walks over rows, keeps its columns' part of the gain's gradient in registers and
// leaves it in partial[block][column] for kf_column_sums.  dh as a product leaves it, unrounded: rounded to 16 bits on the way it moves the
// gain's gradient, a sum over thousands of rows that cancel, by as much as the gradient's own rounding does.
// Bound by memory, 10 bytes an element (dt given), and by the wait of a row for its own sum: three blocks on an SM take turns (four of 64
// registers spill, and gain nothing).  us (at the copy rate; the two passes that there were over dh in 16 bits): 16 384 x 4096 120 (103; 159),
// 4096 x 4096 37 (26; 49), 16 384 x 768 28 (19; 74), 999 x 768 8.2 (1.2; 11.7).
template <int THREADS, int VPT, int BLOCKS>
__global__ void __launch_bounds__(THREADS, BLOCKS)
kf_norm_grads(const float* dh, const __nv_bfloat16* t, const __nv_bfloat16* gain, const float* rstd, const __nv_bfloat16* dt, __nv_bfloat16* dx,
              float* partial, int rows, int D) {
  __shared__ float red[2][32];
  const int nvec = D >> 3;
  wait_for_previous();
  let_next_in();
  float sum[VPT][8] = {};
  int turn = 0;
  for (int row = blockIdx.x; row < rows; row += gridDim.x, turn ^= 1) {
    const size_t at = size_t(row) * D;
    float4 a[VPT][2];
    uint4 tv[VPT], iv[VPT], gv[VPT];
#pragma unroll
    for (int c = 0; c < VPT; ++c) {
      const int i = threadIdx.x + c * THREADS;
      a[c][0] = a[c][1] = make_float4(0.f, 0.f, 0.f, 0.f);
      tv[c] = iv[c] = gv[c] = make_uint4(0, 0, 0, 0);
      if (i < nvec) {
        a[c][0] = *reinterpret_cast<const float4*>(dh + at + i * 8);
        a[c][1] = *reinterpret_cast<const float4*>(dh + at + i * 8 + 4);
        tv[c] = *reinterpret_cast<const uint4*>(t + at + i * 8);
        if (dt) iv[c] = *reinterpret_cast<const uint4*>(dt + at + i * 8);
        gv[c] = *reinterpret_cast<const uint4*>(gain + i * 8);
      }
    }
    const float r = rstd[row];
    float dot = 0.f;
#pragma unroll
    for (int c = 0; c < VPT; ++c) {
      const float d[8] = {a[c][0].x, a[c][0].y, a[c][0].z, a[c][0].w, a[c][1].x, a[c][1].y, a[c][1].z, a[c][1].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 x = pair_at(tv[c], j), g = pair_at(gv[c], j);
        dot += d[2 * j] * (g.x * x.x);
        dot += d[2 * j + 1] * (g.y * x.y);
        sum[c][2 * j] += d[2 * j] * (x.x * r);
        sum[c][2 * j + 1] += d[2 * j + 1] * (x.y * r);
      }
    }
    const float coef = block_sum<THREADS>(dot, red[turn]) / float(D) * r * r * r;
#pragma unroll
    for (int c = 0; c < VPT; ++c) {
      const int i = threadIdx.x + c * THREADS;
      const float d[8] = {a[c][0].x, a[c][0].y, a[c][0].z, a[c][0].w, a[c][1].x, a[c][1].y, a[c][1].z, a[c][1].w};
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 x = pair_at(tv[c], j), g = pair_at(gv[c], j), in = pair_at(iv[c], j);
        w[j] = pack_bf16(in.x + (r * (d[2 * j] * g.x) - x.x * coef), in.y + (r * (d[2 * j + 1] * g.y) - x.y * coef));
      }
      if (i < nvec) *reinterpret_cast<uint4*>(dx + at + i * 8) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
#pragma unroll
  for (int c = 0; c < VPT; ++c) {
    const int i = threadIdx.x + c * THREADS;
    if (i < nvec) {
      float* p = partial + size_t(blockIdx.x) * D + i * 8;
      *reinterpret_cast<float4*>(p) = make_float4(sum[c][0], sum[c][1], sum[c][2], sum[c][3]);
      *reinterpret_cast<float4*>(p + 4) = make_float4(sum[c][4], sum[c][5], sum[c][6], sum[c][7]);
    }
  }
}

// The same of rows of more than 16 384 columns, whose data registers do not hold: the gain's sums are in shared memory, each column's with the one
// thread that has it, and a row is read twice, the second time from L2.  us (at the copy rate): 2048 x 32 768 142 (103).  (1024 threads with the
// data in registers serve up to 16 384 columns: 4096 x 12 288 124 (77), 4096 x 16 384 136 (103).  Rounding dh to bf16 for the two passes over such
// values, as the layers did for more than 8192 columns, lost what cancels in the gain's gradient and took 167, 216 and 245.)
__global__ void __launch_bounds__(1024)
kf_norm_grads_wide(const float* dh, const __nv_bfloat16* t, const __nv_bfloat16* gain, const float* rstd, const __nv_bfloat16* dt, __nv_bfloat16* dx,
                   float* partial, int rows, int D) {
  extern __shared__ float4 sums[];  // [half of a vector of eight][vector]
  __shared__ float red[2][32];
  const int nvec = D >> 3;
  for (int i = threadIdx.x; i < nvec; i += 1024) sums[i] = sums[nvec + i] = make_float4(0.f, 0.f, 0.f, 0.f);
  wait_for_previous();
  let_next_in();
  int turn = 0;
  for (int row = blockIdx.x; row < rows; row += gridDim.x, turn ^= 1) {
    const size_t at = size_t(row) * D;
    const float r = rstd[row];
    float4 a[2][2];
    uint4 tv[2], gv[2], iv[2];
    // two vectors of this thread, dt's too where it is asked for
    auto load = [&](int i0, const __nv_bfloat16* in) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int i = i0 + c * 1024;
        a[c][0] = a[c][1] = make_float4(0.f, 0.f, 0.f, 0.f);
        tv[c] = gv[c] = iv[c] = make_uint4(0, 0, 0, 0);
        if (i < nvec) {
          a[c][0] = *reinterpret_cast<const float4*>(dh + at + i * 8);
          a[c][1] = *reinterpret_cast<const float4*>(dh + at + i * 8 + 4);
          tv[c] = *reinterpret_cast<const uint4*>(t + at + i * 8);
          gv[c] = *reinterpret_cast<const uint4*>(gain + i * 8);
          if (in) iv[c] = *reinterpret_cast<const uint4*>(in + at + i * 8);
        }
      }
    };
    float dot = 0.f;
#pragma unroll 1
    for (int i0 = threadIdx.x; i0 < nvec; i0 += 2048) {
      load(i0, nullptr);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int i = i0 + c * 1024;
        const float d[8] = {a[c][0].x, a[c][0].y, a[c][0].z, a[c][0].w, a[c][1].x, a[c][1].y, a[c][1].z, a[c][1].w};
        float s[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 x = pair_at(tv[c], j), g = pair_at(gv[c], j);
          dot += d[2 * j] * (g.x * x.x);
          dot += d[2 * j + 1] * (g.y * x.y);
          s[2 * j] = d[2 * j] * (x.x * r);
          s[2 * j + 1] = d[2 * j + 1] * (x.y * r);
        }
        if (i < nvec) {
          const float4 lo = sums[i], hi = sums[nvec + i];
          sums[i] = make_float4(lo.x + s[0], lo.y + s[1], lo.z + s[2], lo.w + s[3]);
          sums[nvec + i] = make_float4(hi.x + s[4], hi.y + s[5], hi.z + s[6], hi.w + s[7]);
        }
      }
    }
    const float coef = block_sum<1024>(dot, red[turn]) / float(D) * r * r * r;
#pragma unroll 1
    for (int i0 = threadIdx.x; i0 < nvec; i0 += 2048) {
      load(i0, dt);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int i = i0 + c * 1024;
        const float d[8] = {a[c][0].x, a[c][0].y, a[c][0].z, a[c][0].w, a[c][1].x, a[c][1].y, a[c][1].z, a[c][1].w};
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 x = pair_at(tv[c], j), g = pair_at(gv[c], j), in = pair_at(iv[c], j);
          w[j] = pack_bf16(in.x + (r * (d[2 * j] * g.x) - x.x * coef), in.y + (r * (d[2 * j + 1] * g.y) - x.y * coef));
        }
        if (i < nvec) *reinterpret_cast<uint4*>(dx + at + i * 8) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
  for (int i = threadIdx.x; i < nvec; i += 1024) {
    float* p = partial + size_t(blockIdx.x) * D + i * 8;
    *reinterpret_cast<float4*>(p) = sums[i];
    *reinterpret_cast<float4*>(p + 4) = sums[nvec + i];
  }
}

// out[column] = sum over parts of partial[part][column], 32 columns per block and every 32nd part per warp, in a fixed order
__global__ void __launch_bounds__(1024) kf_column_sums(const float* partial, int parts, int D, __nv_bfloat16* out) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  wait_for_previous();
  let_next_in();
  float v = 0.f;
  if (c < D) {
#pragma unroll 8
    for (int p = warp; p < parts; p += 32) v += partial[size_t(p) * D + c];
  }
  red[warp][lane] = v;
  __syncthreads();
  v = red[lane][warp];  // a warp per column
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (lane == 0 && blockIdx.x * 32 + warp < D) out[blockIdx.x * 32 + warp] = __float2bfloat16(v);
}

// The values that the bytes stand for, in bf16 (exact where bf16 has them): sixteen per thread, blocks of 16 x 16 threads on 256 columns.
// FAR: more of them than the y dimension holds go on in z (of up to z blocks too many no index passes 31 bits).
template <bool E5M2, bool FAR>
__global__ void __launch_bounds__(256)
kf_blocks_values(const uint8_t* q, long long ld, const uint8_t* scales, long long ld_scales, int rows, int cols,
                 __nv_bfloat16* out) {
  const int c = (FAR ? blockIdx.z * gridDim.y + blockIdx.y : blockIdx.y) * 256 + (threadIdx.x & 15) * 16, r = blockIdx.x * 16 + (threadIdx.x >> 4);
  wait_for_previous();
  let_next_in();
  if (c >= cols || r >= rows) return;
  const uint8_t* p = q + r * ld + c;
  __nv_bfloat16* o = out + (size_t)r * cols + c;
  const bool whole = c + 15 < cols;
  uint32_t w[4] = {0, 0, 0, 0};
  const uint32_t b = scales[(c >> 7) * ld_scales + r];
  if (whole && (ld & 15) == 0 && (reinterpret_cast<uintptr_t>(q) & 15) == 0) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (c + e < cols) w[e >> 2] |= uint32_t(p[e]) << (8 * (e & 3));
  }
  // a factor of 2^-127 (byte 0) has no normal 32-bit number: half of the next one, which subnormal arithmetic keeps
  const float f = b == 0 ? __uint_as_float(0x400000u) : b == 255 ? __uint_as_float(0x7fffffffu) : __uint_as_float(b << 23);
  uint32_t packed[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[j >> 1] >> (16 * (j & 1))), E5M2 ? __NV_E5M2 : __NV_E4M3);
    packed[j] = pack_bf16(mul_full(__half2float(__half(__half_raw{h.x})), f), mul_full(__half2float(__half(__half_raw{h.y})), f));
  }
  if (whole && (cols & 7) == 0) {
    *reinterpret_cast<uint4*>(o) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
    *reinterpret_cast<uint4*>(o + 8) = make_uint4(packed[4], packed[5], packed[6], packed[7]);
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (c + e < cols) reinterpret_cast<unsigned short*>(o)[e] = (unsigned short)(packed[e >> 1] >> (16 * (e & 1)));
  }
}

constexpr int GRID_Y = 65535;  // blocks in the y dimension of a grid

}  // namespace f8b
}  // namespace kf

extern "C" {

// Casts bf16 x[rows][cols] (pitch ldx elements), or x * rstd[row] * gain[column] where rstd is given (the transposed copy in e4m3 only).  out /
// scales: row-major copy (pitch ld_out) and its (ceil(cols / 128), rows) scale bytes (pitch ld_scales); out_t / scales_t: the transposed one, (cols,
// rows) and (ceil(rows / 128), cols); either may be null.  square: blocks of 128 x 128.
int kf_fp8_blocks_cast_bf16(const void* x, int rows, int cols, long long ldx, const void* rstd, const void* gain, int e5m2, int square,
                            void* out, long long ld_out, void* scales, long long ld_scales, void* out_t, long long ld_t, void* scales_t,
                            long long ld_scales_t, void* stream) {
  using namespace kf::f8b;
  if (rows <= 0 || cols <= 0 || rows > LARGEST || cols > LARGEST || (rstd == nullptr) != (gain == nullptr) || (!out && !out_t) ||
      (rstd && (square || e5m2 || out)))
    return 5;
  // rows that the y dimension does not hold are the next launch's: with them in a third dimension the cast took 2 % longer at every size
  auto go = [&](auto kern) {
    int rc = 0;
    for (long long r = 0; r < rows && !rc; r += 128 * GRID_Y) {
      const int n = int(rows - r < 128 * GRID_Y ? rows - r : 128 * GRID_Y);
      rc = launch_programmatic(kern, dim3((cols + 127) / 128, (n + 127) / 128), 512, 0, 1, (cudaStream_t)stream, (const __nv_bfloat16*)x + r * ldx, n,
                               cols, ldx, rstd ? (const float*)rstd + r : nullptr, (const __nv_bfloat16*)gain, out ? (uint8_t*)out + r * ld_out : nullptr,
                               ld_out, out ? (uint8_t*)scales + r : nullptr, ld_scales, out_t ? (uint8_t*)out_t + r : nullptr, ld_t,
                               out_t ? (uint8_t*)scales_t + r / 128 * ld_scales_t : nullptr, ld_scales_t);
    }
    return rc;
  };
  auto copies = [&](auto e5, auto sq) {
    constexpr bool E = decltype(e5)::value, S = decltype(sq)::value;
    if (!out_t) return go(kf_cast_blocks<E, PLAIN, S, true, false>);
    return out ? go(kf_cast_blocks<E, PLAIN, S, true, true>) : go(kf_cast_blocks<E, PLAIN, S, false, true>);
  };
  if (rstd) return go(kf_cast_blocks<false, NORMED, false, false, true>);
  if (square) return e5m2 ? copies(std::true_type{}, std::true_type{}) : copies(std::false_type{}, std::true_type{});
  return e5m2 ? copies(std::true_type{}, std::false_type{}) : copies(std::false_type{}, std::false_type{});
}

// t = bf16(x + residual) (x itself, and nothing is written, where residual is null), rstd, and RMSNorm(t) * gain in e4m3.  x, residual, t:
// contiguous rows of D bf16 values on 16 bytes, D a multiple of 8, at most 32 768; pitch ld_out a multiple of 8.
int kf_add_rmsnorm_fp8_blocks(const void* x, const void* residual, const void* gain, void* t, void* rstd, void* out, long long ld_out,
                              void* scales, long long ld_scales, int rows, int D, double eps, void* stream) {
  using namespace kf::f8b;
  if (rows <= 0 || D <= 0 || (D & 7) || D > 32768 || (ld_out & 7) ||
      ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) | reinterpret_cast<uintptr_t>(gain) | reinterpret_cast<uintptr_t>(t)) & 15) ||
      (reinterpret_cast<uintptr_t>(out) & 7) || (residual && !t))
    return 5;
  auto go = [&](auto kern, int threads) {
    return launch_programmatic(kern, dim3(unsigned(rows)), threads, 0, 1, (cudaStream_t)stream, (const __nv_bfloat16*)x, (const __nv_bfloat16*)residual,
                               (const __nv_bfloat16*)gain, (__nv_bfloat16*)t, (float*)rstd, (uint8_t*)out, ld_out, (uint8_t*)scales, ld_scales, D, 1. / D,
                               eps);
  };
  // as many warps as hold a row
  auto pick = [&](auto threads) {
    constexpr int N = decltype(threads)::value;
    return (long long)rows * N <= EARLY_THREADS ? go(kf_add_rmsnorm_blocks<N, 4, true>, N) : go(kf_add_rmsnorm_blocks<N, 4, false>, N);
  };
  const int warps = (D / 8 + 4 * 32 - 1) / (4 * 32);
  switch (warps) {
    case 1: return pick(std::integral_constant<int, 32>{});
    case 2: return pick(std::integral_constant<int, 64>{});
    case 3: return pick(std::integral_constant<int, 96>{});
    case 4: return pick(std::integral_constant<int, 128>{});
    case 5: return pick(std::integral_constant<int, 160>{});
    case 6: return pick(std::integral_constant<int, 192>{});
  }
  return warps <= 8 ? pick(std::integral_constant<int, 256>{})
                    : warps <= 16 ? pick(std::integral_constant<int, 512>{}) : pick(std::integral_constant<int, 1024>{});
}

// Blocks of kf_norm_grads_f32, each of which leaves D floats in `partial`: what the SMs hold, of four rows at least where that fills them.
int kf_norm_grads_blocks(int rows, int D, int num_sms) {
  int blocks = num_sms * (D <= 1024 ? 8 : D <= 4096 ? 3 : D <= 8192 ? 2 : 1);
  if (blocks > rows / 4) blocks = rows / 4 > num_sms ? rows / 4 : num_sms;
  return rows < 1 ? 1 : rows < blocks ? rows : blocks;
}

// dx (bf16) = dt (or 0 where null) + the gradient of RMSNorm at t for dh (fp32); dgain (bf16) of its gain.  Contiguous rows on 16 bytes, D a
// multiple of 8, at most 32 768.
int kf_norm_grads_f32(const void* dh, const void* t, const void* gain, const void* rstd, const void* dt, void* dx, void* partial, void* dgain, int rows,
                      int D, int num_sms, void* stream) {
  using namespace kf::f8b;
  if (rows <= 0 || D <= 0 || (D & 7) || D > 32768 ||
      ((reinterpret_cast<uintptr_t>(dh) | reinterpret_cast<uintptr_t>(t) | reinterpret_cast<uintptr_t>(gain) | reinterpret_cast<uintptr_t>(dt) |
        reinterpret_cast<uintptr_t>(dx) | reinterpret_cast<uintptr_t>(partial)) & 15))
    return 5;
  const int blocks = kf_norm_grads_blocks(rows, D, num_sms);
  cudaStream_t st = (cudaStream_t)stream;
  const size_t wide = D > 16384 ? size_t(D) * 4 : 0;  // bytes of shared memory
  if (wide) {
    static bool attr_set[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 64 || !attr_set[dev]) {
      const cudaError_t e = cudaFuncSetAttribute(kf_norm_grads_wide, cudaFuncAttributeMaxDynamicSharedMemorySize, 32768 * 4);
      if (e != cudaSuccess) return 300 + (int)e;
      if (dev < 64) attr_set[dev] = true;
    }
  }
  auto go = [&](auto kern, int threads) {
    return launch_programmatic(kern, dim3(unsigned(blocks)), threads, wide, 1, st, (const float*)dh, (const __nv_bfloat16*)t, (const __nv_bfloat16*)gain,
                               (const float*)rstd, (const __nv_bfloat16*)dt, (__nv_bfloat16*)dx, (float*)partial, rows, D);
  };
  const int rc = D <= 1024    ? go(kf_norm_grads<128, 1, 8>, 128)
                 : D <= 4096  ? go(kf_norm_grads<256, 2, 3>, 256)
                 : D <= 8192  ? go(kf_norm_grads<512, 2, 2>, 512)
                 : D <= 16384 ? go(kf_norm_grads<1024, 2, 1>, 1024)
                              : go(kf_norm_grads_wide, 1024);
  if (rc) return rc;
  return launch_programmatic(kf_column_sums, dim3((D + 31) / 32), 1024, 0, 1, st, (const float*)partial, blocks, D, (__nv_bfloat16*)dgain);
}

// out[rows][cols] (contiguous bf16) = the values that q (pitch ld) and its scale bytes stand for.
int kf_fp8_blocks_values_bf16(const void* q, long long ld, const void* scales, long long ld_scales, int rows, int cols, int e5m2, void* out,
                              void* stream) {
  using namespace kf::f8b;
  if (rows <= 0 || cols <= 0 || rows > LARGEST || cols > LARGEST || (reinterpret_cast<uintptr_t>(out) & 15)) return 5;
  // (an index of the z dimension, or a pitch apart from cols, in the kernel of all sizes cost it 1 %)
  const int n = (cols + 255) / 256, z = (n + GRID_Y - 1) / GRID_Y;
  auto kern = z > 1 ? (e5m2 ? kf_blocks_values<true, true> : kf_blocks_values<false, true>)
                    : (e5m2 ? kf_blocks_values<true, false> : kf_blocks_values<false, false>);
  return launch_programmatic(kern, dim3((rows + 15) / 16, (n + z - 1) / z, z), 256, 0, 1, (cudaStream_t)stream, (const uint8_t*)q, ld,
                             (const uint8_t*)scales, ld_scales, rows, cols, (__nv_bfloat16*)out);
}

}  // extern "C"
