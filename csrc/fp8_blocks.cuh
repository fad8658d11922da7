// The 8-bit form with a scale for each block of 128: a byte per value (e4m3 or e5m2) and, for every row and 128 columns, a byte b that
// stands for the factor 2^(b - 127).  Scale bytes are stored block-major, (ceil(cols / 128), rows), so that the 128 rows of a tile read
// theirs as one line.
//
// Why powers of two: the tensor cores multiply such factors into the sum of a block themselves (tcgen05.mma kind::mxf8f6f4), a value's
// bits do not depend on how its scale was rounded, and what a byte pair stands for is exact in bf16.
#pragma once
#include "common.cuh"
#include <cuda_fp8.h>

namespace kf {
namespace f8b {

constexpr int BLOCK = 128;
constexpr int LARGEST = 0x7fff0000;  // rows or columns: kernels add a few blocks to an index in 32 bits

// 32-bit arithmetic that keeps subnormal numbers, which the library's flags would flush
__device__ __forceinline__ float mul_full(float a, float b) {
  float r;
  asm("mul.rn.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float add_full(float a, float b) {
  float r;
  asm("add.rn.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_abs(float m, float v) {  // NaN counts for nothing
  float r;
  asm("{\n\t.reg .f32 t;\n\tabs.f32 t, %2;\n\tmax.f32 %0, %1, t;\n\t}" : "=f"(r) : "f"(m), "f"(v));
  return r;
}

// Scale byte of a block whose largest magnitude is a (finite): the least power of two, of at least 2^-126, that brings a to 448 or less
// (e4m3; 57 344 for e5m2).  Both are 1.75 times a power of two, so the exponent and one comparison of a's bits decide it exactly.
template <bool E5M2>
__device__ __forceinline__ uint32_t scale_byte(float a) {
  const uint32_t u = __float_as_uint(a);
  const int e = int(u >> 23) - (E5M2 ? 15 : 8) + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return u == 0 ? 127u : uint32_t(max(e, 1));
}
// the factor that divides by the scale: exact, and a normal number for every byte that scale_byte gives (1 .. 247)
__device__ __forceinline__ float inverse_of(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

__device__ __forceinline__ bool is_inf(float v) { return (__float_as_uint(v) & 0x7fffffffu) == 0x7f800000u; }
__device__ __forceinline__ float nan_if_inf(float v) { return is_inf(v) ? __uint_as_float(0x7fffffffu) : v; }

// two values as two bytes: nearest, ties to even
template <bool E5M2>
__device__ __forceinline__ uint32_t to_bytes(float a, float b) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, E5M2 ? __NV_E5M2 : __NV_E4M3);
}

// ------------------------------------------------------------------ programmatic launches
// A kernel so launched sets itself up while the one before it drains.  It waits before it reads or writes global memory, and lets the next
// one in only after that: whatever starts early finds every kernel but its immediate predecessor complete.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_in() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// kernel<<<grid, block, smem, stream>>>(args ..), in clusters of `cluster` blocks, as a programmatic launch
template <class... P, class... A>
int launch_programmatic(void (*kernel)(P...), dim3 grid, int block, size_t smem, int cluster, cudaStream_t stream, A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(unsigned(block));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = unsigned(cluster);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
  return e == cudaSuccess ? 0 : 400 + (int)e;
}

// ------------------------------------------------------------------ tcgen05
// Instruction descriptor for kind::mxf8f6f4: formats 0 = e4m3, 1 = e5m2, both K-major, scales as exponent bytes, byte 0 of each word; plus
// b of them, byte b.
constexpr uint32_t IDESC_NEXT_BYTE = (1u << 4) | (1u << 29);
__host__ __device__ constexpr uint32_t idesc_blocks(int m, int n, int a_fmt, int b_fmt) {
  return (uint32_t(a_fmt) << 7) | (uint32_t(b_fmt) << 10) | (uint32_t(n >> 3) << 17) | (1u << 23) | (uint32_t(m >> 4) << 24);
}
__device__ __forceinline__ void tmem_st_x4(uint32_t taddr, const uint32_t (&r)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}
__device__ __forceinline__ void tmem_st_x8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// rows x cols bytes, pitch ld -> tensor map with (box_cols x box_rows) boxes
inline int make_map_u8(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_cols, uint32_t box_rows,
                       bool swizzled) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return -1;
  cuuint64_t dims[2] = {cols, rows};
  cuuint64_t strides[1] = {ld};
  cuuint32_t box[2] = {box_cols, box_rows};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  swizzled ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : (int)r;
}

}  // namespace f8b
}  // namespace kf
