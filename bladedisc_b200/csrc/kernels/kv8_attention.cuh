// What the two attention kernels of the 8-bit cache share.
#pragma once
#include "kv8.h"

#include "device_info.h"
#include "kv8_types.cuh"
#include "sm100_ptx.cuh"
#include "tensor_map.h"

namespace disc_b200 {

// One lane of a converged warp, the same each time.  Copies, products and commits behind it, in code that the whole warp
// runs with uniform values, issue back to back; behind `lane == 0` a commit cost 180 cycles of the tensor core and a
// copy 170 of its warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "}\n"
      : "=r"(r));
  return r != 0;
}
// Bytes b (as b + 128) `sel` picks two of them -> two f16 with the values b.
__device__ __forceinline__ uint32_t bytes_to_f16(uint32_t biased, uint32_t sel) {
  const uint32_t w = __byte_perm(biased, 0x64646464u, sel);
  const uint32_t c = 0x64806480u;  // 1152
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&w), *reinterpret_cast<const __half2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Largest magnitude of sixteen values, as its bits.
__device__ __forceinline__ uint32_t top_q16(const __nv_bfloat16* p) {
  float f[16];
  load8(p, f);
  load8(p + 8, f + 8);
  uint32_t t = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) t = max(t, __float_as_uint(f[i]) & 0x7fffffffu);
  return t;
}
// 2^n that brings a row with this largest magnitude to [2^13, 2^14); n stays within what a float holds.
__device__ __forceinline__ float row_power(uint32_t top) {
  const int n = min(max(13 - (static_cast<int>(top >> 23) - 127), -120), 120);
  return __uint_as_float(static_cast<uint32_t>(n + 127) << 23);
}

// One box is `rows` tokens of one block and head.
inline bool make_map(CUtensorMap* tm, const int8_t* base, const Kv8Cache& c, int rows) {
  EncodeTiledFn fn = tensor_map_encode_fn();
  if (!fn) return false;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(c.dim), static_cast<cuuint64_t>(c.block_size),
                        static_cast<cuuint64_t>(c.num_blocks) * c.kv_heads};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(c.dim), static_cast<cuuint64_t>(c.dim) * c.block_size};
  cuuint32_t box[3] = {static_cast<cuuint32_t>(c.dim), static_cast<cuuint32_t>(rows), 1};
  cuuint32_t estr[3] = {1, 1, 1};
  return fn(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<int8_t*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, c.dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Many rows: requests with more than min_rows query rows per kv head (kv8_prefill.cu).
int64_t kv8_prefill_workspace_bytes(const Kv8AttentionParams& p);
cudaError_t kv8_prefill_launch(const Kv8AttentionParams& p, int min_rows, void* workspace, cudaStream_t stream,
                               const char** err);
cudaError_t kv8_prefill_join_launch(const Kv8AttentionParams& p, int min_rows, void* workspace, cudaStream_t stream);

}  // namespace disc_b200
