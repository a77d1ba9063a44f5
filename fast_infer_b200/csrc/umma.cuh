// tcgen05 operand descriptors shared by the tensor-core attention kernels: 128-byte
// swizzled shared-memory tiles and the f16-kind instruction descriptor.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace fi {

// Shared-memory matrix descriptor, 128-byte swizzle (sm_100 "version 1" format):
// start address, leading / stride byte offsets (16-byte units), layout type 2.
__device__ __forceinline__ uint64_t umma_desc_sw128(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr >> 4) & 0x3FFFu);
  d |= (uint64_t)((lbo >> 4) & 0x3FFFu) << 16;
  d |= (uint64_t)((sbo >> 4) & 0x3FFFu) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

// 16-bit storage types of Q, K, V and O.
template <typename T>
struct Half16;
template <>
struct Half16<__half> {
  static constexpr uint32_t kUmmaFormat = 0;
  static constexpr CUtensorMapDataType kTmap = CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  __device__ static __forceinline__ uint32_t pack(float lo, float hi) { return pack_half2(lo, hi); }
};
template <>
struct Half16<__nv_bfloat16> {
  static constexpr uint32_t kUmmaFormat = 1;
  static constexpr CUtensorMapDataType kTmap = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  __device__ static __forceinline__ uint32_t pack(float lo, float hi) {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  }
};

// Instruction descriptor of kind::f16 with fp32 accumulation: operand type T for both A
// and B, operand majorness per argument (0 = K-major, 1 = MN-major).
template <typename T>
__host__ __device__ constexpr uint32_t umma_idesc(uint32_t m, uint32_t n, uint32_t a_mn_major,
                                                  uint32_t b_mn_major) {
  return (1u << 4) | (Half16<T>::kUmmaFormat << 7) | (Half16<T>::kUmmaFormat << 10) |
         (a_mn_major << 15) | (b_mn_major << 16) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

}  // namespace fi
