// Codes of a paged 8-bit cache (quant8.cuh) as operands of the 5th-generation tensor cores: kind::f8f6f4 products, descriptors
// of tiles as TMA leaves them, tensor maps of the pages, and numbers as two codes whose sum they are.
#pragma once
#include "quant8.cuh"
#include "tcgen05.cuh"

// A tile's row is D bytes: one swizzled row of 128 bytes (D = 128) or of 64 (D = 64).
template <int D> struct Q8Tile {
  static_assert(D == 64 || D == 128, "rows of 64 or 128 codes");
  static constexpr int KEYS = 128;
  static constexpr int BYTES = KEYS * D;
  static constexpr int GROUP = 8 * D;                          // eight rows
  static constexpr uint64_t LAYOUT = D == 128 ? 2 : 4;         // 128- or 64-byte swizzle
  // where 16-byte piece `piece` of row `row` lies
  static __device__ __forceinline__ int piece_at(int row, int piece) {
    return row * D + ((D == 128 ? piece ^ (row & 7) : piece ^ ((row >> 1) & 3)) << 4);
  }
};

__device__ __forceinline__ uint64_t q8_desc(uint32_t addr, uint32_t leading, uint32_t stride, uint64_t layout) {
  return (uint64_t)((addr & 0x3FFFF) >> 4) | (uint64_t)(leading >> 4) << 16 | (uint64_t)(stride >> 4) << 32 | (uint64_t)1 << 46 | layout << 61;
}
// e4m3 x e4m3 -> f32, M = m, N = n; a_mn: the A operand lies M-major (a row per k), b_mn: the B operand N-major.
__host__ __device__ constexpr uint32_t q8_instr(int m, int n, bool a_mn, bool b_mn) {
  return (1u << 4) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// D[tmem] (+)= A B over 32 k's, both operands from shared memory.  Called by a converged warp, one lane issues.
__device__ __forceinline__ void umma_q8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(tmem_d),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(0u)
      : "memory");
}

// A number of up to 448 as the sum of two codes: the nearest one, and the one nearest to what is left.  A number of eight
// significant bits (a bfloat16) is hit exactly down to 2^-2, any other to 2^-8 of itself or 2^-10, whichever is more.
__device__ __forceinline__ void q8_split4(const float (&x)[4], uint32_t& high, uint32_t& low) {
  high = q8_encode4(x[0], x[1], x[2], x[3]);
  const float4 h = q8_decode4(high);
  low = q8_encode4(x[0] - h.x, x[1] - h.y, x[2] - h.z, x[3] - h.w);
}

__device__ __forceinline__ float warp_max_number(float v) {      // a NaN is passed over
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// Codes [rows, D]: boxes of `box_rows` whole rows.
template <int D>
static inline int q8_make_map(CUtensorMap* map, const void* base, long long rows, int box_rows) {
  LabEncodeTiledFn fn = lab_encode_fn();
  if (!fn) return (int)cudaErrorNotSupported;
  cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)D};
  cuuint32_t box[2] = {(cuuint32_t)D, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : (int)cudaErrorInvalidValue;
}
static inline bool q8_pages_fit(int page_size, long long pool_rows) {
  return page_size >= 8 && page_size <= 128 && (page_size & (page_size - 1)) == 0 && pool_rows < (1ll << 31);
}
