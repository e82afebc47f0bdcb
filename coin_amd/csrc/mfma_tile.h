// Device helpers of the 32 x 32 matrix-tile kernels (attention.hip, linear.hip), for bfloat16 and float32: swizzled LDS images filled by
// the range-checked LDS-DMA, 16-byte row fragments and transposed fragments, and the matrix instructions that take them.
#pragma once
#include "common.h"
#include "conv_gemm_dev.h"

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

// this wave's DMA has landed and its LDS accesses are complete; behind the barrier everybody's have
#define TILE_WAIT()                                              \
  do {                                                                \
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");      \
    P8_BAR();                                                         \
  } while (0)

__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// 16-byte chunk c of row r of an image with ROWB-byte rows sits at chunk c ^ swz(r).  LDS serves 256 bytes (64 banks) at a time: the chunk c
// of 16 consecutive rows (a row fragment's quarter) and 64 bytes of 4 consecutive rows (half of a transposed fragment) must fall on
// different banks.  Rows of 256 bytes and more all start on bank 0: four bits of the row, the lowest two on the 64-byte segment; shorter rows
// lie on different banks by themselves as far as they go.  (Swizzles of eight 16-byte slots, as 128 bytes at a time would ask for, left every
// second LDS cycle a conflict.)
template <int ROWB>
__device__ __forceinline__ int swz(int r) {
  return ROWB == 64 ? (r >> 2) & 3 : ROWB == 128 ? ((r >> 1) & 1) << 2 | ((r >> 2) & 3) : (r & 3) << 2 | ((r >> 2) & 3);
}

// acc[i][j] += sum over the 16-byte fragments: A row i = lane & 31, B column j = lane & 31, contraction = 8 bf16 / 4 floats per lane half
template <typename T>
__device__ __forceinline__ void mma(f32x16& acc, const f32x4& a, const f32x4& b) {
  if constexpr (sizeof(T) == 2) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], acc, 0, 0, 0);
  }
}

// An image of `ROWS` rows.  PAD: every 1 KiB (one DMA instruction's rows) is followed by 16 bytes, which takes the place of the swizzle's lower
// two bits for 256-byte rows: what is left of the swizzle touches a chunk's upper bits alone, so a fragment's addresses are four registers and
// constant offsets instead of sixteen registers.
template <int ROWB, int ROWS, bool PAD = false>
struct Img {
  static_assert(!PAD || ROWB == 256, "");
  static constexpr int BLOCK = PAD ? 1040 : 1024, BYTES = ROWB * ROWS / 1024 * BLOCK;
  static __device__ __forceinline__ int key(int row) { return PAD ? (row & 3) << 2 : swz<ROWB>(row); }
  static __device__ __forceinline__ int row_at(int row) { return PAD ? (row >> 2) * BLOCK + (row & 3) * ROWB : row * ROWB; }
  // row fragment: 16 bytes of row `row`, chunk `chunk`
  static __device__ __forceinline__ f32x4 frag(const char* img, int row, int chunk) {
    return *reinterpret_cast<const f32x4*>(img + row_at(row) + ((chunk ^ key(row)) << 4));
  }
};

// rows 0 .. ROWS - 1 of a tile -> swizzled LDS image; rows >= nvalid and chunks >= nchunk arrive as zeros.  `off(row)` = byte offset of a
// row behind `base` (below 2^31: checked on the host)
template <int ROWB, int ROWS, int NW, bool PAD = false, typename OFF>
__device__ __forceinline__ void stage_tile(char* dst, const void* base, int nvalid, int nchunk, int wave, int lane, const OFF& off) {
  using I = Img<ROWB, ROWS, PAD>;
  constexpr int LPR = ROWB / 16, RPI = 64 / LPR, NI = ROWS / RPI;
  static_assert(ROWS % RPI == 0 && NI % NW == 0, "");
#pragma unroll
  for (int i = 0; i < NI / NW; ++i) {
    const int inst = wave * (NI / NW) + i;
    const int row = inst * RPI + lane / LPR;
    const int ch = (lane % LPR) ^ I::key(row);
    const unsigned o = row < nvalid && ch < nchunk ? off(row) + (unsigned)ch * 16u : P8_OOB;
    blds16(base, 0x7fffffffu, o, 0, dst + inst * I::BLOCK);
  }
}

template <typename T>
__device__ __forceinline__ void store4(T* p, float a, float b, float c, float d) {
  if constexpr (sizeof(T) == 2) {
    const bf16x4 o = {(bf16_t)a, (bf16_t)b, (bf16_t)c, (bf16_t)d};
    *reinterpret_cast<bf16x4*>(p) = o;
  } else {
    *reinterpret_cast<f32x4*>(p) = (f32x4){a, b, c, d};
  }
}

