// Linear layer with its bias, activation and residual in the epilogue (coin_linear_fwd / _bwd), float32 and bfloat16:
//
//   z = x W^T + b,   y = residual + act(z);      dz = dy o act'(z),   dx = dz W,   dW = dz^T x,   db = sum_rows dz
//
// One matrix-product kernel serves the three products: an operand is read with the contraction along its rows (x and W of the forward,
// dz of dx) or across them (W of dx, both of dW).  Tiles go to LDS by the range-checked LDS-DMA as they lie in memory; the fragments of a
// tile whose contraction runs across the rows come out through the transposing LDS read (bfloat16) or column reads (float32), so no
// operand is ever transposed in memory.
//
// The forward keeps act'(z) where a gradient will be asked for, in half precision for bfloat16 tensors: off by 2^-11 of its value at most, an
// eighth of what rounding dz to bfloat16 costs (2^-8), and within its range for every activation here (|act'| < 1.2).  dz is one pass over dy and act'
// which takes the column sums of db along (partials per row block, added in order: no atomics).
//
// Few tiles and a long contraction (dW of a narrow layer, a product of few rows) are cut along the contraction; the float32 partial tiles
// meet in a second launch, in order, which applies the same epilogue.
#include "common.h"
#include "mfma_tile.h"

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct LinArgs {
  const void *A, *B;
  int64_t lda, ldb;       // elements
  int M, N, K;            // rows and columns of the output, contraction
  void* C; int64_t ldc;
  int c_f32;              // C (and the residual) are float32
  const void* bias; int bias_f32;
  const void* res; int64_t ldr;
  void* slope; int64_t lds_;   // act'(z): half (bfloat16 operands) / float
  int act, vec;           // vec: 16-byte accesses of C, residual and slope rows
  int split; float* part; // K pieces: float32 partials [split][M][N]
  int tiles_m, tiles_n;
};

// Phi(z) and exp(-z^2 / 2) by Abramowitz & Stegun 7.1.26 (erfc x = exp(-x^2) P(t), t = 1 / (1 + p x), absolute error 1.5e-7: a float32 product
// of a few hundred terms is off by as much), which shares its exponential with the slope: 18 instructions a value where the library's erfc and
// exp take 80, and those 80 were 0.25 ms of 0.93 ms on [16381 x 8192] outputs
__device__ __forceinline__ void normal_cdf(float z, float& cdf, float& bell) {
  const float x = fabsf(z) * 0.70710678118654752f;
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, x, 1.f));
  float q = __builtin_fmaf(1.061405429f, t, -1.453152027f);
  q = __builtin_fmaf(q, t, 1.421413741f);
  q = __builtin_fmaf(q, t, -0.284496736f);
  q = __builtin_fmaf(q, t, 0.254829592f);
  bell = __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f);
  q = 0.5f * q * t * bell;   // Phi(-|z|)
  cdf = z < 0.f ? q : 1.f - q;
}

__device__ __forceinline__ float sigmoid_of(float x) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * -1.4426950408889634f)); }

// v <- act(v) for eight values, and act'(v) into sl where SLOPE.  The activation is chosen once for the eight: a choice per value made the
// epilogue's code larger than the instruction cache
template <bool SLOPE>
__device__ __forceinline__ void act8(float (&v)[8], float (&sl)[8], int act) {
  if (act == COIN_ACT_NONE) {
#pragma unroll
    for (int i = 0; i < 8; ++i) sl[i] = 1.f;
  } else if (act == COIN_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      sl[i] = v[i] > 0.f ? 1.f : 0.f;
      v[i] = v[i] > 0.f ? v[i] : (v[i] != v[i] ? v[i] : 0.f);
    }
  } else if (act == COIN_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float cdf, bell;
      normal_cdf(v[i], cdf, bell);
      if (SLOPE) sl[i] = __builtin_fmaf(v[i] * 0.39894228040143268f, bell, cdf);
      v[i] *= cdf;
    }
  } else {
    const float a = act == COIN_ACT_QUICK_GELU ? 1.702f : 1.f;   // z sigmoid(a z)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float s = sigmoid_of(a * v[i]);
      if (SLOPE) sl[i] = s * (1.f + a * v[i] * (1.f - s));
      v[i] *= s;
    }
  }
}

// the residual's eight columns of a row; `raw`: what finish_rows fetched ahead (bfloat16 rows of whole chunks)
__device__ __forceinline__ void residual8(const LinArgs& p, float (&r)[8], const bf16x8& raw, int64_t row, int col) {
  const int left = p.N - col;
  if (p.vec && !p.c_f32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (float)raw[i];
  } else if (p.vec) {
    const f32x4 a = *reinterpret_cast<const f32x4*>((const float*)p.res + row * p.ldr + col);
    const f32x4 b = *reinterpret_cast<const f32x4*>((const float*)p.res + row * p.ldr + col + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r[i] = a[i];
      r[4 + i] = b[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      r[i] = 0.f;
      if (i < left) r[i] = p.c_f32 ? ((const float*)p.res)[row * p.ldr + col + i] : (float)((const bf16_t*)p.res)[row * p.ldr + col + i];
    }
  }
}

__device__ __forceinline__ bf16x8 residual_ahead(const LinArgs& p, int64_t row, int col) {
  bf16x8 r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = (bf16_t)0.f;
  if (p.res && p.vec && !p.c_f32) r = *reinterpret_cast<const bf16x8*>((const bf16_t*)p.res + row * p.ldr + col);
  return r;
}

// eight columns of one row through the epilogue: v holds the product
template <typename T>
__device__ __forceinline__ void finish8(const LinArgs& p, float (&v)[8], const float (&bias)[8], const bf16x8& ahead, int64_t row, int col) {
  const int left = p.N - col;
  float sl[8], r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = 0.f;
  if (p.res) residual8(p, r, ahead, row, col);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] += bias[i];
  if (p.slope) act8<true>(v, sl, p.act);
  else act8<false>(v, sl, p.act);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] += r[i];
  if (p.vec) {
    if (p.c_f32) {
      float* c = (float*)p.C + row * p.ldc + col;
      *reinterpret_cast<f32x4*>(c) = (f32x4){v[0], v[1], v[2], v[3]};
      *reinterpret_cast<f32x4*>(c + 4) = (f32x4){v[4], v[5], v[6], v[7]};
    } else {
      bf16x8 o;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = (bf16_t)v[i];
      *reinterpret_cast<bf16x8*>((bf16_t*)p.C + row * p.ldc + col) = o;
    }
    if (p.slope) {
      if constexpr (sizeof(T) == 2) {
        f16x8 o;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = (_Float16)sl[i];
        *reinterpret_cast<f16x8*>((_Float16*)p.slope + row * p.lds_ + col) = o;
      } else {
        float* c = (float*)p.slope + row * p.lds_ + col;
        *reinterpret_cast<f32x4*>(c) = (f32x4){sl[0], sl[1], sl[2], sl[3]};
        *reinterpret_cast<f32x4*>(c + 4) = (f32x4){sl[4], sl[5], sl[6], sl[7]};
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) {
        if (p.c_f32) ((float*)p.C)[row * p.ldc + col + i] = v[i];
        else ((bf16_t*)p.C)[row * p.ldc + col + i] = (bf16_t)v[i];
        if (p.slope) {
          if constexpr (sizeof(T) == 2) ((_Float16*)p.slope)[row * p.lds_ + col + i] = (_Float16)sl[i];
          else ((float*)p.slope)[row * p.lds_ + col + i] = sl[i];
        }
      }
  }
}

__device__ __forceinline__ void load_bias(const LinArgs& p, float (&b)[8], int col) {
#pragma unroll
  for (int i = 0; i < 8; ++i) b[i] = p.bias && col + i < p.N ? (p.bias_f32 ? ((const float*)p.bias)[col + i] : (float)((const bf16_t*)p.bias)[col + i]) : 0.f;
}

constexpr int BKB = 128;   // bytes of the contraction in a stage: whole cache lines (64-byte rows cost a quarter of the rate)

// One operand of a stage: E rows (or columns) of the output, BKB bytes of the contraction.  ACROSS: the contraction runs across the rows
template <typename T, bool ACROSS, int E, int NW>
struct Operand {
  static constexpr int EL = 16 / (int)sizeof(T), BK = BKB / (int)sizeof(T);
  static constexpr int ROWB = ACROSS ? E * (int)sizeof(T) : BKB, ROWS = ACROSS ? BK : E, BYTES = ROWS * ROWB;
  // e0: first row of the tile (elements of the output), ext: how many there are; k0: first index of the contraction, K: its end
  static __device__ __forceinline__ void stage(char* dst, const T* base, int64_t ld, int e0, int ext, int k0, int K, int wave, int lane) {
    const unsigned st = (unsigned)(ld * sizeof(T));
    if constexpr (ACROSS)
      stage_tile<ROWB, ROWS, NW>(dst, base + (int64_t)k0 * ld + e0, K - k0, (ext - e0 + EL - 1) / EL, wave, lane, [&](int r) { return (unsigned)r * st; });
    else
      stage_tile<ROWB, ROWS, NW>(dst, base + (int64_t)e0 * ld + k0, ext - e0, (K - k0 + EL - 1) / EL, wave, lane, [&](int r) { return (unsigned)r * st; });
  }
  // fragment of the 32 rows from `row0`, step `s` of the contraction (32 bytes): lane & 31 = row, the lane half's 16 bytes
  static __device__ __forceinline__ f32x4 frag_at(const char* img, int row0, int s, int lane) {
    const int half = lane >> 5;
    if constexpr (!ACROSS) {
      return Img<BKB, ROWS>::frag(img, row0 + (lane & 31), 2 * s + half);
    } else if constexpr (sizeof(T) == 2) {
      const int q4 = (lane >> 2) & 3, p4 = lane & 3;
      const int chunk = (row0 >> 3) + ((lane >> 4) & 1) * 2 + (p4 >> 1);
      const int r0 = s * 16 + half * 8 + q4;
      const char* a0 = img + r0 * ROWB + ((chunk ^ swz<ROWB>(r0)) << 4) + (p4 & 1) * 8;
      const char* a1 = img + (r0 + 4) * ROWB + ((chunk ^ swz<ROWB>(r0 + 4)) << 4) + (p4 & 1) * 8;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)a0);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)a1);
      const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      return __builtin_bit_cast(f32x4, v);
    } else {
      f32x4 v;
      const int chunk = (row0 >> 2) + ((lane & 31) >> 2);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = s * 8 + half * 4 + e;
        v[e] = *reinterpret_cast<const float*>(img + r * ROWB + ((chunk ^ swz<ROWB>(r)) << 4) + (lane & 3) * 4);
      }
      return v;
    }
  }
};

// XCD-aware order: workgroups b, b + 8, ... share an XCD and take neighbouring items of a contiguous eighth of the list; the list walks groups
// of 8 tile rows column by column, so what runs together shares 8 row panels and a few column panels in the XCD's L2
__device__ __forceinline__ void tile_of(const LinArgs& p, int& tm, int& tn, int& piece) {
  const int nwg = gridDim.x, q = nwg >> 3, r = nwg & 7, x = blockIdx.x & 7, i = blockIdx.x >> 3;
  const int item = (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + i;
  piece = item % p.split;
  const int tile = item / p.split, per = 8 * p.tiles_n, grp = tile / per, in = tile - grp * per;
  const int gm = p.tiles_m - grp * 8 < 8 ? p.tiles_m - grp * 8 : 8;
  tm = grp * 8 + in % gm;
  tn = in / gm;
}

// rows mp .. mp + ROWS - 1 of the output from the epilogue image (ROWS x TN float32, 16-byte chunk c of row r at c ^ (r & 7)); NT threads
template <typename T, int ROWS, int TN, int NT>
__device__ __forceinline__ void finish_rows(const LinArgs& p, const char* lds, int mp, int n0, int piece) {
  constexpr int TPR = TN / 8, RPP = NT / TPR;
  const int c8 = threadIdx.x % TPR, col = n0 + c8 * 8;
  if (col >= p.N) return;
  float bias[8];
  if (p.split == 1) load_bias(p, bias, col);
  // a rolled loop: unrolled it takes the same time (within 0.2 % with GELU, its slope and a residual on [16381 x 2048 x 8192]) and 0.5 MB more
  // code.  The next row's residual is on its way while this one is finished
  const int r0 = threadIdx.x / TPR;
  bf16x8 ahead = residual_ahead(p, mp + r0 < p.M ? mp + r0 : p.M - 1, col);
#pragma unroll 1
  for (int rr = r0; rr < ROWS && mp + rr < p.M; rr += RPP) {
    const int nx = mp + rr + RPP;
    const bf16x8 next = residual_ahead(p, nx < p.M ? nx : p.M - 1, col);
    const f32x4 x = *reinterpret_cast<const f32x4*>(lds + rr * (TN * 4) + (((2 * c8) ^ (rr & 7)) << 4));
    const f32x4 y = *reinterpret_cast<const f32x4*>(lds + rr * (TN * 4) + (((2 * c8 + 1) ^ (rr & 7)) << 4));
    if (p.split > 1) {
      float* o = p.part + ((int64_t)piece * p.M + mp + rr) * p.N + col;
      if (p.N % 8 == 0) {
        *reinterpret_cast<f32x4*>(o) = x;
        *reinterpret_cast<f32x4*>(o + 4) = y;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (col + i < p.N) o[i] = i < 4 ? x[i & 3] : y[i & 3];
      }
    } else {
      float v[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
      finish8<T>(p, v, bias, ahead, mp + rr, col);
    }
    ahead = next;
  }
}

// one 32 x 32 accumulator into the image: lane & 31 = row, registers = columns
template <int TN>
__device__ __forceinline__ void put_tile(char* lds, const f32x16& acc, int row0, int col0, int lane) {
  const int row = row0 + (lane & 31), half = lane >> 5;
#pragma unroll
  for (int r = 0; r < 16; r += 4) {
    const int ch = (col0 + 2 * r + 4 * half) >> 2;
    *reinterpret_cast<f32x4*>(lds + row * (TN * 4) + ((ch ^ (row & 7)) << 4)) = (f32x4){acc[r], acc[r + 1], acc[r + 2], acc[r + 3]};
  }
}

// C tile TS x TS by four waves (2 x 2), each (TS / 2)^2 in 32 x 32 accumulators, a ring of NST stages.  Bound by the DMA's traffic in bfloat16 (a
// 128 x 128 tile moves twice the bytes a product of a 256 x 256 one: [2048 x 4096 x 1024] 25.3 us, 679 TFLOP/s), by the matrix instructions in float32
// ([4096 x 4096 x 1024] 280 us, 123 TFLOP/s).  128 x 128 x 2 stages: 64 KiB of LDS,
// two workgroups per CU, one's epilogue and barriers under the other's matrix instructions; 64 x 64 x 3: 48 KiB, three per CU
template <typename T, bool AA, bool BA, int TS, int NST>
__global__ __launch_bounds__(256, 2) void linear_gemm_kernel(const LinArgs p) {
  using OA = Operand<T, AA, TS, 4>;
  using OB = Operand<T, BA, TS, 4>;
  constexpr int BK = OA::BK, STAGE = OA::BYTES + OB::BYTES, W = TS / 64;
  __shared__ __attribute__((aligned(1024))) char lds[NST * STAGE];
  static_assert(NST * STAGE >= TS * TS * 4 && (NST == 2 || (NST == 3 && STAGE == 4 * 4096)), "");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wave >> 1, wc = wave & 1;
  int tm, tn, piece;
  tile_of(p, tm, tn, piece);
  const int m0 = tm * TS, n0 = tn * TS;
  const int nk = (p.K + BK - 1) / BK;
  const int kb = (int)((int64_t)piece * nk / p.split), ke = (int)((int64_t)(piece + 1) * nk / p.split);
  auto stage = [&](int kt, int slot) {
    char* d = lds + slot * STAGE;
    OA::stage(d, (const T*)p.A, p.lda, m0, p.M, kt * BK, p.K, wave, lane);
    OB::stage(d + OA::BYTES, (const T*)p.B, p.ldb, n0, p.N, kt * BK, p.K, wave, lane);
  };
  f32x16 acc[W][W];
#pragma unroll
  for (int i = 0; i < W; ++i)
#pragma unroll
    for (int j = 0; j < W; ++j) acc[i][j] = zero16();
#pragma unroll
  for (int s = 0; s < NST - 1; ++s)
    if (kb + s < ke) stage(kb + s, s);
  int slot = 0;
  for (int kt = kb; kt < ke; ++kt) {
    // stage kt has landed: a wave's four DMA instructions of one younger stage may be under way
    if (NST == 3 && kt + 1 < ke) asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    P8_BAR();   // for every wave, and nobody reads the slot of stage kt - 1 any more
    if (kt + NST - 1 < ke) stage(kt + NST - 1, slot == 0 ? NST - 1 : slot - 1);
    const char* la = lds + slot * STAGE;
    const char* lb = la + OA::BYTES;
#pragma unroll
    for (int s = 0; s < BKB / 32; ++s) {
      f32x4 a[W], b[W];
#pragma unroll
      for (int j = 0; j < W; ++j) b[j] = OB::frag_at(lb, wc * (TS / 2) + j * 32, s, lane);
#pragma unroll
      for (int i = 0; i < W; ++i) a[i] = OA::frag_at(la, wr * (TS / 2) + i * 32, s, lane);
#pragma unroll
      for (int i = 0; i < W; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j) mma<T>(acc[i][j], b[j], a[i]);   // swapped: lane = output row, registers = 4 consecutive columns
    }
    slot = slot == NST - 1 ? 0 : slot + 1;
  }
  P8_LDS_SYNC();   // every wave is done with the ring: it becomes the epilogue image
#pragma unroll
  for (int i = 0; i < W; ++i)
#pragma unroll
    for (int j = 0; j < W; ++j) put_tile<TS>(lds, acc[i][j], wr * (TS / 2) + i * 32, wc * (TS / 2) + j * 32, lane);
  P8_LDS_SYNC();
  finish_rows<T, TS, TS, 256>(p, lds, m0, n0, piece);
}

// C tile 256 x 256 by eight waves in two groups of four (one wave of each per SIMD), one workgroup per CU, two K-tiles of 64 in LDS, each of
// four half-tiles (A or B, low or high 128 rows, 16 KiB).  A wave owns a 64 x 32 piece of every (A half, B half) quadrant and walks them in
// four phases {read fragments, issue one half-tile's DMA; barrier; eight matrix instructions; barrier}:
//   1: reads B low, A low     2: reads B high     3: reads A high     4: reads nothing;   products  Al Bl, Al Bh, Ah Bh, Ah Bl
// Group 1 runs one barrier behind group 0: one group's matrix instructions run while the other reads.  In barrier intervals, group 0's phase
// i of K-tile g reads at 8 g + 2 (i - 1), group 1 one later; so A low and B low are free from 8 g + 2 on, B high from 8 g + 4, A high from
// 8 g + 6, and their K-tile g + 2 is issued in phases 3, 2, 4 of K-tile g and 1 of K-tile g + 1.  The order of issue is Bl Al Bh Ah, and each is
// read by everybody in the phase after the wait that leaves the five youngest half-tiles (ten instructions of a wave) under way: fourteen
// intervals to land.  K-tiles behind the last are issued too, out of range: they write zeros that nobody reads and keep the count.
// [16381 x 2048 x 8192]: dx 530 us (1036 TFLOP/s), dW 507 us (1085), forward 510 us without an epilogue and 700 us with GELU, its slope and a
// residual (0.8 GB of rows that nobody's matrix instructions cover).  Bound by LDS, which the DMA and the fragment reads contend for: dx takes
// 340 us with every DMA out of range, 500 us without the matrix instructions, 310 us with the DMA alone.  128 x 128 tiles: 887 / 751 / 698 us (forward / dx / dW).
// (bfloat16 alone: float32 matrix instructions are sixteen times slower, and 128 x 128 tiles already feed them)
template <bool AA, bool BA>
__global__ __launch_bounds__(512, 2) void linear_gemm256_kernel(const LinArgs p) {
  using T = bf16_t;
  using OA = Operand<T, AA, 128, 8>;
  using OB = Operand<T, BA, 128, 8>;
  constexpr int BK = OA::BK, HALF = OA::BYTES, STAGE = 4 * HALF;   // Al | Ah | Bl | Bh
  __shared__ __attribute__((aligned(1024))) char lds[2 * STAGE];
  static_assert(HALF == 16384 && OB::BYTES == HALF, "two DMA instructions of a wave a half-tile");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = wave >> 2, wr = group, wc = wave & 3;
  int tm, tn, piece;
  tile_of(p, tm, tn, piece);
  const int m0 = tm * 256, n0 = tn * 256;
  const int nk = (p.K + BK - 1) / BK;
  auto stage_a = [&](int kt, int hi) {
    OA::stage(lds + (kt & 1) * STAGE + hi * HALF, (const T*)p.A, p.lda, m0 + hi * 128, p.M, kt * BK, p.K, wave, lane);
  };
  auto stage_b = [&](int kt, int hi) {
    OB::stage(lds + (kt & 1) * STAGE + (2 + hi) * HALF, (const T*)p.B, p.ldb, n0 + hi * 128, p.N, kt * BK, p.K, wave, lane);
  };
  f32x16 acc[2][2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j][0] = acc[i][j][1] = zero16();
  f32x4 a[2][4], b[2][4];
  // `landed`: for group 0 behind the products, for group 1 behind the reads -- in either case ahead of the barrier that ends an odd interval
  auto multiply = [&](int ah, int bh) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (group) asm volatile("s_waitcnt vmcnt(10)" ::: "memory");
    P8_BAR();
    P8_SCHED();
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i) mma<T>(acc[ah][bh][i], b[bh][s], a[i][s]);
    __builtin_amdgcn_s_setprio(0);
    P8_SCHED();
    if (!group) asm volatile("s_waitcnt vmcnt(10)" ::: "memory");
    P8_BAR();
    P8_SCHED();
  };
  auto read_a = [&](const char* img) {
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i) a[i][s] = OA::frag_at(img, wr * 64 + i * 32, s, lane);
  };
  auto read_b = [&](const char* img, int bh) {
#pragma unroll
    for (int s = 0; s < 4; ++s) b[bh][s] = OB::frag_at(img, wc * 32, s, lane);
  };
  stage_b(0, 0);
  stage_a(0, 0);
  stage_b(0, 1);
  stage_a(0, 1);
  stage_b(1, 0);
  stage_a(1, 0);
  stage_b(1, 1);
  asm volatile("s_waitcnt vmcnt(10)" ::: "memory");
  P8_BAR();
  if (group) P8_BAR();
  for (int kt = 0; kt < nk; ++kt) {
    const char* img = lds + (kt & 1) * STAGE;
    read_b(img + 2 * HALF, 0);
    read_a(img);
    stage_a(kt + 1, 1);
    multiply(0, 0);
    read_b(img + 3 * HALF, 1);
    stage_b(kt + 2, 0);
    multiply(0, 1);
    read_a(img + HALF);
    stage_a(kt + 2, 0);
    multiply(1, 1);
    stage_b(kt + 2, 1);
    multiply(1, 0);
  }
  if (!group) P8_BAR();
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  // epilogue image: 128 rows (the low, then the high half of A) of 256 float32 columns
  auto half_rows = [&](const f32x16 (&c)[2][2], int mp) {
    P8_LDS_SYNC();
#pragma unroll
    for (int bh = 0; bh < 2; ++bh)
#pragma unroll
      for (int i = 0; i < 2; ++i) put_tile<256>(lds, c[bh][i], wr * 64 + i * 32, bh * 128 + wc * 32, lane);
    P8_LDS_SYNC();
    finish_rows<T, 128, 256, 512>(p, lds, mp, n0, piece);
  };
  half_rows(acc[0], m0);
  half_rows(acc[1], m0 + 128);
}

// the K pieces of eight columns of a row, in order, and the epilogue
template <typename T>
__global__ __launch_bounds__(256) void linear_join_kernel(const LinArgs p) {
  const int n8 = (p.N + 7) / 8;
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= (int64_t)p.M * n8) return;
  const int64_t row = at / n8;
  const int col = (int)(at - row * n8) * 8;
  float v[8], bias[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = 0.f;
  for (int s = 0; s < p.split; ++s) {
    const float* o = p.part + ((int64_t)s * p.M + row) * p.N + col;
    if (p.N % 8 == 0) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(o), y = *reinterpret_cast<const f32x4*>(o + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] += x[i];
        v[4 + i] += y[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (col + i < p.N) v[i] += o[i];
    }
  }
  load_bias(p, bias, col);
  finish8<T>(p, v, bias, residual_ahead(p, row, col), row, col);
}

// dz = dy o act' (rows of ldz elements, zeros behind N) and the column sums of dz per block of rows.  32 threads x 8 columns, 8 rows at a time.
// Bound by memory: [16381 x 8192] bfloat16 186 us at 4.3 TB/s
struct DzArgs {
  const void* dy; int64_t ldy; int dy_f32;
  const void* slope; int64_t lds_;
  void* dz; int64_t ldz;     // null: dz is dy itself, only its column sums are wanted
  float* part;               // [row blocks][N] or null
  int64_t M; int N, rows, vec;   // rows of a block; vec: 16-byte accesses of dy and slope rows
};

template <typename T>
__global__ __launch_bounds__(256) void linear_dz_kernel(const DzArgs p) {
  __shared__ float red[8][256];
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5, col = (blockIdx.x * 32 + cx) * 8, left = p.N - col;
  float s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = 0.f;
  const int64_t r0 = (int64_t)blockIdx.y * p.rows, r1 = r0 + p.rows < p.M ? r0 + p.rows : p.M;
  if (left > 0)
    for (int64_t r = r0 + ry; r < r1; r += 8) {
      float d[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i] = 0.f;
      if (p.vec) {
        if (p.dy_f32) {
          const f32x4 a = *reinterpret_cast<const f32x4*>((const float*)p.dy + r * p.ldy + col);
          const f32x4 b = *reinterpret_cast<const f32x4*>((const float*)p.dy + r * p.ldy + col + 4);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            d[i] = a[i];
            d[4 + i] = b[i];
          }
        } else {
          const bf16x8 a = *reinterpret_cast<const bf16x8*>((const bf16_t*)p.dy + r * p.ldy + col);
#pragma unroll
          for (int i = 0; i < 8; ++i) d[i] = (float)a[i];
        }
        if (p.slope) {
          if constexpr (sizeof(T) == 2) {
            const f16x8 a = *reinterpret_cast<const f16x8*>((const _Float16*)p.slope + r * p.lds_ + col);
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] *= (float)a[i];
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] *= ((const float*)p.slope)[r * p.lds_ + col + i];
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < left) {
            d[i] = p.dy_f32 ? ((const float*)p.dy)[r * p.ldy + col + i] : (float)((const bf16_t*)p.dy)[r * p.ldy + col + i];
            if (p.slope) {
              if constexpr (sizeof(T) == 2) d[i] *= (float)((const _Float16*)p.slope)[r * p.lds_ + col + i];
              else d[i] *= ((const float*)p.slope)[r * p.lds_ + col + i];
            }
          }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] += d[i];
      if (p.dz) {   // ldz is a multiple of 8 and covers whole chunks
        if constexpr (sizeof(T) == 2) {
          bf16x8 o;
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] = (bf16_t)d[i];
          *reinterpret_cast<bf16x8*>((bf16_t*)p.dz + r * p.ldz + col) = o;
        } else {
          float* o = (float*)p.dz + r * p.ldz + col;
          *reinterpret_cast<f32x4*>(o) = (f32x4){d[0], d[1], d[2], d[3]};
          *reinterpret_cast<f32x4*>(o + 4) = (f32x4){d[4], d[5], d[6], d[7]};
        }
      }
    }
  if (!p.part) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) red[ry][cx * 8 + i] = s[i];
  __syncthreads();
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= p.N) return;
  float t = red[0][threadIdx.x];
#pragma unroll
  for (int y = 1; y < 8; ++y) t += red[y][threadIdx.x];
  p.part[(int64_t)blockIdx.y * p.N + c] = t;
}

// db: the row blocks' column sums, in order; 64 columns x 4 runs of blocks
__global__ __launch_bounds__(256) void linear_db_kernel(const float* part, void* db, int db_f32, int blocks, int N) {
  __shared__ float red[4][64];
  const int lane = threadIdx.x & 63, run = threadIdx.x >> 6, col = blockIdx.x * 64 + lane;
  const int per = (blocks + 3) / 4, b0 = run * per, b1 = b0 + per < blocks ? b0 + per : blocks;
  float s = 0.f;
  if (col < N)
    for (int b = b0; b < b1; ++b) s += part[(int64_t)b * N + col];
  red[run][lane] = s;
  __syncthreads();
  if (run || col >= N) return;
  s = ((red[0][lane] + red[1][lane]) + red[2][lane]) + red[3][lane];
  if (db_f32) ((float*)db)[col] = s;
  else ((bf16_t*)db)[col] = (bf16_t)s;
}

// rows of `cols` elements -> rows of `ldd` elements, zeros behind the columns (bound by memory; only rows that are not whole 16-byte chunks come here)
template <typename T>
__global__ __launch_bounds__(256) void pad_rows_kernel(const T* src, int64_t lds_, T* dst, int64_t ldd, int64_t rows, int cols) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, n8 = ldd / 8;
  if (at >= rows * n8) return;
  const int64_t r = at / n8;
  const int c = (int)(at - r * n8) * 8;
#pragma unroll
  for (int i = 0; i < 8; ++i) dst[r * ldd + c + i] = c + i < cols ? src[r * lds_ + c + i] : (T)0.f;
}

constexpr int64_t SPAN = 0x7fffffff;
constexpr int CUS = 256;   // MI355X

struct Tiling {
  int ts, split;
};

// Tile size and K pieces of one product; us measured with each size forced, 256 / 128 / 64:
//   bfloat16: 256 x 256 tiles where at least 7 of 8 CUs work in every round.  [4096 x 4096 x 1024], one full round, 42 / 47 / 66; 192 tiles
//     ([3000 x 4096]) 38 / 38 / 49; one and a half rounds ([6000 x 4096]) 72 / 66 / 92.  (float32 gains nothing: 304 / 280 / 302)
//   128 x 128 where they are as many as the CUs: [2048 x 2048 x 2048] - / 30 / 32, float32 - / 139 / 146;
//   fewer of them, with the contraction cut to two workgroups per CU, where the pieces keep 16 stages: [512 x 2048 x 8192] - / 38 / 83, float32
//     - / 148 / 216; [2048 x 1024 x 8192] - / 49 / 56; shorter pieces pay for the join: [1024 x 2048 x 2048], 8 stages, - / 27 / 17;
//   else 64 x 64; fewer than the CUs are cut the same way, in pieces of at least four stages
static Tiling plan(int64_t M, int64_t N, int64_t K, int es) {
  const int64_t nk = (K * es + BKB - 1) / BKB;
  const int64_t t256 = (M + 255) / 256 * ((N + 255) / 256), t128 = (M + 127) / 128 * ((N + 127) / 128), t64 = (M + 63) / 64 * ((N + 63) / 64);
  const int64_t rounds = (t256 + CUS - 1) / CUS;
  if (es == 2 && 8 * t256 >= 7 * rounds * CUS) return {256, 1};
  if (t128 >= CUS) return {128, 1};
  int64_t s = 2 * CUS / t128;
  if (s <= 64 && nk / s >= 16) return {128, (int)s};
  s = t64 >= CUS ? 1 : 2 * CUS / t64;
  if (s > nk / 4) s = nk / 4;
  if (s > 64) s = 64;
  return {64, s < 1 ? 1 : (int)s};
}

static size_t part_bytes(int64_t M, int64_t N, int64_t K, int es) {
  const int s = plan(M, N, K, es).split;
  return s > 1 ? (size_t)s * M * N * sizeof(float) : 0;
}

template <typename T, bool AA, bool BA>
static void run_gemm(LinArgs a, hipStream_t st) {
  const Tiling t = plan(a.M, a.N, a.K, sizeof(T));
  a.split = t.split;
  a.tiles_m = (a.M + t.ts - 1) / t.ts;
  a.tiles_n = (a.N + t.ts - 1) / t.ts;
  const unsigned grid = (unsigned)(a.tiles_m * a.tiles_n * a.split);
  if constexpr (sizeof(T) == 2) {
    if (t.ts == 256) linear_gemm256_kernel<AA, BA><<<grid, 512, 0, st>>>(a);
  }
  if (t.ts == 256) return;
  if (t.ts == 128) linear_gemm_kernel<T, AA, BA, 128, 2><<<grid, 256, 0, st>>>(a);
  else linear_gemm_kernel<T, AA, BA, 64, 3><<<grid, 256, 0, st>>>(a);
  if (a.split > 1) linear_join_kernel<T><<<(unsigned)(((int64_t)a.M * ((a.N + 7) / 8) + 255) / 256), 256, 0, st>>>(a);
}

static int dz_blocks(int64_t M, int N, int* rows) {
  // about four workgroups per CU; at least 32 rows of a block, so that the column sums stay small beside the rows
  const int64_t cols = (N + 255) / 256;
  int64_t b = (4 * CUS + cols - 1) / cols;
  if (b > (M + 31) / 32) b = (M + 31) / 32;
  int64_t r = ((M + b - 1) / b + 7) / 8 * 8;
  *rows = (int)r;
  return (int)((M + r - 1) / r);
}

static bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

static int check_lin(int64_t M, int N, int K, int dtype) {
  if (M < 0 || N <= 0 || K <= 0 || (dtype != COIN_F32 && dtype != COIN_BF16)) return COIN_EINVAL;
  if (M > (1 << 30) || N > (1 << 24) || K > (1 << 24)) return COIN_ESHAPE;
  const int es = dtype == COIN_BF16 ? 2 : 4;
  const int64_t dims[3][3] = {{M, N, K}, {M, K, N}, {N, K, M}};
  for (auto& d : dims) {   // grids below 2^31
    const int s = plan(d[0] > 0 ? d[0] : 1, d[1], d[2] > 0 ? d[2] : 1, es).split;
    if (((d[0] + 63) / 64) * ((d[1] + 63) / 64) * s >= SPAN || d[0] * ((d[1] + 7) / 8) / 256 >= SPAN - 1) return COIN_ESHAPE;
  }
  return COIN_OK;
}

// an operand: 16-byte rows (the last chunk of a row may be read whole: `cols` rounded up to chunks fits the row pitch), offsets of a tile below 2^31
static int check_op(const void* p, int64_t ld, int64_t cols, int es) {
  if (!p) return COIN_EINVAL;
  const int el = 16 / es;
  if (!al16(p) || ld % el || ld < (cols + el - 1) / el * el) return COIN_EALIGN;
  if (ld >= SPAN || 260 * ld * es + cols * es + 4096 >= SPAN) return COIN_ESHAPE;
  return COIN_OK;
}

static bool act_ok(int act) { return act == COIN_ACT_NONE || act == COIN_ACT_RELU || act == COIN_ACT_GELU || act == COIN_ACT_QUICK_GELU || act == COIN_ACT_SILU; }

}  // namespace

extern "C" int coin_pad_rows(const void* src, int64_t ld_src, void* dst, int64_t ld_dst, int64_t rows, int cols, int dtype, void* stream) {
  if (!src || !dst || rows < 0 || cols <= 0 || ld_dst < cols || (dtype != COIN_F32 && dtype != COIN_BF16)) return COIN_EINVAL;
  if (ld_dst % 8 || rows * (ld_dst / 8) / 256 >= SPAN - 1) return COIN_ESHAPE;
  if (rows == 0) return COIN_OK;
  const unsigned grid = (unsigned)((rows * (ld_dst / 8) + 255) / 256);
  if (dtype == COIN_BF16) pad_rows_kernel<bf16_t><<<grid, 256, 0, (hipStream_t)stream>>>((const bf16_t*)src, ld_src, (bf16_t*)dst, ld_dst, rows, cols);
  else pad_rows_kernel<float><<<grid, 256, 0, (hipStream_t)stream>>>((const float*)src, ld_src, (float*)dst, ld_dst, rows, cols);
  return coin_launch_status();
}

static size_t up256(size_t n) { return (n + 255) / 256 * 256; }

static size_t dz_bytes(int64_t M, int N, int es) { return up256((size_t)M * ((N + 7) / 8 * 8) * es); }

// what the products and the column sums of a backward share, one after the other
static size_t bwd_part_bytes(int64_t M, int N, int K, int es) {
  int rows;
  size_t n = (size_t)dz_blocks(M, N, &rows) * N * sizeof(float);
  const size_t a = part_bytes(M, K, N, es), b = part_bytes(N, K, M, es);
  n = a > n ? a : n;
  return b > n ? b : n;
}

extern "C" size_t coin_linear_workspace_bytes(int64_t M, int N, int K, int dtype, int backward) {
  if (check_lin(M, N, K, dtype) != COIN_OK || M == 0) return 0;
  const int es = dtype == COIN_BF16 ? 2 : 4;
  if (!backward) return part_bytes(M, N, K, es);
  return (backward > 1 ? dz_bytes(M, N, es) : 0) + bwd_part_bytes(M, N, K, es);
}

extern "C" int coin_linear_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, int bias_dtype, int act, const void* residual,
                               int64_t ldr, void* y, int64_t ldy, int y_dtype, void* slope, int64_t ld_slope, int64_t M, int N, int K, int dtype,
                               void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_lin(M, N, K, dtype);
  if (rc != COIN_OK) return rc;
  if (!act_ok(act) || (y_dtype != COIN_F32 && y_dtype != COIN_BF16) || (dtype == COIN_F32 && y_dtype != COIN_F32)) return COIN_EINVAL;
  if (bias && bias_dtype != COIN_F32 && bias_dtype != COIN_BF16) return COIN_EINVAL;
  if (M == 0) return COIN_OK;
  const int es = dtype == COIN_BF16 ? 2 : 4;
  if (!y || ldy < N || (residual && ldr < N) || (slope && ld_slope < N)) return COIN_EINVAL;
  if ((rc = check_op(x, ldx, K, es)) != COIN_OK || (rc = check_op(w, ldw, K, es)) != COIN_OK) return rc;
  const size_t need = part_bytes(M, N, K, es);
  if (need && (!workspace || workspace_bytes < need)) return COIN_EINVAL;
  if (!al16(workspace)) return COIN_EALIGN;
  LinArgs a = {};
  a.A = x; a.lda = ldx; a.B = w; a.ldb = ldw; a.M = (int)M; a.N = N; a.K = K; a.C = y; a.ldc = ldy; a.c_f32 = y_dtype == COIN_F32;
  a.bias = bias; a.bias_f32 = bias_dtype == COIN_F32; a.res = residual; a.ldr = ldr; a.slope = slope; a.lds_ = ld_slope; a.act = act;
  a.vec = N % 8 == 0 && ldy % 8 == 0 && al16(y) && (!residual || (ldr % 8 == 0 && al16(residual))) && (!slope || (ld_slope % 8 == 0 && al16(slope)));
  a.part = (float*)workspace;
  if (dtype == COIN_BF16) run_gemm<bf16_t, false, false>(a, (hipStream_t)stream);
  else run_gemm<float, false, false>(a, (hipStream_t)stream);
  return coin_launch_status();
}

extern "C" int coin_linear_bwd(const void* dy, int64_t ldy, int dy_dtype, const void* slope, int64_t ld_slope, const void* x, int64_t ldx, const void* w,
                               int64_t ldw, void* dx, int64_t lddx, void* dw, int64_t lddw, int dw_dtype, void* db, int db_dtype, int64_t M, int N, int K,
                               int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_lin(M, N, K, dtype);
  if (rc != COIN_OK) return rc;
  if (!dy || (!dx && !dw && !db) || M == 0 || ldy < N || (slope && ld_slope < N)) return COIN_EINVAL;
  if ((dy_dtype != COIN_F32 && dy_dtype != COIN_BF16) || (dtype == COIN_F32 && dy_dtype != COIN_F32)) return COIN_EINVAL;
  if (db && db_dtype != COIN_F32 && db_dtype != COIN_BF16) return COIN_EINVAL;
  if (dw && dw_dtype != COIN_F32 && (dw_dtype != COIN_BF16 || dtype == COIN_F32)) return COIN_EINVAL;
  if ((dx && lddx < K) || (dw && lddw < K)) return COIN_EINVAL;
  const int es = dtype == COIN_BF16 ? 2 : 4;
  if (dx && (rc = check_op(w, ldw, K, es)) != COIN_OK) return rc;
  if (dw && (rc = check_op(x, ldx, K, es)) != COIN_OK) return rc;
  // dz is dy itself where there is no activation, its type is the products' and its rows are whole chunks
  const bool products = dx || dw;
  const bool own = products && (slope || dy_dtype != dtype || N % (16 / es) || check_op(dy, ldy, N, es) != COIN_OK);
  if (!workspace || workspace_bytes < (own ? dz_bytes(M, N, es) : 0) + bwd_part_bytes(M, N, K, es)) return COIN_EINVAL;
  if (!al16(workspace)) return COIN_EALIGN;
  hipStream_t st = (hipStream_t)stream;
  float* part = (float*)((char*)workspace + (own ? dz_bytes(M, N, es) : 0));
  const void* dz = own ? workspace : dy;
  const int64_t ldz = own ? (N + 7) / 8 * 8 : ldy;
  if (products && (rc = check_op(dz, ldz, N, es)) != COIN_OK) return rc;
  if (own || db) {
    DzArgs a = {};
    a.dy = dy; a.ldy = ldy; a.dy_f32 = dy_dtype == COIN_F32; a.slope = slope; a.lds_ = ld_slope; a.dz = own ? workspace : nullptr; a.ldz = ldz;
    a.M = M; a.N = N; a.part = db ? part : nullptr;
    a.vec = N % 8 == 0 && ldy % 8 == 0 && al16(dy) && (!slope || (ld_slope % 8 == 0 && al16(slope)));
    const int blocks = dz_blocks(M, N, &a.rows);
    const dim3 grid((N + 255) / 256, blocks);
    if (dtype == COIN_BF16) linear_dz_kernel<bf16_t><<<grid, 256, 0, st>>>(a);
    else linear_dz_kernel<float><<<grid, 256, 0, st>>>(a);
    if (db) linear_db_kernel<<<(N + 63) / 64, 256, 0, st>>>(part, db, db_dtype == COIN_F32, blocks, N);
  }
  if (dx) {
    LinArgs a = {};
    a.A = dz; a.lda = ldz; a.B = w; a.ldb = ldw; a.M = (int)M; a.N = K; a.K = N; a.C = dx; a.ldc = lddx; a.c_f32 = dtype == COIN_F32;
    a.vec = K % 8 == 0 && lddx % 8 == 0 && al16(dx);
    a.part = part;
    if (dtype == COIN_BF16) run_gemm<bf16_t, false, true>(a, st);
    else run_gemm<float, false, true>(a, st);
  }
  if (dw) {
    LinArgs a = {};
    a.A = dz; a.lda = ldz; a.B = x; a.ldb = ldx; a.M = N; a.N = K; a.K = (int)M; a.C = dw; a.ldc = lddw; a.c_f32 = dw_dtype == COIN_F32;
    a.vec = K % 8 == 0 && lddw % 8 == 0 && al16(dw);
    a.part = part;
    if (dtype == COIN_BF16) run_gemm<bf16_t, true, true>(a, st);
    else run_gemm<float, true, true>(a, st);
  }
  return coin_launch_status();
}
