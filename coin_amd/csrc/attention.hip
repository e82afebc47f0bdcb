// Attention of a transformer block (coin_attention_fwd / _bwd), forward and backward, float32 and bfloat16, for gfx950.
//
//   s_ij = scale * q_i . k_j   for the keys j that query i sees:  j < n_b  and, causal, j <= i + n_b - Lq     (n_b = the sequence's keys)
//   p_ij = exp(s_ij) / sum_j exp(s_ij),   o_i = sum_j p_ij v_j;   a query that sees no key gives o_i = 0 and no gradient
//
// The g = Hq / Hkv query heads that share a key head are rows of ONE product: row t = i * g + head, R = Lq * g rows per (sequence, key
// head), so a key or value tile is staged once for all of them and a single new token still fills g rows of a matrix instruction.
//
// Forward: one pass over the keys with the running maximum m and sum l of each row.  A wave owns 32 rows; S^T = K Q^T on 32 x 32 matrix
// tiles leaves, per lane, ONE query (lane & 31) and 16 keys, so the row statistics are per-lane values plus one exchange between the two
// lane halves, and the probabilities, rounded to the tensors' type, ARE the B operand of O^T += V^T P^T (the contraction index is
// permuted the same way on both operands).  m moves only when a score passes it by more than 8 (log2): p stays below 2^8 and the
// accumulator is rescaled a few times per row instead of once per tile.
//
// D_i takes what rounding took from o_i back: bfloat16 training keeps that part beside o (`out_lo`).  Rows of few keys have o_i near a v_j, and
// the rounded o_i alone made dQ and dK of a causal [77 x 77] head 8 % less exact
// (2-norm, 2.61e-3 against 2.41e-3).
//
// Backward, from L_i = log2 sum_j exp2(s_ij log2 e) that the forward keeps: P is recomputed, never stored.
//   D_i = do_i . o_i,   dS = P (dO V^T - D),   dQ = scale dS K,   dK = scale dS^T Q,   dV = P^T dO
// in two launches: one owns query rows (dQ and D), one owns keys and walks the rows (dK, dV; S is formed with the queries in the
// registers, so P and dS are B operands again).  That is 7 products where one launch would take 5, but every sum has one owner: no atomics,
// the same bits every time, and the heads that share a key head are summed in registers.
//
// K, V, Q, dO tiles go to LDS by the range-checked LDS-DMA into swizzled images (mfma_tile.h), two buffers, one barrier per tile.
// float32 tensors take the same kernels with 32x32x2 float32 matrix instructions: four of them use one 16-byte fragment.
#include "common.h"
#include "mfma_tile.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESCALE = 8.0f;   // log2: how far a score may pass the running maximum before the accumulator is rescaled

struct AttnArgs {
  const void *q, *k, *v, *o, *dout;   // o / dout: backward inputs
  bf16_t* lo;                         // [B][Lq][Hq][D]: what rounding took from out
  void *out, *dq, *dk, *dv;
  float *lse, *delta;                 // [B * Hkv][R]
  const int* lengths;                 // [B] or null
  int64_t qs[3], ks[3], vs[3], os[3], dos[3], dqs[3], dks[3], dvs[3];   // element strides: sequence, token, head
  int B, Lq, Lk, Hkv, g, D, R;
  unsigned magic;                     // ceil(2^32 / g)
  int causal, splits, chunk;          // splits of the keys (forward; `chunk` keys each) or of the rows (dK, dV)
  float scale, c;                     // c = scale * log2 e
  float *part, *part_ml;
};

// acc[dt]^T[d][col] += sum over the 32 image rows row0 .. row0 + 31 of image[row][d] * p[row][col], p in accumulator registers:
// register r of lane half h holds row 8 (r >> 2) + 4 h + (r & 3).  SUM (bfloat16): sum[.][col] += the same with an image of ones
template <typename T, typename I, int ND, bool SUM = false>
__device__ __forceinline__ void mma_t(f32x16 (&acc)[ND], const char* img, int row0, const f32x16& p, int lane, f32x16* sum = nullptr) {
  const int half = lane >> 5;
  if constexpr (sizeof(T) == 2) {
    const int q4 = (lane >> 2) & 3, p4 = lane & 3, lrow = half * 4 + q4;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      bf16x8 pf;
#pragma unroll
      for (int e = 0; e < 8; ++e) pf[e] = (bf16_t)p[8 * s + e];
      if constexpr (SUM) {
        const s16x8 one = {0x3f80, 0x3f80, 0x3f80, 0x3f80, 0x3f80, 0x3f80, 0x3f80, 0x3f80};
        *sum = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, one), pf, *sum, 0, 0, 0);
      }
#pragma unroll
      for (int dt = 0; dt < ND; ++dt) {
        const int chunk = dt * 4 + ((lane >> 4) & 1) * 2 + (p4 >> 1);
        const char* a0 = img + I::row_at(row0 + 16 * s) + I::row_at(lrow) + ((chunk ^ I::key(lrow)) << 4) + (p4 & 1) * 8;
        const char* a1 = img + I::row_at(row0 + 16 * s + 8) + I::row_at(lrow) + ((chunk ^ I::key(lrow + 8)) << 4) + (p4 & 1) * 8;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)a0);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)a1);
        const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, v), pf, acc[dt], 0, 0, 0);
      }
    }
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int lrow = 8 * (r >> 2) + 4 * half + (r & 3);
#pragma unroll
      for (int dt = 0; dt < ND; ++dt) {
        const int chunk = dt * 8 + ((lane & 31) >> 2);
        const float a = *reinterpret_cast<const float*>(img + I::row_at(row0) + I::row_at(lrow) + ((chunk ^ I::key(lrow)) << 4) + (lane & 3) * 4);
        acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, p[r], acc[dt], 0, 0, 0);
      }
    }
  }
}

// 32 rows x DP of a row-major tensor as register fragments: lane & 31 = row, chunk 2 c + half
template <int NC>
__device__ __forceinline__ void load_frags(f32x4 (&f)[NC], const char* rowp, bool live, int nchunk, int half) {
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    f[c] = (f32x4){0.f, 0.f, 0.f, 0.f};
    if (live && 2 * c + half < nchunk) f[c] = *reinterpret_cast<const f32x4*>(rowp + (2 * c + half) * 16);
  }
}

__device__ __forceinline__ int keys_of(const AttnArgs& p, int b) {
  if (!p.lengths) return p.Lk;
  const int n = p.lengths[b];
  return n < 0 ? 0 : (n > p.Lk ? p.Lk : n);
}

// t / g.  umulhi(t, magic) is the quotient or one more (the excess t (magic g - 2^32) / (g 2^32) is below 1 for 32-bit t)
__device__ __forceinline__ int row_token(const AttnArgs& p, int t) {
  if (p.g == 1) return t;
  const int q = (int)__umulhi((unsigned)t, p.magic);
  return q * p.g > t ? q - 1 : q;
}

// first key that row t does not see
__device__ __forceinline__ int row_limit(const AttnArgs& p, int t, int n) {
  if (t >= p.R) return 0;
  if (!p.causal) return n;
  const int i = row_token(p, t);
  const int l = i + n - p.Lq + 1;
  return l < 0 ? 0 : (l > n ? n : l);
}

template <typename T, int DP>
struct Cfg {
  static constexpr int ROWB = DP * (int)sizeof(T);
  static constexpr int NC = ROWB / 32;              // 16-byte chunk pairs of a row
  static constexpr int KT = ROWB <= 256 ? 64 : 32;  // rows of a staged tile: two double-buffered tiles stay within 64 KiB
  static constexpr int NS = KT / 32, ND = DP / 32;
  static constexpr int EL = 16 / (int)sizeof(T);    // elements of a chunk
  using I = Img<ROWB, KT, ROWB == 256>;             // row0 of a fragment is a multiple of 8: row_at adds up
  static constexpr int TILE = I::BYTES;
};

// ------------------------------------------------------------------------------------------------------------------------------ forward
// 128 rows by four waves, or up to 32 rows by one; a wave's 32 rows keep Q (32 registers at D 128), the scores of 64 keys (32) and O (64) within
// the 256 that let two waves on a SIMD (workgroups of one wave, each with its own tiles, take 2.4 times as long on the long case below).
// Bound by issue as it stands (a tile's scores, its exponentials and its second product follow one another within a wave): on that case the
// matrix units are busy 49 % of the SIMDs' cycles and vector instructions (exponentials, sums, conversions and the
// issue of the products) 47 %, with two waves to cover one another.
// 2 x 4001 causal tokens, 16 heads over 4, D 128, bfloat16: 179 us, 732 TFLOP/s.  One row per sequence over a long cache is bound by memory:
// 16 ragged caches of up to 32768 keys, 276 us at 4.1 TB/s.
template <typename T, int DP, int NW, bool SPLIT>
__global__ __launch_bounds__(NW * 64, (sizeof(T) == 4 && DP == 128 ? 1 : 2)) void attention_fwd_kernel(const AttnArgs p) {
  using C = Cfg<T, DP>;
  using I = typename C::I;
  constexpr int ROWB = C::ROWB, KT = C::KT;
  __shared__ __attribute__((aligned(1024))) char lds[4 * C::TILE];
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nbh = p.B * p.Hkv, tiles = (p.R + NW * 32 - 1) / (NW * 32);
  int id = blockIdx.x, split = 0;
  if (SPLIT) {
    split = id % p.splits;
    id /= p.splits;
  }
  // the tiles with the most keys first (causal: the last rows); the tiles of one key head stay on one XCD where 8 divides their number
  const int tile = tiles - 1 - id / nbh, bh = id % nbh;
  const int b = bh / p.Hkv, hk = bh - b * p.Hkv;
  const int n = keys_of(p, b), nchunk = p.D / C::EL;
  const int t = (tile * NW + wave) * 32 + (lane & 31);
  const bool live = t < p.R;
  const int i = row_token(p, t), gi = t - i * p.g;
  const int lim = row_limit(p, t, n);
  const int wt = (tile * NW + wave) * 32, wlast = wt + 31 < p.R ? wt + 31 : p.R - 1;
  const int wmax = wt < p.R ? row_limit(p, wlast, n) : 0;                       // keys any row of the wave sees
  const int wmin = wt + 31 < p.R ? row_limit(p, wt, n) : 0;                     // keys every row sees
  const int tlast = (tile + 1) * NW * 32 - 1 < p.R ? (tile + 1) * NW * 32 - 1 : p.R - 1;
  const int kb = SPLIT ? split * p.chunk : 0;
  int ke = row_limit(p, tlast, n);
  if (SPLIT && ke > kb + p.chunk) ke = kb + p.chunk;

  f32x4 qf[C::NC];
  load_frags<C::NC>(qf, (const char*)((const T*)p.q + b * p.qs[0] + (int64_t)i * p.qs[1] + (int64_t)(hk * p.g + gi) * p.qs[2]), live, nchunk, half);
  const T* kbase = (const T*)p.k + b * p.ks[0] + hk * p.ks[2];
  const T* vbase = (const T*)p.v + b * p.vs[0] + hk * p.vs[2];
  const unsigned kst = (unsigned)(p.ks[1] * sizeof(T)), vst = (unsigned)(p.vs[1] * sizeof(T));
  auto stage = [&](int kt, int buf) {
    char* d = lds + buf * 2 * C::TILE;
    stage_tile<ROWB, KT, NW, ROWB == 256>(d, kbase + (int64_t)kt * p.ks[1], n - kt, nchunk, wave, lane, [&](int r) { return (unsigned)r * kst; });
    stage_tile<ROWB, KT, NW, ROWB == 256>(d + C::TILE, vbase + (int64_t)kt * p.vs[1], n - kt, nchunk, wave, lane, [&](int r) { return (unsigned)r * vst; });
  };
  f32x16 o[C::ND];
#pragma unroll
  for (int d = 0; d < C::ND; ++d) o[d] = zero16();
  // l: the sum that L is made of.  lw[0]: the sum of the rounded probabilities that the product takes; o = sum p~ v / sum p~ is off by the
  // roundings times (v_j - o) instead of v_j, which is what D and through it dQ and dK see.  It comes from the matrix units, as one more row
  // of V^T that holds ones: the vector unit is the busier one (3.5 % of the long case's time)
  float m = -INFINITY, l = 0.f;
  f32x16 lw = zero16();
  const float c = p.c;
  if (kb < ke) stage(kb, 0);
  int buf = 0;
  for (int kt = kb; kt < ke; kt += KT, buf ^= 1) {
    TILE_WAIT();   // this tile has landed for every wave; the other buffer is no longer read
    if (kt + KT < ke) stage(kt + KT, buf ^ 1);
    if (kt >= wmax) continue;
    const char* kimg = lds + buf * 2 * C::TILE;
    const char* vimg = kimg + C::TILE;
    f32x16 st[C::NS];
#pragma unroll
    for (int s = 0; s < C::NS; ++s) {
      st[s] = zero16();
      if (sizeof(T) == 2 || kt + s * 32 < wmax)   // float32 products are dear: 32 keys that no row of the wave sees cost their mask alone
#pragma unroll
        for (int cc = 0; cc < C::NC; ++cc) mma<T>(st[s], I::frag(kimg, s * 32 + (lane & 31), 2 * cc + half), qf[cc]);
    }
    if (kt + KT > wmin) {
#pragma unroll
      for (int s = 0; s < C::NS; ++s)
#pragma unroll
        for (int r = 0; r < 16; ++r) st[s][r] = kt + s * 32 + 8 * (r >> 2) + 4 * half + (r & 3) < lim ? st[s][r] : -INFINITY;
    }
    float mx = st[0][0];
#pragma unroll
    for (int s = 0; s < C::NS; ++s)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, st[s][r]);
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    if (__any((mx - m) * c > RESCALE || (m == -INFINITY && mx > m))) {
      const float mn = fmaxf(m, mx);
      const float al = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - mn) * c);
      m = mn;
      l *= al;
      lw[0] *= al;
#pragma unroll
      for (int d = 0; d < C::ND; ++d) o[d] *= al;
    }
    const float mc = m == -INFINITY ? 0.f : m * c;
    float ls = 0.f;
#pragma unroll
    for (int s = 0; s < C::NS; ++s)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        st[s][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[s][r], c, -mc));
        ls += st[s][r];
      }
    l += ls;
#pragma unroll
    for (int s = 0; s < C::NS; ++s)
      if (sizeof(T) == 2 || kt + s * 32 < wmax) mma_t<T, I, C::ND, sizeof(T) == 2>(o, vimg, s * 32, st[s], lane, &lw);
  }
  l += __shfl_xor(l, 32, 64);
  const float lsum = sizeof(T) == 4 ? l : lw[0];
  if (!live) return;
  const size_t row = (size_t)bh * p.R + t;
  if (SPLIT) {   // unnormalised sums with their maximum; joined by attention_join_kernel.  A split without keys leaves l = 0 and no sums
    const size_t prow = (size_t)split * nbh * p.R + row;
    if (half == 0) {
      *reinterpret_cast<f32x4*>(p.part_ml + prow * 4) = (f32x4){m == -INFINITY ? 0.f : m * c, l, lsum, 0.f};
    }
    if (kb < wmax && l > 0.f) {
#pragma unroll
      for (int d = 0; d < C::ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
          const int dd = d * 32 + 2 * r + 4 * half;
          if (dd < p.D) *reinterpret_cast<f32x4*>(p.part + prow * p.D + dd) = (f32x4){o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]};
        }
    }
    return;
  }
  const float inv = lsum > 0.f ? 1.f / lsum : (lsum == 0.f ? 0.f : lsum);   // no key: zeros; NaN stays
  if (p.lse && half == 0) p.lse[row] = l == 0.f ? INFINITY : m * c + __builtin_amdgcn_logf(l);
  T* op = (T*)p.out + b * p.os[0] + (int64_t)i * p.os[1] + (int64_t)(hk * p.g + gi) * p.os[2];
  bf16_t* lp = p.lo ? p.lo + (((size_t)b * p.Lq + i) * p.Hkv * p.g + hk * p.g + gi) * p.D : nullptr;
#pragma unroll
  for (int d = 0; d < C::ND; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int dd = d * 32 + 2 * r + 4 * half;
      if (dd >= p.D) continue;
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = o[d][r + e] * inv;
      store4<T>(op + dd, v[0], v[1], v[2], v[3]);
      if (sizeof(T) == 2 && lp) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] -= (float)(bf16_t)v[e];
        store4<bf16_t>(lp + dd, v[0], v[1], v[2], v[3]);
      }
    }
}

// one wave per row: the splits' sums joined with their maxima, in split order.  Lane s first holds split s's maximum and sum, so that the loads
// of the partial rows do not wait for one another
template <typename T>
__global__ __launch_bounds__(256) void attention_join_kernel(const AttnArgs p) {
  const int lane = threadIdx.x & 63;
  const int64_t rows = (int64_t)p.B * p.Hkv * p.R, row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  float m = -INFINITY;
  bool bad = false;
  for (int s = lane; s < p.splits; s += 64) {
    const f32x4 ml = *reinterpret_cast<const f32x4*>(p.part_ml + (s * rows + row) * 4);
    if (ml[1] != 0.f) m = fmaxf(m, ml[0]);
    bad |= !(ml[1] == ml[1]);
  }
  m = wave_reduce_max(m);
  bad = __any(bad);
  float a0 = 0.f, a1 = 0.f, l = 0.f, lw = 0.f;
  const int d = lane * 2;   // head dimensions are even and <= 128
  for (int s0 = 0; s0 < p.splits; s0 += 64) {
    float w = 0.f, ls = 0.f, lr = 0.f;
    if (s0 + lane < p.splits) {
      const f32x4 ml = *reinterpret_cast<const f32x4*>(p.part_ml + ((s0 + lane) * rows + row) * 4);
      if (ml[1] > 0.f) {
        w = __builtin_amdgcn_exp2f(ml[0] - m);
        ls = ml[1] * w;
        lr = ml[2] * w;
      }
    }
    l += wave_reduce_sum(ls);
    lw += wave_reduce_sum(lr);
    const int ns = p.splits - s0 < 64 ? p.splits - s0 : 64;
#pragma unroll 8
    for (int s = 0; s < ns; ++s) {
      const float ws = __shfl(w, s, 64);
      float2 v = make_float2(0.f, 0.f);
      if (ws != 0.f && d < p.D) v = *reinterpret_cast<const float2*>(p.part + ((s0 + s) * rows + row) * p.D + d);   // sums of a split without keys are not there
      a0 = __builtin_fmaf(v.x, ws, a0);
      a1 = __builtin_fmaf(v.y, ws, a1);
    }
  }
  if (bad) l = lw = __builtin_nanf("");
  const float inv = lw == 0.f ? 0.f : 1.f / lw;
  const int bh = (int)(row / p.R), t = (int)(row - (int64_t)bh * p.R), b = bh / p.Hkv, hk = bh - b * p.Hkv, i = row_token(p, t), gi = t - i * p.g;
  if (p.lse && lane == 0) p.lse[row] = l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l);
  if (d < p.D) {
    T* op = (T*)p.out + b * p.os[0] + (int64_t)i * p.os[1] + (int64_t)(hk * p.g + gi) * p.os[2] + d;
    a0 *= inv;
    a1 *= inv;
    op[0] = (T)a0;
    op[1] = (T)a1;
    if (sizeof(T) == 2 && p.lo) {
      bf16_t* lp = p.lo + (((size_t)b * p.Lq + i) * p.Hkv * p.g + hk * p.g + gi) * p.D + d;
      lp[0] = (bf16_t)(a0 - (float)(bf16_t)a0);
      lp[1] = (bf16_t)(a1 - (float)(bf16_t)a1);
    }
  }
}

// ----------------------------------------------------------------------------------------------------------------------- backward: dQ, D
// The forward's split and tiles with dO beside Q; 2 x 4001 causal tokens as above: 216 us, 912 TFLOP/s over its three products,
// matrix units busy 57 % of the cycles.
template <typename T, int DP>
__global__ __launch_bounds__(256, (sizeof(T) == 4 && DP == 128 ? 1 : 2)) void attention_dq_kernel(const AttnArgs p) {
  using C = Cfg<T, DP>;
  constexpr int NW = 4;
  using I = typename C::I;
  constexpr int ROWB = C::ROWB, KT = C::KT;
  __shared__ __attribute__((aligned(1024))) char lds[4 * C::TILE];
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nbh = p.B * p.Hkv, tiles = (p.R + NW * 32 - 1) / (NW * 32);
  const int tile = tiles - 1 - (int)blockIdx.x / nbh, bh = (int)blockIdx.x % nbh;
  const int b = bh / p.Hkv, hk = bh - b * p.Hkv;
  const int n = keys_of(p, b), nchunk = p.D / C::EL;
  const int t = (tile * NW + wave) * 32 + (lane & 31);
  const bool live = t < p.R;
  const int i = row_token(p, t), gi = t - i * p.g;
  const int lim = row_limit(p, t, n);
  const int wt = (tile * NW + wave) * 32, wlast = wt + 31 < p.R ? wt + 31 : p.R - 1;
  const int wmax = wt < p.R ? row_limit(p, wlast, n) : 0;
  const int wmin = wt + 31 < p.R ? row_limit(p, wt, n) : 0;
  const int tlast = (tile + 1) * NW * 32 - 1 < p.R ? (tile + 1) * NW * 32 - 1 : p.R - 1;
  const int ke = row_limit(p, tlast, n);
  const int h = hk * p.g + gi;
  const size_t row = (size_t)bh * p.R + t;

  const T* kbase = (const T*)p.k + b * p.ks[0] + hk * p.ks[2];
  const T* vbase = (const T*)p.v + b * p.vs[0] + hk * p.vs[2];
  const unsigned kst = (unsigned)(p.ks[1] * sizeof(T)), vst = (unsigned)(p.vs[1] * sizeof(T));
  auto stage = [&](int kt, int buf) {
    char* d = lds + buf * 2 * C::TILE;
    stage_tile<ROWB, KT, NW, ROWB == 256>(d, kbase + (int64_t)kt * p.ks[1], n - kt, nchunk, wave, lane, [&](int r) { return (unsigned)r * kst; });
    stage_tile<ROWB, KT, NW, ROWB == 256>(d + C::TILE, vbase + (int64_t)kt * p.vs[1], n - kt, nchunk, wave, lane, [&](int r) { return (unsigned)r * vst; });
  };
  if (ke > 0) stage(0, 0);
  f32x4 qf[C::NC], gf[C::NC];
  load_frags<C::NC>(qf, (const char*)((const T*)p.q + b * p.qs[0] + (int64_t)i * p.qs[1] + (int64_t)h * p.qs[2]), live, nchunk, half);
  load_frags<C::NC>(gf, (const char*)((const T*)p.dout + b * p.dos[0] + (int64_t)i * p.dos[1] + (int64_t)h * p.dos[2]), live, nchunk, half);
  float dl = 0.f;
  {
    const char* orow = (const char*)((const T*)p.o + b * p.os[0] + (int64_t)i * p.os[1] + (int64_t)h * p.os[2]);
    const char* lrow = (const char*)(p.lo + (((size_t)b * p.Lq + i) * p.Hkv * p.g + h) * p.D);
#pragma unroll
    for (int cc = 0; cc < C::NC; ++cc)
      if (live && 2 * cc + half < nchunk) {
        const f32x4 of = *reinterpret_cast<const f32x4*>(orow + (2 * cc + half) * 16);
        if constexpr (sizeof(T) == 2) {
          const bf16x8 x = __builtin_bit_cast(bf16x8, of), y = __builtin_bit_cast(bf16x8, gf[cc]);
          const bf16x8 z = *reinterpret_cast<const bf16x8*>(lrow + (2 * cc + half) * 16);
#pragma unroll
          for (int e = 0; e < 8; ++e) dl = __builtin_fmaf((float)x[e] + (float)z[e], (float)y[e], dl);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) dl = __builtin_fmaf(of[e], gf[cc][e], dl);
        }
      }
    dl += __shfl_xor(dl, 32, 64);
    if (live && half == 0) p.delta[row] = dl;
  }
  const float lse = live ? p.lse[row] : INFINITY;
  f32x16 dq[C::ND];
#pragma unroll
  for (int d = 0; d < C::ND; ++d) dq[d] = zero16();
  const float c = p.c;
  int buf = 0;
  for (int kt = 0; kt < ke; kt += KT, buf ^= 1) {
    TILE_WAIT();
    if (kt + KT < ke) stage(kt + KT, buf ^ 1);
    if (kt >= wmax) continue;
    const char* kimg = lds + buf * 2 * C::TILE;
    const char* vimg = kimg + C::TILE;
    const bool masked = kt + KT > wmin;
#pragma unroll
    for (int s = 0; s < C::NS; ++s) {
      if (sizeof(T) == 4 && kt + s * 32 >= wmax) break;
      f32x16 st = zero16(), dp = zero16();
#pragma unroll
      for (int cc = 0; cc < C::NC; ++cc) {
        mma<T>(st, I::frag(kimg, s * 32 + (lane & 31), 2 * cc + half), qf[cc]);
        mma<T>(dp, I::frag(vimg, s * 32 + (lane & 31), 2 * cc + half), gf[cc]);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(st[r], c, -lse));
        st[r] = pr * (dp[r] - dl);
      }
      if (masked) {
#pragma unroll
        for (int r = 0; r < 16; ++r) st[r] = kt + s * 32 + 8 * (r >> 2) + 4 * half + (r & 3) < lim ? st[r] : 0.f;
      }
      mma_t<T, I, C::ND>(dq, kimg, s * 32, st, lane);
    }
  }
  if (!live) return;
  T* op = (T*)p.dq + b * p.dqs[0] + (int64_t)i * p.dqs[1] + (int64_t)h * p.dqs[2];
  const float sc = p.scale;
#pragma unroll
  for (int d = 0; d < C::ND; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int dd = d * 32 + 2 * r + 4 * half;
      if (dd < p.D) store4<T>(op + dd, dq[d][r] * sc, dq[d][r + 1] * sc, dq[d][r + 2] * sc, dq[d][r + 3] * sc);
    }
}

// -------------------------------------------------------------------------------------------------------------------- backward: dK and dV
// A wave owns 32 keys and both accumulators (128 registers at D 128) and walks the rows; bound by the little room that leaves: 246 registers, two
// waves a SIMD, matrix units busy 39 % of the cycles.  2 x 4001 causal tokens as above: 358 us, 732 TFLOP/s over its four products.
template <typename T, int DP, bool SPLIT>
__global__ __launch_bounds__(256, (sizeof(T) == 4 && DP == 128 ? 1 : 2)) void attention_dkv_kernel(const AttnArgs p) {
  using C = Cfg<T, DP>;
  constexpr int NW = 4;
  // D 128: the fragments of K (32 registers in bfloat16, 64 in float32), of V (as many) and the two accumulators (128) leave too little of 256 or
  // 512 registers.  With V in LDS and no spill: 2 x 4001 causal tokens, bfloat16, 3 % faster (V's 32 KiB beside tiles of 32 rows still let
  // two workgroups on a CU); 4000 causal tokens, 32 heads over 8, float32, 2919 -> 2478 us.  Four waves at any size: workgroups of one wave took
  // 347 us instead of 133 ([2 x 2001], 16 heads over 4, D 128, causal, bfloat16), and as long where there are few tokens
  constexpr bool VL = DP == 128;
  constexpr int ROWB = C::ROWB, KT = VL ? 32 : C::KT, NS = KT / 32;
  using I = Img<ROWB, KT, ROWB == 256>;
  using IV = Img<ROWB, NW * 32, ROWB == 256>;
  constexpr int TILE = I::BYTES;
  __shared__ __attribute__((aligned(1024))) char lds[4 * TILE + (VL ? IV::BYTES : 0)];
  char* const vimg = lds + 4 * TILE;
  __shared__ __attribute__((aligned(16))) float stat[2][3][KT];   // L, D and the limit of each staged row
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nbh = p.B * p.Hkv;
  int id = blockIdx.x, split = 0;   // causal: the first keys have the most rows, so their workgroups come first
  const int tile = id / (nbh * (SPLIT ? p.splits : 1));
  id -= tile * (nbh * (SPLIT ? p.splits : 1));
  if (SPLIT) {
    split = id / nbh;
    id -= split * nbh;
  }
  const int bh = id;
  const int b = bh / p.Hkv, hk = bh - b * p.Hkv;
  const int n = keys_of(p, b), nchunk = p.D / C::EL;
  const int k0 = tile * NW * 32, kw = k0 + wave * 32, key = kw + (lane & 31);
  const bool live = key < n;
  // rows that see a key of this tile: i >= k0 - n + Lq (below Lq, so i g fits: a tile behind the sequence's length has no rows to start from)
  int t0 = 0;
  if (p.causal && k0 < n) {
    const int i0 = k0 - n + p.Lq;
    t0 = i0 > 0 ? i0 * p.g : 0;
  }
  int te = k0 < n ? p.R : 0;
  if (SPLIT && t0 < te) {   // this split's share of the tile's rows
    const int share = ((te - t0 + p.splits - 1) / p.splits + 31) / 32 * 32, first = t0;
    t0 = first + split * share < te ? first + split * share : te;
    te = t0 + share < te ? t0 + share : te;
  }
  const int h0 = hk * p.g;
  f32x4 kf[C::NC], vf[VL ? 1 : C::NC];
  load_frags<C::NC>(kf, (const char*)((const T*)p.k + b * p.ks[0] + (int64_t)key * p.ks[1] + hk * p.ks[2]), live, nchunk, half);
  if constexpr (VL) {
    const unsigned vst = (unsigned)(p.vs[1] * sizeof(T));
    stage_tile<ROWB, NW * 32, NW, ROWB == 256>(vimg, (const T*)p.v + b * p.vs[0] + (int64_t)k0 * p.vs[1] + hk * p.vs[2], n - k0, nchunk, wave, lane,
                                               [&](int r) { return (unsigned)r * vst; });
  } else {
    load_frags<C::NC>(vf, (const char*)((const T*)p.v + b * p.vs[0] + (int64_t)key * p.vs[1] + hk * p.vs[2]), live, nchunk, half);
  }
  const T* qbase = (const T*)p.q + b * p.qs[0] + h0 * p.qs[2];
  const T* gbase = (const T*)p.dout + b * p.dos[0] + h0 * p.dos[2];
  const unsigned ql = (unsigned)(p.qs[1] * sizeof(T)), qh = (unsigned)(p.qs[2] * sizeof(T));
  const unsigned gl = (unsigned)(p.dos[1] * sizeof(T)), gh = (unsigned)(p.dos[2] * sizeof(T));
  auto stage = [&](int tt, int buf) {
    char* d = lds + buf * 2 * TILE;
    const int i0 = row_token(p, tt);
    stage_tile<ROWB, KT, NW, ROWB == 256>(d, qbase + (int64_t)i0 * p.qs[1], te - tt, nchunk, wave, lane, [&](int r) {
      if (p.g == 1) return (unsigned)r * ql;
      const int x = tt + r, i = row_token(p, x);
      return (unsigned)(i - i0) * ql + (unsigned)(x - i * p.g) * qh;
    });
    stage_tile<ROWB, KT, NW, ROWB == 256>(d + TILE, gbase + (int64_t)i0 * p.dos[1], te - tt, nchunk, wave, lane, [&](int r) {
      if (p.g == 1) return (unsigned)r * gl;
      const int x = tt + r, i = row_token(p, x);
      return (unsigned)(i - i0) * gl + (unsigned)(x - i * p.g) * gh;
    });
  };
  const float* lsep = p.lse + (size_t)bh * p.R;
  const float* delp = p.delta + (size_t)bh * p.R;
  auto put_stat = [&](int tt, int buf, float ls, float de) {
    if ((int)threadIdx.x < KT) {
      stat[buf][0][threadIdx.x] = ls;
      stat[buf][1][threadIdx.x] = de;
      stat[buf][2][threadIdx.x] = __int_as_float(tt + (int)threadIdx.x < te ? row_limit(p, tt + (int)threadIdx.x, n) : 0);
    }
  };
  auto get_stat = [&](int tt, float& ls, float& de) {
    const int x = tt + (int)threadIdx.x;
    ls = INFINITY;
    de = 0.f;
    if ((int)threadIdx.x < KT && x < te) {
      ls = lsep[x];
      de = delp[x];
    }
  };
  f32x16 dk[C::ND], dv[C::ND];
#pragma unroll
  for (int d = 0; d < C::ND; ++d) dk[d] = dv[d] = zero16();
  const float c = p.c;
  if (t0 < te) {
    float ls, de;
    stage(t0, 0);
    get_stat(t0, ls, de);
    put_stat(t0, 0, ls, de);
  }
  int buf = 0;
  for (int tt = t0; tt < te; tt += KT, buf ^= 1) {
    TILE_WAIT();
    const bool more = tt + KT < te;
    float ls = 0.f, de = 0.f;
    if (more) {
      stage(tt + KT, buf ^ 1);
      get_stat(tt + KT, ls, de);
    }
    const int last = tt + KT - 1 < te ? tt + KT - 1 : te - 1;
    if (kw < row_limit(p, last, n)) {
      const char* qimg = lds + buf * 2 * TILE;
      const char* gimg = qimg + TILE;
      const bool masked = kw + 32 > row_limit(p, tt, n);   // rows behind `te` have L = inf: their P is 0 without a mask
#pragma unroll 1
      for (int s = 0; s < NS; ++s) {
        const int end = tt + s * 32 + 31 < last ? tt + s * 32 + 31 : last;
        if (NS > 1 && (tt + s * 32 > last || kw >= row_limit(p, end, n))) continue;   // no row of these 32 sees a key of the wave
        f32x16 st = zero16();
#pragma unroll
        for (int cc = 0; cc < C::NC; ++cc) mma<T>(st, I::frag(qimg, s * 32 + (lane & 31), 2 * cc + half), kf[cc]);
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const int at = s * 32 + 8 * r4 + 4 * half;
          const f32x4 L = *reinterpret_cast<const f32x4*>(&stat[buf][0][at]);
#pragma unroll
          for (int e = 0; e < 4; ++e) st[r4 * 4 + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[r4 * 4 + e], c, -L[e]));
          if (masked) {   // a masked P is 0, and so is its dS
            const f32x4 lm = *reinterpret_cast<const f32x4*>(&stat[buf][2][at]);
#pragma unroll
            for (int e = 0; e < 4; ++e) st[r4 * 4 + e] = key < __float_as_int(lm[e]) ? st[r4 * 4 + e] : 0.f;
          }
        }
        mma_t<T, I, C::ND>(dv, gimg, s * 32, st, lane);
        f32x16 dp = zero16();
#pragma unroll
        for (int cc = 0; cc < C::NC; ++cc) mma<T>(dp, I::frag(gimg, s * 32 + (lane & 31), 2 * cc + half), VL ? IV::frag(vimg, wave * 32 + (lane & 31), 2 * cc + half) : vf[VL ? 0 : cc]);
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const f32x4 De = *reinterpret_cast<const f32x4*>(&stat[buf][1][s * 32 + 8 * r4 + 4 * half]);
#pragma unroll
          for (int e = 0; e < 4; ++e) dp[r4 * 4 + e] = st[r4 * 4 + e] * (dp[r4 * 4 + e] - De[e]);
        }
        mma_t<T, I, C::ND>(dk, qimg, s * 32, dp, lane);
      }
    }
    if (more) put_stat(tt + KT, buf ^ 1, ls, de);
  }
  if (key >= p.Lk) return;   // keys behind the sequence's length get zeros
  const float sc = p.scale;
  if (SPLIT) {   // fp32 partials [split][bh][key][dK | dV][D]
    float* pp = p.part + (((size_t)split * nbh + bh) * p.Lk + key) * 2 * p.D;
#pragma unroll
    for (int d = 0; d < C::ND; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int dd = d * 32 + 2 * r + 4 * half;
        if (dd < p.D) {
          store4<float>(pp + dd, dk[d][r] * sc, dk[d][r + 1] * sc, dk[d][r + 2] * sc, dk[d][r + 3] * sc);
          store4<float>(pp + p.D + dd, dv[d][r], dv[d][r + 1], dv[d][r + 2], dv[d][r + 3]);
        }
      }
    return;
  }
  T* kp = (T*)p.dk + b * p.dks[0] + (int64_t)key * p.dks[1] + hk * p.dks[2];
  T* vp = (T*)p.dv + b * p.dvs[0] + (int64_t)key * p.dvs[1] + hk * p.dvs[2];
#pragma unroll
  for (int d = 0; d < C::ND; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int dd = d * 32 + 2 * r + 4 * half;
      if (dd < p.D) {
        store4<T>(kp + dd, dk[d][r] * sc, dk[d][r + 1] * sc, dk[d][r + 2] * sc, dk[d][r + 3] * sc);
        store4<T>(vp + dd, dv[d][r], dv[d][r + 1], dv[d][r + 2], dv[d][r + 3]);
      }
    }
}

// the splits' dK and dV summed in split order; a thread owns four values
template <typename T>
__global__ __launch_bounds__(256) void attention_dkv_join_kernel(const AttnArgs p) {
  const int64_t per = (int64_t)p.B * p.Hkv * p.Lk * 2 * p.D, at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= per) return;
  f32x4 a = *reinterpret_cast<const f32x4*>(p.part + at);
  for (int s = 1; s < p.splits; ++s) a += *reinterpret_cast<const f32x4*>(p.part + s * per + at);
  const int d = (int)(at % p.D), kv = (int)(at / p.D) & 1;
  const int64_t rest = at / (2 * p.D);
  const int key = (int)(rest % p.Lk), bh = (int)(rest / p.Lk), b = bh / p.Hkv, hk = bh - b * p.Hkv;
  T* op = kv ? (T*)p.dv + b * p.dvs[0] + (int64_t)key * p.dvs[1] + hk * p.dvs[2] : (T*)p.dk + b * p.dks[0] + (int64_t)key * p.dks[1] + hk * p.dks[2];
  store4<T>(op + d, a[0], a[1], a[2], a[3]);
}

// --------------------------------------------------------------------------------------------------------------------------------- host
constexpr int64_t SPAN = 0x7fffffff;

static int cus() { return 256; }   // MI355X

// Keys per split of the forward.  Up to 32 rows (a few tokens over a cache): one wave a workgroup, 8 workgroups a CU where fewer than 2 a CU
// would run.  Measured on one token over 16 ragged caches of up to 32768 keys, 32 heads over 8, join included: 4 workgroups a CU take as
// long as 8, 16 take 5 % longer; the lengths are ragged, so the finer of the two that tie.  More rows: four waves, 4 workgroups a CU where fewer than
// one would run.  [1 x 16000] tokens, one head of 128, bfloat16: 277 us with one-wave workgroups in 5 splits, 123 with four waves in 9;
// [1 x 500] over 20000 keys, 8 heads of 64: 74, 55; float32 [1 x 2048], 8 heads over 2 of 64: 152 unsplit, 99.  Pieces under 256 keys would pay
// more for the join than they gain
static int fwd_splits(int64_t wgs, int waves, int Lk, int* chunk) {
  *chunk = Lk;
  if (wgs <= 0 || wgs >= (waves == 4 ? 1 : 2) * cus() || Lk <= 512) return 1;
  int64_t s = ((waves == 4 ? 4 : 8) * cus() + wgs - 1) / wgs, most = (Lk + 255) / 256;
  if (s > most) s = most;
  if (s <= 1) return 1;
  int c = (int)((Lk + s - 1) / s);
  c = (c + 63) / 64 * 64;
  *chunk = c;
  return (Lk + c - 1) / c;
}

// Row splits of the dK, dV launch: its workgroups (128 keys of a head) run two to a CU (D 128 float32: one), and a causal head's are unequal, so
// two rounds' worth are wanted while there are 512 rows for each; where half the chip would idle, one round's worth down to 128 rows each.
// 2 x 4001 causal tokens, 16 heads over 4, D 128 (256 workgroups unsplit), join included, relative to four splits: none 2.35, two 1.39, eight
// 1.10.  [1 x 1000], 8 heads of 64 (64 workgroups): unsplit 42 us, 7 splits 23 with the join; [4 x 333], 16 heads of 128 (192): unsplit 29, two 36
static int dkv_splits(int64_t wgs, int64_t R) {
  if (wgs <= 0) return 1;
  int64_t s = (4 * cus() + wgs - 1) / wgs, fill = 2 * wgs <= cus() ? 2 * cus() / wgs : 1;
  if (s > R / 512) s = R / 512;
  if (fill > R / 128) fill = R / 128;
  if (s < fill) s = fill;
  return s < 1 ? 1 : (int)s;
}

struct Plan {
  int fw, fsplits, fchunk, ksplits;
  size_t fwd_bytes, bwd_bytes;
};

static Plan make_plan(int64_t B, int64_t Lq, int64_t Lk, int64_t Hq, int64_t Hkv, int64_t D) {
  Plan p;
  const int64_t nbh = B * Hkv, R = Lq * (Hq / Hkv);
  p.fw = R > 32 ? 4 : 1;
  p.fsplits = fwd_splits((R + p.fw * 32 - 1) / (p.fw * 32) * nbh, p.fw, (int)Lk, &p.fchunk);
  if (p.fsplits == 1) p.fw = 4;   // four waves stage a tile together, however few of them have rows ([4 x 333], 16 heads of 128: 32 us, 18)
  p.fwd_bytes = p.fsplits > 1 ? (size_t)p.fsplits * nbh * R * (D + 4) * sizeof(float) : 0;
  p.ksplits = dkv_splits((Lk + 127) / 128 * nbh, R);
  p.bwd_bytes = (size_t)nbh * R * sizeof(float);
  p.bwd_bytes = (p.bwd_bytes + 255) / 256 * 256;
  if (p.ksplits > 1) p.bwd_bytes += (size_t)p.ksplits * nbh * Lk * 2 * D * sizeof(float);
  return p;
}

static int check_shape(int B, int Lq, int Lk, int Hq, int Hkv, int D, int dtype) {
  if (B < 0 || Lq < 0 || Lk < 0 || Hq <= 0 || Hkv <= 0 || (dtype != COIN_F32 && dtype != COIN_BF16)) return COIN_EINVAL;
  if (Hq % Hkv || D <= 0 || D > 128 || D % (dtype == COIN_BF16 ? 8 : 4)) return COIN_ESHAPE;
  const int64_t g = Hq / Hkv, nbh = (int64_t)B * Hkv, R = (int64_t)Lq * g;
  if (Lk > (1 << 30) || R > (1 << 30) || nbh > (1 << 24)) return COIN_ESHAPE;
  // grids stay below 2^31 workgroups (the joins: one per four rows / 1024 values)
  if (((R + 31) / 32 + 1) * nbh * 64 >= SPAN || ((int64_t)Lk / 32 + 1) * nbh * 64 >= SPAN || nbh * R >= SPAN || nbh * Lk * 2 * D / 1024 >= SPAN) return COIN_ESHAPE;
  return COIN_OK;
}

// strides of a [B, L, H, D] tensor: multiples of 16 bytes, a staged tile's offsets below 2^31
static int check_tensor(const void* p, const int64_t* s, int es, int64_t g) {
  if (!p || !s) return COIN_EINVAL;
  if ((uintptr_t)p & 15) return COIN_EALIGN;
  for (int i = 0; i < 3; ++i)
    if (s[i] < 0 || (s[i] * es) & 15) return COIN_EALIGN;
  if (s[1] >= SPAN || s[2] >= SPAN || 130 * s[1] * es + g * s[2] * es >= SPAN) return COIN_ESHAPE;
  return COIN_OK;
}

template <typename T, int DP>
static void launch_fwd(const AttnArgs& a, const Plan& pl, hipStream_t st) {
  const int64_t nbh = (int64_t)a.B * a.Hkv;
  const unsigned grid = (unsigned)((a.R + pl.fw * 32 - 1) / (pl.fw * 32) * nbh * pl.fsplits);
  if (pl.fsplits > 1) {
    if (pl.fw == 1) attention_fwd_kernel<T, DP, 1, true><<<grid, 64, 0, st>>>(a);
    else attention_fwd_kernel<T, DP, 4, true><<<grid, 256, 0, st>>>(a);
    attention_join_kernel<T><<<(unsigned)((nbh * a.R + 3) / 4), 256, 0, st>>>(a);
  } else {
    attention_fwd_kernel<T, DP, 4, false><<<grid, 256, 0, st>>>(a);
  }
}

template <typename T, int DP>
static void launch_bwd(const AttnArgs& a, const Plan& pl, hipStream_t st) {
  const int64_t nbh = (int64_t)a.B * a.Hkv;
  if (a.R > 0) {
    attention_dq_kernel<T, DP><<<(unsigned)((a.R + 127) / 128 * nbh), 256, 0, st>>>(a);
  }
  if (a.Lk > 0) {
    const unsigned grid = (unsigned)((a.Lk + 127) / 128 * nbh * pl.ksplits);
    if (pl.ksplits > 1) {
      attention_dkv_kernel<T, DP, true><<<grid, 256, 0, st>>>(a);
      attention_dkv_join_kernel<T><<<(unsigned)((nbh * a.Lk * 2 * a.D / 4 + 255) / 256), 256, 0, st>>>(a);
    } else {
      attention_dkv_kernel<T, DP, false><<<grid, 256, 0, st>>>(a);
    }
  }
}

template <typename T>
static void launch(const AttnArgs& a, const Plan& pl, bool bwd, hipStream_t st) {
  if (a.D <= 32) bwd ? launch_bwd<T, 32>(a, pl, st) : launch_fwd<T, 32>(a, pl, st);
  else if (a.D <= 64) bwd ? launch_bwd<T, 64>(a, pl, st) : launch_fwd<T, 64>(a, pl, st);
  else bwd ? launch_bwd<T, 128>(a, pl, st) : launch_fwd<T, 128>(a, pl, st);
}

static void set3(int64_t (&d)[3], const int64_t* s) {
  for (int i = 0; i < 3; ++i) d[i] = s[i];
}

}  // namespace

extern "C" size_t coin_attention_workspace_bytes(int B, int Lq, int Lk, int Hq, int Hkv, int D, int dtype, int backward) {
  if (check_shape(B, Lq, Lk, Hq, Hkv, D, dtype) != COIN_OK || B == 0) return 0;
  const Plan pl = make_plan(B, Lq, Lk, Hq, Hkv, D);
  return backward ? pl.bwd_bytes : pl.fwd_bytes;
}

extern "C" int coin_attention_fwd(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                                  void* out, const int64_t* out_strides, void* out_lo, float* lse, const int* key_lengths, int B, int Lq, int Lk, int Hq, int Hkv,
                                  int D, int causal, float scale, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_shape(B, Lq, Lk, Hq, Hkv, D, dtype);
  if (rc != COIN_OK) return rc;
  if (!(scale > 0.f) || scale > 1.0e30f) return COIN_EINVAL;
  if (B == 0 || Lq == 0) return COIN_OK;
  const int es = dtype == COIN_BF16 ? 2 : 4, g = Hq / Hkv;
  if ((rc = check_tensor(q, q_strides, es, g)) != COIN_OK || (rc = check_tensor(out, out_strides, es, g)) != COIN_OK) return rc;
  if (Lk > 0 && ((rc = check_tensor(k, k_strides, es, 1)) != COIN_OK || (rc = check_tensor(v, v_strides, es, 1)) != COIN_OK)) return rc;
  const Plan pl = make_plan(B, Lq, Lk, Hq, Hkv, D);
  if (pl.fwd_bytes && (!workspace || workspace_bytes < pl.fwd_bytes)) return COIN_EINVAL;
  if (((uintptr_t)workspace | (uintptr_t)out_lo) & 15) return COIN_EALIGN;
  AttnArgs a = {};
  a.lo = dtype == COIN_BF16 ? (bf16_t*)out_lo : nullptr;
  a.q = q; a.k = k; a.v = v; a.out = out; a.lse = lse; a.lengths = key_lengths;
  set3(a.qs, q_strides); set3(a.os, out_strides);
  if (Lk > 0) { set3(a.ks, k_strides); set3(a.vs, v_strides); }
  a.B = B; a.Lq = Lq; a.Lk = Lk; a.Hkv = Hkv; a.g = g; a.D = D; a.R = Lq * g; a.magic = (unsigned)(((1ull << 32) + g - 1) / g);
  a.causal = causal != 0; a.splits = pl.fsplits; a.chunk = pl.fchunk; a.scale = scale; a.c = scale * LOG2E;
  a.part = (float*)workspace;
  a.part_ml = a.part + (size_t)pl.fsplits * B * Hkv * a.R * D;
  if (dtype == COIN_BF16) launch<bf16_t>(a, pl, false, (hipStream_t)stream);
  else launch<float>(a, pl, false, (hipStream_t)stream);
  return coin_launch_status();
}

extern "C" int coin_attention_bwd(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                                  const void* out, const int64_t* out_strides, const void* out_lo, const void* dout, const int64_t* dout_strides, const float* lse,
                                  const int* key_lengths, void* dq, const int64_t* dq_strides, void* dk, const int64_t* dk_strides, void* dv,
                                  const int64_t* dv_strides, int B, int Lq, int Lk, int Hq, int Hkv, int D, int causal, float scale, int dtype,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_shape(B, Lq, Lk, Hq, Hkv, D, dtype);
  if (rc != COIN_OK) return rc;
  if (!(scale > 0.f) || scale > 1.0e30f) return COIN_EINVAL;
  if (B == 0 || (Lq == 0 && Lk == 0)) return COIN_OK;
  const int es = dtype == COIN_BF16 ? 2 : 4, g = Hq / Hkv;
  AttnArgs a = {};
  if (Lq > 0) {
    if (!lse || (dtype == COIN_BF16 && !out_lo)) return COIN_EINVAL;
    if ((rc = check_tensor(q, q_strides, es, g)) != COIN_OK || (rc = check_tensor(out, out_strides, es, g)) != COIN_OK ||
        (rc = check_tensor(dout, dout_strides, es, g)) != COIN_OK || (rc = check_tensor(dq, dq_strides, es, g)) != COIN_OK)
      return rc;
    set3(a.qs, q_strides); set3(a.os, out_strides); set3(a.dos, dout_strides); set3(a.dqs, dq_strides);
  }
  if (Lk > 0) {
    if ((rc = check_tensor(k, k_strides, es, 1)) != COIN_OK || (rc = check_tensor(v, v_strides, es, 1)) != COIN_OK ||
        (rc = check_tensor(dk, dk_strides, es, 1)) != COIN_OK || (rc = check_tensor(dv, dv_strides, es, 1)) != COIN_OK)
      return rc;
    set3(a.ks, k_strides); set3(a.vs, v_strides); set3(a.dks, dk_strides); set3(a.dvs, dv_strides);
  }
  const Plan pl = make_plan(B, Lq, Lk, Hq, Hkv, D);
  if (pl.bwd_bytes && (!workspace || workspace_bytes < pl.bwd_bytes)) return COIN_EINVAL;
  if (((uintptr_t)workspace | (uintptr_t)out_lo) & 15) return COIN_EALIGN;
  a.lo = (bf16_t*)const_cast<void*>(out_lo);
  a.q = q; a.k = k; a.v = v; a.o = out; a.dout = dout; a.dq = dq; a.dk = dk; a.dv = dv; a.lse = const_cast<float*>(lse); a.lengths = key_lengths;
  a.B = B; a.Lq = Lq; a.Lk = Lk; a.Hkv = Hkv; a.g = g; a.D = D; a.R = Lq * g; a.magic = (unsigned)(((1ull << 32) + g - 1) / g);
  a.causal = causal != 0; a.splits = pl.ksplits; a.scale = scale; a.c = scale * LOG2E;
  a.delta = (float*)workspace;
  a.part = (float*)((char*)workspace + ((size_t)B * Hkv * a.R * sizeof(float) + 255) / 256 * 256);
  if (dtype == COIN_BF16) launch<bf16_t>(a, pl, true, (hipStream_t)stream);
  else launch<float>(a, pl, true, (hipStream_t)stream);
  return coin_launch_status();
}
