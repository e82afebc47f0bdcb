// Residual add of a transformer block with the norm behind the block's branch, its gate and scale, and the norm before the next branch
// (coin_residual_norm_fwd / _bwd):
//
//   r = x + scale * gate o N_post(y),   h = N_pre(r),      N(u) = (u - mu) / sqrt(var + eps) o w + b   (RMSNorm: u / sqrt(mean u^2 + eps) o w)
//
// each of y, gate, N_post, N_pre may be absent.  Backward with e = dr + N_pre'(dh):  dx = e,  dgate = sum_rows scale e N_post(y),
// df = scale gate o e,  dy = N_post'(df);   N'(g) = (gw - mean(gw) - n mean(gw n)) / sigma with gw = g o w, n the normalised row (RMSNorm:
// without mean(gw));  dw = sum_rows g n,  db = sum_rows g.
//
// Bound by memory: x and y are read once and r and h written once; the backward reads x, y, dr, dh and writes dx, dy.  It computes r again
// from x and y (not from the rounded r), so its normalised rows are exactly the forward's; only the rows' means and deviations (four
// floats a row) are kept from the forward.  A row lives in the registers of TPR threads, two passes over registers give mean and variance.
// 32768 rows of 2048, float32 stream, bfloat16 branch, gate and both norms: forward 156 us at 5.2 TB/s, backward 298 us at 4.05 TB/s (a copy of
// 2 GiB: 4.8), its column sums 15 + 7 us.  All sums are float32.  The backward's `walkers` (TPR threads each) own contiguous rows and hold
// the column sums of dw, db and dgate in registers; the walkers of a workgroup meet in LDS, the workgroups in a second launch that adds them
// in order: no atomics, the same bits every time.
#include "common.h"

namespace {

struct NormArgs {
  const void *x, *y, *gate, *dr, *dh;
  void *r, *h, *dx, *dy;
  const float *post_w, *post_b, *pre_w, *pre_b;
  float* stats;                   // [M][4]: mean, 1 / deviation behind the branch, mean, 1 / deviation before the next
  float* part;                    // [workgroups][5][D]: dw_post, db_post, dw_pre, db_pre, dgate (one gate for all rows)
  float* gpart;                   // [walkers][2][D]: a walker's first and last group of dgate
  void* dgate;
  int64_t M, group;               // group = rows that share a gate row
  int64_t rows;                   // rows of a walker
  int D, gate_bf16, has_post, has_pre, want_gate;   // want_gate: 0 no, 1 one row of gate for all, 2 groups
  int want_param, rms;
  float scale, post_eps, pre_eps;
};

// eight columns from `col` on; VECT: D and every pointer allow 16-byte accesses, else column by column up to D
template <bool VECT, typename T>
__device__ __forceinline__ void load8(float (&o)[8], const T* p, int left) {
  if constexpr (VECT && sizeof(T) == 2) {
    const bf16x8 v = *reinterpret_cast<const bf16x8*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (float)v[i];
  } else if constexpr (VECT) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[i] = a[i];
      o[4 + i] = b[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = i < left ? (float)p[i] : 0.f;
  }
}

template <bool VECT, typename T>
__device__ __forceinline__ void store8(T* p, const float (&o)[8], int left) {
  if constexpr (VECT && sizeof(T) == 2) {
    bf16x8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (bf16_t)o[i];
    *reinterpret_cast<bf16x8*>(p) = v;
  } else if constexpr (VECT) {
    *reinterpret_cast<f32x4*>(p) = (f32x4){o[0], o[1], o[2], o[3]};
    *reinterpret_cast<f32x4*>(p + 4) = (f32x4){o[4], o[5], o[6], o[7]};
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = (T)o[i];
  }
}

// sums of a and b over the TPR threads of a row, in every one of them; `red`: this use's own 8 floats of LDS (TPR == 256)
template <int TPR>
__device__ __forceinline__ void row_sum2(float& a, float& b, float* red) {
#pragma unroll
  for (int o = (TPR > 64 ? 32 : TPR / 2); o > 0; o >>= 1) {
    a += __shfl_xor(a, o, 64);
    b += __shfl_xor(b, o, 64);
  }
  if constexpr (TPR == 256) {
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
      red[w * 2] = a;
      red[w * 2 + 1] = b;
    }
    __syncthreads();
    a = (red[0] + red[2]) + (red[4] + red[6]);
    b = (red[1] + red[3]) + (red[5] + red[7]);
  }
}

// mean and 1 / deviation of a row held as v[NV][8] (whole chunks behind D hold zeros)
template <bool VECT, int TPR, int NV>
__device__ __forceinline__ void row_stats(const float (&v)[NV][8], int D, int sub, float eps, bool rms, float& mean, float& rstd, float* red) {
  float s = 0.f, q = 0.f;
  mean = 0.f;
  if (!rms) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) s += VECT || (sub + k * TPR) * 8 + i < D ? v[k][i] : 0.f;
    row_sum2<TPR>(s, q, red);
    mean = s / (float)D;
  }
  s = q = 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k)
    if ((sub + k * TPR) * 8 < D) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = VECT || (sub + k * TPR) * 8 + i < D ? v[k][i] - mean : 0.f;
        q = __builtin_fmaf(d, d, q);
      }
    }
  row_sum2<TPR>(q, s, red + 8);
  rstd = 1.f / __builtin_sqrtf(q / (float)D + eps);
}

template <bool VECT>
__device__ __forceinline__ void load_gate(float (&g)[8], const NormArgs& p, int64_t at, int left) {
  if (p.gate_bf16) load8<VECT>(g, (const bf16_t*)p.gate + at, left);
  else load8<VECT>(g, (const float*)p.gate + at, left);
}

template <typename TS, typename TB, bool VECT, int TPR, int NV>
__global__ __launch_bounds__(256) void residual_norm_fwd_kernel(const NormArgs p) {
  __shared__ float buf[2][32];   // the row sums of even and of odd turns: a turn's barriers are all that keeps the next but one off its buffer
  const int sub = threadIdx.x % TPR;
  constexpr int RPW = 256 / TPR;
  const int64_t step = (int64_t)gridDim.x * RPW;
  // a workgroup-wide trip count: the barriers inside the row sums are reached by every thread
  int turn = 0;
  for (int64_t base = (int64_t)blockIdx.x * RPW; base < p.M; base += step, turn ^= 1) {
    float* red = buf[turn];
    const int64_t row = base + threadIdx.x / TPR;
    const bool live = row < p.M;
    float r[NV][8], f[NV][8];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int col = (sub + k * TPR) * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) r[k][i] = f[k][i] = 0.f;
      if (live && col < p.D) {
        load8<VECT>(r[k], (const TS*)p.x + row * p.D + col, p.D - col);
        if (p.y) load8<VECT>(f[k], (const TB*)p.y + row * p.D + col, p.D - col);
      }
    }
    float mp = 0.f, sp = 0.f, mr = 0.f, sr = 0.f;
    if (p.y) {
      if (p.has_post) row_stats<VECT, TPR, NV>(f, p.D, sub, p.post_eps, p.rms, mp, sp, red);
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int col = (sub + k * TPR) * 8;
        if (!live || col >= p.D) continue;
        if (p.has_post) {
          float w[8], b[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            w[i] = 1.f;
            b[i] = 0.f;
          }
          if (p.post_w) load8<VECT>(w, p.post_w + col, p.D - col);
          if (p.post_b) load8<VECT>(b, p.post_b + col, p.D - col);
#pragma unroll
          for (int i = 0; i < 8; ++i) f[k][i] = __builtin_fmaf((f[k][i] - mp) * sp, w[i], b[i]);
        }
        if (p.gate) {
          float g[8];
          load_gate<VECT>(g, p, row / p.group * p.D + col, p.D - col);
#pragma unroll
          for (int i = 0; i < 8; ++i) f[k][i] *= g[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) r[k][i] = __builtin_fmaf(p.scale, f[k][i], r[k][i]);
        if (p.r) store8<VECT>((TS*)p.r + row * p.D + col, r[k], p.D - col);
      }
    }
    if (p.has_pre) {
      row_stats<VECT, TPR, NV>(r, p.D, sub, p.pre_eps, p.rms, mr, sr, red + 16);
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int col = (sub + k * TPR) * 8;
        if (!live || col >= p.D) continue;
        float w[8], b[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          w[i] = 1.f;
          b[i] = 0.f;
        }
        if (p.pre_w) load8<VECT>(w, p.pre_w + col, p.D - col);
        if (p.pre_b) load8<VECT>(b, p.pre_b + col, p.D - col);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = __builtin_fmaf((r[k][i] - mr) * sr, w[i], b[i]);
        store8<VECT>((TB*)p.h + row * p.D + col, w, p.D - col);
      }
    }
    if (p.stats && live && sub == 0) *reinterpret_cast<f32x4*>(p.stats + row * 4) = (f32x4){mp, sp, mr, sr};
  }
}

template <typename TS, typename TB, bool VECT, int TPR, int NV>
__global__ __launch_bounds__(256) void residual_norm_bwd_kernel(const NormArgs p) {
  constexpr int RPW = 256 / TPR;
  __shared__ float red[32];
  __shared__ float comb[RPW > 1 ? RPW * TPR * 8 : 1];
  const int sub = threadIdx.x % TPR, slot = threadIdx.x / TPR;
  const int64_t walker = (int64_t)blockIdx.x * RPW + slot;
  const int64_t r0 = walker * p.rows;
  float a_pw[NV][8], a_pb[NV][8], a_nw[NV][8], a_nb[NV][8], a_g[NV][8];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) a_pw[k][i] = a_pb[k][i] = a_nw[k][i] = a_nb[k][i] = a_g[k][i] = 0.f;
  const int64_t head = r0 / p.group;
  int64_t cur = head;
  const float invd = 1.f / (float)p.D;
  for (int64_t j = 0; j < p.rows; ++j) {   // every walker of a workgroup makes the same number of turns: the barriers match
    const int64_t row = r0 + j;
    const bool live = row < p.M;
    if (p.want_gate == 2 && live) {
      const int64_t g = row / p.group;
      if (g != cur) {   // the group that ends here: the walker's first goes to its slot, one in between is whole
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          const int col = (sub + k * TPR) * 8;
          if (col < p.D) {
            if (cur == head) store8<VECT>(p.gpart + walker * 2 * p.D + col, a_g[k], p.D - col);
            else if (p.gate_bf16) store8<VECT>((bf16_t*)p.dgate + cur * p.D + col, a_g[k], p.D - col);
            else store8<VECT>((float*)p.dgate + cur * p.D + col, a_g[k], p.D - col);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) a_g[k][i] = 0.f;
        }
        cur = g;
      }
    }
    float r[NV][8], f[NV][8], e[NV][8];
    f32x4 st = (f32x4){0.f, 0.f, 0.f, 0.f};
    if (live) st = *reinterpret_cast<const f32x4*>(p.stats + row * 4);
    const float mp = st[0], sp = st[1], mr = st[2], sr = st[3];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int col = (sub + k * TPR) * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) r[k][i] = f[k][i] = e[k][i] = 0.f;
      if (!live || col >= p.D) continue;
      const int64_t at = row * p.D + col;
      if (p.y) {
        load8<VECT>(f[k], (const TB*)p.y + at, p.D - col);
        if (p.has_post) {
#pragma unroll
          for (int i = 0; i < 8; ++i) f[k][i] = (f[k][i] - mp) * sp;   // the normalised row from here on
        }
      }
      if (p.dr) load8<VECT>(e[k], (const TS*)p.dr + at, p.D - col);
      if (p.dh) {
        load8<VECT>(r[k], (const TS*)p.x + at, p.D - col);
        if (p.y) {
          float b[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) b[i] = f[k][i];
          if (p.has_post) {
            float w[8], c[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              w[i] = 1.f;
              c[i] = 0.f;
            }
            if (p.post_w) load8<VECT>(w, p.post_w + col, p.D - col);
            if (p.post_b) load8<VECT>(c, p.post_b + col, p.D - col);
#pragma unroll
            for (int i = 0; i < 8; ++i) b[i] = __builtin_fmaf(b[i], w[i], c[i]);
          }
          if (p.gate) {
            float g[8];
            load_gate<VECT>(g, p, row / p.group * p.D + col, p.D - col);
#pragma unroll
            for (int i = 0; i < 8; ++i) b[i] *= g[i];
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) r[k][i] = __builtin_fmaf(p.scale, b[i], r[k][i]);
        }
        float dh[8], w[8];
        load8<VECT>(dh, (const TB*)p.dh + at, p.D - col);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = 1.f;
        if (p.pre_w) load8<VECT>(w, p.pre_w + col, p.D - col);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          r[k][i] = (r[k][i] - mr) * sr;
          a_nw[k][i] = __builtin_fmaf(dh[i], r[k][i], a_nw[k][i]);
          a_nb[k][i] += dh[i];
          const float gw = dh[i] * w[i];
          s1 += gw;
          s2 = __builtin_fmaf(gw, r[k][i], s2);
          e[k][i] = __builtin_fmaf(sr, gw, e[k][i]);
        }
      }
    }
    if (p.dh) {
      row_sum2<TPR>(s1, s2, red + (j & 1) * 8);   // one barrier a sum: the buffers of even and odd turns alternate
      s1 = p.rms ? 0.f : s1 * invd * sr;
      s2 = s2 * invd * sr;
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) e[k][i] -= __builtin_fmaf(r[k][i], s2, s1);
    }
    if (p.dx && live) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int col = (sub + k * TPR) * 8;
        if (col < p.D) store8<VECT>((TS*)p.dx + row * p.D + col, e[k], p.D - col);
      }
    }
    if (!p.y) continue;
    s1 = s2 = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int col = (sub + k * TPR) * 8;
      if (!live || col >= p.D) continue;
#pragma unroll
      for (int i = 0; i < 8; ++i) e[k][i] = VECT || col + i < p.D ? e[k][i] * p.scale : 0.f;
      float w[8], c[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        w[i] = 1.f;
        c[i] = 0.f;
      }
      if (p.post_w) load8<VECT>(w, p.post_w + col, p.D - col);
      if (p.gate) {
        float g[8];
        load_gate<VECT>(g, p, row / p.group * p.D + col, p.D - col);
        if (p.has_post && p.want_gate && p.post_b) load8<VECT>(c, p.post_b + col, p.D - col);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          a_g[k][i] = __builtin_fmaf(e[k][i], p.has_post ? __builtin_fmaf(f[k][i], w[i], c[i]) : f[k][i], a_g[k][i]);
          e[k][i] *= g[i];
        }
      }
      if (p.has_post) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          a_pw[k][i] = __builtin_fmaf(e[k][i], f[k][i], a_pw[k][i]);
          a_pb[k][i] += e[k][i];
          e[k][i] *= w[i];
          s1 += e[k][i];
          s2 = __builtin_fmaf(e[k][i], f[k][i], s2);
        }
      }
    }
    if (p.has_post) {
      row_sum2<TPR>(s1, s2, red + 16 + (j & 1) * 8);
      s1 = p.rms ? 0.f : s1 * invd;
      s2 = s2 * invd;
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) e[k][i] = sp * (e[k][i] - __builtin_fmaf(f[k][i], s2, s1));
    }
    if (p.dy && live) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int col = (sub + k * TPR) * 8;
        if (col < p.D) store8<VECT>((TB*)p.dy + row * p.D + col, e[k], p.D - col);
      }
    }
  }
  if (p.want_gate == 2 && r0 < p.M) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int col = (sub + k * TPR) * 8;
      if (col < p.D) store8<VECT>(p.gpart + (walker * 2 + (cur == head ? 0 : 1)) * p.D + col, a_g[k], p.D - col);
    }
  }
  if (!p.want_param && p.want_gate != 1) return;
  // the workgroup's column sums: its walkers meet in LDS, in order
  auto put = [&](int which, float (&a)[NV][8]) {
    float* out = p.part + ((int64_t)blockIdx.x * 5 + which) * p.D;
    if constexpr (RPW > 1) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) comb[(slot * 8 + i) * TPR + sub] = a[k][i];
        __syncthreads();
        if (slot == 0) {
          const int col = (sub + k * TPR) * 8;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float s = comb[i * TPR + sub];
#pragma unroll
            for (int w = 1; w < RPW; ++w) s += comb[(w * 8 + i) * TPR + sub];
            if (col + i < p.D) out[col + i] = s;
          }
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int col = (sub + k * TPR) * 8;
        if (col < p.D) store8<VECT>(out + col, a[k], p.D - col);
      }
    }
  };
  if (p.want_param && p.has_post) {
    put(0, a_pw);
    put(1, a_pb);
  }
  if (p.want_param && p.has_pre && p.dh) {
    put(2, a_nw);
    put(3, a_nb);
  }
  if (p.want_gate == 1) put(4, a_g);
}

struct NormSums {
  const float* part;
  float* out[4];        // dw_post, db_post, dw_pre, db_pre; null: not wanted
  void* dgate;          // one gate row for all
  int gate_bf16, nwg, D;
};

// columns' sums over the workgroups, in order: 64 columns x 16 runs of workgroups, the runs meet in LDS.  grid.y = which sum
__global__ __launch_bounds__(1024) void residual_norm_sums_kernel(const NormSums p) {
  __shared__ float red[16][64];
  const int which = blockIdx.y, lane = threadIdx.x & 63, run = threadIdx.x >> 6, col = blockIdx.x * 64 + lane;
  if (which < 4 ? p.out[which] == nullptr : p.dgate == nullptr) return;
  const int per = (p.nwg + 15) / 16, w0 = run * per, w1 = w0 + per < p.nwg ? w0 + per : p.nwg;
  float s = 0.f;
  if (col < p.D)
    for (int w = w0; w < w1; ++w) s += p.part[((int64_t)w * 5 + which) * p.D + col];
  red[run][lane] = s;
  __syncthreads();
  if (run || col >= p.D) return;
  s = red[0][lane];
#pragma unroll
  for (int r = 1; r < 16; ++r) s += red[r][lane];
  if (which < 4) p.out[which][col] = s;
  else if (p.gate_bf16) ((bf16_t*)p.dgate)[col] = (bf16_t)s;
  else ((float*)p.dgate)[col] = s;
}

// dgate of one group: the walkers that hold a part of it, in order.  A group inside one walker's rows, with rows of other groups on both
// sides, was stored by that walker.  grid = (columns / 64, groups, up to 65535 at a time); 16 runs of walkers as above
__global__ __launch_bounds__(1024) void residual_norm_gate_kernel(const float* gpart, void* dgate, int gate_bf16, int64_t M, int64_t group, int64_t rows, int D, int64_t g0) {
  __shared__ float red[16][64];
  const int lane = threadIdx.x & 63, run = threadIdx.x >> 6, col = blockIdx.x * 64 + lane;
  const int64_t g = g0 + blockIdx.y, first = g * group, last = first + group - 1;
  const int64_t w0 = first / rows, w1 = last / rows;
  if (w0 == w1) {
    const int64_t b = w0 * rows, e = b + rows < M ? b + rows : M;
    if (first / group != b / group && last / group != (e - 1) / group) return;
  }
  const int64_t n = w1 - w0 + 1, per = (n + 15) / 16;
  float s = 0.f;
  if (col < D)
    for (int64_t w = w0 + run * per; w < w0 + (run + 1) * per && w <= w1; ++w) s += gpart[(w * 2 + (w * rows / group == g ? 0 : 1)) * D + col];
  red[run][lane] = s;
  __syncthreads();
  if (run || col >= D) return;
  s = red[0][lane];
#pragma unroll
  for (int r = 1; r < 16; ++r) s += red[r][lane];
  if (gate_bf16) ((bf16_t*)dgate)[g * D + col] = (bf16_t)s;
  else ((float*)dgate)[g * D + col] = s;
}

constexpr int MAX_D = 8192;

// threads per row: the fewest that hold it in eight values each, up to a workgroup; column by column a wave at least
static int threads_per_row(int D, bool vec) {
  if (!vec) return D <= 512 ? 64 : 256;
  return D <= 128 ? 16 : D <= 256 ? 32 : D <= 1024 ? 64 : 256;
}

static bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

// backward: workgroups and rows of a walker.  1024 workgroups fill the chip four deep; more would only add column sums to join
static void bwd_shape(int64_t M, int D, bool vec, int64_t* wgs, int64_t* rows) {
  const int rpw = 256 / threads_per_row(D, vec);
  int64_t w = (M + rpw - 1) / rpw;
  if (w > 1024) w = 1024;
  *rows = (M + w * rpw - 1) / (w * rpw);
  *wgs = (M + *rows * rpw - 1) / (*rows * rpw);
}

template <typename TS, typename TB, bool VECT, int TPR, int NV>
static void launch(const NormArgs& a, bool bwd, int64_t grid, hipStream_t st) {
  if (bwd) residual_norm_bwd_kernel<TS, TB, VECT, TPR, NV><<<(unsigned)grid, 256, 0, st>>>(a);
  else residual_norm_fwd_kernel<TS, TB, VECT, TPR, NV><<<(unsigned)grid, 256, 0, st>>>(a);
}

template <typename TS, typename TB>
static void dispatch(const NormArgs& a, bool vec, bool bwd, int64_t grid, hipStream_t st) {
  const int D = a.D;
  if (vec) {
    if (D <= 128) launch<TS, TB, true, 16, 1>(a, bwd, grid, st);
    else if (D <= 256) launch<TS, TB, true, 32, 1>(a, bwd, grid, st);
    else if (D <= 512) launch<TS, TB, true, 64, 1>(a, bwd, grid, st);
    else if (D <= 1024) launch<TS, TB, true, 64, 2>(a, bwd, grid, st);
    else if (D <= 2048) launch<TS, TB, true, 256, 1>(a, bwd, grid, st);
    else if (D <= 4096) launch<TS, TB, true, 256, 2>(a, bwd, grid, st);
    else launch<TS, TB, true, 256, 4>(a, bwd, grid, st);
  } else {
    if (D <= 512) launch<TS, TB, false, 64, 1>(a, bwd, grid, st);
    else if (D <= 2048) launch<TS, TB, false, 256, 1>(a, bwd, grid, st);
    else launch<TS, TB, false, 256, 4>(a, bwd, grid, st);
  }
}

static int check_args(int64_t M, int D, int stream_dtype, int branch_dtype, int64_t group, const void* gate, int gate_dtype) {
  if (M < 0 || D <= 0 || group <= 0 || (stream_dtype != COIN_F32 && stream_dtype != COIN_BF16) || (branch_dtype != COIN_F32 && branch_dtype != COIN_BF16))
    return COIN_EINVAL;
  if (gate && gate_dtype != COIN_F32 && gate_dtype != COIN_BF16) return COIN_EINVAL;
  if (D > MAX_D || M > ((int64_t)1 << 31) || (stream_dtype == COIN_BF16 && branch_dtype == COIN_F32) || M % group) return COIN_ESHAPE;
  return COIN_OK;
}

}  // namespace

extern "C" int coin_residual_norm_fwd(const void* x, const void* y, const void* gate, int64_t rows_per_gate, const float* post_weight, const float* post_bias,
                                      int has_post, float post_eps, const float* pre_weight, const float* pre_bias, int has_pre, float pre_eps, int rms,
                                      float scale, void* r, void* h, float* stats, int64_t M, int D, int stream_dtype, int branch_dtype, int gate_dtype,
                                      void* stream) {
  const int rc = check_args(M, D, stream_dtype, branch_dtype, rows_per_gate, gate, gate_dtype);
  if (rc != COIN_OK) return rc;
  if (M == 0) return COIN_OK;
  if (!x || (has_pre && !h) || (y && !r) || (!y && !has_pre) || (!y && (gate || has_post))) return COIN_EINVAL;
  if ((uintptr_t)stats & 15) return COIN_EALIGN;
  NormArgs a = {};
  a.x = x; a.y = y; a.gate = gate; a.r = r; a.h = h; a.stats = stats;
  a.post_w = post_weight; a.post_b = post_bias; a.pre_w = pre_weight; a.pre_b = pre_bias;
  a.M = M; a.group = rows_per_gate; a.D = D; a.gate_bf16 = gate_dtype == COIN_BF16; a.has_post = has_post; a.has_pre = has_pre;
  a.rms = rms != 0; a.scale = scale; a.post_eps = post_eps; a.pre_eps = pre_eps;
  const bool vec = D % 8 == 0 && aligned(x) && aligned(y) && aligned(gate) && aligned(r) && aligned(h) && aligned(post_weight) && aligned(post_bias) &&
                   aligned(pre_weight) && aligned(pre_bias);
  const int rpw = 256 / threads_per_row(D, vec);
  int64_t grid = (M + rpw - 1) / rpw;
  if (grid > 8192) grid = 8192;
  hipStream_t st = (hipStream_t)stream;
  if (stream_dtype == COIN_BF16) dispatch<bf16_t, bf16_t>(a, vec, false, grid, st);
  else if (branch_dtype == COIN_BF16) dispatch<float, bf16_t>(a, vec, false, grid, st);
  else dispatch<float, float>(a, vec, false, grid, st);
  return coin_launch_status();
}

extern "C" size_t coin_residual_norm_bwd_workspace_bytes(int64_t M, int D) {
  if (M <= 0 || D <= 0 || D > MAX_D) return 0;
  size_t most = 0;   // whichever of the two row layouts the pointers' alignment chooses
  for (int v = 0; v < 2; ++v) {
    if (v && D % 8) break;
    int64_t wgs, rows;
    bwd_shape(M, D, v, &wgs, &rows);
    const size_t b = (size_t)wgs * (5 + 2 * (256 / threads_per_row(D, v))) * D * sizeof(float);
    if (b > most) most = b;
  }
  return most;
}

extern "C" int coin_residual_norm_bwd(const void* x, const void* y, const void* gate, int64_t rows_per_gate, const float* post_weight, const float* post_bias,
                                      int has_post, const float* pre_weight, int has_pre, int rms, float scale, const float* stats, const void* dr,
                                      const void* dh, void* dx, void* dy, void* dgate, float* dpost_weight, float* dpost_bias, float* dpre_weight,
                                      float* dpre_bias, int64_t M, int D, int stream_dtype, int branch_dtype, int gate_dtype, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  const int rc = check_args(M, D, stream_dtype, branch_dtype, rows_per_gate, gate, gate_dtype);
  if (rc != COIN_OK) return rc;
  if (!x || !stats || (!y && (gate || has_post || dy)) || (dgate && !gate) || (dh && !has_pre) || (!dr && !dh)) return COIN_EINVAL;
  if ((dpost_weight || dpost_bias) && !has_post) return COIN_EINVAL;
  if ((dpre_weight || dpre_bias) && !dh) return COIN_EINVAL;
  if (M == 0) return COIN_EINVAL;   // the sums over no rows are the caller's zeros
  NormArgs a = {};
  a.x = x; a.y = y; a.gate = gate; a.dr = dr; a.dh = dh; a.dx = dx; a.dy = dy; a.stats = const_cast<float*>(stats);
  a.post_w = post_weight; a.post_b = post_bias; a.pre_w = pre_weight;
  a.M = M; a.group = rows_per_gate; a.D = D; a.gate_bf16 = gate_dtype == COIN_BF16; a.has_post = has_post; a.has_pre = has_pre; a.rms = rms != 0; a.scale = scale;
  a.dgate = dgate;
  a.want_gate = !dgate ? 0 : (rows_per_gate == M ? 1 : 2);
  a.want_param = dpost_weight || dpost_bias || dpre_weight || dpre_bias;
  const bool vec = D % 8 == 0 && aligned(x) && aligned(y) && aligned(gate) && aligned(dr) && aligned(dh) && aligned(dx) && aligned(dy) && aligned(dgate) &&
                   aligned(post_weight) && aligned(post_bias) && aligned(pre_weight);
  if (((uintptr_t)stats | (uintptr_t)workspace) & 15) return COIN_EALIGN;
  int64_t wgs;
  bwd_shape(M, D, vec, &wgs, &a.rows);
  if (a.want_param || a.want_gate) {
    if (!workspace || workspace_bytes < coin_residual_norm_bwd_workspace_bytes(M, D)) return COIN_EINVAL;
    a.part = (float*)workspace;
    a.gpart = a.part + wgs * 5 * D;
  }
  hipStream_t st = (hipStream_t)stream;
  if (stream_dtype == COIN_BF16) dispatch<bf16_t, bf16_t>(a, vec, true, wgs, st);
  else if (branch_dtype == COIN_BF16) dispatch<float, bf16_t>(a, vec, true, wgs, st);
  else dispatch<float, float>(a, vec, true, wgs, st);
  if (a.want_param || a.want_gate == 1) {
    NormSums s = {};
    s.part = a.part; s.nwg = (int)wgs; s.D = D; s.gate_bf16 = a.gate_bf16;
    s.out[0] = dpost_weight; s.out[1] = dpost_bias; s.out[2] = dpre_weight; s.out[3] = dpre_bias;
    s.dgate = a.want_gate == 1 ? dgate : nullptr;
    residual_norm_sums_kernel<<<dim3((D + 63) / 64, 5), 1024, 0, st>>>(s);
  }
  if (a.want_gate == 2) {
    const int64_t groups = M / rows_per_gate;
    for (int64_t g0 = 0; g0 < groups; g0 += 65535) {
      const int64_t n = groups - g0 < 65535 ? groups - g0 : 65535;
      residual_norm_gate_kernel<<<dim3((D + 63) / 64, (unsigned)n), 1024, 0, st>>>(a.gpart, dgate, a.gate_bf16, M, rows_per_gate, a.rows, D, g0);
    }
  }
  return coin_launch_status();
}
