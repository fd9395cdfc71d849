// The norms around a block, with its gate and residual scale, in one pass over the rows:
//   u  = post(y)                    post: none, RMS or layer norm, optional weight / bias
//   h' = rs h + gate_g u            g = row / rows_per_mod: the row's adaLN group (gate null: 1)
//   xn = pre(h') (1 + scale_g) + shift_g      the next block's input (pre none: not formed)
// and its backward from dh' and dxn.  With n1, n2 the normalised rows, r1, r2 their 1 / std,
// z = n2 w2 + b2, and (g, a) the gradients of (h', z):
//   a = dxn (1 + scale),  g = dh' + r2 (a w2 - mean(a w2) - n2 mean(a w2 n2))     (RMS: no mean term)
//   dh = rs g,  e = gate g w1,  dy = r1 (e - mean(e) - n1 mean(e n1))
// and four column sums per group give every parameter's gradient:
//   S1 = sum dxn, S2 = sum dxn n2, S3 = sum g, S4 = sum g n1
//   dshift = S1, dscale = w2 S2 + b2 S1, dgate = w1 S4 + b1 S3   (per group)
//   dw2 = sum_g (1 + scale) S2, db2 = sum_g (1 + scale) S1, dw1 = sum_g gate S4, db1 = sum_g gate S3
// Bound by memory: forward 37-38 us at [32000, 384] (fp32 residual, bf16 branch: 147 MB, 3.9 TB/s of a copy's 5.1; 27-30
// where the rows are still in cache), 131 us at [16383, 4096] in bf16 (537 MB, 4.1 TB/s); backward 59-60 us at
// [32000, 384] (221 MB, 3.7 TB/s; 160 registers, three waves per SIMD), its column sums 5 + 5 us, and 92 us in all
// at [8000, 2048] (295 MB).
// The backward takes one block per group at least, so short groups are slow: forward and backward of 32000 rows of
// 384 take 96 us in groups of 4000, 195 of 32, 916 of 4 and 4606 of one row (all but one of a block's teams idle, 32
// bytes of partials per element).
// A row lives in the registers of TPR threads (32 or 64 lanes of a wave, or the whole block of 256, or of
// 1024 for long rows of odd length; in the backward also 512 and 1024 for wide ones), NV vectors of V elements each,
// so it is read once; statistics are
// fp32, the variance from the centred row.  xn is formed from h' before h' is rounded, and the backward recomputes h' from h
// and y instead of reading the rounded one.  Column sums: registers over the block's rows, then LDS
// over its teams, fp32 partials per block, summed in a fixed order: results repeat bit for bit.
#include "../../include/mdgen_hip.h"
#include "common.h"

namespace mdg {
namespace {

struct GrnP {
  const void *h, *y;
  void *ho, *xn;
  const float *gate, *shift, *scale;
  long long mod_stride;
  const float *w1, *b1, *w2, *b2;
  float rs, eps, invC;
  int M, C, R, post, pre;  // R = rows_per_mod, at most M
  long long ldh, ldy;      // row strides of h and y (outputs are contiguous)
  // backward
  const void *dho, *dxn;
  void *dh, *dy;
  float* part;  // [group][chunk][4][C]
  int chunks, rows_per_chunk, want_y_sums, want_x_sums;
};

template <typename T, int V>
__device__ __forceinline__ void ldv(const T* p, float (&o)[V]) {
  if constexpr (sizeof(T) == 4 && V >= 4) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      const float4 t = reinterpret_cast<const float4*>(p)[i];
      o[4 * i] = t.x, o[4 * i + 1] = t.y, o[4 * i + 2] = t.z, o[4 * i + 3] = t.w;
    }
  } else if constexpr (sizeof(T) == 2 && V == 8) {
    const bf16x8 t = *reinterpret_cast<const bf16x8*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (float)t[i];
  } else if constexpr (sizeof(T) == 2 && V == 4) {
    const bf16x4 t = *reinterpret_cast<const bf16x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = (float)t[i];
  } else {
    static_assert(V == 1, "");
    o[0] = (float)p[0];
  }
}
template <typename T, int V>
__device__ __forceinline__ void stv(T* p, const float (&o)[V]) {
  if constexpr (sizeof(T) == 4 && V >= 4) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i)
      reinterpret_cast<float4*>(p)[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
  } else if constexpr (sizeof(T) == 2 && V == 8) {
    bf16x8 t;
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = (bf16_t)o[i];
    *reinterpret_cast<bf16x8*>(p) = t;
  } else if constexpr (sizeof(T) == 2 && V == 4) {
    st4<bf16_t>(p, o[0], o[1], o[2], o[3]);
  } else {
    p[0] = (T)o[0];
  }
}

// Scratch of the block-wide sums: two areas in turn, so that one barrier per sum is enough (an area
// is written again only after the barrier of the sum between).
struct Red {
  float* at;
  int turn;
};

// sums of N values over the TPR threads of a row's team, the same in every one of them
template <int TPR, int N>
__device__ __forceinline__ void team_sum(float (&v)[N], Red& rd) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lane_sum<(TPR < 64 ? TPR : 64)>(v[i]);
  if constexpr (TPR >= 256) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float* red = rd.at + rd.turn * 32;
    rd.turn ^= 1;
    if (lane == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) red[wave * N + i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = red[i];
#pragma unroll
      for (int w = 1; w < TPR / 64; ++w) v[i] += red[w * N + i];
    }
  }
}

// ROWS rows of a team at once: x <- normalised x, r <- 1 / std.  Columns past C hold 0 and stay 0.
template <int TPR, int ROWS, int NV, int V>
__device__ __forceinline__ void normalise(float (&x)[ROWS][NV][V], float (&r)[ROWS], int kind, float eps, float invC,
                                          const bool (&in)[NV], Red& red) {
  if (kind == MDG_NORM_LAYER) {
    float s[ROWS];
#pragma unroll
    for (int w = 0; w < ROWS; ++w) {
      s[w] = 0.f;
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) s[w] += x[w][k][i];
    }
    team_sum<TPR, ROWS>(s, red);
#pragma unroll
    for (int w = 0; w < ROWS; ++w) {
      const float mean = s[w] * invC;
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) x[w][k][i] = in[k] ? x[w][k][i] - mean : 0.f;
    }
  }
#pragma unroll
  for (int w = 0; w < ROWS; ++w) {
    r[w] = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) r[w] = fmaf(x[w][k][i], x[w][k][i], r[w]);
  }
  team_sum<TPR, ROWS>(r, red);
#pragma unroll
  for (int w = 0; w < ROWS; ++w) {
    r[w] = 1.0f / sqrtf(fmaf(r[w], invC, eps));
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) x[w][k][i] *= r[w];
  }
}

// g <- r (g - [mean(g)] - n mean(g n)): the gradient of the row before its norm.  Columns past C stay 0.
template <int TPR, int NV, int V>
__device__ __forceinline__ void normalise_bwd(float (&g)[NV][V], const float (&n)[NV][V], float r, int kind, float invC,
                                              const bool (&in)[NV], Red& red) {
  float s[2] = {0.f, 0.f};
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) s[0] += g[k][i], s[1] = fmaf(g[k][i], n[k][i], s[1]);
  team_sum<TPR, 2>(s, red);
  const float m = kind == MDG_NORM_LAYER ? s[0] * invC : 0.f, q = s[1] * invC;
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) g[k][i] = in[k] ? r * (g[k][i] - m - n[k][i] * q) : 0.f;
}

template <int V>
__device__ __forceinline__ void ldopt(const float* p, long long at, float dflt, float (&o)[V]) {
  if (p) {
    ldv<float, V>(p + at, o);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = dflt;
  }
}

// ROWS consecutive rows per team: the parameters' rows (up to seven of them, fp32, from L2) are read
// once for all that share them, which bounds wide rows, and a block's sums share their barriers.
template <typename RT, typename CT, int V, int TPR, int NV, int ROWS>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void grn_fwd_kernel(const GrnP p) {
  __shared__ float red_[64];
  Red red{red_, 0};
  constexpr int TEAMS = TPR < 256 ? 256 / TPR : 1;
  const int team = threadIdx.x / TPR, t = threadIdx.x % TPR;
  const int row0 = (blockIdx.x * TEAMS + team) * ROWS;
  if (TPR < 256 && row0 >= p.M) return;
  float h[ROWS][NV][V], y[ROWS][NV][V], r[ROWS];
  long long mo[ROWS];
  bool in[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) in[k] = (t + k * TPR) * V < p.C;
#pragma unroll
  for (int w = 0; w < ROWS; ++w) {
    const int row = min(row0 + w, p.M - 1);  // (past the last row: the last one, not stored)
    mo[w] = (long long)(row / p.R) * p.mod_stride;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (t + k * TPR) * V;
#pragma unroll
      for (int i = 0; i < V; ++i) h[w][k][i] = y[w][k][i] = 0.f;
      if (in[k]) {
        ldv<RT, V>(reinterpret_cast<const RT*>(p.h) + row * p.ldh + c, h[w][k]);
        if (p.y) ldv<CT, V>(reinterpret_cast<const CT*>(p.y) + row * p.ldy + c, y[w][k]);
      }
    }
  }
  if (p.post != MDG_NORM_NONE) normalise<TPR, ROWS, NV, V>(y, r, p.post, p.eps, p.invC, in, red);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (t + k * TPR) * V;
    if (!in[k]) continue;
    float wt[V], b[V], g[V];
    if (p.y) {
      ldopt<V>(p.w1, c, 1.f, wt);
      ldopt<V>(p.b1, c, 0.f, b);
    }
#pragma unroll
    for (int w = 0; w < ROWS; ++w) {
      if (p.y) {
        if (w == 0 || mo[w] != mo[w - 1]) ldopt<V>(p.gate, mo[w] + c, 1.f, g);
#pragma unroll
        for (int i = 0; i < V; ++i) h[w][k][i] = fmaf(g[i], fmaf(y[w][k][i], wt[i], b[i]), p.rs * h[w][k][i]);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) h[w][k][i] *= p.rs;
      }
      if (p.ho && row0 + w < p.M) stv<RT, V>(reinterpret_cast<RT*>(p.ho) + (long long)(row0 + w) * p.C + c, h[w][k]);
    }
  }
  if (p.pre == MDG_NORM_NONE) return;
  normalise<TPR, ROWS, NV, V>(h, r, p.pre, p.eps, p.invC, in, red);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (t + k * TPR) * V;
    if (!in[k]) continue;
    float wt[V], b[V], sc[V], sh[V], o[V];
    ldopt<V>(p.w2, c, 1.f, wt);
    ldopt<V>(p.b2, c, 0.f, b);
#pragma unroll
    for (int w = 0; w < ROWS; ++w) {
      if (w == 0 || mo[w] != mo[w - 1]) {
        ldopt<V>(p.scale, mo[w] + c, 0.f, sc);
        ldopt<V>(p.shift, mo[w] + c, 0.f, sh);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = fmaf(fmaf(h[w][k][i], wt[i], b[i]), 1.0f + sc[i], sh[i]);
      if (row0 + w < p.M) stv<CT, V>(reinterpret_cast<CT*>(p.xn) + (long long)(row0 + w) * p.C + c, o);
    }
  }
}

// One block: rows_per_chunk rows of one group.
template <typename RT, typename CT, int V, int TPR, int NV>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void grn_bwd_kernel(const GrnP p) {
  constexpr int TEAMS = TPR < 256 ? 256 / TPR : 1;
  __shared__ float red_[64];
  Red red{red_, 0};
  __shared__ __attribute__((aligned(16))) float cols[TEAMS > 1 ? TPR * NV * V : 1];
  const int team = threadIdx.x / TPR, t = threadIdx.x % TPR;
  const int grp = blockIdx.x / p.chunks, chunk = blockIdx.x % p.chunks;
  // (ends from what is left: a group's first row plus its rows may pass 31 bits)
  const int g0 = grp * p.R, g1 = g0 + min(p.R, p.M - g0);
  const int r0 = g0 + min(g1 - g0, chunk * p.rows_per_chunk), r1 = r0 + min(g1 - r0, p.rows_per_chunk);
  const long long mo = (long long)grp * p.mod_stride;
  float S[4][NV][V];
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) S[s][k][i] = 0.f;
  bool in[NV];
  // the group's rows of parameters: gate w1, gate b1, (1 + scale) w2
  float gw[NV][V], gb[NV][V], sw[NV][V];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (t + k * TPR) * V;
    in[k] = c < p.C;
#pragma unroll
    for (int i = 0; i < V; ++i) gw[k][i] = gb[k][i] = sw[k][i] = 0.f;
    if (in[k]) {
      float g[V], w2[V], sc[V];
      ldopt<V>(p.gate, mo + c, 1.f, g);
      ldopt<V>(p.w1, c, 1.f, gw[k]);
      ldopt<V>(p.b1, c, 0.f, gb[k]);
      ldopt<V>(p.w2, c, 1.f, w2);
      ldopt<V>(p.scale, mo + c, 0.f, sc);
#pragma unroll
      for (int i = 0; i < V; ++i) gw[k][i] *= g[i], gb[k][i] *= g[i], sw[k][i] = (1.0f + sc[i]) * w2[i];
    }
  }

  // every team of the block makes the same number of turns (the sums of a whole block hold barriers)
  for (int rb = r0; rb < r1; rb += TEAMS) {
    const int row = rb + team;
    if (TPR < 256 && row >= r1) break;
    float h[1][NV][V], y[1][NV][V], g[NV][V], a[NV][V], r1y[1], r2[1];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (t + k * TPR) * V;
#pragma unroll
      for (int i = 0; i < V; ++i) h[0][k][i] = y[0][k][i] = g[k][i] = a[k][i] = 0.f;
      if (in[k]) {
        if (p.dxn) ldv<RT, V>(reinterpret_cast<const RT*>(p.h) + row * p.ldh + c, h[0][k]);
        if (p.y) ldv<CT, V>(reinterpret_cast<const CT*>(p.y) + row * p.ldy + c, y[0][k]);
        if (p.dxn) ldv<CT, V>(reinterpret_cast<const CT*>(p.dxn) + (long long)row * p.C + c, a[k]);
        if (p.dho) ldv<RT, V>(reinterpret_cast<const RT*>(p.dho) + (long long)row * p.C + c, g[k]);
      }
    }
    r1y[0] = 1.f;
    if (p.post != MDG_NORM_NONE) normalise<TPR, 1, NV, V>(y, r1y, p.post, p.eps, p.invC, in, red);  // y is n1
    if (p.dxn) {
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i)
          h[0][k][i] = p.y ? fmaf(y[0][k][i], gw[k][i], fmaf(p.rs, h[0][k][i], gb[k][i])) : p.rs * h[0][k][i];
      normalise<TPR, 1, NV, V>(h, r2, p.pre, p.eps, p.invC, in, red);  // h is n2
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          S[0][k][i] += a[k][i];
          S[1][k][i] = fmaf(a[k][i], h[0][k][i], S[1][k][i]);
          a[k][i] *= sw[k][i];
        }
      normalise_bwd<TPR, NV, V>(a, h[0], r2[0], p.pre, p.invC, in, red);
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) g[k][i] += a[k][i];
    }
    if (p.dh) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        if (!in[k]) continue;
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = p.rs * g[k][i];
        stv<RT, V>(reinterpret_cast<RT*>(p.dh) + (long long)row * p.C + (t + k * TPR) * V, o);
      }
    }
    if (!p.y) continue;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        S[2][k][i] += g[k][i];
        S[3][k][i] = fmaf(g[k][i], y[0][k][i], S[3][k][i]);
        g[k][i] *= gw[k][i];
      }
    if (!p.dy) continue;
    if (p.post != MDG_NORM_NONE) normalise_bwd<TPR, NV, V>(g, y[0], r1y[0], p.post, p.invC, in, red);
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (in[k]) stv<CT, V>(reinterpret_cast<CT*>(p.dy) + (long long)row * p.C + (t + k * TPR) * V, g[k]);
  }
  if (!p.part) return;
  float* out = p.part + ((long long)grp * p.chunks + chunk) * 4 * p.C;
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    if (s < 2 ? !p.want_x_sums : !p.want_y_sums) continue;
    if constexpr (TEAMS > 1) {
      for (int tm = 0; tm < TEAMS; ++tm) {  // teams one after the other: a fixed order
        if (team == tm) {
#pragma unroll
          for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) {
              float* at = cols + (t + k * TPR) * V + i;
              *at = tm == 0 ? S[s][k][i] : *at + S[s][k][i];
            }
        }
        __syncthreads();
      }
      for (int c = threadIdx.x; c < p.C; c += 256) out[s * p.C + c] = cols[c];
      __syncthreads();
    } else {
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (in[k]) stv<float, V>(out + s * p.C + (t + k * TPR) * V, S[s][k]);
    }
  }
}

// Column sums of the blocks' partials: one block = 64 columns of one group and one norm (blockIdx.z 0: the
// pre norm's S1, S2; 1: the post norm's S3, S4), 16 lanes along the chunks; then the group's modulation
// gradients, and its sums S [G][4][C] for grn_weights_kernel.
__global__ __launch_bounds__(1024) void grn_cols_kernel(const GrnP p, float* sums, float* dgate, float* dshift, float* dscale,
                                                        long long dmod_stride) {
  __shared__ float red[2][16][64];
  const int x = threadIdx.x & 63, c = blockIdx.y * 64 + x, lane = threadIdx.x >> 6, grp = blockIdx.x, half = blockIdx.z;
  if (half ? !p.want_y_sums : !p.want_x_sums) return;
  const float* base = p.part + ((long long)grp * p.chunks * 4 + 2 * half) * p.C + c;
  float u = 0.f, v = 0.f;
  if (c < p.C) {
#pragma unroll 4
    for (int k = lane; k < p.chunks; k += 16) {
      u += base[(long long)k * 4 * p.C];
      v += base[((long long)k * 4 + 1) * p.C];
    }
  }
  red[0][lane][x] = u, red[1][lane][x] = v;
  __syncthreads();
  if (lane != 0 || c >= p.C) return;
  u = v = 0.f;
#pragma unroll
  for (int k = 0; k < 16; ++k) u += red[0][k][x], v += red[1][k][x];
  sums[((long long)grp * 4 + 2 * half) * p.C + c] = u;
  sums[((long long)grp * 4 + 2 * half + 1) * p.C + c] = v;
  const long long at = (long long)grp * dmod_stride + c;
  if (half) {
    if (dgate) dgate[at] = (p.w1 ? p.w1[c] : 1.f) * v + (p.b1 ? p.b1[c] * u : 0.f);
  } else {
    if (dshift) dshift[at] = u;
    if (dscale) dscale[at] = (p.w2 ? p.w2[c] : 1.f) * v + (p.b2 ? p.b2[c] * u : 0.f);
  }
}

// The weights' gradients: one block = 64 columns, 16 lanes along the groups.
__global__ __launch_bounds__(1024) void grn_weights_kernel(const GrnP p, const float* sums, int G, float* dw1, float* db1,
                                                           float* dw2, float* db2) {
  __shared__ float red[4][16][64];
  const int x = threadIdx.x & 63, c = blockIdx.x * 64 + x, lane = threadIdx.x >> 6;
  float a[4] = {0.f, 0.f, 0.f, 0.f};  // db2, dw2, db1, dw1
  if (c < p.C) {
    for (int g = lane; g < G; g += 16) {
      const float* s = sums + (long long)g * 4 * p.C + c;
      if (p.want_x_sums) {
        const float sc = 1.0f + (p.scale ? p.scale[g * p.mod_stride + c] : 0.f);
        a[0] = fmaf(sc, s[0], a[0]), a[1] = fmaf(sc, s[p.C], a[1]);
      }
      if (p.want_y_sums) {
        const float gt = p.gate ? p.gate[g * p.mod_stride + c] : 1.f;
        a[2] = fmaf(gt, s[2 * (long long)p.C], a[2]), a[3] = fmaf(gt, s[3 * (long long)p.C], a[3]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) red[i][lane][x] = a[i];
  __syncthreads();
  if (lane >= 4 || c >= p.C) return;
  float v = 0.f;
#pragma unroll
  for (int k = 0; k < 16; ++k) v += red[lane][k][x];
  float* out = lane == 0 ? db2 : lane == 1 ? dw2 : lane == 2 ? db1 : dw1;
  if (out) out[c] = v;
}

// rows of a modulation group; a longer run than there are rows is one group of them all
int group_rows(const mdg_gate_res_norm_desc& d) { return d.rows_per_mod < d.M ? d.rows_per_mod : d.M; }

GrnP grn_params(const mdg_gate_res_norm_desc& d) {
  GrnP p;
  p.h = d.h, p.y = d.y, p.ho = d.h_out, p.xn = d.xn;
  p.gate = d.gate, p.shift = d.shift, p.scale = d.scale, p.mod_stride = d.mod_stride;
  p.w1 = d.post_w, p.b1 = d.post_b, p.w2 = d.pre_w, p.b2 = d.pre_b;
  p.rs = d.resid_scale, p.eps = d.eps, p.invC = 1.0f / d.C;
  p.M = d.M, p.C = d.C, p.R = group_rows(d), p.post = d.post, p.pre = d.pre;
  p.ldh = d.ldh, p.ldy = d.ldy;
  p.dho = d.dh_out, p.dxn = d.dxn, p.dh = d.dh, p.dy = d.dy;
  p.part = nullptr, p.chunks = 1, p.rows_per_chunk = p.R;
  p.want_y_sums = p.want_x_sums = 0;
  return p;
}

int grn_vec(const mdg_gate_res_norm_desc& d) {
  const int re = d.res_dtype == MDG_BF16 ? 2 : 4, ce = d.dtype == MDG_BF16 ? 2 : 4;
  for (int v = ce == 2 && re == 2 ? 8 : 4; v >= 4; v /= 2) {
    if (d.C % v) continue;
    uintptr_t r = (uintptr_t)d.h | (uintptr_t)d.h_out | (uintptr_t)d.dh_out | (uintptr_t)d.dh | (uintptr_t)(d.ldh * re);
    uintptr_t c = (uintptr_t)d.y | (uintptr_t)d.xn | (uintptr_t)d.dxn | (uintptr_t)d.dy | (uintptr_t)(d.ldy * ce);
    uintptr_t f = (uintptr_t)d.gate | (uintptr_t)d.shift | (uintptr_t)d.scale | (uintptr_t)d.post_w | (uintptr_t)d.post_b |
                  (uintptr_t)d.pre_w | (uintptr_t)d.pre_b;
    if (d.gate || d.shift || d.scale) f |= (uintptr_t)(d.mod_stride * 4);
    const uintptr_t rm = (re == 4 ? 16 : v * 2) - 1, cm = (ce == 4 ? 16 : v * 2) - 1;
    if ((r & rm) == 0 && (c & cm) == 0 && (f & 15) == 0) return v;
  }
  return 1;
}

// Threads per row and vectors per thread: the smallest team that holds the row in few vectors.
struct Shape {
  int tpr, nv;
};
Shape grn_shape(int C, int V) {
  const int n = (C + V - 1) / V;
  if (V == 1) return n <= 256 ? Shape{64, 4} : n <= 1024 ? Shape{256, 4} : n <= 2048 ? Shape{256, 8} : Shape{1024, 8};
  for (int nv = 1; nv <= 3; ++nv)
    if (n <= 32 * nv) return {32, nv};
  for (int nv = 2; nv <= 4; ++nv)
    if (n <= 64 * nv) return {64, nv};
  for (int nv = 2; nv <= 4; ++nv)
    if (n <= 256 * nv) return {256, nv};
  return {256, 8};
}

// The backward's: four sums per column beside the row, so fewer vectors per thread and larger teams (registers,
// waves per SIMD: one vector 71, 7; two 118, 4; three 162, 3; four 218, 2).  [3 x 1500, 4096] bf16 99 us, with the
// forward's four vectors of 256 threads 135, with 1024 threads 174; [8 x 4000, 384] the same with two vectors of 64 lanes.
Shape grn_back_shape(int C, int V) {
  const int n = (C + V - 1) / V;
  if (V == 1) return grn_shape(C, 1);
  for (int nv = 1; nv <= 3; ++nv)
    if (n <= 32 * nv) return {32, nv};
  if (n <= 128) return {64, 2};
  for (int nv = 1; nv <= 2; ++nv)
    if (n <= 256 * nv) return {256, nv};
  return n <= 1024 ? Shape{512, 2} : Shape{1024, 2};
}

template <typename RT, typename CT, int V, int TPR, int NV>
void grn_go(const GrnP& p, hipStream_t s) {
  constexpr int BD = TPR < 256 ? 256 : TPR, TEAMS = BD / TPR, ROWS = TPR == 256 ? 2 : 1;
  hipLaunchKernelGGL((grn_fwd_kernel<RT, CT, V, TPR, NV, ROWS>), dim3((unsigned)((p.M + TEAMS * ROWS - 1) / (TEAMS * ROWS))),
                          dim3(BD), 0, s, p);
}
template <typename RT, typename CT, int V, int TPR, int NV>
void grn_back(const GrnP& p, int G, hipStream_t s) {
  hipLaunchKernelGGL((grn_bwd_kernel<RT, CT, V, TPR, NV>), dim3((unsigned)(G * p.chunks)), dim3(TPR < 256 ? 256 : TPR), 0, s, p);
}

template <typename RT, typename CT, int V>
void grn_by_shape(const GrnP& p, hipStream_t s) {
  const Shape sh = grn_shape(p.C, V);
  if constexpr (V == 1) {
    if (sh.tpr == 64) grn_go<RT, CT, 1, 64, 4>(p, s);
    else if (sh.nv == 4) grn_go<RT, CT, 1, 256, 4>(p, s);
    else if (sh.tpr == 256) grn_go<RT, CT, 1, 256, 8>(p, s);
    else grn_go<RT, CT, 1, 1024, 8>(p, s);
  } else {
    switch (sh.tpr * 16 + sh.nv) {
      case 32 * 16 + 1: grn_go<RT, CT, V, 32, 1>(p, s); break;
      case 32 * 16 + 2: grn_go<RT, CT, V, 32, 2>(p, s); break;
      case 32 * 16 + 3: grn_go<RT, CT, V, 32, 3>(p, s); break;
      case 64 * 16 + 2: grn_go<RT, CT, V, 64, 2>(p, s); break;
      case 64 * 16 + 3: grn_go<RT, CT, V, 64, 3>(p, s); break;
      case 64 * 16 + 4: grn_go<RT, CT, V, 64, 4>(p, s); break;
      case 256 * 16 + 2: grn_go<RT, CT, V, 256, 2>(p, s); break;
      case 256 * 16 + 3: grn_go<RT, CT, V, 256, 3>(p, s); break;
      case 256 * 16 + 4: grn_go<RT, CT, V, 256, 4>(p, s); break;
      default:
        if constexpr (V == 4) grn_go<RT, CT, V, 256, 8>(p, s);
        break;
    }
  }
}
template <typename RT, typename CT, int V>
void grn_back_by_shape(const GrnP& p, int G, hipStream_t s) {
  const Shape sh = grn_back_shape(p.C, V);
  if constexpr (V == 1) {
    if (sh.tpr == 64) grn_back<RT, CT, 1, 64, 4>(p, G, s);
    else if (sh.nv == 4) grn_back<RT, CT, 1, 256, 4>(p, G, s);
    else if (sh.tpr == 256) grn_back<RT, CT, 1, 256, 8>(p, G, s);
    else grn_back<RT, CT, 1, 1024, 8>(p, G, s);
  } else {
    switch (sh.tpr * 16 + sh.nv) {
      case 32 * 16 + 1: grn_back<RT, CT, V, 32, 1>(p, G, s); break;
      case 32 * 16 + 2: grn_back<RT, CT, V, 32, 2>(p, G, s); break;
      case 32 * 16 + 3: grn_back<RT, CT, V, 32, 3>(p, G, s); break;
      case 64 * 16 + 2: grn_back<RT, CT, V, 64, 2>(p, G, s); break;
      case 256 * 16 + 1: grn_back<RT, CT, V, 256, 1>(p, G, s); break;
      case 256 * 16 + 2: grn_back<RT, CT, V, 256, 2>(p, G, s); break;
      case 512 * 16 + 2: grn_back<RT, CT, V, 512, 2>(p, G, s); break;
      default: grn_back<RT, CT, V, 1024, 2>(p, G, s); break;
    }
  }
}

template <typename RT, typename CT, int V>
void grn_dispatch_v(const GrnP& p, bool back, int G, hipStream_t s) {
  if (!back) grn_by_shape<RT, CT, V>(p, s);
  else if constexpr (V <= 4) grn_back_by_shape<RT, CT, V>(p, G, s);
}

void grn_dispatch(const mdg_gate_res_norm_desc& d, const GrnP& p, bool back, int G, hipStream_t s) {
  // (the backward's rows, sums and parameters fill the registers at 4 columns per vector)
  const int v = back ? (grn_vec(d) < 4 ? 1 : 4) : grn_vec(d);
  if (d.res_dtype == MDG_BF16) {
    if (v == 8) grn_dispatch_v<bf16_t, bf16_t, 8>(p, back, G, s);
    else if (v == 4) grn_dispatch_v<bf16_t, bf16_t, 4>(p, back, G, s);
    else grn_dispatch_v<bf16_t, bf16_t, 1>(p, back, G, s);
  } else if (d.dtype == MDG_BF16) {
    if (v == 4) grn_dispatch_v<float, bf16_t, 4>(p, back, G, s);
    else grn_dispatch_v<float, bf16_t, 1>(p, back, G, s);
  } else {
    if (v == 4) grn_dispatch_v<float, float, 4>(p, back, G, s);
    else grn_dispatch_v<float, float, 1>(p, back, G, s);
  }
}

bool want_y(const mdg_gate_res_norm_desc& d) { return d.dgate || d.dpost_w || d.dpost_b; }
bool want_x(const mdg_gate_res_norm_desc& d) { return d.dshift || d.dscale || d.dpre_w || d.dpre_b; }
int groups(const mdg_gate_res_norm_desc& d) { return (int)(((long long)d.M + group_rows(d) - 1) / group_rows(d)); }

// Chunks of a group's rows: about 768 blocks in all (three per CU), each with four turns of its teams or more, or
// eight rows of a whole block (a chunk's partial sums cost about as much as two rows).  [8 x 1000, 2048] 92 us against
// 180 with 32 rows at least, [1 x 300, 2000] 38 / 79; four rows at least are no faster.
int grn_chunks(const mdg_gate_res_norm_desc& d) {
  const int G = groups(d);
  const int least = d.C > 512 ? 8 : d.C > 384 ? 16 : 32;
  const long long want = (768LL + G - 1) / G, most = ((long long)group_rows(d) + least - 1) / least;
  return (int)(want < most ? want : most);
}

}  // namespace

size_t gate_res_norm_ws_bytes(const mdg_gate_res_norm_desc& d) {
  if (!want_y(d) && !want_x(d)) return 0;
  return (size_t)groups(d) * (grn_chunks(d) + 1) * 4 * d.C * sizeof(float);
}

// every launch within the 2^32 threads of a grid, row numbers (the last blocks', past the end) within 31 bits
bool gate_res_norm_grid_ok(const mdg_gate_res_norm_desc& d, bool back) {
  const long long threads = (1LL << 32) - 4096, v = grn_vec(d);
  const long long tpr = (back ? grn_back_shape(d.C, v < 4 ? 1 : 4) : grn_shape(d.C, (int)v)).tpr;
  if (d.M > (1LL << 31) - 4096) return false;
  if (!back) return d.M * tpr <= threads;
  const long long G = groups(d);
  return G * grn_chunks(d) * (tpr > 256 ? tpr : 256) <= threads && (!(want_y(d) || want_x(d)) || G * 1024 <= threads);
}

hipError_t gate_res_norm_fwd_launch(const mdg_gate_res_norm_desc& d, hipStream_t s) {
  grn_dispatch(d, grn_params(d), false, 0, s);
  return hipGetLastError();
}

hipError_t gate_res_norm_bwd_launch(const mdg_gate_res_norm_desc& d, void* ws, hipStream_t s) {
  GrnP p = grn_params(d);
  const int G = groups(d);
  p.chunks = grn_chunks(d);
  p.rows_per_chunk = (p.R + p.chunks - 1) / p.chunks;
  p.want_y_sums = want_y(d), p.want_x_sums = want_x(d);
  const bool sums = p.want_y_sums || p.want_x_sums;
  float* S = nullptr;
  if (sums) {
    p.part = reinterpret_cast<float*>(ws);
    S = p.part + (size_t)G * p.chunks * 4 * d.C;
  }
  grn_dispatch(d, p, true, G, s);
  if (sums) {
    hipLaunchKernelGGL(grn_cols_kernel, dim3(G, (d.C + 63) / 64, 2), dim3(1024), 0, s, p, S, d.dgate, d.dshift, d.dscale,
                       (long long)d.dmod_stride);
    if (d.dpost_w || d.dpost_b || d.dpre_w || d.dpre_b)
      hipLaunchKernelGGL(grn_weights_kernel, dim3((d.C + 63) / 64), dim3(1024), 0, s, p, (const float*)S, G, d.dpost_w, d.dpost_b,
                         d.dpre_w, d.dpre_b);
  }
  return hipGetLastError();
}

}  // namespace mdg
