// Rotary positions with several axes: pair p of a head's rotated columns belongs to one axis (frame,
// residue, height, ...) and turns by pos[token][axis[p]] * freq[p]; columns past the pairs pass through.
//   y1 = x1 cos - x2 sin,  y2 = x2 cos + x1 sin      (inverse: -sin; it is the backward)
// Bound by memory: every element is read and written once.  A block takes a few tokens: first their cos /
// sin per pair into LDS, once for all heads (the angle is formed in double as a number of turns and
// reduced there: a position of 10^6 in fp32 would lose it), then a sweep over the tokens' rows in
// memory order.  q and k go in one launch: their heads are one list.
// fp32 [2, 50001] tokens of 16 heads x 64 columns (820 MB): 201-204 us, 4.0 TB/s; one token 3 us.  A large copy
// reaches 5.1 TB/s.  Tried: token bases in LDS (57 -> 69 us for both directions: a dependent read before every
// load), the division by N as a multiplication, half and a quarter of the LDS entries (the same),
// non-temporal accesses and heads unrolled per thread (slower).
#include "../../include/mdgen_hip.h"
#include "common.h"

#include <initializer_list>

namespace mdg {
namespace {

struct RopeSeg {
  const void* x;
  void* y;
  long long xb, xn, xh, yb, yn, yh;
};
struct RopeP {
  RopeSeg seg[2];
  int H0, HT;  // heads of the first tensor, of both
  int N, D, np;
  unsigned tokens;  // B * N
  const void* pos;
  long long pb, pn;
  const double* turns;
  const int* axis;
  const int* cols;  // first columns of the pairs, then second columns
  int inverse, i64;
  int rot_tasks, tasks;  // per head row: rotations of V pairs, then copies of copy_w columns (2V or V)
  int copy_w;
  int T;  // tokens per block
  int lds;  // rope_tile_kernel's bytes, 0: the other kernel
  float inv_np, inv_tasks, inv_row;  // 1 / pairs, tasks, tasks of a token
};

constexpr int kRopeLds = 2048;  // (token, pair) entries of a block

// i / d for 0 <= i < 2^21 and d < 2^21: (i + 1/2) / d is at least 1 / (2 d) from a whole number, well
// beyond the products' rounding there
__device__ __forceinline__ int small_div(int i, float inv_d) { return (int)(((float)i + 0.5f) * inv_d); }

// cos and (signed) sin of pair pr at token (b, n)
__device__ __forceinline__ void turn_of(const RopeP& p, unsigned b, unsigned n, int pr, float& cs, float& sn) {
  const long long at = b * p.pb + n * p.pn + p.axis[pr];
  const double ps = p.i64 ? (double)reinterpret_cast<const long long*>(p.pos)[at]
                          : (double)reinterpret_cast<const int*>(p.pos)[at];
  const double turn = ps * p.turns[pr];
  float s, c;
  sincospif(2.0f * (float)(turn - rint(turn)), &s, &c);  // half turns in [-1, 1]
  cs = c, sn = p.inverse ? -s : s;
}

template <typename CT, int W> struct Pack { CT v[W]; };
template <typename CT, int W>
__device__ __forceinline__ Pack<CT, W> ldw(const CT* p) {
  Pack<CT, W> r;
  if constexpr (W * sizeof(CT) >= 16) {
#pragma unroll
    for (int i = 0; i < (int)(W * sizeof(CT) / 16); ++i) {
      const uint4 u = reinterpret_cast<const uint4*>(p)[i];
      __builtin_memcpy(&r.v[i * (16 / sizeof(CT))], &u, 16);
    }
  } else if constexpr (W * sizeof(CT) == 8) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    __builtin_memcpy(r.v, &u, 8);
  } else if constexpr (W * sizeof(CT) == 4) {
    const unsigned u = *reinterpret_cast<const unsigned*>(p);
    __builtin_memcpy(r.v, &u, 4);
  } else {
    r.v[0] = p[0];
  }
  return r;
}
template <typename CT, int W>
__device__ __forceinline__ void stw(CT* p, const Pack<CT, W>& r) {
  if constexpr (W * sizeof(CT) >= 16) {
#pragma unroll
    for (int i = 0; i < (int)(W * sizeof(CT) / 16); ++i) {
      uint4 u;
      __builtin_memcpy(&u, &r.v[i * (16 / sizeof(CT))], 16);
      reinterpret_cast<uint4*>(p)[i] = u;
    }
  } else if constexpr (W * sizeof(CT) == 8) {
    uint2 u;
    __builtin_memcpy(&u, r.v, 8);
    *reinterpret_cast<uint2*>(p) = u;
  } else if constexpr (W * sizeof(CT) == 4) {
    unsigned u;
    __builtin_memcpy(&u, r.v, 4);
    *reinterpret_cast<unsigned*>(p) = u;
  } else {
    p[0] = r.v[0];
  }
}

// V pairs per item.  INTER: the pair's columns are neighbours (one run of 2V columns); otherwise two runs
// of V columns, cols[p] .. and cols[np + p] ..  (the host picks V so that no run crosses a section
// and every run is aligned to its bytes).  Items run over (token, head, task), task fastest.
template <typename CT, int V, bool INTER>
__global__ __launch_bounds__(256) void rope_axes_kernel(const RopeP p) {
  __shared__ __attribute__((aligned(16))) float cs[kRopeLds], sn[kRopeLds];
  const int tid = threadIdx.x;
  const unsigned t0 = blockIdx.x * (unsigned)p.T;
  const int T = (int)min((unsigned)p.T, p.tokens - t0);
  for (int i = tid; i < T * p.np; i += 256) {
    const int t = small_div(i, p.inv_np), pr = i - t * p.np;
    const unsigned b = (t0 + t) / (unsigned)p.N, n = t0 + t - b * p.N;
    turn_of(p, b, n, pr, cs[i], sn[i]);
  }
  __syncthreads();
  constexpr int W = INTER ? 2 * V : V;
  const int per = p.HT * p.tasks, items = T * per;
#pragma unroll 2
  for (int i = tid; i < items; i += 256) {
    const int t = small_div(i, p.inv_row), j = i - t * per, hd = small_div(j, p.inv_tasks), task = j - hd * p.tasks;
    const unsigned b = (t0 + t) / (unsigned)p.N, n = t0 + t - b * p.N;
    const RopeSeg& g = p.seg[hd >= p.H0];
    const int h = hd >= p.H0 ? hd - p.H0 : hd;
    const CT* x = reinterpret_cast<const CT*>(g.x) + b * g.xb + n * g.xn + h * g.xh;
    CT* y = reinterpret_cast<CT*>(g.y) + b * g.yb + n * g.yn + h * g.yh;
    if (task >= p.rot_tasks) {
      const int c = 2 * p.np + (task - p.rot_tasks) * p.copy_w;
      for (int k = 0; k < p.copy_w; k += V) stw<CT, V>(y + c + k, ldw<CT, V>(x + c + k));
      continue;
    }
    const int p0 = task * V, at = t * p.np + p0;
    const int c1 = INTER ? 2 * p0 : p.cols[p0], c2 = INTER ? 0 : p.cols[p.np + p0];
    const Pack<float, V> c = ldw<float, V>(cs + at), s = ldw<float, V>(sn + at);
    if constexpr (INTER) {
      const Pack<CT, W> a = ldw<CT, W>(x + c1);
      Pack<CT, W> r;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float v = (float)a.v[2 * k], w = (float)a.v[2 * k + 1];
        r.v[2 * k] = (CT)(v * c.v[k] - w * s.v[k]);
        r.v[2 * k + 1] = (CT)(w * c.v[k] + v * s.v[k]);
      }
      stw<CT, W>(y + c1, r);
    } else {
      const Pack<CT, V> a = ldw<CT, V>(x + c1), d = ldw<CT, V>(x + c2);
      Pack<CT, V> r, q;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float v = (float)a.v[k], w = (float)d.v[k];
        r.v[k] = (CT)(v * c.v[k] - w * s.v[k]);
        q.v[k] = (CT)(w * c.v[k] + v * s.v[k]);
      }
      stw<CT, V>(y + c1, r);
      stw<CT, V>(y + c2, q);
    }
  }
}

// The same where an item would be one or two pairs but head rows are whole 16-byte pieces (sections of 6 or 5
// pairs, odd pair counts): rows go through LDS, in and out 16 bytes per lane, and are rotated there.  A
// thread keeps its (token, run) and walks the heads, so its cos, sin and columns stay in registers.
// [8, 4000] tokens of 16 heads x 64, us with the kernel above / this one: bf16 axis 11 + 11 + 10 pairs 56 / 31,
// interleaved 10 + 12 39 / 28 and 9 + 8 69 / 27; fp32 axis 11 + 11 + 10 57 / 49, 10 + 6 57 / 50, interleaved 9 + 6 69 / 47
// (5.5 TB/s, partly from cache); 32 heads x 24 bf16, axis 6 + 6, 27 / 23.  bf16 axis 12 + 20, four pairs at a time: 26 / 30.
// Bytes of rows per block: 16 KiB, ten blocks per CU (of 24 or 12 KiB within 5 %, 32: bf16 axis 35.7 against 31 us), where one
// token needs more than that up to twice as much.
constexpr int kRopeTile = 16384;
template <typename CT, int V>
__global__ __launch_bounds__(256) void rope_tile_kernel(const RopeP p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int N = 16 / sizeof(CT);
  const int tid = threadIdx.x, pieces = p.D / N;
  const int t0 = blockIdx.x * p.T, T = min(p.T, (int)p.tokens - t0);
  // a token's rows, one piece apart from a multiple of the banks
  const int per = p.HT * pieces, step = (per | 1) * N;
  CT* tile = reinterpret_cast<CT*>(smem);
  for (int i = tid; i < T * per; i += 256) {
    const int t = small_div(i, p.inv_row), j = i - t * per, hd = small_div(j, p.inv_tasks), c = j - hd * pieces;
    const unsigned b = (unsigned)(t0 + t) / (unsigned)p.N, n = t0 + t - b * p.N;
    const int second = hd >= p.H0, h = second ? hd - p.H0 : hd;
    const RopeSeg& g = p.seg[second];
    const CT* x = reinterpret_cast<const CT*>(g.x) + b * g.xb + n * g.xn + h * g.xh;
    *reinterpret_cast<uint4*>(tile + t * step + j * N) = *reinterpret_cast<const uint4*>(x + c * N);
  }
  __syncthreads();
  const int runs = p.np / V, combos = T * runs, groups = combos < 256 ? 256 / combos : 1;
  for (int c = tid; c < combos * groups; c += 256) {
    const int grp = c / combos, cc = c - grp * combos, t = cc / runs, p0 = (cc - t * runs) * V;
    const unsigned b = (unsigned)(t0 + t) / (unsigned)p.N, n = t0 + t - b * p.N;
    float cs[V], sn[V];
#pragma unroll
    for (int k = 0; k < V; ++k) turn_of(p, b, n, p0 + k, cs[k], sn[k]);
    const int c1 = p.cols[p0], c2 = p.cols[p.np + p0];
    CT* row = tile + t * step + grp * p.D;
    for (int hd = grp; hd < p.HT; hd += groups, row += groups * p.D) {
      const Pack<CT, V> a = ldw<CT, V>(row + c1), d = ldw<CT, V>(row + c2);
      Pack<CT, V> r, q;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float v = (float)a.v[k], w = (float)d.v[k];
        r.v[k] = (CT)(v * cs[k] - w * sn[k]);
        q.v[k] = (CT)(w * cs[k] + v * sn[k]);
      }
      stw<CT, V>(row + c1, r);
      stw<CT, V>(row + c2, q);
    }
  }
  __syncthreads();
  for (int i = tid; i < T * per; i += 256) {
    const int t = small_div(i, p.inv_row), j = i - t * per, hd = small_div(j, p.inv_tasks), c = j - hd * pieces;
    const unsigned b = (unsigned)(t0 + t) / (unsigned)p.N, n = t0 + t - b * p.N;
    const int second = hd >= p.H0, h = second ? hd - p.H0 : hd;
    const RopeSeg& g = p.seg[second];
    CT* y = reinterpret_cast<CT*>(g.y) + b * g.yb + n * g.yn + h * g.yh;
    *reinterpret_cast<uint4*>(y + c * N) = *reinterpret_cast<const uint4*>(tile + t * step + j * N);
  }
}

}  // namespace

// largest run V (columns) such that every run starts at a multiple of V and V elements are aligned
static int rope_v(const mdg_rope_axes_desc& d, int e) {
  const bool inter = d.pairs == MDG_ROPE_INTERLEAVED;
  const int vmax = 16 / e / (inter ? 2 : 1);
  for (int v = vmax; v > 1; v /= 2) {
    const int run = inter ? 2 * v : v;
    bool ok = (d.D - 2 * d.npairs) % v == 0 && (2 * d.npairs) % v == 0 && d.npairs % v == 0;
    if (d.pairs == MDG_ROPE_AXIS)
      for (int a = 0; a < d.naxes; ++a) ok = ok && d.section[a] % v == 0;
    for (int i = 0; ok && i < d.nseg; ++i) {
      const mdg_heads* t[2] = {&d.x[i], &d.out[i]};
      for (int j = 0; j < 2; ++j)
        ok = ok && (((uintptr_t)t[j]->p | (uintptr_t)(t[j]->sb * e) | (uintptr_t)(t[j]->sn * e) | (uintptr_t)(t[j]->sh * e)) &
                    (uintptr_t)(run * e - 1)) == 0;
    }
    if (ok) return v;
  }
  return 1;
}

// Items of one or two pairs, shorter than 16 bytes, whole 16-byte pieces per head row, and a token's rows in a tile
static bool rope_tiled(const mdg_rope_axes_desc& d, int V, int heads) {
  const int e = d.dtype == MDG_BF16 ? 2 : 4, run = V * e * (d.pairs == MDG_ROPE_INTERLEAVED ? 2 : 1);
  if (V > 2 || run >= 16 || d.D * e % 16 || heads * d.D * e > 2 * kRopeTile - 16) return false;
  for (int i = 0; i < d.nseg; ++i)
    for (const mdg_heads* t : {&d.x[i], &d.out[i]})
      if (((uintptr_t)t->p | (uintptr_t)(t->sb * e) | (uintptr_t)(t->sn * e) | (uintptr_t)(t->sh * e)) & 15) return false;
  return true;
}

static RopeP rope_params(const mdg_rope_axes_desc& d, int& V) {
  const int e = d.dtype == MDG_BF16 ? 2 : 4;
  V = rope_v(d, e);
  // (one interleaved pair is a run of two: its two columns must be readable as one word)
  RopeP p;
  p.HT = 0;
  for (int i = 0; i < d.nseg; ++i) {
    p.seg[i] = RopeSeg{d.x[i].p, const_cast<void*>(d.out[i].p), d.x[i].sb, d.x[i].sn, d.x[i].sh, d.out[i].sb, d.out[i].sn, d.out[i].sh};
    p.HT += d.H[i];
  }
  if (d.nseg == 1) p.seg[1] = p.seg[0];
  p.H0 = d.H[0], p.N = d.N, p.D = d.D, p.np = d.npairs;
  p.tokens = (unsigned)d.B * (unsigned)d.N;
  p.pos = d.pos, p.pb = d.pos_sb, p.pn = d.pos_sn, p.i64 = d.pos_i64;
  p.turns = d.turns, p.axis = d.axis, p.cols = d.cols, p.inverse = d.inverse;
  const int tail = d.D - 2 * d.npairs;
  p.rot_tasks = d.npairs / V;
  p.copy_w = tail % (2 * V) == 0 ? 2 * V : V;
  p.tasks = p.rot_tasks + tail / p.copy_w;
  p.lds = 0;
  if (rope_tiled(d, V, p.HT)) {
    if (d.pairs == MDG_ROPE_INTERLEAVED) V = 1;  // (two runs of one column)
    const int per = p.HT * d.D * e / 16, row = (per | 1) * 16;
    int T = kRopeTile / row, few = (int)((p.tokens + 1023) / 1024);
    if (T > few) T = few;
    p.T = T < 1 ? 1 : T, p.lds = p.T * row;
    p.inv_np = 0.f, p.inv_tasks = 1.0f / (d.D * e / 16), p.inv_row = 1.0f / per;  // of pieces
    return p;
  }
  // tokens per block: about 2048 items, and 1024 blocks where there are that many tokens
  const int row = p.HT * p.tasks;
  int T = 2048 / row, few = (int)((p.tokens + 1023) / 1024);
  if (T > few) T = few;
  if (T * p.np > kRopeLds) T = kRopeLds / p.np;
  p.T = T < 1 ? 1 : T;
  p.inv_np = 1.0f / p.np, p.inv_tasks = 1.0f / p.tasks, p.inv_row = 1.0f / row;
  return p;
}

// whether one interleaved pair can be read as a run of two elements
bool rope_axes_pair_aligned(const mdg_rope_axes_desc& d) {
  const int e = d.dtype == MDG_BF16 ? 2 : 4;
  for (int i = 0; i < d.nseg; ++i) {
    const mdg_heads* t[2] = {&d.x[i], &d.out[i]};
    for (int j = 0; j < 2; ++j)
      if (((uintptr_t)t[j]->p | (uintptr_t)(t[j]->sb * e) | (uintptr_t)(t[j]->sn * e) | (uintptr_t)(t[j]->sh * e)) & (uintptr_t)(2 * e - 1))
        return false;
  }
  return true;
}

static void rope_tile_go(const RopeP& p, int dtype, int V, unsigned grid, hipStream_t s) {
#define ROPE_GO(CT, V_) hipLaunchKernelGGL((rope_tile_kernel<CT, V_>), dim3(grid), dim3(256), p.lds, s, p)
  if (dtype == MDG_BF16) {
    if (V == 2) ROPE_GO(bf16_t, 2);
    else ROPE_GO(bf16_t, 1);
  } else {
    if (V == 2) ROPE_GO(float, 2);
    else ROPE_GO(float, 1);
  }
#undef ROPE_GO
}

static void rope_go(const RopeP& p, int dtype, int V, bool inter, unsigned grid, hipStream_t s) {
#define ROPE_GO(CT, V_, I) hipLaunchKernelGGL((rope_axes_kernel<CT, V_, I>), dim3(grid), dim3(256), 0, s, p)
  if (dtype == MDG_BF16) {
    if (inter) {
      if (V == 4) ROPE_GO(bf16_t, 4, true);
      else if (V == 2) ROPE_GO(bf16_t, 2, true);
      else ROPE_GO(bf16_t, 1, true);
    } else {
      if (V == 8) ROPE_GO(bf16_t, 8, false);
      else if (V == 4) ROPE_GO(bf16_t, 4, false);
      else if (V == 2) ROPE_GO(bf16_t, 2, false);
      else ROPE_GO(bf16_t, 1, false);
    }
  } else {
    if (inter) {
      if (V == 2) ROPE_GO(float, 2, true);
      else ROPE_GO(float, 1, true);
    } else {
      if (V == 4) ROPE_GO(float, 4, false);
      else if (V == 2) ROPE_GO(float, 2, false);
      else ROPE_GO(float, 1, false);
    }
  }
#undef ROPE_GO
}

// within the 2^32 threads of a grid
bool rope_axes_grid_ok(const mdg_rope_axes_desc& d) {
  int V;
  const RopeP p = rope_params(d, V);
  return (p.tokens - 1) / p.T < ((1LL << 32) - 1) / 256 - 1;
}

hipError_t rope_axes_launch(const mdg_rope_axes_desc& d, hipStream_t s) {
  int V;
  const RopeP p = rope_params(d, V);
  // (interleaved pairs that do not lie on a word of two elements take the two-run kernel: V is 1 then)
  const bool inter = d.pairs == MDG_ROPE_INTERLEAVED && rope_axes_pair_aligned(d);
  const unsigned grid = (p.tokens + p.T - 1) / p.T;
  if (p.lds) rope_tile_go(p, d.dtype, V, grid, s);
  else rope_go(p, d.dtype, V, inter, grid, s);
  return hipGetLastError();
}

}  // namespace mdg
