// Rotary positions with several axes: pair p of a head's rotated columns belongs to one axis (frame,
// residue, height, ...) and turns by pos[token][axis[p]] * freq[p]; columns past the pairs pass through.
//   y1 = x1 cos - x2 sin,  y2 = x2 cos + x1 sin      (inverse: -sin; it is the backward)
// Bound by memory: every element is read and written once.  The angle is formed in double as a number
// of turns and reduced there (a position of 10^6 in fp32 would lose the angle), then cos / sin in
// fp32, once per (token, pair) and thread for all the heads that thread walks.  q and k go in one
// launch: their heads are one list.
#include "../../include/mdgen_hip.h"
#include "common.h"

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
  int N, D, np, pairs;
  long long tokens;  // B * N
  const void* pos;
  long long pb, pn;
  const double* turns;
  const int* axis;
  const int* cols;  // first columns of the pairs, then second columns
  int inverse, i64;
  int rot_tasks, tasks;  // per head row: rotations of V pairs, then copies of 2V (or V) columns
  int copy_w;
  int hpt, hs;  // heads per thread, threads along the heads
};

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

// V pairs per thread and head.  INTER: the pair's columns are neighbours (one run of 2V columns);
// otherwise two runs of V columns, cols[p] .. and cols[np + p] ..  (the host picks V so that no run
// crosses a section and every run is aligned to its bytes).
template <typename CT, int V, bool INTER>
__global__ __launch_bounds__(256) void rope_axes_kernel(const RopeP p) {
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  const int task = (int)(id % p.tasks);
  const long long rest = id / p.tasks;
  const int hslot = (int)(rest % p.hs);
  const long long tok = rest / p.hs;
  if (tok >= p.tokens) return;
  const long long b = tok / p.N, n = tok % p.N;

  const bool rot = task < p.rot_tasks;
  float cs[V], sn[V];
  int c1, c2;
  if (rot) {
    const int p0 = task * V;
    c1 = INTER ? 2 * p0 : p.cols[p0];
    c2 = INTER ? 2 * p0 : p.cols[p.np + p0];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const long long at = b * p.pb + n * p.pn + p.axis[p0 + i];
      const double ps = p.i64 ? (double)reinterpret_cast<const long long*>(p.pos)[at]
                              : (double)reinterpret_cast<const int*>(p.pos)[at];
      const double t = ps * p.turns[p0 + i];
      const float f = 2.0f * (float)(t - rint(t));  // half turns in [-1, 1]
      sincospif(f, &sn[i], &cs[i]);
      if (p.inverse) sn[i] = -sn[i];
    }
  } else {
    c1 = c2 = 2 * p.np + (task - p.rot_tasks) * p.copy_w;
  }
  for (int j = 0; j < p.hpt; ++j) {
    const int hd = j * p.hs + hslot;
    if (hd >= p.HT) break;
    const RopeSeg& g = p.seg[hd >= p.H0];
    const int h = hd >= p.H0 ? hd - p.H0 : hd;
    const CT* x = reinterpret_cast<const CT*>(g.x) + b * g.xb + n * g.xn + h * g.xh;
    CT* y = reinterpret_cast<CT*>(g.y) + b * g.yb + n * g.yn + h * g.yh;
    if (!rot) {
      for (int i = 0; i < p.copy_w; i += V) stw<CT, V>(y + c1 + i, ldw<CT, V>(x + c1 + i));
    } else if constexpr (INTER) {
      Pack<CT, 2 * V> a = ldw<CT, 2 * V>(x + c1), r;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float u = (float)a.v[2 * i], w = (float)a.v[2 * i + 1];
        r.v[2 * i] = (CT)(u * cs[i] - w * sn[i]);
        r.v[2 * i + 1] = (CT)(w * cs[i] + u * sn[i]);
      }
      stw<CT, 2 * V>(y + c1, r);
    } else {
      const Pack<CT, V> a = ldw<CT, V>(x + c1), c = ldw<CT, V>(x + c2);
      Pack<CT, V> r, q;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float u = (float)a.v[i], w = (float)c.v[i];
        r.v[i] = (CT)(u * cs[i] - w * sn[i]);
        q.v[i] = (CT)(w * cs[i] + u * sn[i]);
      }
      stw<CT, V>(y + c1, r);
      stw<CT, V>(y + c2, q);
    }
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
  p.H0 = d.H[0], p.N = d.N, p.D = d.D, p.np = d.npairs, p.pairs = d.pairs;
  p.tokens = (long long)d.B * d.N;
  p.pos = d.pos, p.pb = d.pos_sb, p.pn = d.pos_sn, p.i64 = d.pos_i64;
  p.turns = d.turns, p.axis = d.axis, p.cols = d.cols, p.inverse = d.inverse;
  const int tail = d.D - 2 * d.npairs;
  p.rot_tasks = d.npairs / V;
  p.copy_w = tail % (2 * V) == 0 ? 2 * V : V;
  p.tasks = p.rot_tasks + tail / p.copy_w;
  // heads per thread: 8 share one set of cos / sin once the launch fills the chip without that
  p.hpt = p.tokens * p.tasks * p.HT >= 256LL * 2048 * 4 ? (p.HT < 8 ? p.HT : 8) : 1;
  p.hs = (p.HT + p.hpt - 1) / p.hpt;
  return p;
}

bool rope_axes_grid_ok(const mdg_rope_axes_desc& d) {
  int V;
  const RopeP p = rope_params(d, V);
  return (p.tokens * p.tasks * p.hs + 255) / 256 < (1LL << 31);
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

hipError_t rope_axes_launch(const mdg_rope_axes_desc& d, hipStream_t s) {
  int V;
  const RopeP p = rope_params(d, V);
  // (interleaved pairs that do not lie on a word of two elements take the two-run kernel: V is 1 then)
  const bool inter = d.pairs == MDG_ROPE_INTERLEAVED && rope_axes_pair_aligned(d);
  const unsigned grid = (unsigned)((p.tokens * p.tasks * p.hs + 255) / 256);
#define ROPE_GO(CT, V_, I) hipLaunchKernelGGL((rope_axes_kernel<CT, V_, I>), dim3(grid), dim3(256), 0, s, p)
  if (d.dtype == MDG_BF16) {
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
  return hipGetLastError();
}

}  // namespace mdg
