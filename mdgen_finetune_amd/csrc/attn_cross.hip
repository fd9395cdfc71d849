// Cross attention: queries [B][Nq][H][D] over an encoder's k / v [B][Nk][Hk][D] of another length
// (H % Hk == 0: H / Hk query heads share a key head), softmax over the keys that are there
// (key < kv_len[b] and mask[b][key] != 0), and its backward.
//
//   S_ij = scale q_i . k_j,  P = softmax_j S,  o_i = sum_j P_ij v_j        (a row without keys: o = 0)
//   delta_i = do_i . o_i,  dS_ij = P_ij (do_i . v_j - delta_i)
//   dq_i = scale sum_j dS_ij k_j,  dk_j = scale sum_i dS_ij q_i,  dv_j = sum_i P_ij do_i
//
// Rows: the query heads of one key head are packed, row r = n * G + g (G = H / Hk), so a k / v tile
// is read once for all of them and a single token of a grouped model still fills a matrix tile.
//
// Matrix products: 32x32 tiles, K = 16 per step (v_mfma_f32_32x32x16_bf16, or eight
// v_mfma_f32_32x32x2_f32).  Lane l = (c = l & 31, h = l >> 5).  An operand fragment is 8 elements:
// element j of half h is k-index 8h + j; for fp32 MFMA j sums the k-indices j and 8 + j.  The
// accumulator's register 4a + i of half h is row 8a + 4h + i, column c.  Eight consecutive accumulator
// registers are then the next product's second operand as they are, if its first operand's element j
// is row 8 (j >> 2) + 4h + (j & 3) of the 16-row step: col_frag reads it so, and no probability ever
// moves between lanes.  Forward and dq hold S^T (one query per lane: its maximum, sum and offsets
// are lane scalars); dk / dv hold S (one key per lane).
#include "../../include/mdgen_hip.h"
#include "common.h"

#include <cfloat>
#include <cmath>

namespace mdg {
namespace {

typedef __attribute__((ext_vector_type(16))) float f32x16;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNoMax = -FLT_MAX;  // running maximum before the first key

struct View {  // element strides of batch, token, head; the head dim is contiguous
  const void* p;
  long long sb, sn, sh;
};
struct CrossP {
  View q, k, v, o, olo, dout, dq, dk, dv;
  const int *qlen, *klen;
  const void* mask;
  long long mb, mn;
  int mask_f32;
  int B, Nq, Nk, H, Hk, G, D;
  float c;      // scale * log2 e: scores in log2 units
  float scale;
  float* lse;   // [B][H][Nq] log2 of the row's softmax normaliser; -inf: a row without keys
  float* delta; // [B][H][Nq]
  float* part;  // split partials
  float* part_ml;
  int nsplit;
  int vec;      // 16-byte pieces: D a multiple of a piece, every base and stride 16-byte aligned
};

template <typename CT>
__device__ __forceinline__ f32x16 mma(const typename V8<CT>::T& a, const typename V8<CT>::T& b, f32x16 acc) {
  if constexpr (is_bf16<CT>()) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc, 0, 0, 0);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], acc, 0, 0, 0);
    return acc;
  }
}

// LDS row stride: 32 bytes of padding put 8 consecutive rows on different banks for 16-byte reads
template <typename CT, int DP>
constexpr int lds_ld() { return DP + 32 / (int)sizeof(CT); }

// element j: tile[k0 + 8 (j >> 2) + 4h + (j & 3)][c0 + (lane & 31)] of a row-major LDS tile
template <typename CT, int LD>
__device__ __forceinline__ typename V8<CT>::T col_frag(const CT* tile, int k0, int c0, int lane) {
  typename V8<CT>::T r;
  const int h = lane >> 5;
  if constexpr (is_bf16<CT>()) {
    // ds_read_b64_tr_b16: in each group of 16 lanes, lane 4q + p supplies columns 4p..4p+3 of row q and
    // receives column (lane & 15) of the four rows
    typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;
    const CT* a = tile + (k0 + 4 * h + ((lane & 15) >> 2)) * LD + c0 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)a);
    const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(a + 8 * LD));
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = lo[j], r[4 + j] = hi[j];
  } else {
    const CT* a = tile + (k0 + 4 * h) * LD + c0 + (lane & 31);
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = a[j * LD], r[4 + j] = a[(8 + j) * LD];
  }
  return r;
}

template <typename CT, int LD>
__device__ __forceinline__ typename V8<CT>::T row_frag(const CT* tile, int row, int k0, int lane) {
  return ld8<CT>(tile + row * LD + k0 + 8 * (lane >> 5));
}

// one 16-byte piece (columns c0 ..) of a row of D elements, zero past D
template <typename CT>
__device__ __forceinline__ uint4 ld_piece(const CT* row, int c0, int D, int vec) {
  constexpr int N = 16 / sizeof(CT);
  uint4 r = make_uint4(0, 0, 0, 0);
  if (vec) {
    if (c0 < D) r = *reinterpret_cast<const uint4*>(row + c0);
  } else {
    CT e[N];
#pragma unroll
    for (int j = 0; j < N; ++j) e[j] = c0 + j < D ? row[c0 + j] : (CT)0.f;
    __builtin_memcpy(&r, e, 16);
  }
  return r;
}
template <typename CT>
__device__ __forceinline__ typename V8<CT>::T ld_frag(const CT* row, int c0, int D, int vec) {
  typename V8<CT>::T r;
  constexpr int N = 16 / sizeof(CT);
#pragma unroll
  for (int j = 0; j < 8; j += N) {
    const uint4 u = ld_piece<CT>(row, c0 + j, D, vec);
    CT e[N];
    __builtin_memcpy(e, &u, 16);
#pragma unroll
    for (int i = 0; i < N; ++i) r[j + i] = e[i];
  }
  return r;
}

// four consecutive outputs d0 .. d0 + 3 of a row (vec: 8- / 16-byte stores, D a multiple of 4)
template <typename CT>
__device__ __forceinline__ void st_out(CT* row, int d0, int D, int vec, float a, float b, float c, float d) {
  if (vec) {
    if (d0 < D) st4<CT>(row + d0, a, b, c, d);
  } else {
    if (d0 < D) row[d0] = (CT)a;
    if (d0 + 1 < D) row[d0 + 1] = (CT)b;
    if (d0 + 2 < D) row[d0 + 2] = (CT)c;
    if (d0 + 3 < D) row[d0 + 3] = (CT)d;
  }
}

template <typename CT>
__device__ __forceinline__ const CT* vrow(const View& v, int b, int n, int h) {
  return reinterpret_cast<const CT*>(v.p) + b * v.sb + n * v.sn + h * v.sh;
}
template <typename CT>
__device__ __forceinline__ CT* wrow(const View& v, int b, int n, int h) {
  return const_cast<CT*>(vrow<CT>(v, b, n, h));
}

__device__ __forceinline__ int clamp_len(const int* len, int b, int n) {
  return len ? min(max(len[b], 0), n) : n;
}
__device__ __forceinline__ bool key_kept(const CrossP& p, int b, int key) {
  if (!p.mask) return true;
  const long long i = b * p.mb + key * p.mn;
  return p.mask_f32 ? reinterpret_cast<const float*>(p.mask)[i] != 0.f
                    : reinterpret_cast<const unsigned char*>(p.mask)[i] != 0;
}

__device__ __forceinline__ float half_max(float v) { return fmaxf(v, __shfl_xor(v, 32, 64)); }
__device__ __forceinline__ float half_sum(float v) { return v + __shfl_xor(v, 32, 64); }

// The softmax of one 32-key tile: raises the lane's maximum when a score outgrows it by 2^8 (a lagging
// maximum costs no precision: P is floating point and stays below 2^8, sums are fp32), turns the
// scores into P and adds their sum.  s: raw scores, -inf where the key is masked.
template <int NT, int DT>
__device__ __forceinline__ void softmax_tile(f32x16 (&s)[NT], f32x16 (&o)[DT], float& m, float& l, float c) {
  const float grow = 8.0f / c;
  float mx = s[0][0];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[t][i]);
  mx = half_max(mx);
  if (__any(mx > m + grow)) {
    const float nm = mx > m + grow ? mx : m;
    const float alpha = m == kNoMax ? 0.f : __builtin_amdgcn_exp2f((m - nm) * c);
    m = nm;
    l *= alpha;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[t][i] *= alpha;
  }
  const float mc = m == kNoMax ? 0.f : m * c;
  float sum = 0.f;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[t][i] = __builtin_amdgcn_exp2f(fmaf(s[t][i], c, -mc));
      sum += s[t][i];
    }
  l += sum;
}

// A tile of k / v rows on its way from memory to LDS through registers, by NT threads.
template <typename CT, int DP, int ROWS, int NT>
struct Stage {
  static constexpr int LD = lds_ld<CT, DP>(), VEC = 16 / sizeof(CT), PPR = DP / VEC, P = ROWS * PPR / NT;
  static_assert(ROWS * PPR % NT == 0, "whole pieces per thread");
  uint4 r[P];
  // rows key0 .. key0 + ROWS of one (b, kv head); keys >= end are zero
  __device__ __forceinline__ void load(const CT* base, long long sn, int key0, int end, int D, int vec, int tid) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int idx = tid + i * NT, row = idx / PPR, cc = (idx % PPR) * VEC, key = key0 + row;
      r[i] = key < end ? ld_piece<CT>(base + key * sn, cc, D, vec) : make_uint4(0, 0, 0, 0);
    }
  }
  __device__ __forceinline__ void store(CT* tile, int tid) const {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int idx = tid + i * NT, row = idx / PPR, cc = (idx % PPR) * VEC;
      *reinterpret_cast<uint4*>(tile + row * LD + cc) = r[i];
    }
  }
};

// Masked keys' k / v rows are zero in LDS (what lies there, NaN too, never reaches a product) and their
// scores start at -inf: kb holds 0 or -inf per key and is the product's initial accumulator.
template <typename CT, int DP, int ROWS, int NT>
struct KvStage {
  Stage<CT, DP, ROWS, NT> k, v;
  float keep[Stage<CT, DP, ROWS, NT>::P];
  float kb;
  __device__ __forceinline__ void load(const CrossP& p, const CT* kbase, const CT* vbase, int b, int key0, int end,
                                       int tid) {
    using S = Stage<CT, DP, ROWS, NT>;
    k.load(kbase, p.k.sn, key0, end, p.D, p.vec, tid);
    v.load(vbase, p.v.sn, key0, end, p.D, p.vec, tid);
    if (p.mask) {
#pragma unroll
      for (int i = 0; i < S::P; ++i) {
        const int key = key0 + (tid + i * NT) / S::PPR;
        keep[i] = key < end && key_kept(p, b, key) ? 1.f : 0.f;
      }
    }
    const int key = key0 + tid;
    kb = tid < ROWS && key < end && key_kept(p, b, key) ? 0.f : -INFINITY;
  }
  // flag: some key of the tile is not there (one wave holds all of kb: ROWS <= 64)
  __device__ __forceinline__ void store(const CrossP& p, CT* Ks, CT* Vs, float* kbs, int* flag, int tid) {
    using S = Stage<CT, DP, ROWS, NT>;
    if (p.mask) {
#pragma unroll
      for (int i = 0; i < S::P; ++i)
        if (keep[i] == 0.f) k.r[i] = v.r[i] = make_uint4(0, 0, 0, 0);
    }
    k.store(Ks, tid);
    v.store(Vs, tid);
    if (tid < 64) {
      if (tid < ROWS) kbs[tid] = kb;
      const bool any = __any(tid < ROWS && kb != 0.f);
      if (tid == 0) *flag = any;
    }
  }
};

// initial accumulator of a 32-key tile of S^T: the keys' kb, rows 8a + 4h + i
__device__ __forceinline__ f32x16 kb_init(const float* kbs, int flag, int lane) {
  f32x16 s;
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    const float4 t = flag ? *reinterpret_cast<const float4*>(kbs + 8 * a + 4 * (lane >> 5)) : make_float4(0, 0, 0, 0);
    s[4 * a] = t.x, s[4 * a + 1] = t.y, s[4 * a + 2] = t.z, s[4 * a + 3] = t.w;
  }
  return s;
}

template <typename CT>
__device__ __forceinline__ typename V8<CT>::T half_frag(const f32x16& s, int s2) {
  typename V8<CT>::T r;
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = (CT)s[8 * s2 + j];
  return r;
}

// keys [k0, k1) of split `sp`: the sequence's own length shared out in multiples of 32
__device__ __forceinline__ void split_range(int klen, int nsplit, int sp, int& k0, int& k1) {
  const int per = ((klen + nsplit - 1) / nsplit + 31) / 32 * 32;
  k0 = min(klen, sp * per);
  k1 = min(klen, k0 + per);
}

struct BlockId {
  int tile, split, b, hk;
};
__device__ __forceinline__ BlockId block_id(const CrossP& p, int tiles) {
  BlockId r;
  int id = blockIdx.x;
  r.tile = id % tiles;
  id /= tiles;
  r.split = id % p.nsplit;
  id /= p.nsplit;
  r.hk = id % p.Hk;
  r.b = id / p.Hk;
  return r;
}

// rows of partial `sp`: ((b * Hk + hk) * rows + r), rows = Nq * G
__device__ __forceinline__ long long part_row(const CrossP& p, int sp, int b, int hk, int r) {
  const long long rows = (long long)p.Nq * p.G;
  return ((long long)sp * p.B * p.Hk + (long long)b * p.Hk + hk) * rows + r;
}

// ------------------------------------------------------------------------------------------ forward
// One block = 4 waves x 32 rows of one (b, key head); k / v tiles of KT keys go through LDS, double
// buffered through registers, one barrier per tile.
template <typename CT, int DP, int KT>
__global__ __launch_bounds__(256, 2) void cross_fwd_kernel(const CrossP p, int tiles) {
  constexpr int LD = lds_ld<CT, DP>(), DT = DP / 32, KS = DP / 16, NT = KT / 32;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  CT* Ks = reinterpret_cast<CT*>(smem);
  CT* Vs = Ks + 2 * KT * LD;
  float* kbs = reinterpret_cast<float*>(Vs + 2 * KT * LD);
  int* flag = reinterpret_cast<int*>(kbs + 2 * KT);

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
  const BlockId id = block_id(p, tiles);
  const int rows = p.Nq * p.G, r = id.tile * 128 + wave * 32 + (lane & 31);
  const int n = r / p.G, head = id.hk * p.G + r % p.G;
  const int qlen = clamp_len(p.qlen, id.b, p.Nq), klen = clamp_len(p.klen, id.b, p.Nk);
  const bool live = r < rows && n < qlen;

  typename V8<CT>::T qf[KS];
  const CT* qrow = vrow<CT>(p.q, id.b, live ? n : 0, live ? head : 0);
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) qf[ks] = live ? ld_frag<CT>(qrow, 16 * ks + 8 * h, p.D, p.vec) : zero8<CT>();

  f32x16 o[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[t][i] = 0.f;
  float m = kNoMax, l = 0.f;

  int k0, k1;
  split_range(klen, p.nsplit, id.split, k0, k1);
  const CT* kbase = vrow<CT>(p.k, id.b, 0, id.hk);
  const CT* vbase = vrow<CT>(p.v, id.b, 0, id.hk);
  KvStage<CT, DP, KT, 256> st;
  const int nt = (k1 - k0 + KT - 1) / KT;
  if (nt > 0) {
    st.load(p, kbase, vbase, id.b, k0, k1, tid);
    st.store(p, Ks, Vs, kbs, flag, tid);
  }
  __syncthreads();
  for (int t = 0; t < nt; ++t) {
    const int cur = t & 1;
    if (t + 1 < nt) st.load(p, kbase, vbase, id.b, k0 + (t + 1) * KT, k1, tid);
    const CT* Kc = Ks + cur * KT * LD;
    const CT* Vc = Vs + cur * KT * LD;
    f32x16 s[NT];
#pragma unroll
    for (int kt = 0; kt < NT; ++kt) {
      s[kt] = kb_init(kbs + cur * KT + 32 * kt, flag[cur], lane);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        s[kt] = mma<CT>(row_frag<CT, LD>(Kc, 32 * kt + (lane & 31), 16 * ks, lane), qf[ks], s[kt]);
    }
    softmax_tile<NT, DT>(s, o, m, l, p.c);
#pragma unroll
    for (int kt = 0; kt < NT; ++kt)
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        const typename V8<CT>::T pf = half_frag<CT>(s[kt], s2);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
          o[dt] = mma<CT>(col_frag<CT, LD>(Vc, 32 * kt + 16 * s2, 32 * dt, lane), pf, o[dt]);
      }
    if (t + 1 < nt) st.store(p, Ks + (cur ^ 1) * KT * LD, Vs + (cur ^ 1) * KT * LD, kbs + (cur ^ 1) * KT, flag + (cur ^ 1), tid);
    __syncthreads();
  }

  l = half_sum(l);
  if (r >= rows) return;
  if (p.nsplit > 1) {
    const long long pr = part_row(p, id.split, id.b, id.hk, r);
    if (h == 0) {
      p.part_ml[2 * pr] = m;
      p.part_ml[2 * pr + 1] = l;
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int a = 0; a < 4; ++a)
        *reinterpret_cast<float4*>(p.part + pr * DP + 32 * dt + 8 * a + 4 * h) =
            make_float4(o[dt][4 * a], o[dt][4 * a + 1], o[dt][4 * a + 2], o[dt][4 * a + 3]);
    return;
  }
  const bool some = live && l != 0.f;  // (a NaN among the keys that are there stays one)
  const float inv = some ? 1.0f / l : 0.f;
  if (p.lse && h == 0) p.lse[((long long)id.b * p.H + head) * p.Nq + n] = some ? m * p.c + log2f(l) : -INFINITY;
  CT* orow = wrow<CT>(p.o, id.b, n, head);
  CT* lrow = p.olo.p ? wrow<CT>(p.olo, id.b, n, head) : nullptr;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = some ? o[dt][4 * a + i] * inv : 0.f;
      const int d0 = 32 * dt + 8 * a + 4 * h;
      st_out<CT>(orow, d0, p.D, p.vec, v[0], v[1], v[2], v[3]);
      if (lrow)  // the rounding residual of o, for an exact delta in the backward
        st_out<CT>(lrow, d0, p.D, p.vec, v[0] - (float)(CT)v[0], v[1] - (float)(CT)v[1], v[2] - (float)(CT)v[2],
                   v[3] - (float)(CT)v[3]);
    }
}

// At most 32 rows per (b, key head), the single-token form: the 4 waves split the keys instead of
// the rows.  Each wave stages its own 32-key tiles (no block barrier in the loop: a wave's LDS
// operations are in order), and the four partial softmaxes are joined in LDS at the end.
template <typename CT, int DP>
__global__ __launch_bounds__(256) void cross_few_kernel(const CrossP p, int tiles) {
  constexpr int LD = lds_ld<CT, DP>(), DT = DP / 32, KS = DP / 16, LO = DP + 4;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
  CT* Ks = reinterpret_cast<CT*>(smem) + wave * 2 * 32 * LD;
  CT* Vs = Ks + 32 * LD;
  float* kbs = reinterpret_cast<float*>(reinterpret_cast<CT*>(smem) + 4 * 2 * 32 * LD) + wave * 32;
  int* flag = reinterpret_cast<int*>(reinterpret_cast<float*>(reinterpret_cast<CT*>(smem) + 4 * 2 * 32 * LD) + 128) + wave;

  const BlockId id = block_id(p, tiles);
  const int rows = p.Nq * p.G, r = lane & 31;
  const int n = r / p.G, head = id.hk * p.G + r % p.G;
  const int qlen = clamp_len(p.qlen, id.b, p.Nq), klen = clamp_len(p.klen, id.b, p.Nk);
  const bool live = r < rows && n < qlen;
  typename V8<CT>::T qf[KS];
  const CT* qrow = vrow<CT>(p.q, id.b, live ? n : 0, live ? head : 0);
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) qf[ks] = live ? ld_frag<CT>(qrow, 16 * ks + 8 * h, p.D, p.vec) : zero8<CT>();
  f32x16 o[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[t][i] = 0.f;
  float m = kNoMax, l = 0.f;

  int k0, k1;
  split_range(klen, p.nsplit, id.split, k0, k1);
  const CT* kbase = vrow<CT>(p.k, id.b, 0, id.hk);
  const CT* vbase = vrow<CT>(p.v, id.b, 0, id.hk);
  KvStage<CT, DP, 32, 64> st;
  int key = k0 + 32 * wave;
  if (key < k1) st.load(p, kbase, vbase, id.b, key, k1, lane);
  for (; key < k1; key += 128) {
    st.store(p, Ks, Vs, kbs, flag, lane);
    if (key + 128 < k1) st.load(p, kbase, vbase, id.b, key + 128, k1, lane);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    f32x16 s[1] = {kb_init(kbs, *flag, lane)};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) s[0] = mma<CT>(row_frag<CT, LD>(Ks, lane & 31, 16 * ks, lane), qf[ks], s[0]);
    softmax_tile<1, DT>(s, o, m, l, p.c);
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2) {
      const typename V8<CT>::T pf = half_frag<CT>(s[0], s2);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] = mma<CT>(col_frag<CT, LD>(Vs, 16 * s2, 32 * dt, lane), pf, o[dt]);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
  l = half_sum(l);

  // join: [4][32] maxima and sums, then the rescaled outputs [4][32][DP + 4] over the staging area
  __syncthreads();
  float* jm = reinterpret_cast<float*>(smem);
  float* jl = jm + 128;
  float* js = jl + 128;  // [32] the rows' joined sums
  float* jo = js + 32;
  if (h == 0) jm[32 * wave + r] = m, jl[32 * wave + r] = l;
  __syncthreads();
  float M = kNoMax, L = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) M = fmaxf(M, jm[32 * w + r]);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float mw = jm[32 * w + r];
    L += jl[32 * w + r] * (mw == kNoMax ? 1.f : __builtin_amdgcn_exp2f((mw - M) * p.c));
  }
  const float f = m == kNoMax ? 1.f : __builtin_amdgcn_exp2f((m - M) * p.c);  // (no keys: sums of 0)
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int a = 0; a < 4; ++a)
      *reinterpret_cast<float4*>(jo + (32 * wave + r) * LO + 32 * dt + 8 * a + 4 * h) =
          make_float4(o[dt][4 * a] * f, o[dt][4 * a + 1] * f, o[dt][4 * a + 2] * f, o[dt][4 * a + 3] * f);
  if (wave == 0 && h == 0 && r < rows) {
    if (p.nsplit > 1) {
      const long long pr = part_row(p, id.split, id.b, id.hk, r);
      p.part_ml[2 * pr] = M;
      p.part_ml[2 * pr + 1] = L;
    } else if (p.lse) {
      p.lse[((long long)id.b * p.H + head) * p.Nq + n] = live && L != 0.f ? M * p.c + log2f(L) : -INFINITY;
    }
  }
  if (wave == 0 && h == 0) js[r] = L;
  __syncthreads();
  for (int i = tid; i < rows * (DP / 4); i += 256) {
    const int row = i / (DP / 4), d0 = (i % (DP / 4)) * 4;
    float4 v = make_float4(0, 0, 0, 0);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float4 t = *reinterpret_cast<const float4*>(jo + (32 * w + row) * LO + d0);
      v.x += t.x, v.y += t.y, v.z += t.z, v.w += t.w;
    }
    if (p.nsplit > 1) {
      *reinterpret_cast<float4*>(p.part + part_row(p, id.split, id.b, id.hk, row) * DP + d0) = v;
    } else {
      const int rn = row / p.G, rh = id.hk * p.G + row % p.G;
      const float Lr = js[row];
      const bool some = rn < qlen && Lr != 0.f;
      const float inv = some ? 1.0f / Lr : 0.f;
      v = some ? make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv) : make_float4(0, 0, 0, 0);
      st_out<CT>(wrow<CT>(p.o, id.b, rn, rh), d0, p.D, p.vec, v.x, v.y, v.z, v.w);
      if (p.olo.p)
        st_out<CT>(wrow<CT>(p.olo, id.b, rn, rh), d0, p.D, p.vec, v.x - (float)(CT)v.x, v.y - (float)(CT)v.y,
                   v.z - (float)(CT)v.z, v.w - (float)(CT)v.w);
    }
  }
}

// Joins the splits' partial softmaxes: 32 lanes per row, fixed order over the splits.
template <typename CT, int DP>
__global__ __launch_bounds__(256) void cross_join_kernel(const CrossP p) {
  const long long rows = (long long)p.Nq * p.G, total = rows * p.B * p.Hk;
  const long long pr = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int d0 = (threadIdx.x & 31) * 4;
  if (pr >= total) return;
  float M = kNoMax, L = 0.f;
  for (int s = 0; s < p.nsplit; ++s) M = fmaxf(M, p.part_ml[2 * (s * total + pr)]);
  float4 v = make_float4(0, 0, 0, 0);
  for (int s = 0; s < p.nsplit; ++s) {
    const float ms = p.part_ml[2 * (s * total + pr)];
    const float f = ms == kNoMax ? 1.f : __builtin_amdgcn_exp2f((ms - M) * p.c);  // (no keys: sums of 0)
    L += f * p.part_ml[2 * (s * total + pr) + 1];
    if (d0 < DP) {
      const float4 t = *reinterpret_cast<const float4*>(p.part + (s * total + pr) * DP + d0);
      v.x = fmaf(f, t.x, v.x), v.y = fmaf(f, t.y, v.y), v.z = fmaf(f, t.z, v.z), v.w = fmaf(f, t.w, v.w);
    }
  }
  const int bh = (int)(pr / rows), r = (int)(pr % rows), b = bh / p.Hk, n = r / p.G, head = (bh % p.Hk) * p.G + r % p.G;
  const bool some = n < clamp_len(p.qlen, b, p.Nq) && L != 0.f;
  const float inv = some ? 1.0f / L : 0.f;
  if (p.lse && d0 == 0) p.lse[((long long)b * p.H + head) * p.Nq + n] = some ? M * p.c + log2f(L) : -INFINITY;
  if (d0 >= DP) return;
  v = some ? make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv) : make_float4(0, 0, 0, 0);
  st_out<CT>(wrow<CT>(p.o, b, n, head), d0, p.D, p.vec, v.x, v.y, v.z, v.w);
  if (p.olo.p)
    st_out<CT>(wrow<CT>(p.olo, b, n, head), d0, p.D, p.vec, v.x - (float)(CT)v.x, v.y - (float)(CT)v.y,
               v.z - (float)(CT)v.z, v.w - (float)(CT)v.w);
}

// ------------------------------------------------------------------------------------------ backward
// dq: the forward's layout (one query per lane).  delta = do . (o + o_lo) is formed here from the
// fragments in registers and left for the dk / dv pass.
template <typename CT, int DP, int KT>
__global__ __launch_bounds__(256, sizeof(CT) * DP >= 512 ? 1 : 2) void cross_dq_kernel(const CrossP p, int tiles) {
  constexpr int LD = lds_ld<CT, DP>(), DT = DP / 32, KS = DP / 16, NT = KT / 32;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  CT* Ks = reinterpret_cast<CT*>(smem);
  CT* Vs = Ks + 2 * KT * LD;
  float* kbs = reinterpret_cast<float*>(Vs + 2 * KT * LD);
  int* flag = reinterpret_cast<int*>(kbs + 2 * KT);

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
  const BlockId id = block_id(p, tiles);
  const int rows = p.Nq * p.G, r = id.tile * 128 + wave * 32 + (lane & 31);
  const int n = r / p.G, head = id.hk * p.G + r % p.G;
  const int qlen = clamp_len(p.qlen, id.b, p.Nq), klen = clamp_len(p.klen, id.b, p.Nk);
  const bool live = r < rows && n < qlen;
  const int ln = live ? n : 0, lh = live ? head : 0;
  const long long srow = ((long long)id.b * p.H + lh) * p.Nq + ln;

  typename V8<CT>::T qf[KS], gf[KS];
  float delta = 0.f;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const int c0 = 16 * ks + 8 * h;
    qf[ks] = live ? ld_frag<CT>(vrow<CT>(p.q, id.b, ln, lh), c0, p.D, p.vec) : zero8<CT>();
    gf[ks] = live ? ld_frag<CT>(vrow<CT>(p.dout, id.b, ln, lh), c0, p.D, p.vec) : zero8<CT>();
    const typename V8<CT>::T of = live ? ld_frag<CT>(vrow<CT>(p.o, id.b, ln, lh), c0, p.D, p.vec) : zero8<CT>();
    if (p.olo.p) {
      const typename V8<CT>::T lo = live ? ld_frag<CT>(vrow<CT>(p.olo, id.b, ln, lh), c0, p.D, p.vec) : zero8<CT>();
#pragma unroll
      for (int j = 0; j < 8; ++j) delta = fmaf((float)gf[ks][j], (float)of[j] + (float)lo[j], delta);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) delta = fmaf((float)gf[ks][j], (float)of[j], delta);
    }
  }
  delta = half_sum(delta);
  float lse = live ? p.lse[srow] : -INFINITY;
  if (lse == -INFINITY) lse = INFINITY;  // a row without keys: every P is 0
  if (p.delta && id.split == 0 && r < rows && h == 0) p.delta[((long long)id.b * p.H + head) * p.Nq + n] = delta;

  f32x16 acc[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[t][i] = 0.f;

  int k0, k1;
  split_range(klen, p.nsplit, id.split, k0, k1);
  const CT* kbase = vrow<CT>(p.k, id.b, 0, id.hk);
  const CT* vbase = vrow<CT>(p.v, id.b, 0, id.hk);
  KvStage<CT, DP, KT, 256> st;
  const int nt = (k1 - k0 + KT - 1) / KT;
  if (nt > 0) {
    st.load(p, kbase, vbase, id.b, k0, k1, tid);
    st.store(p, Ks, Vs, kbs, flag, tid);
  }
  __syncthreads();
  for (int t = 0; t < nt; ++t) {
    const int cur = t & 1;
    if (t + 1 < nt) st.load(p, kbase, vbase, id.b, k0 + (t + 1) * KT, k1, tid);
    const CT* Kc = Ks + cur * KT * LD;
    const CT* Vc = Vs + cur * KT * LD;
#pragma unroll
    for (int kt = 0; kt < NT; ++kt) {
      f32x16 s = kb_init(kbs + cur * KT + 32 * kt, flag[cur], lane), g;
#pragma unroll
      for (int i = 0; i < 16; ++i) g[i] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        s = mma<CT>(row_frag<CT, LD>(Kc, 32 * kt + (lane & 31), 16 * ks, lane), qf[ks], s);
        g = mma<CT>(row_frag<CT, LD>(Vc, 32 * kt + (lane & 31), 16 * ks, lane), gf[ks], g);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], p.c, -lse)) * (g[i] - delta);
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        const typename V8<CT>::T df = half_frag<CT>(s, s2);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
          acc[dt] = mma<CT>(col_frag<CT, LD>(Kc, 32 * kt + 16 * s2, 32 * dt, lane), df, acc[dt]);
      }
    }
    if (t + 1 < nt) st.store(p, Ks + (cur ^ 1) * KT * LD, Vs + (cur ^ 1) * KT * LD, kbs + (cur ^ 1) * KT, flag + (cur ^ 1), tid);
    __syncthreads();
  }
  if (r >= rows) return;
  if (p.nsplit > 1) {
    const long long pr = part_row(p, id.split, id.b, id.hk, r);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int a = 0; a < 4; ++a)
        *reinterpret_cast<float4*>(p.part + pr * DP + 32 * dt + 8 * a + 4 * h) =
            make_float4(acc[dt][4 * a], acc[dt][4 * a + 1], acc[dt][4 * a + 2], acc[dt][4 * a + 3]);
    return;
  }
  CT* row = wrow<CT>(p.dq, id.b, n, head);
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int a = 0; a < 4; ++a)
      st_out<CT>(row, 32 * dt + 8 * a + 4 * h, p.D, p.vec, acc[dt][4 * a] * p.scale, acc[dt][4 * a + 1] * p.scale,
                 acc[dt][4 * a + 2] * p.scale, acc[dt][4 * a + 3] * p.scale);
}

// dk, dv: one key per lane; a block owns 4 x 32 keys of one (b, key head) and walks the rows in tiles
// of 32 (q and do through LDS, double buffered); splits share the rows, their fp32 partials summed in
// order by cross_sum_kernel.
template <typename CT, int DP>
__global__ __launch_bounds__(256) void cross_dkv_kernel(const CrossP p, int tiles) {
  constexpr int LD = lds_ld<CT, DP>(), DT = DP / 32, KS = DP / 16, QT = 32;
  using S = Stage<CT, DP, QT, (QT * DP * (int)sizeof(CT) / 16 < 256 ? 128 : 256)>;
  constexpr int SN = QT * DP * (int)sizeof(CT) / 16 < 256 ? 128 : 256;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  CT* Qs = reinterpret_cast<CT*>(smem);
  CT* Gs = Qs + 2 * QT * LD;
  float* ls = reinterpret_cast<float*>(Gs + 2 * QT * LD);  // [2][QT]
  float* ds = ls + 2 * QT;

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
  const BlockId id = block_id(p, tiles);
  const int qlen = clamp_len(p.qlen, id.b, p.Nq), klen = clamp_len(p.klen, id.b, p.Nk);
  const int rows = qlen * p.G;
  const int key = id.tile * 128 + wave * 32 + (lane & 31);
  const bool live = key < klen && key_kept(p, id.b, key);

  typename V8<CT>::T kf[KS], vf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const int c0 = 16 * ks + 8 * h;
    kf[ks] = live ? ld_frag<CT>(vrow<CT>(p.k, id.b, key, id.hk), c0, p.D, p.vec) : zero8<CT>();
    vf[ks] = live ? ld_frag<CT>(vrow<CT>(p.v, id.b, key, id.hk), c0, p.D, p.vec) : zero8<CT>();
  }
  f32x16 dk[DT], dv[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) dk[t][i] = dv[t][i] = 0.f;

  const int per = ((rows + p.nsplit - 1) / p.nsplit + QT - 1) / QT * QT;
  const int r0 = min(rows, id.split * per), r1 = min(rows, r0 + per);
  const int nt = (r1 - r0 + QT - 1) / QT;
  // a block whose keys all lie past the sequence has nothing to sum
  const int todo = id.tile * 128 < klen ? nt : 0;

  uint4 rq[S::P], rg[S::P];
  float rl = INFINITY, rd = 0.f;
  auto load = [&](int row0) {
#pragma unroll
    for (int i = 0; i < S::P; ++i) {
      const int idx = tid + i * SN, row = row0 + idx / S::PPR, cc = (idx % S::PPR) * S::VEC;
      rq[i] = rg[i] = make_uint4(0, 0, 0, 0);
      if (tid < SN && row < r1) {
        const int n = row / p.G, hd = id.hk * p.G + row % p.G;
        rq[i] = ld_piece<CT>(vrow<CT>(p.q, id.b, n, hd), cc, p.D, p.vec);
        rg[i] = ld_piece<CT>(vrow<CT>(p.dout, id.b, n, hd), cc, p.D, p.vec);
      }
    }
    rl = INFINITY, rd = 0.f;
    if (tid < QT && row0 + tid < r1) {
      const int row = row0 + tid, n = row / p.G, hd = id.hk * p.G + row % p.G;
      const long long i = ((long long)id.b * p.H + hd) * p.Nq + n;
      rl = p.lse[i], rd = p.delta[i];
      if (rl == -INFINITY) rl = INFINITY;
    }
  };
  auto store = [&](int buf) {
    if (tid < SN) {
#pragma unroll
      for (int i = 0; i < S::P; ++i) {
        const int idx = tid + i * SN, row = idx / S::PPR, cc = (idx % S::PPR) * S::VEC;
        *reinterpret_cast<uint4*>(Qs + buf * QT * LD + row * LD + cc) = rq[i];
        *reinterpret_cast<uint4*>(Gs + buf * QT * LD + row * LD + cc) = rg[i];
      }
    }
    if (tid < QT) ls[buf * QT + tid] = rl, ds[buf * QT + tid] = rd;
  };
  if (todo > 0) {
    load(r0);
    store(0);
  }
  __syncthreads();
  for (int t = 0; t < todo; ++t) {
    const int cur = t & 1;
    if (t + 1 < todo) load(r0 + (t + 1) * QT);
    const CT* Qc = Qs + cur * QT * LD;
    const CT* Gc = Gs + cur * QT * LD;
    f32x16 s, g;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = g[i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      s = mma<CT>(row_frag<CT, LD>(Qc, lane & 31, 16 * ks, lane), kf[ks], s);
      g = mma<CT>(row_frag<CT, LD>(Gc, lane & 31, 16 * ks, lane), vf[ks], g);
    }
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const float4 lv = *reinterpret_cast<const float4*>(ls + cur * QT + 8 * a + 4 * h);
      const float4 dl = *reinterpret_cast<const float4*>(ds + cur * QT + 8 * a + 4 * h);
      const float lw[4] = {lv.x, lv.y, lv.z, lv.w}, dw[4] = {dl.x, dl.y, dl.z, dl.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float pr = __builtin_amdgcn_exp2f(fmaf(s[4 * a + i], p.c, -lw[i]));
        s[4 * a + i] = pr;
        g[4 * a + i] = pr * (g[4 * a + i] - dw[i]);
      }
    }
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2) {
      const typename V8<CT>::T pf = half_frag<CT>(s, s2), df = half_frag<CT>(g, s2);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        dv[dt] = mma<CT>(col_frag<CT, LD>(Gc, 16 * s2, 32 * dt, lane), pf, dv[dt]);
        dk[dt] = mma<CT>(col_frag<CT, LD>(Qc, 16 * s2, 32 * dt, lane), df, dk[dt]);
      }
    }
    if (t + 1 < todo) store(cur ^ 1);
    __syncthreads();
  }
  if (key >= p.Nk) return;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int d0 = 32 * dt + 8 * a + 4 * h;
      float x[4], y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = live ? dk[dt][4 * a + i] * p.scale : 0.f, y[i] = live ? dv[dt][4 * a + i] : 0.f;
      if (p.nsplit > 1) {
        const long long total = (long long)p.B * p.Hk * p.Nk;
        const long long pr = ((long long)id.split * 2 * total + ((long long)id.b * p.Hk + id.hk) * p.Nk + key) * DP + d0;
        *reinterpret_cast<float4*>(p.part + pr) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(p.part + pr + total * DP) = make_float4(y[0], y[1], y[2], y[3]);
      } else {
        st_out<CT>(wrow<CT>(p.dk, id.b, key, id.hk), d0, p.D, p.vec, x[0], x[1], x[2], x[3]);
        st_out<CT>(wrow<CT>(p.dv, id.b, key, id.hk), d0, p.D, p.vec, y[0], y[1], y[2], y[3]);
      }
    }
}

// sums the splits' fp32 partials in order: nout planes [rows][DP] per split -> the strided outputs.
// kv: rows (b, hk, key), planes dk | dv; else rows (b, hk, n * G + g), dq scaled here.
template <typename CT, int DP>
__global__ __launch_bounds__(256) void cross_sum_kernel(const CrossP p, int kv) {
  constexpr int Q = DP / 4;
  const long long rows = kv ? (long long)p.Nk : (long long)p.Nq * p.G, total = rows * p.B * p.Hk;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long row = i / Q;
  const int d0 = (int)(i % Q) * 4, nout = kv ? 2 : 1;
  if (row >= total * nout) return;
  float4 v = make_float4(0, 0, 0, 0);
  for (int s = 0; s < p.nsplit; ++s) {
    const float4 t = *reinterpret_cast<const float4*>(p.part + (s * nout * total + row) * DP + d0);
    v.x += t.x, v.y += t.y, v.z += t.z, v.w += t.w;
  }
  const long long r0 = row % total;
  const int bh = (int)(r0 / rows), r = (int)(r0 % rows), b = bh / p.Hk, hk = bh % p.Hk;
  if (kv) {
    st_out<CT>(wrow<CT>(row < total ? p.dk : p.dv, b, r, hk), d0, p.D, p.vec, v.x, v.y, v.z, v.w);
  } else {
    st_out<CT>(wrow<CT>(p.dq, b, r / p.G, hk * p.G + r % p.G), d0, p.D, p.vec, v.x * p.scale, v.y * p.scale,
               v.z * p.scale, v.w * p.scale);
  }
}

// ------------------------------------------------------------------------------------------ host
int dp_of_head(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }

// Splits: enough blocks to fill 256 CUs several times over, none with less than `least` of the long axis.
int pick_split(long long blocks, long long len, int least, int want) {
  if (blocks <= 0 || blocks >= want || len <= least) return 1;
  const long long s = (want + blocks - 1) / blocks, most = (len + least - 1) / least;
  return (int)(s < most ? s : most);
}

template <typename F>
hipError_t allow_lds(F f, size_t bytes) {
  return bytes > 65536 ? hipFuncSetAttribute(reinterpret_cast<const void*>(f), hipFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)bytes)
                       : hipSuccess;
}

View view(const mdg_heads& t) { return View{t.p, t.sb, t.sn, t.sh}; }

bool aligned16(const mdg_heads& t, int e) {
  return !t.p || ((reinterpret_cast<uintptr_t>(t.p) | (uintptr_t)(t.sb * e) | (uintptr_t)(t.sn * e) | (uintptr_t)(t.sh * e)) & 15) == 0;
}

CrossP params(const mdg_attn_cross& a, bool bwd) {
  CrossP p;
  p.q = view(a.q), p.k = view(a.k), p.v = view(a.v), p.o = view(a.o), p.olo = view(a.o_lo);
  p.dout = view(a.dout), p.dq = view(a.dq), p.dk = view(a.dk), p.dv = view(a.dv);
  p.qlen = a.q_len, p.klen = a.kv_len, p.mask = a.mask, p.mask_f32 = a.mask_type == MDG_MASK_F32;
  p.mb = a.mask_sb, p.mn = a.mask_sn;
  p.B = a.B, p.Nq = a.Nq, p.Nk = a.Nk, p.H = a.H, p.Hk = a.Hk, p.G = a.H / a.Hk, p.D = a.D;
  p.c = a.scale * kLog2e, p.scale = a.scale, p.lse = a.lse;
  p.delta = nullptr, p.part = p.part_ml = nullptr, p.nsplit = 1;
  const int e = a.dtype == MDG_BF16 ? 2 : 4;
  p.vec = a.D % (16 / e) == 0 && aligned16(a.q, e) && aligned16(a.k, e) && aligned16(a.v, e) && aligned16(a.o, e) &&
          aligned16(a.o_lo, e);
  if (bwd) p.vec = p.vec && aligned16(a.dout, e) && aligned16(a.dq, e) && aligned16(a.dk, e) && aligned16(a.dv, e);
  return p;
}

struct Plan {
  bool few;
  long long tiles;
  int split;
  size_t part, ml, bytes;  // byte offsets / total
};
size_t al(size_t n) { return (n + 255) / 256 * 256; }

Plan fwd_plan(const mdg_attn_cross& a) {
  Plan w;
  const long long rows = (long long)a.Nq * (a.H / a.Hk), bh = (long long)a.B * a.Hk;
  w.few = rows <= 32;
  w.tiles = w.few ? 1 : (rows + 127) / 128;
  w.split = pick_split(w.tiles * bh, a.Nk, w.few ? 256 : 512, w.few ? 1024 : 512);
  w.part = 0, w.ml = w.bytes = 0;
  if (w.split > 1) {
    w.ml = al((size_t)w.split * rows * bh * dp_of_head(a.D) * 4);
    w.bytes = w.ml + al((size_t)w.split * rows * bh * 8);
  }
  return w;
}

struct BwdPlan {
  long long qtiles, ktiles;
  int qsplit, ksplit;  // splits of the dq pass (over keys) and of the dk / dv pass (over rows)
  size_t delta, part, bytes;
};
BwdPlan bwd_plan(const mdg_attn_cross& a) {
  BwdPlan w;
  const long long rows = (long long)a.Nq * (a.H / a.Hk), bh = (long long)a.B * a.Hk;
  w.qtiles = (rows + 127) / 128, w.ktiles = ((long long)a.Nk + 127) / 128;
  w.qsplit = pick_split(w.qtiles * bh, a.Nk, 512, 512);
  w.ksplit = pick_split(w.ktiles * bh, rows, 256, 512);
  w.delta = 0;
  w.part = al((size_t)a.B * a.H * a.Nq * 4);
  const size_t dp = dp_of_head(a.D);
  const size_t pq = w.qsplit > 1 ? (size_t)w.qsplit * rows * bh * dp * 4 : 0;
  const size_t pk = w.ksplit > 1 ? (size_t)w.ksplit * 2 * a.Nk * bh * dp * 4 : 0;
  w.bytes = w.part + al(pq > pk ? pq : pk);
  return w;
}

template <typename CT, int DP>
hipError_t fwd(const mdg_attn_cross& a, void* ws, hipStream_t s) {
  constexpr int KT = sizeof(CT) == 2 ? 64 : 32, LD = lds_ld<CT, DP>();
  const Plan w = fwd_plan(a);
  CrossP p = params(a, false);
  p.nsplit = w.split;
  if (w.split > 1) {
    p.part = reinterpret_cast<float*>(ws);
    p.part_ml = reinterpret_cast<float*>(static_cast<char*>(ws) + w.ml);
  }
  const unsigned grid = (unsigned)(w.tiles * w.split * a.B * a.Hk);
  hipError_t e;
  if (w.few) {
    const size_t stage = (size_t)4 * 2 * 32 * LD * sizeof(CT) + 4 * 32 * 4 + 16;
    const size_t join = (size_t)(288 + 128 * (DP + 4)) * 4, sm = stage > join ? stage : join;
    if ((e = allow_lds(cross_few_kernel<CT, DP>, sm)) != hipSuccess) return e;
    hipLaunchKernelGGL((cross_few_kernel<CT, DP>), dim3(grid), dim3(256), sm, s, p, 1);
  } else {
    const size_t sm = (size_t)4 * KT * LD * sizeof(CT) + 2 * KT * 4 + 16;
    if ((e = allow_lds(cross_fwd_kernel<CT, DP, KT>, sm)) != hipSuccess) return e;
    hipLaunchKernelGGL((cross_fwd_kernel<CT, DP, KT>), dim3(grid), dim3(256), sm, s, p, (int)w.tiles);
  }
  if (w.split > 1) {
    const long long total = (long long)a.B * a.H * a.Nq;
    hipLaunchKernelGGL((cross_join_kernel<CT, DP>), dim3((unsigned)((total + 7) / 8)), dim3(256), 0, s, p);
  }
  return hipGetLastError();
}

template <typename CT, int DP>
hipError_t bwd(const mdg_attn_cross& a, void* ws, hipStream_t s) {
  constexpr int KT = sizeof(CT) == 2 ? 64 : 32, LD = lds_ld<CT, DP>(), QT = 32;
  const BwdPlan w = bwd_plan(a);
  CrossP p = params(a, true);
  p.delta = reinterpret_cast<float*>(static_cast<char*>(ws) + w.delta);
  p.part = reinterpret_cast<float*>(static_cast<char*>(ws) + w.part);
  hipError_t e;
  const size_t smq = (size_t)4 * KT * LD * sizeof(CT) + 2 * KT * 4 + 16;
  const size_t smk = (size_t)4 * QT * LD * sizeof(CT) + 4 * QT * 4;
  if ((e = allow_lds(cross_dq_kernel<CT, DP, KT>, smq)) != hipSuccess) return e;
  if ((e = allow_lds(cross_dkv_kernel<CT, DP>, smk)) != hipSuccess) return e;
  p.nsplit = w.qsplit;
  hipLaunchKernelGGL((cross_dq_kernel<CT, DP, KT>), dim3((unsigned)(w.qtiles * w.qsplit * a.B * a.Hk)), dim3(256), smq, s, p,
                     (int)w.qtiles);
  if (w.qsplit > 1) {
    const long long n = (long long)a.B * a.H * a.Nq * (DP / 4);
    hipLaunchKernelGGL((cross_sum_kernel<CT, DP>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, p, 0);
  }
  if (!a.dk.p || a.Nk == 0) return hipGetLastError();  // a frozen encoder, or none
  p.nsplit = w.ksplit;
  hipLaunchKernelGGL((cross_dkv_kernel<CT, DP>), dim3((unsigned)(w.ktiles * w.ksplit * a.B * a.Hk)), dim3(256), smk, s, p,
                     (int)w.ktiles);
  if (w.ksplit > 1) {
    const long long n = (long long)a.B * a.Hk * a.Nk * 2 * (DP / 4);
    hipLaunchKernelGGL((cross_sum_kernel<CT, DP>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, p, 1);
  }
  return hipGetLastError();
}

template <typename CT>
hipError_t by_head(const mdg_attn_cross& a, bool back, void* ws, hipStream_t s) {
  switch (dp_of_head(a.D)) {
    case 32: return back ? bwd<CT, 32>(a, ws, s) : fwd<CT, 32>(a, ws, s);
    case 64: return back ? bwd<CT, 64>(a, ws, s) : fwd<CT, 64>(a, ws, s);
    default: return back ? bwd<CT, 128>(a, ws, s) : fwd<CT, 128>(a, ws, s);
  }
}

}  // namespace

size_t attn_cross_ws_bytes(const mdg_attn_cross& a, bool back) { return back ? bwd_plan(a).bytes : fwd_plan(a).bytes; }

// grid sizes of every launch, for the host-side check (each must stay below 2^31)
bool attn_cross_grid_ok(const mdg_attn_cross& a, bool back) {
  const long long lim = (1LL << 31) - 1, bh = (long long)a.B * a.Hk, dp4 = dp_of_head(a.D) / 4;
  const long long rows = (long long)a.Nq * (a.H / a.Hk);
  if (rows > lim || rows * bh > lim || (long long)a.Nk * bh > lim) return false;
  if (!back) {
    const Plan w = fwd_plan(a);
    return w.tiles * w.split * bh <= lim;
  }
  const BwdPlan w = bwd_plan(a);
  return w.qtiles * w.qsplit * bh <= lim && w.ktiles * w.ksplit * bh <= lim && rows * bh * dp4 / 256 < lim &&
         (long long)a.Nk * bh * 2 * dp4 / 256 < lim;
}

hipError_t attn_cross_launch(const mdg_attn_cross& a, bool back, void* ws, hipStream_t s) {
  return a.dtype == MDG_BF16 ? by_head<bf16_t>(a, back, ws, s) : by_head<float>(a, back, ws, s);
}

}  // namespace mdg
