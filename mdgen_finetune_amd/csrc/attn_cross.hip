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
//
// What rounds: with bf16 inputs P and dS go to bf16 as operands of their second products (half a step of
// 2^-8 each, the type of v and k beside them); scores, statistics, sums and every accumulator are fp32.
// delta is formed with o + o_lo, o's own rounding residual: dP - delta cancels, and o's rounding would show.
#include "../../include/mdgen_hip.h"
#include "common.h"

#include <cfloat>
#include <cmath>
#include <initializer_list>
#include <type_traits>

namespace mdg {
namespace {

typedef __attribute__((ext_vector_type(16))) float f32x16;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNoMax = -FLT_MAX;  // running maximum before the first key

struct View {  // element strides of batch, token, head; the head dim is contiguous
  const void* p;
  long long sb, sn, sh;
};
// n / d for 0 <= n < 2^31 by one multiplication (d >= 1): mul = floor(2^32 (2^shift - d) / d) + 1 with
// shift = ceil(log2 d); the sum below stays under 2^32
struct Divisor {
  unsigned mul, shift;
};
inline Divisor divisor(long long d) {
  unsigned s = 0;
  while ((1LL << s) < d) ++s;
  return Divisor{(unsigned)((((1ULL << s) - (unsigned long long)d) << 32) / (unsigned long long)d + 1), s};
}
__device__ __forceinline__ int quot(int n, const Divisor& d) { return (int)((__umulhi((unsigned)n, d.mul) + (unsigned)n) >> d.shift); }

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
  Divisor by_g, by_hk, by_split, by_tiles, by_rows;
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

// LDS tiles are rows of DP elements without padding (what an asynchronous load can fill: a wave writes
// 1024 consecutive bytes); the 16-byte chunk c of row r lies at chunk c ^ chunk_xor(r).  The XOR puts
// the 8 rows that one pass of a 16-byte row read covers, and the 4 rows of a transposing read, on
// different banks.
template <typename CT, int DP>
__device__ __forceinline__ int chunk_xor(int r) {
  if constexpr (sizeof(CT) == 2) {
    if constexpr (DP >= 128) return ((r & 3) << 2) | ((r >> 2) & 3);
    else if constexpr (DP == 64) return ((r & 2) << 1) | ((r >> 2) & 3);
    else return (r >> 2) & 3;
  } else {
    if constexpr (DP >= 64) return (r & 3) | ((r & 4) << 1);
    else return (r >> 1) & 7;
  }
}
// element offset of chunk c of row r
template <typename CT, int DP>
__device__ __forceinline__ int lds_at(int r, int c) {
  return r * DP + (c ^ chunk_xor<CT, DP>(r)) * (16 / (int)sizeof(CT));
}

// element j: tile[k0 + 8 (j >> 2) + 4h + (j & 3)][c0 + (lane & 31)]
template <typename CT, int DP>
__device__ __forceinline__ typename V8<CT>::T col_frag(const CT* tile, int k0, int c0, int lane) {
  typename V8<CT>::T r;
  const int h = lane >> 5;
  if constexpr (is_bf16<CT>()) {
    // ds_read_b64_tr_b16: in each group of 16 lanes, lane 4q + p supplies columns 4p..4p+3 of row q and
    // receives column (lane & 15) of the four rows
    typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;
    const int row = k0 + 4 * h + ((lane & 15) >> 2), c = c0 / 8 + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), e = 4 * (lane & 1);
    const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(tile + lds_at<CT, DP>(row, c) + e));
    const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(tile + lds_at<CT, DP>(row + 8, c) + e));
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = lo[j], r[4 + j] = hi[j];
  } else {
    const int c = (c0 + (lane & 31)) / 4, e = lane & 3;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = tile[lds_at<CT, DP>(k0 + 8 * (j >> 2) + 4 * h + (j & 3), c) + e];
  }
  return r;
}

template <typename CT, int DP>
__device__ __forceinline__ typename V8<CT>::T row_frag(const CT* tile, int row, int k0, int lane) {
  const int c = (k0 + 8 * (lane >> 5)) * (int)sizeof(CT) / 16;
  if constexpr (is_bf16<CT>()) {
    return *reinterpret_cast<const bf16x8*>(tile + lds_at<CT, DP>(row, c));
  } else {
    const f32x4 a = *reinterpret_cast<const f32x4*>(tile + lds_at<CT, DP>(row, c));
    const f32x4 b = *reinterpret_cast<const f32x4*>(tile + lds_at<CT, DP>(row, c + 1));
    f32x8 r;
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = a[j], r[4 + j] = b[j];
    return r;
  }
}

// one 16-byte piece (columns c0 .., c0 < D) of a row of D elements, zero past D.  VEC: D is a multiple of a
// piece and every base and stride is 16-byte aligned; otherwise element by element.
template <typename CT, bool VEC>
__device__ __forceinline__ uint4 ld_piece(const CT* row, int c0, int D) {
  constexpr int N = 16 / sizeof(CT);
  uint4 r = make_uint4(0, 0, 0, 0);
  if constexpr (VEC) {
    r = *reinterpret_cast<const uint4*>(row + c0);
  } else {
    CT e[N];
#pragma unroll
    for (int j = 0; j < N; ++j) e[j] = c0 + j < D ? row[c0 + j] : (CT)0.f;
    __builtin_memcpy(&r, e, 16);
  }
  return r;
}
template <typename CT, bool VEC>
__device__ __forceinline__ typename V8<CT>::T ld_frag(const CT* row, int c0, int D) {
  typename V8<CT>::T r;
  constexpr int N = 16 / sizeof(CT);
#pragma unroll
  for (int j = 0; j < 8; j += N) {
    const uint4 u = c0 + j < D ? ld_piece<CT, VEC>(row, c0 + j, D) : make_uint4(0, 0, 0, 0);
    CT e[N];
    __builtin_memcpy(e, &u, 16);
#pragma unroll
    for (int i = 0; i < N; ++i) r[j + i] = e[i];
  }
  return r;
}

// and back: the columns c0 .. (c0 < D) of a row
template <typename CT, bool VEC>
__device__ __forceinline__ void st_piece(CT* row, int c0, int D, const uint4& u) {
  constexpr int N = 16 / sizeof(CT);
  if constexpr (VEC) {
    *reinterpret_cast<uint4*>(row + c0) = u;
  } else {
    CT e[N];
    __builtin_memcpy(e, &u, 16);
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (c0 + j < D) row[c0 + j] = e[j];
  }
}

// four consecutive outputs d0 .. d0 + 3 of a row
template <typename CT, bool VEC>
__device__ __forceinline__ void st_out(CT* row, int d0, int D, float a, float b, float c, float d) {
  if constexpr (VEC) {
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


// The softmax of NT 32-key tiles: raises the lane's maximum when a score outgrows it by 2^8 (a lagging
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
  mx = other_half_max(mx);
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

// Asynchronous loads, memory -> LDS, 16 bytes per lane at lds + 16 * lane.  Offsets outside the
// resource's bytes read zeros, so a lane whose piece is not there is sent out of range.  (In assembly:
// for the builtin the compiler waits for every such load before any later LDS read.  There is no
// register result; async_wait below comes before the barrier after which the tile is read.)
constexpr unsigned kNowhere = 0x80000000u;
__device__ __forceinline__ u32x4 resource(uint64_t base, unsigned bytes) {
  u32x4 r;
  r[0] = (unsigned)base, r[1] = (unsigned)(base >> 32) & 0xffffu, r[2] = bytes, r[3] = 0x00020000u;
  return r;
}
__device__ __forceinline__ uint64_t uniform64(uint64_t v) {
  // (readfirstlane gives an int: the low word must not be widened with its sign)
  return ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) |
         (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v);
}
__device__ __forceinline__ unsigned lds_address(const void* p) {
  return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}
// (m0 is written right before each use, by the compiler too.  Five wait states before the load, which
// the compiler does not count into assembly: the vector unit may just have written the resource's
// scalar registers.)
__device__ __forceinline__ void async_load16(const u32x4& res, unsigned lds, unsigned off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(off), "s"(res)
               : "memory");
}
// all but this wave's N youngest loads have landed
template <int N = 0>
__device__ __forceinline__ void async_wait() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// k and v tiles of ROWS keys of one (b, key head), by NT threads.  Masked keys' rows are zero in LDS (what
// lies there, NaN too, never reaches a product) and their scores start at -inf: kb holds 0 or
// -inf per key and is the products' initial accumulator; a tile whose keys are all there (flag 0) skips that.
//   begin(key0): starts the tile (ASYNC: straight into LDS; else into registers)
//   finish(...): completes it in LDS; the caller's barrier follows
// Tiles come in order, `step` keys apart, init with the first.
template <typename CT, int DP, int ROWS, int NT, bool VEC, bool ASYNC>
struct KvStage {
  static constexpr int N = 16 / sizeof(CT), CPR = DP / N, P = ROWS * CPR / NT;
  static_assert(ROWS * CPR % NT == 0 && ROWS <= 64, "whole pieces per thread");
  uint4 k[ASYNC ? 1 : P], v[ASYNC ? 1 : P];
  unsigned ko[ASYNC ? P : 1], vo[ASYNC ? P : 1];  // byte offsets of this thread's pieces in a tile
  bool keep[P];  // ASYNC: of the tile to begin next; else of the begun one
  float kb;
  const CT *kp, *vp;           // the tile's first row
  uint64_t ka, va;             // ASYNC: its address, and the strides from tile to tile, in bytes
  int64_t kstep, vstep;
  unsigned first;              // ASYNC: this wave's first slot in a tile, in bytes
  // ASYNC: piece i is slot (wave * P + i) * 64 + lane of the tile's 16-byte slots; else i * NT + tid
  __device__ __forceinline__ static int slot(int i, int tid) {
    return ASYNC ? ((tid >> 6) * P + i) * 64 + (tid & 63) : i * NT + tid;
  }
  __device__ __forceinline__ void init(const CrossP& p, int b, int hk, int key0, int end, int step, int tid) {
    kp = vrow<CT>(p.k, b, key0, hk);
    vp = vrow<CT>(p.v, b, key0, hk);
    if constexpr (ASYNC) {
      ka = uniform64((uint64_t)kp), va = uniform64((uint64_t)vp);
      kstep = step * p.k.sn * (int)sizeof(CT), vstep = step * p.v.sn * (int)sizeof(CT);
      first = __builtin_amdgcn_readfirstlane(tid >> 6) * P * 1024;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const int row = slot(i, tid) / CPR, c = slot(i, tid) % CPR ^ chunk_xor<CT, DP>(row);
        ko[i] = c * N < p.D ? (unsigned)(row * p.k.sn * sizeof(CT)) + c * 16 : kNowhere;
        vo[i] = c * N < p.D ? (unsigned)(row * p.v.sn * sizeof(CT)) + c * 16 : kNowhere;
      }
    }
    if constexpr (ASYNC) look(p, b, key0, end, tid);
  }
  __device__ __forceinline__ void look(const CrossP& p, int b, int key0, int end, int tid) {
    if (!p.mask) return;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int key = key0 + slot(i, tid) / CPR;
      keep[i] = key < end && key_kept(p, b, key);
    }
  }
  __device__ __forceinline__ void begin(const CrossP& p, CT* Ks, CT* Vs, int b, int key0, int end, int step, int tid) {
    const int here = min(ROWS, end - key0);
    if constexpr (ASYNC) {
      const u32x4 kr = resource(ka, (unsigned)(((here - 1) * p.k.sn + p.D) * (int)sizeof(CT)));
      const u32x4 vr = resource(va, (unsigned)(((here - 1) * p.v.sn + p.D) * (int)sizeof(CT)));
      const unsigned kl = lds_address(Ks) + first, vl = lds_address(Vs) + first;
      if (p.mask) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
          async_load16(kr, kl + i * 1024, keep[i] ? ko[i] : kNowhere);
          async_load16(vr, vl + i * 1024, keep[i] ? vo[i] : kNowhere);
        }
      } else {
#pragma unroll
        for (int i = 0; i < P; ++i) {
          async_load16(kr, kl + i * 1024, ko[i]);
          async_load16(vr, vl + i * 1024, vo[i]);
        }
      }
      ka += kstep, va += vstep;
    } else {
      look(p, b, key0, end, tid);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const int row = slot(i, tid) / CPR, cc = slot(i, tid) % CPR * N;
        const bool in = row < here && cc < p.D;
        k[i] = in ? ld_piece<CT, VEC>(kp + row * p.k.sn, cc, p.D) : make_uint4(0, 0, 0, 0);
        v[i] = in ? ld_piece<CT, VEC>(vp + row * p.v.sn, cc, p.D) : make_uint4(0, 0, 0, 0);
      }
    }
    if constexpr (!ASYNC) kp += step * p.k.sn, vp += step * p.v.sn;
    kb = 0.f;
    if (p.mask || here < ROWS) {  // (uniform)
      if (tid < ROWS) kb = tid < here && key_kept(p, b, key0 + tid) ? 0.f : -INFINITY;
      if constexpr (ASYNC) look(p, b, key0 + step, end, tid);
    }
  }
  __device__ __forceinline__ void finish_rows(const CrossP& p, CT* Ks, CT* Vs, int tid) {
    if constexpr (!ASYNC) {
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const int at = lds_at<CT, DP>(slot(i, tid) / CPR, slot(i, tid) % CPR);
        const bool drop = p.mask && !keep[i];
        *reinterpret_cast<uint4*>(Ks + at) = drop ? make_uint4(0, 0, 0, 0) : k[i];
        *reinterpret_cast<uint4*>(Vs + at) = drop ? make_uint4(0, 0, 0, 0) : v[i];
      }
    }
  }
  __device__ __forceinline__ void finish_kb(float* kbs, int* flag, int tid) {
    if (tid < 64) {
      if (tid < ROWS) kbs[tid] = kb;
      const bool any = __any(kb != 0.f);
      if (tid == 0) *flag = any;
    }
  }
  __device__ __forceinline__ void finish(const CrossP& p, CT* Ks, CT* Vs, float* kbs, int* flag, int tid) {
    finish_rows(p, Ks, Vs, tid);
    finish_kb(kbs, flag, tid);
    if constexpr (ASYNC) async_wait();
  }
};

// initial accumulator of a 32-key tile of S^T with keys that are not there: their kb (rows 8a + 4h + i)
__device__ __forceinline__ f32x16 kb_init(const float* kbs, int lane) {
  f32x16 s;
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    const float4 t = *reinterpret_cast<const float4*>(kbs + 8 * a + 4 * (lane >> 5));
    s[4 * a] = t.x, s[4 * a + 1] = t.y, s[4 * a + 2] = t.z, s[4 * a + 3] = t.w;
  }
  return s;
}
__device__ __forceinline__ f32x16 zero16() {
  f32x16 s;
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = 0.f;
  return s;
}

// A product's steps of 16 past D are zeros.  fp32, eight MFMA of 64 cycles each, leaves them out; for bf16,
// one of 32 cycles, the branches would cost more than they save.
template <typename CT, int DP>
__device__ __forceinline__ bool step_there(int ks, int D) {
  return is_bf16<CT>() || 32 * ks < DP || 16 * ks < D;  // (D > DP / 2, or DP is 32 and D > 0)
}

// S^T of a tile of NT * 32 keys.  (The products stand in both branches: an accumulator that is one of two
// things would be copied, one that starts at a literal zero is not.)
template <typename CT, int DP, int NT>
__device__ __forceinline__ void key_scores(f32x16 (&s)[NT], const CT* Kt, const typename V8<CT>::T (&qf)[DP / 16],
                                           const float* kbs, bool holes, int D, int lane) {
  if (holes) {
#pragma unroll
    for (int kt = 0; kt < NT; ++kt) {
      s[kt] = kb_init(kbs + 32 * kt, lane);
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks)
        if (step_there<CT, DP>(ks, D)) s[kt] = mma<CT>(row_frag<CT, DP>(Kt, 32 * kt + (lane & 31), 16 * ks, lane), qf[ks], s[kt]);
    }
  } else {
#pragma unroll
    for (int kt = 0; kt < NT; ++kt) {
      s[kt] = zero16();
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks)
        if (step_there<CT, DP>(ks, D)) s[kt] = mma<CT>(row_frag<CT, DP>(Kt, 32 * kt + (lane & 31), 16 * ks, lane), qf[ks], s[kt]);
    }
  }
}

template <typename CT>
__device__ __forceinline__ typename V8<CT>::T half_frag(const f32x16& s, int s2) {
  typename V8<CT>::T r;
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = (CT)s[8 * s2 + j];
  return r;
}

// keys [k0, k1) of split `sp`: the sequence's own length shared out in multiples of 32 (k0 + per may pass 31 bits)
__device__ __forceinline__ void split_range(const CrossP& p, int klen, int sp, int& k0, int& k1) {
  const int per = (quot(klen + p.nsplit - 1, p.by_split) + 31) / 32 * 32;
  k0 = min(klen, sp * per);
  k1 = k0 + min(klen - k0, per);
}

struct BlockId {
  int tile, split, b, hk;
};
__device__ __forceinline__ BlockId block_id(const CrossP& p, int tiles) {
  BlockId r;
  int id = blockIdx.x, q = quot(id, p.by_tiles);
  r.tile = id - q * tiles;
  id = q, q = quot(id, p.by_split);
  r.split = id - q * p.nsplit;
  r.b = quot(q, p.by_hk);
  r.hk = q - r.b * p.Hk;
  return r;
}
// packed row r: token n, query head g of the key head's G
struct PackedRow {
  int n, g;
};
__device__ __forceinline__ PackedRow packed(const CrossP& p, int r) {
  const int n = quot(r, p.by_g);
  return PackedRow{n, r - n * p.G};
}

// rows of partial `sp`: ((b * Hk + hk) * rows + r), rows = Nq * G
__device__ __forceinline__ long long part_row(const CrossP& p, int sp, int b, int hk, int r) {
  const long long rows = (long long)p.Nq * p.G;
  return ((long long)sp * p.B * p.Hk + (long long)b * p.Hk + hk) * rows + r;
}

// Where a mask leaves no key the sums are 0, but -inf + 0 q is NaN for a query that is not finite.  So a wave that
// ends with a NaN looks over the mask of its keys [k0, k1); others pay nothing (a flag kept in the loop cost 2 % at D = 24).
__device__ __forceinline__ bool no_key(const CrossP& p, int b, int k0, int k1, bool nan, int lane) {
  if (!p.mask || !__any(nan)) return false;
  for (int key = k0; key < k1; key += 64)
    if (__any(key + lane < k1 && key_kept(p, b, key + lane))) return false;
  return true;
}
// Scores past fp32 once scaled: a maximum was seen and yet every P is exp2(-inf).  NaN, not a row without keys.
__device__ __forceinline__ float sum_in_range(float m, float l) { return l == 0.f && m != kNoMax ? __builtin_nanf("") : l; }
template <int DT>
__device__ __forceinline__ bool has_nan(const f32x16 (&x)[DT]) {
  bool r = false;
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) r |= x[t][i] != x[t][i];
  return r;
}

// a lane's row of outputs, O^T rows 32 dt + 8a + 4h + i: normalised, or a split's partial
template <typename CT, int DP, bool VEC>
__device__ __forceinline__ void store_rows(const CrossP& p, const BlockId& id, int r, int rows, bool live,
                                           const f32x16* o, float m, float l, int lane) {
  constexpr int DT = DP / 32;
  const int h = lane >> 5;
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
  const PackedRow pk = packed(p, r);
  const int n = pk.n, head = id.hk * p.G + pk.g;
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
      st_out<CT, VEC>(orow, d0, p.D, v[0], v[1], v[2], v[3]);
      if (lrow)  // the rounding residual of o, for an exact delta in the backward
        st_out<CT, VEC>(lrow, d0, p.D, v[0] - (float)(CT)v[0], v[1] - (float)(CT)v[1], v[2] - (float)(CT)v[2],
                        v[3] - (float)(CT)v[3]);
    }
}

// ------------------------------------------------------------------------------------------ forward
// One block = 4 waves x 32 rows of one (b, key head), tiles of KT keys through two LDS buffers, one barrier per
// tile; a tile's loads run under the products of the one before.  The running maximum and sum make it one
// pass; no score is stored.
// Narrow heads are bound by the vector unit (per 32 x 32 tile about 320 cycles of max, fma, exp, add and
// convert against 128 of MFMA at D <= 32): [8, 4000, 16, 24] on 256 keys takes 48 us alone, 42 in a row of passes whose
// ends overlap; 27 of them grow with the keys and 10 are its 51 MB.  D = 64, [4, 4096, 16] on 2048 ragged keys (110
// GFLOP): 139-144 us, 770 TFLOP/s.
// Tried: two row groups per wave (the registers cost a wave per SIMD: 700 against 610 us at D = 128), 32-key
// tiles (697), all keys in LDS with waves walking the rows (46 -> 42 us masked, equal unmasked, and
// 37 -> 47 at D = 64 with 64 keys), row sums by a product with ones (1-2 % slower).
template <typename CT, int DP, int KT, bool VEC>
__global__ __launch_bounds__(256, 2) void cross_fwd_kernel(const CrossP p, int tiles) {
  constexpr int TILE = KT * DP, DT = DP / 32, KS = DP / 16, NT = KT / 32;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  CT* Ks = reinterpret_cast<CT*>(smem);
  CT* Vs = Ks + 2 * TILE;
  float* kbs = reinterpret_cast<float*>(Vs + 2 * TILE);
  int* flag = reinterpret_cast<int*>(kbs + 2 * KT);

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const BlockId id = block_id(p, tiles);
  const int rows = p.Nq * p.G, r = id.tile * 128 + wave * 32 + (lane & 31);
  const PackedRow pk = packed(p, r);
  const int n = pk.n, head = id.hk * p.G + pk.g;
  const int qlen = clamp_len(p.qlen, id.b, p.Nq), klen = clamp_len(p.klen, id.b, p.Nk);
  const bool live = r < rows && n < qlen;

  typename V8<CT>::T qf[KS];
  const CT* qrow = vrow<CT>(p.q, id.b, live ? n : 0, live ? head : 0);
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) qf[ks] = live ? ld_frag<CT, VEC>(qrow, 16 * ks + 8 * h, p.D) : zero8<CT>();

  f32x16 o[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) o[t] = zero16();
  float m = kNoMax, l = 0.f;

  int k0, k1;
  split_range(p, klen, id.split, k0, k1);
  KvStage<CT, DP, KT, 256, VEC, VEC> st;
  const int nt = (k1 - k0 + KT - 1) / KT;
  const bool busy = id.tile * 128 + wave * 32 < qlen * p.G;  // (otherwise the wave has no row, and only loads)
  if (nt > 0) {
    st.init(p, id.b, id.hk, k0, k1, KT, tid);
    st.begin(p, Ks, Vs, id.b, k0, k1, KT, tid);
    st.finish(p, Ks, Vs, kbs, flag, tid);
  }
  __syncthreads();
  for (int t = 0; t < nt; ++t) {
    const int cur = t & 1;
    const int other = (cur ^ 1) * TILE;
    if (t + 1 < nt) st.begin(p, Ks + other, Vs + other, id.b, k0 + (t + 1) * KT, k1, KT, tid);
    const CT* Kc = Ks + cur * TILE;
    const CT* Vc = Vs + cur * TILE;
    if (busy) {
      f32x16 s[NT];
      key_scores<CT, DP, NT>(s, Kc, qf, kbs + cur * KT, __builtin_amdgcn_readfirstlane(flag[cur]), p.D, lane);
      softmax_tile<NT, DT>(s, o, m, l, p.c);
#pragma unroll
      for (int kt = 0; kt < NT; ++kt)
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) {
          const typename V8<CT>::T pf = half_frag<CT>(s[kt], s2);
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
            o[dt] = mma<CT>(col_frag<CT, DP>(Vc, 32 * kt + 16 * s2, 32 * dt, lane), pf, o[dt]);
        }
    }
    if (t + 1 < nt) st.finish(p, Ks + other, Vs + other, kbs + (cur ^ 1) * KT, flag + (cur ^ 1), tid);
    __syncthreads();
  }

  l = sum_in_range(m, other_half_sum(l));
  if (no_key(p, id.b, k0, k1, l != l, lane)) {
    m = kNoMax, l = 0.f;
#pragma unroll
    for (int t = 0; t < DT; ++t) o[t] = zero16();
  }
  store_rows<CT, DP, VEC>(p, id, r, rows, live, o, m, l, lane);
}

// The same with two groups of four waves (256 rows per block), one phase apart, each SIMD holding one wave
// of either group: while one group's waves run their matrix products (M), the other's run their softmax
// (V), and a barrier ends every phase.  (Left to themselves, waves of equal code drift into step and the
// matrix cores and the vector unit take turns.)
//   M(t): O += V(t-1)^T P(t-1), S = K(t) Q^T;   V(t): P(t) = softmax of S
// Group 0 loads: K(t+1) and V(t+1) start at its M(t) and are awaited at the end of its V(t); K lies in two
// buffers, V, read a phase later, in three.
// [2, 4096, 16, 128] on 4 heads of 8192 keys: 511-528 us, 1040-1075 TFLOP/s (592 us with the kernel above; a large
// library product reaches 1130-1165).  For D <= 64 it is no faster (654 against 654 us of training at D = 64, 51 against 52
// at D = 24): fewer MFMA per score leave too little to run under the other phase.
template <int DP, int KT>
__global__ __launch_bounds__(512, 2) void cross_fwd_pp_kernel(const CrossP p, int tiles) {
  using CT = bf16_t;
  constexpr int TILE = KT * DP, DT = DP / 32, KS = DP / 16, NT = KT / 32;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  CT* Ks = reinterpret_cast<CT*>(smem);
  CT* Vs = Ks + 2 * TILE;
  float* kbs = reinterpret_cast<float*>(Vs + 3 * TILE);
  int* flag = reinterpret_cast<int*>(kbs + 2 * KT);

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const bool second = wave >= 4;
  const BlockId id = block_id(p, tiles);
  const int rows = p.Nq * p.G, r = id.tile * 256 + wave * 32 + (lane & 31);
  const PackedRow pk = packed(p, r);
  const int n = pk.n, head = id.hk * p.G + pk.g;
  const int qlen = clamp_len(p.qlen, id.b, p.Nq), klen = clamp_len(p.klen, id.b, p.Nk);
  const bool live = r < rows && n < qlen;

  bf16x8 qf[KS];
  const CT* qrow = vrow<CT>(p.q, id.b, live ? n : 0, live ? head : 0);
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) qf[ks] = live ? ld_frag<CT, true>(qrow, 16 * ks + 8 * h, p.D) : zero8<CT>();
  f32x16 o[DT], s[NT];
#pragma unroll
  for (int t = 0; t < DT; ++t) o[t] = zero16();
  float m = kNoMax, l = 0.f;
  bf16x8 pf[NT][2];

  int k0, k1;
  split_range(p, klen, id.split, k0, k1);
  KvStage<CT, DP, KT, 256, true, true> st;
  const int nt = (k1 - k0 + KT - 1) / KT;
  if (nt > 0 && !second) {
    st.init(p, id.b, id.hk, k0, k1, KT, tid);
    st.begin(p, Ks, Vs, id.b, k0, k1, KT, tid);
    st.finish(p, Ks, Vs, kbs, flag, tid);
  }
  __syncthreads();
  if (second) __syncthreads();
  int vprev = 0, vnext = 1;  // buffers of V(t-1) and V(t+1)
  for (int t = 0; t <= nt; ++t) {
    const bool loads = !second && t + 1 < nt;
    if (loads) st.begin(p, Ks + ((t + 1) & 1) * TILE, Vs + vnext * TILE, id.b, k0 + (t + 1) * KT, k1, KT, tid);
    if (t > 0) {
#pragma unroll
      for (int kt = 0; kt < NT; ++kt)
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
            o[dt] = mma<CT>(col_frag<CT, DP>(Vs + vprev * TILE, 32 * kt + 16 * s2, 32 * dt, lane), pf[kt][s2], o[dt]);
      vprev = vprev == 2 ? 0 : vprev + 1;
    }
    if (t < nt)
      key_scores<CT, DP, NT>(s, Ks + (t & 1) * TILE, qf, kbs + (t & 1) * KT, __builtin_amdgcn_readfirstlane(flag[t & 1]), p.D, lane);
    __syncthreads();
    if (t < nt) {
      softmax_tile<NT, DT>(s, o, m, l, p.c);
#pragma unroll
      for (int kt = 0; kt < NT; ++kt) pf[kt][0] = half_frag<CT>(s[kt], 0), pf[kt][1] = half_frag<CT>(s[kt], 1);
    }
    if (loads) st.finish(p, Ks, Vs, kbs + ((t + 1) & 1) * KT, flag + ((t + 1) & 1), tid);
    vnext = vnext == 2 ? 0 : vnext + 1;
    __syncthreads();
  }
  if (!second) __syncthreads();
  l = sum_in_range(m, other_half_sum(l));
  if (no_key(p, id.b, k0, k1, l != l, lane)) {
    m = kNoMax, l = 0.f;
#pragma unroll
    for (int t = 0; t < DT; ++t) o[t] = zero16();
  }
  store_rows<CT, DP, true>(p, id, r, rows, live, o, m, l, lane);
}

// At most 32 rows per (b, key head), the single-token form: the 4 waves split the keys instead of
// the rows.  Each wave stages its own 32-key tiles in two buffers of its own (no block barrier in the
// loop: a wave's LDS operations are in order), and the four partial softmaxes are joined in LDS at the end.
// Bound by memory, for which the splits keep four blocks per CU in flight: 16 sequences of one token, 32 heads
// on 8 of 16384 keys (ragged, 806 MB) take 151 us (5.3 TB/s) and 4.5 of the join.  One short sequence: 4.6 us, a launch.
// (fp32 at 128 columns: two buffers per wave would not fit, it stages through registers)
template <typename CT, int DP, bool VEC>
constexpr bool few_async() { return VEC && sizeof(CT) * DP <= 256; }
template <typename CT, int DP, bool VEC>
__global__ __launch_bounds__(256) void cross_few_kernel(const CrossP p, int tiles) {
  constexpr int TILE = 32 * DP, DT = DP / 32, KS = DP / 16, LO = DP + 4, BUFS = few_async<CT, DP, VEC>() ? 2 : 1;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  CT* Ks = reinterpret_cast<CT*>(smem) + wave * 2 * BUFS * TILE;
  CT* Vs = Ks + BUFS * TILE;
  float* kbs = reinterpret_cast<float*>(reinterpret_cast<CT*>(smem) + 4 * 2 * BUFS * TILE) + wave * 32;
  int* flag = reinterpret_cast<int*>(reinterpret_cast<float*>(reinterpret_cast<CT*>(smem) + 4 * 2 * BUFS * TILE) + 128) + wave;

  const BlockId id = block_id(p, tiles);
  const int rows = p.Nq * p.G, r = lane & 31;
  const PackedRow pk = packed(p, r);
  const int n = pk.n, head = id.hk * p.G + pk.g;
  const int qlen = clamp_len(p.qlen, id.b, p.Nq), klen = clamp_len(p.klen, id.b, p.Nk);
  const bool live = r < rows && n < qlen;
  typename V8<CT>::T qf[KS];
  f32x16 o[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) o[t] = zero16();
  float m = kNoMax, l = 0.f;

  int k0, k1;
  split_range(p, klen, id.split, k0, k1);
  using S = KvStage<CT, DP, 32, 64, VEC, BUFS == 2>;
  S st;
  int key = k0 + 32 * wave, cur = 0;
  if (key < k1) {
    st.init(p, id.b, id.hk, key, k1, 128, lane);
    st.begin(p, Ks, Vs, id.b, key, k1, 128, lane);
  }
  const CT* qrow = vrow<CT>(p.q, id.b, live ? n : 0, live ? head : 0);
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) qf[ks] = live ? ld_frag<CT, VEC>(qrow, 16 * ks + 8 * h, p.D) : zero8<CT>();
  for (; key < k1; key += 128) {
    st.finish_kb(kbs, flag, lane);
    const bool more = key + 128 < k1;
    if constexpr (BUFS == 2) {
      if (more) {
        st.begin(p, Ks + (cur ^ 1) * TILE, Vs + (cur ^ 1) * TILE, id.b, key + 128, k1, 128, lane);
        async_wait<2 * S::P>();  // this tile's loads, not the next one's
      } else {
        async_wait();
      }
    } else {
      st.finish_rows(p, Ks, Vs, lane);
      if (more) st.begin(p, Ks, Vs, id.b, key + 128, k1, 128, lane);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    f32x16 s[1];
    key_scores<CT, DP, 1>(s, Ks + cur * TILE, qf, kbs, __builtin_amdgcn_readfirstlane(*flag), p.D, lane);
    softmax_tile<1, DT>(s, o, m, l, p.c);
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2) {
      const typename V8<CT>::T pf = half_frag<CT>(s[0], s2);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] = mma<CT>(col_frag<CT, DP>(Vs + cur * TILE, 16 * s2, 32 * dt, lane), pf, o[dt]);
    }
    // the next turn's loads overwrite this buffer: its reads are done before they start
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    if constexpr (BUFS == 2) cur ^= 1;
  }
  l = sum_in_range(m, other_half_sum(l));
  if (no_key(p, id.b, k0, k1, l != l, lane)) {
    m = kNoMax, l = 0.f;
#pragma unroll
    for (int t = 0; t < DT; ++t) o[t] = zero16();
  }

  // join: [4][32] maxima and sums, then the rescaled outputs [4][32][DP + 4] over the staging area
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the last tile's reads are done
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
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
      const PackedRow pr = packed(p, row);
      const int rn = pr.n, rh = id.hk * p.G + pr.g;
      const float Lr = js[row];
      const bool some = rn < qlen && Lr != 0.f;
      const float inv = some ? 1.0f / Lr : 0.f;
      v = some ? make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv) : make_float4(0, 0, 0, 0);
      st_out<CT, VEC>(wrow<CT>(p.o, id.b, rn, rh), d0, p.D, v.x, v.y, v.z, v.w);
      if (p.olo.p)
        st_out<CT, VEC>(wrow<CT>(p.olo, id.b, rn, rh), d0, p.D, v.x - (float)(CT)v.x, v.y - (float)(CT)v.y,
                   v.z - (float)(CT)v.z, v.w - (float)(CT)v.w);
    }
  }
}

// Joins the splits' partial softmaxes: 32 lanes per row.  A lane reads the statistics of the splits
// lane, lane + 32, ...; then the lanes walk the splits in order, four columns each.  5.9 us for 16016 rows of
// 64 columns in 4 splits (16 MB), 4.5 for 512 rows of 128 in 8.
template <typename CT, int DP, bool VEC>
__global__ __launch_bounds__(256) void cross_join_kernel(const CrossP p) {
  const long long rows = (long long)p.Nq * p.G, total = rows * p.B * p.Hk;
  const int pr = (int)min(blockIdx.x * 8LL + (threadIdx.x >> 5), total);  // (total < 2^31)
  const int sub = threadIdx.x & 31, d0 = sub * 4;
  if (pr >= total) return;  // (all 32 lanes of the row)
  float M = kNoMax;
  for (int s = sub; s < p.nsplit; s += 32) M = fmaxf(M, p.part_ml[2 * (s * total + pr)]);
#pragma unroll
  for (int x = 16; x >= 1; x >>= 1) M = fmaxf(M, __shfl_xor(M, x, 64));
  float L = 0.f;
  float4 v = make_float4(0, 0, 0, 0);
  for (int s0 = 0; s0 < p.nsplit; s0 += 32) {
    float f = 0.f, lf = 0.f;
    if (s0 + sub < p.nsplit) {
      const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + 2 * ((s0 + sub) * total + pr));
      f = ml.x == kNoMax ? 1.f : __builtin_amdgcn_exp2f((ml.x - M) * p.c);  // (no keys: sums of 0)
      lf = f * ml.y;
    }
    const int n = min(32, p.nsplit - s0);
    for (int s = 0; s < n; s += 4) {  // four loads in flight; past the last split f is 0
      float4 t[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        t[j] = d0 < DP && s + j < n ? *reinterpret_cast<const float4*>(p.part + ((s0 + s + j) * total + pr) * DP + d0) : make_float4(0, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float fs = __shfl(f, (threadIdx.x & 32) + s + j, 64);
        L += __shfl(lf, (threadIdx.x & 32) + s + j, 64);
        v.x = fmaf(fs, t[j].x, v.x), v.y = fmaf(fs, t[j].y, v.y), v.z = fmaf(fs, t[j].z, v.z), v.w = fmaf(fs, t[j].w, v.w);
      }
    }
  }
  const int bh = quot(pr, p.by_rows), b = quot(bh, p.by_hk);
  const PackedRow pk = packed(p, pr - bh * (int)rows);
  const int n = pk.n, head = (bh - b * p.Hk) * p.G + pk.g;
  const bool some = n < clamp_len(p.qlen, b, p.Nq) && L != 0.f;
  const float inv = some ? 1.0f / L : 0.f;
  if (p.lse && d0 == 0) p.lse[((long long)b * p.H + head) * p.Nq + n] = some ? M * p.c + log2f(L) : -INFINITY;
  if (d0 >= p.D) return;
  v = some ? make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv) : make_float4(0, 0, 0, 0);
  st_out<CT, VEC>(wrow<CT>(p.o, b, n, head), d0, p.D, v.x, v.y, v.z, v.w);
  if (p.olo.p)
    st_out<CT, VEC>(wrow<CT>(p.olo, b, n, head), d0, p.D, v.x - (float)(CT)v.x, v.y - (float)(CT)v.y,
                    v.z - (float)(CT)v.z, v.w - (float)(CT)v.w);
}

// ------------------------------------------------------------------------------------------ backward
// delta = do . (o + o_lo) of a lane's row, from memory; h: the lane's half of the columns
template <typename CT, int KS, bool VEC>
__device__ __forceinline__ float row_delta(const CrossP& p, int b, int n, int head, bool live, int h) {
  float delta = 0.f;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const int c0 = 16 * ks + 8 * h;
    const typename V8<CT>::T g = live ? ld_frag<CT, VEC>(vrow<CT>(p.dout, b, n, head), c0, p.D) : zero8<CT>();
    const typename V8<CT>::T o = live ? ld_frag<CT, VEC>(vrow<CT>(p.o, b, n, head), c0, p.D) : zero8<CT>();
    if (p.olo.p) {
      const typename V8<CT>::T lo = live ? ld_frag<CT, VEC>(vrow<CT>(p.olo, b, n, head), c0, p.D) : zero8<CT>();
#pragma unroll
      for (int j = 0; j < 8; ++j) delta = fmaf((float)g[j], (float)o[j] + (float)lo[j], delta);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) delta = fmaf((float)g[j], (float)o[j], delta);
    }
  }
  return other_half_sum(delta);
}

// S, dP of 32 rows (8a + 4h + i) by one key per lane -> P, dS; ls, ds: the rows' lse and delta
__device__ __forceinline__ void grad_scores(f32x16& s, f32x16& g, const float* ls, const float* ds, float c, int h) {
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    const float4 lv = *reinterpret_cast<const float4*>(ls + 8 * a + 4 * h);
    const float4 dl = *reinterpret_cast<const float4*>(ds + 8 * a + 4 * h);
    const float lw[4] = {lv.x, lv.y, lv.z, lv.w}, dw[4] = {dl.x, dl.y, dl.z, dl.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float pr = __builtin_amdgcn_exp2f(fmaf(s[4 * a + i], c, -lw[i]));
      s[4 * a + i] = pr;
      g[4 * a + i] = pr * (g[4 * a + i] - dw[i]);
    }
  }
}

// dq: the forward's layout (one query per lane).  delta = do . (o + o_lo) is formed here from the
// fragments in registers and left for the dk / dv pass.  Scores are formed anew from q, k and lse where a
// stored P would be Nq x Nk of traffic.  dq and dk / dv are two kernels, each the sole writer of its
// sums, so results repeat bit for bit (one kernel would have to add dq by atomics).
// D = 64, [4, 4096, 16] on 2048 ragged keys (165 GFLOP): 186-192 us, 860 TFLOP/s; MFMA and vector unit 45 and 60 % busy.
template <typename CT, int DP, int KT, bool VEC>
__global__ __launch_bounds__(256, sizeof(CT) * DP >= 512 ? 1 : 2) void cross_dq_kernel(const CrossP p, int tiles) {
  constexpr int TILE = KT * DP, DT = DP / 32, KS = DP / 16, NT = KT / 32;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  CT* Ks = reinterpret_cast<CT*>(smem);
  CT* Vs = Ks + 2 * TILE;
  float* kbs = reinterpret_cast<float*>(Vs + 2 * TILE);
  int* flag = reinterpret_cast<int*>(kbs + 2 * KT);

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const BlockId id = block_id(p, tiles);
  const int rows = p.Nq * p.G, r = id.tile * 128 + wave * 32 + (lane & 31);
  const PackedRow pk = packed(p, r);
  const int n = pk.n, head = id.hk * p.G + pk.g;
  const int qlen = clamp_len(p.qlen, id.b, p.Nq), klen = clamp_len(p.klen, id.b, p.Nk);
  const bool live = r < rows && n < qlen, busy = id.tile * 128 + wave * 32 < qlen * p.G;
  const int ln = live ? n : 0, lh = live ? head : 0;
  const long long srow = ((long long)id.b * p.H + lh) * p.Nq + ln;

  int k0, k1;
  split_range(p, klen, id.split, k0, k1);
  KvStage<CT, DP, KT, 256, VEC, VEC> st;
  const int nt = (k1 - k0 + KT - 1) / KT;
  if (nt > 0) {  // (the first tile's loads start before delta waits for its own)
    st.init(p, id.b, id.hk, k0, k1, KT, tid);
    st.begin(p, Ks, Vs, id.b, k0, k1, KT, tid);
  }
  typename V8<CT>::T qf[KS], gf[KS];
  float delta = 0.f;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const int c0 = 16 * ks + 8 * h;
    qf[ks] = live ? ld_frag<CT, VEC>(vrow<CT>(p.q, id.b, ln, lh), c0, p.D) : zero8<CT>();
    gf[ks] = live ? ld_frag<CT, VEC>(vrow<CT>(p.dout, id.b, ln, lh), c0, p.D) : zero8<CT>();
    const typename V8<CT>::T of = live ? ld_frag<CT, VEC>(vrow<CT>(p.o, id.b, ln, lh), c0, p.D) : zero8<CT>();
    if (p.olo.p) {
      const typename V8<CT>::T lo = live ? ld_frag<CT, VEC>(vrow<CT>(p.olo, id.b, ln, lh), c0, p.D) : zero8<CT>();
#pragma unroll
      for (int j = 0; j < 8; ++j) delta = fmaf((float)gf[ks][j], (float)of[j] + (float)lo[j], delta);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) delta = fmaf((float)gf[ks][j], (float)of[j], delta);
    }
  }
  delta = other_half_sum(delta);
  float lse = live ? p.lse[srow] : -INFINITY;
  if (lse == -INFINITY) lse = INFINITY;  // a row without keys: every P is 0
  if (id.split == 0 && r < rows && h == 0) p.delta[((long long)id.b * p.H + head) * p.Nq + n] = delta;

  f32x16 acc[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[t][i] = 0.f;

  if (nt > 0) st.finish(p, Ks, Vs, kbs, flag, tid);
  __syncthreads();
  for (int t = 0; t < nt; ++t) {
    const int cur = t & 1;
    const int other = (cur ^ 1) * TILE;
    if (t + 1 < nt) st.begin(p, Ks + other, Vs + other, id.b, k0 + (t + 1) * KT, k1, KT, tid);
    const CT* Kc = Ks + cur * TILE;
    const CT* Vc = Vs + cur * TILE;
    const bool holes = __builtin_amdgcn_readfirstlane(flag[cur]);
#pragma unroll
    for (int kt = 0; kt < NT; ++kt) {
      if (!busy) break;  // (a wave without rows only loads)
      f32x16 s1[1], g = zero16();
      f32x16& s = s1[0];
      key_scores<CT, DP, 1>(s1, Kc + 32 * kt * DP, qf, kbs + cur * KT + 32 * kt, holes, p.D, lane);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        if (step_there<CT, DP>(ks, p.D)) g = mma<CT>(row_frag<CT, DP>(Vc, 32 * kt + (lane & 31), 16 * ks, lane), gf[ks], g);
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], p.c, -lse)) * (g[i] - delta);
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        const typename V8<CT>::T df = half_frag<CT>(s, s2);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
          acc[dt] = mma<CT>(col_frag<CT, DP>(Kc, 32 * kt + 16 * s2, 32 * dt, lane), df, acc[dt]);
      }
    }
    if (t + 1 < nt) st.finish(p, Ks + other, Vs + other, kbs + (cur ^ 1) * KT, flag + (cur ^ 1), tid);
    __syncthreads();
  }
  const bool none = no_key(p, id.b, k0, k1, has_nan(acc), lane);
  if (r >= rows) return;
  if (!live || none) {  // 0, whatever keys, query and its gradient hold
#pragma unroll
    for (int t = 0; t < DT; ++t) acc[t] = zero16();
  }
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
      st_out<CT, VEC>(row, 32 * dt + 8 * a + 4 * h, p.D, acc[dt][4 * a] * p.scale, acc[dt][4 * a + 1] * p.scale,
                 acc[dt][4 * a + 2] * p.scale, acc[dt][4 * a + 3] * p.scale);
}

// Packed rows of q and do, QT at a time, on their way to LDS (as KvStage), with their lse and delta.
template <typename CT, int DP, int QT, bool VEC, bool ASYNC>
struct RowStage {
  static constexpr int N = 16 / sizeof(CT), CPR = DP / N, P = QT * CPR / 256;
  static_assert(QT * CPR % 256 == 0 && QT <= 64, "whole pieces per thread");
  uint4 q[ASYNC ? 1 : P], g[ASYNC ? 1 : P];
  float lse, delta;
  __device__ __forceinline__ static int slot(int i, int tid) {
    return ASYNC ? ((tid >> 6) * P + i) * 64 + (tid & 63) : i * 256 + tid;
  }
  __device__ __forceinline__ void begin(const CrossP& p, CT* Qs, CT* Gs, int b, int hk, int row0, int end, int tid) {
    const int n0 = packed(p, row0).n;
    const CT* qb = vrow<CT>(p.q, b, n0, hk * p.G);
    const CT* gb = vrow<CT>(p.dout, b, n0, hk * p.G);
    u32x4 qr, gr;
    if constexpr (ASYNC) qr = resource(uniform64((uint64_t)qb), 0x7fffffffu), gr = resource(uniform64((uint64_t)gb), 0x7fffffffu);
    const unsigned first = __builtin_amdgcn_readfirstlane(tid >> 6) * P * 1024;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int lr = slot(i, tid) / CPR, row = row0 + lr;
      const PackedRow pk = packed(p, row);
      const int n = pk.n, hd = pk.g;
      if constexpr (ASYNC) {
        const int c = slot(i, tid) % CPR ^ chunk_xor<CT, DP>(lr);
        const bool in = row < end && c * N < p.D;
        const int dn = n - n0;
        async_load16(qr, lds_address(Qs) + first + i * 1024,
                     in ? (unsigned)((dn * p.q.sn + hd * p.q.sh) * sizeof(CT)) + c * 16 : kNowhere);
        async_load16(gr, lds_address(Gs) + first + i * 1024,
                     in ? (unsigned)((dn * p.dout.sn + hd * p.dout.sh) * sizeof(CT)) + c * 16 : kNowhere);
      } else {
        const int cc = slot(i, tid) % CPR * N;
        const bool in = row < end && cc < p.D;
        q[i] = in ? ld_piece<CT, VEC>(qb + (n - n0) * p.q.sn + hd * p.q.sh, cc, p.D) : make_uint4(0, 0, 0, 0);
        g[i] = in ? ld_piece<CT, VEC>(gb + (n - n0) * p.dout.sn + hd * p.dout.sh, cc, p.D) : make_uint4(0, 0, 0, 0);
      }
    }
    lse = INFINITY, delta = 0.f;  // (every P of a row past the end, or without keys, is 0)
    if (tid < QT && row0 + tid < end) {
      const PackedRow pk = packed(p, row0 + tid);
      const int n = pk.n, hd = hk * p.G + pk.g;
      const long long i = ((long long)b * p.H + hd) * p.Nq + n;
      lse = p.lse[i], delta = p.delta[i];
      if (lse == -INFINITY) lse = INFINITY;
    }
  }
  __device__ __forceinline__ void finish(CT* Qs, CT* Gs, float* ls, float* ds, int tid) {
    if constexpr (!ASYNC) {
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const int at = lds_at<CT, DP>(slot(i, tid) / CPR, slot(i, tid) % CPR);
        *reinterpret_cast<uint4*>(Qs + at) = q[i];
        *reinterpret_cast<uint4*>(Gs + at) = g[i];
      }
    }
    if (tid < QT) ls[tid] = lse, ds[tid] = delta;
    if constexpr (ASYNC) async_wait();
  }
};

// dk, dv: one key per lane; a block owns 4 x 32 keys of one (b, key head) and walks the rows in tiles
// of QT (q and do through LDS, double buffered); splits share the rows, their fp32 partials summed in
// order by cross_sum_kernel.
// D = 64, [4, 4096, 16] on 2048 ragged keys (221 GFLOP): 288-290 us, 760 TFLOP/s: four accumulator tiles, the key
// fragments and two tiles of scores take 204 registers, two waves per SIMD.  Held to 168 registers (three
// waves) it takes 5 % longer, with an interleave of MFMA and vector instructions forced on the scheduler 1-2 %,
// with more splits 5-8 %, also where the blocks past a sequence's end are dealt out evenly over the CUs.
template <typename CT, int DP, int QT, bool VEC>
__global__ __launch_bounds__(256) void cross_dkv_kernel(const CrossP p, int tiles) {
  constexpr int TILE = QT * DP, DT = DP / 32, KS = DP / 16;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  CT* Qs = reinterpret_cast<CT*>(smem);
  CT* Gs = Qs + 2 * TILE;
  float* ls = reinterpret_cast<float*>(Gs + 2 * TILE);  // [2][QT]
  float* ds = ls + 2 * QT;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const BlockId id = block_id(p, tiles);
  const int qlen = clamp_len(p.qlen, id.b, p.Nq), klen = clamp_len(p.klen, id.b, p.Nk);
  const int rows = qlen * p.G;
  const int key = id.tile * 128 + wave * 32 + (lane & 31);
  const bool live = key < klen && key_kept(p, id.b, key), busy = id.tile * 128 + wave * 32 < klen;

  typename V8<CT>::T kf[KS], vf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const int c0 = 16 * ks + 8 * h;
    kf[ks] = live ? ld_frag<CT, VEC>(vrow<CT>(p.k, id.b, key, id.hk), c0, p.D) : zero8<CT>();
    vf[ks] = live ? ld_frag<CT, VEC>(vrow<CT>(p.v, id.b, key, id.hk), c0, p.D) : zero8<CT>();
  }
  f32x16 dk[DT], dv[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) dk[t] = dv[t] = zero16();

  const int per = ((rows + p.nsplit - 1) / p.nsplit + QT - 1) / QT * QT;
  const int r0 = min(rows, id.split * per), r1 = min(rows, r0 + per);
  // a block whose keys all lie past the sequence has nothing to sum
  const int todo = id.tile * 128 < klen ? (r1 - r0 + QT - 1) / QT : 0;

  RowStage<CT, DP, QT, VEC, VEC> st;
  if (todo > 0) {
    st.begin(p, Qs, Gs, id.b, id.hk, r0, r1, tid);
    st.finish(Qs, Gs, ls, ds, tid);
  }
  __syncthreads();
  for (int t = 0; t < todo; ++t) {
    const int cur = t & 1, other = (cur ^ 1) * TILE;
    if (t + 1 < todo) st.begin(p, Qs + other, Gs + other, id.b, id.hk, r0 + (t + 1) * QT, r1, tid);
    const CT* Qc = Qs + cur * TILE;
    const CT* Gc = Gs + cur * TILE;
#pragma unroll
    for (int qt = 0; qt < QT; qt += 32) {
      if (!busy) break;  // (a wave without keys only loads)
      f32x16 s = zero16(), g = zero16();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if (!step_there<CT, DP>(ks, p.D)) continue;
        s = mma<CT>(row_frag<CT, DP>(Qc, qt + (lane & 31), 16 * ks, lane), kf[ks], s);
        g = mma<CT>(row_frag<CT, DP>(Gc, qt + (lane & 31), 16 * ks, lane), vf[ks], g);
      }
      grad_scores(s, g, ls + cur * QT + qt, ds + cur * QT + qt, p.c, h);
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        const typename V8<CT>::T pf = half_frag<CT>(s, s2), df = half_frag<CT>(g, s2);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          dv[dt] = mma<CT>(col_frag<CT, DP>(Gc, qt + 16 * s2, 32 * dt, lane), pf, dv[dt]);
          dk[dt] = mma<CT>(col_frag<CT, DP>(Qc, qt + 16 * s2, 32 * dt, lane), df, dk[dt]);
        }
      }
    }
    if (t + 1 < todo) st.finish(Qs + other, Gs + other, ls + (cur ^ 1) * QT, ds + (cur ^ 1) * QT, tid);
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
        st_out<CT, VEC>(wrow<CT>(p.dk, id.b, key, id.hk), d0, p.D, x[0], x[1], x[2], x[3]);
        st_out<CT, VEC>(wrow<CT>(p.dv, id.b, key, id.hk), d0, p.D, y[0], y[1], y[2], y[3]);
      }
    }
}

// The whole backward for at most 32 rows per (b, key head): one pass over the keys.  As in cross_few_kernel
// the waves split the keys, each with 32-key tiles of its own; q and do lie in LDS for all of them.  Per tile
//   S^T, dP^T (one query per lane) -> dS^T -> dq^T += K^T dS^T,    summed over tiles, waves and splits;
//   S, dP (one key per lane) -> P, dS -> dv^T = dO^T P, dk^T = Q^T dS,   complete here: all rows are in the tile.
// The same two fragments in either order give the two score tiles, and k and v are read once: bound by memory.
// 8 sequences of one token, 16 heads of 128 on 8192 bf16 keys (k and v read, dk and dv written, 1.07 GB): 228 us,
// 4.7 TB/s, against 102 + 460 us of the two kernels above; 4 of 7 tokens, 32 heads of 64 on 8 of 4000 keys 21 against
// 13.6 + 24.2; fp32, 4 of 20 tokens, 8 heads of 64 on 3000 keys 56 against 47 + 33 (its products).  dk and dv leave
// through LDS, 16 bytes per lane.  fp32 wider than 64 columns would spill (160 us against 78 + 64): not built.
template <typename CT, int DP>
constexpr bool few_bwd() { return sizeof(CT) * DP <= 256; }
template <typename CT, int DP, bool VEC>
__global__ __launch_bounds__(256) void cross_few_bwd_kernel(const CrossP p) {
  constexpr int W = 4, TILE = 32 * DP, DT = DP / 32, KS = DP / 16, LO = DP + 4;
  constexpr int BUFS = few_async<CT, DP, VEC>() ? 2 : 1, N = 16 / sizeof(CT), CPR = DP / N;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  CT* Qs = reinterpret_cast<CT*>(smem);
  CT* Gs = Qs + TILE;
  CT* Ks = Gs + TILE + wave * 2 * BUFS * TILE;
  CT* Vs = Ks + BUFS * TILE;
  float* ls = reinterpret_cast<float*>(Qs + (2 + 2 * BUFS * W) * TILE);  // [32], then delta [32]
  float* ds = ls + 32;
  float* kbs = ds + 32 + wave * 32;
  int* flag = reinterpret_cast<int*>(ds + 32 + W * 32) + wave;

  const BlockId id = block_id(p, 1);
  const int rows = p.Nq * p.G, r = lane & 31;
  const PackedRow pk = packed(p, r);
  const int qlen = clamp_len(p.qlen, id.b, p.Nq), klen = clamp_len(p.klen, id.b, p.Nk);
  const bool live = r < rows && pk.n < qlen;
  const int n = live ? pk.n : 0, head = live ? id.hk * p.G + pk.g : 0;

  int k0, kend;  // this block's keys; those past the sequence's end have gradients too, zeros
  split_range(p, p.Nk, id.split, k0, kend);
  const int k1 = min(kend, klen);
  using S = KvStage<CT, DP, 32, 64, VEC, BUFS == 2>;
  S st;
  int key = k0 + 32 * wave, cur = 0;
  if (key < k1) {
    st.init(p, id.b, id.hk, key, k1, 32 * W, lane);
    st.begin(p, Ks, Vs, id.b, key, k1, 32 * W, lane);
  }
  for (int i = tid; i < 32 * CPR; i += 64 * W) {
    const int row = i / CPR, c = i % CPR;
    const PackedRow q = packed(p, row);
    const bool in = row < rows && q.n < qlen && c * N < p.D;
    const int hd = id.hk * p.G + q.g;
    *reinterpret_cast<uint4*>(Qs + lds_at<CT, DP>(row, c)) =
        in ? ld_piece<CT, VEC>(vrow<CT>(p.q, id.b, q.n, hd), c * N, p.D) : make_uint4(0, 0, 0, 0);
    *reinterpret_cast<uint4*>(Gs + lds_at<CT, DP>(row, c)) =
        in ? ld_piece<CT, VEC>(vrow<CT>(p.dout, id.b, q.n, hd), c * N, p.D) : make_uint4(0, 0, 0, 0);
  }
  const float delta = row_delta<CT, KS, VEC>(p, id.b, n, head, live, h);
  float lse = live ? p.lse[((long long)id.b * p.H + head) * p.Nq + n] : -INFINITY;
  if (lse == -INFINITY) lse = INFINITY;  // a row without keys, or none: every P is 0
  if (wave == 0 && h == 0) ls[r] = lse, ds[r] = delta;
  __syncthreads();

  f32x16 acc[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) acc[t] = zero16();
  for (; key < k1; key += 32 * W) {
    st.finish_kb(kbs, flag, lane);
    const bool more = key + 32 * W < k1;
    if constexpr (BUFS == 2) {
      if (more) {
        st.begin(p, Ks + (cur ^ 1) * TILE, Vs + (cur ^ 1) * TILE, id.b, key + 32 * W, k1, 32 * W, lane);
        async_wait<2 * S::P>();  // this tile's loads, not the next one's
      } else {
        async_wait();
      }
    } else {
      st.finish_rows(p, Ks, Vs, lane);
      if (more) st.begin(p, Ks, Vs, id.b, key + 32 * W, k1, 32 * W, lane);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    const CT* Kt = Ks + cur * TILE;
    const CT* Vt = Vs + cur * TILE;
    const bool holes = __builtin_amdgcn_readfirstlane(*flag);
    {
      typename V8<CT>::T qf[KS];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) qf[ks] = row_frag<CT, DP>(Qs, r, 16 * ks, lane);
      f32x16 s[1], g = zero16();
      key_scores<CT, DP, 1>(s, Kt, qf, kbs, holes, p.D, lane);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        if (step_there<CT, DP>(ks, p.D)) g = mma<CT>(row_frag<CT, DP>(Vt, r, 16 * ks, lane), row_frag<CT, DP>(Gs, r, 16 * ks, lane), g);
#pragma unroll
      for (int i = 0; i < 16; ++i) s[0][i] = __builtin_amdgcn_exp2f(fmaf(s[0][i], p.c, -lse)) * (g[i] - delta);
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        const typename V8<CT>::T df = half_frag<CT>(s[0], s2);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[dt] = mma<CT>(col_frag<CT, DP>(Kt, 16 * s2, 32 * dt, lane), df, acc[dt]);
      }
    }
    if (p.dk.p) {
      f32x16 s = zero16(), g = zero16();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if (!step_there<CT, DP>(ks, p.D)) continue;
        s = mma<CT>(row_frag<CT, DP>(Qs, r, 16 * ks, lane), row_frag<CT, DP>(Kt, r, 16 * ks, lane), s);
        g = mma<CT>(row_frag<CT, DP>(Gs, r, 16 * ks, lane), row_frag<CT, DP>(Vt, r, 16 * ks, lane), g);
      }
      const bool there = kbs[r] == 0.f;  // (key `key + r`)
      grad_scores(s, g, ls, ds, p.c, h);
      typename V8<CT>::T pf[2], df[2];
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) pf[s2] = half_frag<CT>(s, s2), df[s2] = half_frag<CT>(g, s2);
      // over the k and v tiles, which are done with, then out by whole rows
      CT* Kw = Ks + cur * TILE;
      CT* Vw = Vs + cur * TILE;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        f32x16 x = zero16(), y = zero16();
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) {
          if (16 * s2 >= rows) continue;  // (the rows past them are zeros)
          x = mma<CT>(col_frag<CT, DP>(Qs, 16 * s2, 32 * dt, lane), df[s2], x);
          y = mma<CT>(col_frag<CT, DP>(Gs, 16 * s2, 32 * dt, lane), pf[s2], y);
        }
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const int d0 = 32 * dt + 8 * a + 4 * h, at = lds_at<CT, DP>(r, d0 / N) + d0 % N;
          st4<CT>(Kw + at, there ? x[4 * a] * p.scale : 0.f, there ? x[4 * a + 1] * p.scale : 0.f,
                  there ? x[4 * a + 2] * p.scale : 0.f, there ? x[4 * a + 3] * p.scale : 0.f);
          st4<CT>(Vw + at, there ? y[4 * a] : 0.f, there ? y[4 * a + 1] : 0.f, there ? y[4 * a + 2] : 0.f, there ? y[4 * a + 3] : 0.f);
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      CT* dk = wrow<CT>(p.dk, id.b, key, id.hk);
      CT* dv = wrow<CT>(p.dv, id.b, key, id.hk);
      for (int i = lane; i < 32 * CPR; i += 64) {
        const int row = i / CPR, c = i % CPR, at = lds_at<CT, DP>(row, c);
        if (key + row < kend && c * N < p.D) {
          st_piece<CT, VEC>(dk + row * p.dk.sn, c * N, p.D, *reinterpret_cast<const uint4*>(Kw + at));
          st_piece<CT, VEC>(dv + row * p.dv.sn, c * N, p.D, *reinterpret_cast<const uint4*>(Vw + at));
        }
      }
    }
    // the next turn's loads overwrite this buffer: its reads are done before they start
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    if constexpr (BUFS == 2) cur ^= 1;
  }
  if (p.dk.p)
    for (; key < kend; key += 32 * W)
      for (int i = lane; i < 32 * CPR; i += 64) {
        const int at = key + i / CPR, c0 = i % CPR * N;
        if (at < kend && c0 < p.D) {
          st_piece<CT, VEC>(wrow<CT>(p.dk, id.b, at, id.hk), c0, p.D, make_uint4(0, 0, 0, 0));
          st_piece<CT, VEC>(wrow<CT>(p.dv, id.b, at, id.hk), c0, p.D, make_uint4(0, 0, 0, 0));
        }
      }

  if (no_key(p, id.b, k0, k1, has_nan(acc), lane)) {
#pragma unroll
    for (int t = 0; t < DT; ++t) acc[t] = zero16();
  }
  // dq of the waves, [W][32][DP + 4] over the tiles, summed in order
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the last tile's reads are done
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
  float* jo = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int a = 0; a < 4; ++a)
      *reinterpret_cast<float4*>(jo + (32 * wave + r) * LO + 32 * dt + 8 * a + 4 * h) =
          make_float4(acc[dt][4 * a], acc[dt][4 * a + 1], acc[dt][4 * a + 2], acc[dt][4 * a + 3]);
  __syncthreads();
  for (int i = tid; i < rows * (DP / 4); i += 64 * W) {
    const int row = i / (DP / 4), d0 = (i % (DP / 4)) * 4;
    float4 v = make_float4(0, 0, 0, 0);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float4 t = *reinterpret_cast<const float4*>(jo + (32 * w + row) * LO + d0);
      v.x += t.x, v.y += t.y, v.z += t.z, v.w += t.w;
    }
    const PackedRow q = packed(p, row);
    if (q.n >= qlen) v = make_float4(0, 0, 0, 0);  // (whatever the keys hold)
    if (p.nsplit > 1) {
      *reinterpret_cast<float4*>(p.part + part_row(p, id.split, id.b, id.hk, row) * DP + d0) = v;
    } else {
      st_out<CT, VEC>(wrow<CT>(p.dq, id.b, q.n, id.hk * p.G + q.g), d0, p.D, v.x * p.scale, v.y * p.scale, v.z * p.scale,
                      v.w * p.scale);
    }
  }
}

// sums the splits' fp32 partials in order: nout planes [rows][DP] per split -> the strided outputs.
// kv: rows (b, hk, key), planes dk | dv; else rows (b, hk, n * G + g), dq scaled here.
template <typename CT, int DP, bool VEC>
__global__ __launch_bounds__(256) void cross_sum_kernel(const CrossP p, int kv) {
  constexpr int Q = DP / 4;
  const long long rows = kv ? (long long)p.Nk : (long long)p.Nq * p.G, total = rows * p.B * p.Hk;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long row = i / Q;
  const int d0 = (int)(i % Q) * 4, nout = kv ? 2 : 1;
  if (row >= total * nout) return;
  float4 v = make_float4(0, 0, 0, 0);
#pragma unroll 4
  for (int s = 0; s < p.nsplit; ++s) {
    const float4 t = *reinterpret_cast<const float4*>(p.part + (s * nout * total + row) * DP + d0);
    v.x += t.x, v.y += t.y, v.z += t.z, v.w += t.w;
  }
  const int r0 = (int)(row < total ? row : row - total), bh = quot(r0, p.by_rows), r = r0 - bh * (int)rows;
  const int b = quot(bh, p.by_hk), hk = bh - b * p.Hk;
  if (kv) {
    st_out<CT, VEC>(wrow<CT>(row < total ? p.dk : p.dv, b, r, hk), d0, p.D, v.x, v.y, v.z, v.w);
  } else {
    const PackedRow pk = packed(p, r);
    st_out<CT, VEC>(wrow<CT>(p.dq, b, pk.n, hk * p.G + pk.g), d0, p.D, v.x * p.scale, v.y * p.scale,
               v.z * p.scale, v.w * p.scale);
  }
}

// ------------------------------------------------------------------------------------------ host
int dp_of_head(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }

// Splits: enough blocks to fill 256 CUs `want` / 256 times over, none with less than `least` of the long axis.
// want: 512 for blocks of four waves (dk / dv at D = 64: 1024 costs 679 against 658 us of training, the partials'
// traffic; fp32: 768 the same as 512), 1024 for single tokens (memory), 256 for the eight waves of the
// two-phase kernel.  least: 256, or 96 for fp32, whose products take sixteen times as long.
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

CrossP params(const mdg_attn_cross& a) {
  CrossP p;
  p.q = view(a.q), p.k = view(a.k), p.v = view(a.v), p.o = view(a.o), p.olo = view(a.o_lo);
  p.dout = view(a.dout), p.dq = view(a.dq), p.dk = view(a.dk), p.dv = view(a.dv);
  p.qlen = a.q_len, p.klen = a.kv_len, p.mask = a.mask, p.mask_f32 = a.mask_type == MDG_MASK_F32;
  p.mb = a.mask_sb, p.mn = a.mask_sn;
  p.B = a.B, p.Nq = a.Nq, p.Nk = a.Nk, p.H = a.H, p.Hk = a.Hk, p.G = a.H / a.Hk, p.D = a.D;
  p.c = a.scale * kLog2e, p.scale = a.scale, p.lse = a.lse;
  p.delta = nullptr, p.part = p.part_ml = nullptr;
  p.by_g = divisor(p.G), p.by_hk = divisor(p.Hk);
  return p;
}
// one launch's blocks: tiles x splits x (batch, key head), each of `rows` rows
void shape(CrossP& p, long long tiles, int split, long long rows) {
  p.nsplit = split;
  p.by_split = divisor(split), p.by_tiles = divisor(tiles), p.by_rows = divisor(rows);
}

// 16-byte pieces: the head dim a multiple of a piece, every base and stride 16-byte aligned; and a tile's
// rows apart, within the 2^30 bytes that an asynchronous load's offset spans (64 keys, or 65 tokens)
// (element by element instead: 693 against 610 us at D = 128)
bool pieces(const mdg_attn_cross& a, bool bwd) {
  const int e = a.dtype == MDG_BF16 ? 2 : 4;
  const int64_t span = (int64_t)1 << 30;
  bool ok = a.D % (16 / e) == 0;
  for (const mdg_heads* t : {&a.q, &a.k, &a.v, &a.o, &a.o_lo}) ok = ok && aligned16(*t, e);
  for (const mdg_heads* t : {&a.k, &a.v}) ok = ok && t->sn >= a.D && 64 * t->sn * e < span;
  if (bwd) {
    for (const mdg_heads* t : {&a.dout, &a.dq, &a.dk, &a.dv}) ok = ok && aligned16(*t, e);
    for (const mdg_heads* t : {&a.q, &a.dout}) ok = ok && (65 * t->sn + a.H * t->sh) * e < span;
  }
  return ok;
}

struct Plan {
  bool few, pp;  // the single-token kernel; the two-phase kernel
  long long tiles;
  int split;
  size_t part, ml, bytes;  // byte offsets / total
};
size_t al(size_t n) { return (n + 255) / 256 * 256; }

Plan fwd_plan(const mdg_attn_cross& a, bool vec) {
  Plan w;
  const long long rows = (long long)a.Nq * (a.H / a.Hk), bh = (long long)a.B * a.Hk;
  // one 32-row tile: the waves split the keys.  (As 32-row blocks under more rows, fp32 [2, 1001, 8, 48] on 333
  // keys: 26.8 us against 21.8 + 5.9 of the join, for four times the k / v reads: not used.)
  w.few = rows <= 32;
  // wide bf16 heads: [8, 256, 16, 128] on 1024 keys 40.7 us against 44.3 of the plain kernel, [4, 1024, 16, 96] on 1024
  // keys 46.0 / 47.1; below 256 rows half of its waves would idle
  w.pp = a.dtype == MDG_BF16 && vec && dp_of_head(a.D) == 128 && rows >= 256;
  w.tiles = w.few ? 1 : w.pp ? (rows + 255) / 256 : (rows + 127) / 128;
  w.split = pick_split(w.tiles * bh, a.Nk, a.dtype == MDG_F32 && !w.few ? 96 : 256, w.few ? 1024 : w.pp ? 256 : 512);
  w.part = 0, w.ml = w.bytes = 0;
  if (w.split > 1) {
    w.ml = al((size_t)w.split * rows * bh * dp_of_head(a.D) * 4);
    w.bytes = w.ml + al((size_t)w.split * rows * bh * 8);
  }
  return w;
}

struct BwdPlan {
  bool few;  // one pass over the keys for one 32-row tile
  long long qtiles, ktiles;
  int qsplit, ksplit;  // splits of the dq pass (over keys) and of the dk / dv pass (over rows)
  size_t delta, part, bytes;
};
BwdPlan bwd_plan(const mdg_attn_cross& a) {
  BwdPlan w;
  const long long rows = (long long)a.Nq * (a.H / a.Hk), bh = (long long)a.B * a.Hk;
  w.qtiles = (rows + 127) / 128, w.ktiles = ((long long)a.Nk + 127) / 128;
  w.few = rows <= 32 && dp_of_head(a.D) * (a.dtype == MDG_F32 ? 4 : 2) <= 256;
  w.qsplit = w.few ? pick_split(bh, a.Nk, 256, 1024) : pick_split(w.qtiles * bh, a.Nk, a.dtype == MDG_F32 ? 96 : 256, 512);
  w.ksplit = w.few ? 1 : pick_split(w.ktiles * bh, rows, a.dtype == MDG_F32 ? 96 : 256, 512);
  w.delta = 0;
  w.part = al((size_t)a.B * a.H * a.Nq * 4);
  const size_t dp = dp_of_head(a.D);
  const size_t pq = w.qsplit > 1 ? (size_t)w.qsplit * rows * bh * dp * 4 : 0;
  const size_t pk = w.ksplit > 1 ? (size_t)w.ksplit * 2 * a.Nk * bh * dp * 4 : 0;
  w.bytes = w.part + al(pq > pk ? pq : pk);
  return w;
}

template <typename CT, int DP, bool VEC>
hipError_t fwd(const mdg_attn_cross& a, void* ws, hipStream_t s) {
  constexpr int KT = sizeof(CT) == 2 ? 64 : 32;
  const Plan w = fwd_plan(a, VEC);
  CrossP p = params(a);
  shape(p, w.tiles, w.split, (long long)a.Nq * p.G);
  if (w.split > 1) {
    p.part = reinterpret_cast<float*>(ws);
    p.part_ml = reinterpret_cast<float*>(static_cast<char*>(ws) + w.ml);
  }
  const unsigned grid = (unsigned)(w.tiles * w.split * a.B * a.Hk);
  hipError_t e;
  if (w.few) {
    const size_t stage = (size_t)4 * 2 * (few_async<CT, DP, VEC>() ? 2 : 1) * 32 * DP * sizeof(CT) + 4 * 32 * 4 + 16;
    const size_t join = (size_t)(288 + 128 * (DP + 4)) * 4, sm = stage > join ? stage : join;
    if ((e = allow_lds(cross_few_kernel<CT, DP, VEC>, sm)) != hipSuccess) return e;
    hipLaunchKernelGGL((cross_few_kernel<CT, DP, VEC>), dim3(grid), dim3(256), sm, s, p, 1);
  } else if (w.pp) {
    if constexpr (VEC && sizeof(CT) == 2 && DP == 128) {
      const size_t sm = (size_t)5 * KT * DP * sizeof(CT) + 2 * KT * 4 + 16;
      if ((e = allow_lds(cross_fwd_pp_kernel<DP, KT>, sm)) != hipSuccess) return e;
      hipLaunchKernelGGL((cross_fwd_pp_kernel<DP, KT>), dim3(grid), dim3(512), sm, s, p, (int)w.tiles);
    }
  } else {
    const size_t sm = (size_t)4 * KT * DP * sizeof(CT) + 2 * KT * 4 + 16;
    if ((e = allow_lds(cross_fwd_kernel<CT, DP, KT, VEC>, sm)) != hipSuccess) return e;
    hipLaunchKernelGGL((cross_fwd_kernel<CT, DP, KT, VEC>), dim3(grid), dim3(256), sm, s, p, (int)w.tiles);
  }
  if (w.split > 1) {
    const long long total = (long long)a.B * a.H * a.Nq;
    hipLaunchKernelGGL((cross_join_kernel<CT, DP, VEC>), dim3((unsigned)((total + 7) / 8)), dim3(256), 0, s, p);
  }
  return hipGetLastError();
}

template <typename CT, int DP, bool VEC>
hipError_t bwd(const mdg_attn_cross& a, void* ws, hipStream_t s) {
  constexpr int KT = sizeof(CT) == 2 ? 64 : 32, QT = sizeof(CT) == 2 && DP <= 64 ? 64 : 32;
  const BwdPlan w = bwd_plan(a);
  CrossP p = params(a);
  p.delta = reinterpret_cast<float*>(static_cast<char*>(ws) + w.delta);
  p.part = reinterpret_cast<float*>(static_cast<char*>(ws) + w.part);
  hipError_t e;
  if (w.few) {
    if constexpr (few_bwd<CT, DP>()) {
    const size_t tiles = (size_t)(2 + 8 * (few_async<CT, DP, VEC>() ? 2 : 1)) * 32 * DP * sizeof(CT) + (64 + 128 + 4) * 4;
    const size_t join = (size_t)128 * (DP + 4) * 4, sm = tiles > join ? tiles : join;
    if ((e = allow_lds(cross_few_bwd_kernel<CT, DP, VEC>, sm)) != hipSuccess) return e;
    shape(p, 1, w.qsplit, (long long)a.Nq * p.G);
    hipLaunchKernelGGL((cross_few_bwd_kernel<CT, DP, VEC>), dim3((unsigned)(w.qsplit * a.B * a.Hk)), dim3(256), sm, s, p);
    if (w.qsplit > 1) {
      const long long n = (long long)a.B * a.H * a.Nq * (DP / 4);
      hipLaunchKernelGGL((cross_sum_kernel<CT, DP, VEC>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, p, 0);
    }
    return hipGetLastError();
    }
  }
  const size_t smq = (size_t)4 * KT * DP * sizeof(CT) + 2 * KT * 4 + 16;
  const size_t smk = (size_t)4 * QT * DP * sizeof(CT) + 4 * QT * 4;
  if ((e = allow_lds(cross_dq_kernel<CT, DP, KT, VEC>, smq)) != hipSuccess) return e;
  if ((e = allow_lds(cross_dkv_kernel<CT, DP, QT, VEC>, smk)) != hipSuccess) return e;
  shape(p, w.qtiles, w.qsplit, (long long)a.Nq * p.G);
  hipLaunchKernelGGL((cross_dq_kernel<CT, DP, KT, VEC>), dim3((unsigned)(w.qtiles * w.qsplit * a.B * a.Hk)), dim3(256), smq, s, p,
                     (int)w.qtiles);
  if (w.qsplit > 1) {
    const long long n = (long long)a.B * a.H * a.Nq * (DP / 4);
    hipLaunchKernelGGL((cross_sum_kernel<CT, DP, VEC>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, p, 0);
  }
  if (!a.dk.p || a.Nk == 0) return hipGetLastError();  // a frozen encoder, or none
  shape(p, w.ktiles, w.ksplit, a.Nk);
  hipLaunchKernelGGL((cross_dkv_kernel<CT, DP, QT, VEC>), dim3((unsigned)(w.ktiles * w.ksplit * a.B * a.Hk)), dim3(256), smk, s, p,
                     (int)w.ktiles);
  if (w.ksplit > 1) {
    const long long n = (long long)a.B * a.Hk * a.Nk * 2 * (DP / 4);
    hipLaunchKernelGGL((cross_sum_kernel<CT, DP, VEC>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, p, 1);
  }
  return hipGetLastError();
}

template <typename CT, bool VEC>
hipError_t by_head(const mdg_attn_cross& a, bool back, void* ws, hipStream_t s) {
  switch (dp_of_head(a.D)) {
    case 32: return back ? bwd<CT, 32, VEC>(a, ws, s) : fwd<CT, 32, VEC>(a, ws, s);
    case 64: return back ? bwd<CT, 64, VEC>(a, ws, s) : fwd<CT, 64, VEC>(a, ws, s);
    default: return back ? bwd<CT, 128, VEC>(a, ws, s) : fwd<CT, 128, VEC>(a, ws, s);
  }
}
template <typename CT>
hipError_t by_layout(const mdg_attn_cross& a, bool back, void* ws, hipStream_t s) {
  return pieces(a, back) ? by_head<CT, true>(a, back, ws, s) : by_head<CT, false>(a, back, ws, s);
}

}  // namespace

// (for either layout: a size query need not know the tensors)
size_t attn_cross_ws_bytes(const mdg_attn_cross& a, bool back) {
  if (back) return bwd_plan(a).bytes;
  const size_t x = fwd_plan(a, false).bytes, y = fwd_plan(a, true).bytes;
  return x > y ? x : y;
}

// Every launch within the 2^32 threads of a grid, and row and key numbers (the last tile's, past the end, and a
// length rounded up to splits) within 31 bits.  (The joins' and sums' grids are small: splits come with
// fewer than 1024 blocks.)
bool attn_cross_grid_ok(const mdg_attn_cross& a, bool back) {
  const long long lim = (1LL << 31) - 8192, blocks = ((1LL << 32) - 1) / 512, bh = (long long)a.B * a.Hk;
  const long long rows = (long long)a.Nq * (a.H / a.Hk);
  if (rows > lim || rows * bh > lim || (long long)a.Nk * bh > lim) return false;
  if (!back) {
    const Plan w = fwd_plan(a, false);  // (the other has half the tiles)
    return w.tiles * w.split * bh <= blocks;
  }
  const BwdPlan w = bwd_plan(a);
  return w.qtiles * w.qsplit * bh <= blocks && w.ktiles * w.ksplit * bh <= blocks;
}

hipError_t attn_cross_launch(const mdg_attn_cross& a, bool back, void* ws, hipStream_t s) {
  return a.dtype == MDG_BF16 ? by_layout<bf16_t>(a, back, ws, s) : by_layout<float>(a, back, ws, s);
}

}  // namespace mdg
