// Per-head RMS norm of queries and keys with the position rotation in the same pass, and its backward.
//
//   n = x / sqrt(mean(x^2) + eps),   y = R(pos) (w n)        x: one head of one token, D values
//   R turns the pairs of the first `rot` columns: (a, b) -> (a c - b s, b c + a s) with c, s of (pos, pair) from a f32 table
//   backward:  g = R^T dy,  dw = sum g n,  dx = (g w - n mean(g w n)) / sqrt(mean(x^2) + eps)
//
// HBM-bound: forward reads x and writes y, backward reads x and dy and writes dx (the norm is made again from x: nothing is saved).
// One lane owns V PAIRS of a head (2 V values), so the rotation is lane-local in both pair layouts and each access is 16 bytes for
// V = 8; the LPR lanes of a head exchange one sum forward, two backward.  Rows (token, head) of one side follow each other, so the
// lanes of a wave cover heads of one token and share its angles.  Everything is f32 between the load and the one rounding at the store.
// The weight gradient is summed in registers over the rows a workgroup walks, through LDS over its lane groups, and by a second
// kernel over the workgroups: a fixed order, no atomics.
// 256 x 197 tokens, 12 + 12 heads of 64, bf16: forward 76 us (4.1 TB/s), backward 102 us (4.6 TB/s) and 5 us for the sums over workgroups; f32:
// 131 us (4.7 TB/s) and 181 (5.1).
#include <hip/hip_ext.h>

#include <algorithm>

#include "common.h"

namespace mmk {

constexpr int QKN_THREADS = 256;
constexpr int QKN_MAX_BLOCKS = 1024;   // workgroups per side of the persistent backward = rows of a side's weight-gradient partials

struct QkSide {
  const void* x;
  const void* w;    // [D], may be null (ones)
  void* y;          // forward: [B, L, H, D] contiguous
  const void* dy;   // backward: strided like x, own strides
  void* dx;         // backward: [B, L, H, D] contiguous
  float* part;      // backward: [blocks][D] partial sums of dw; null: dw is not wanted
  void* dw;
  int64_t sb, sl, sh;      // element strides of x
  int64_t gsb, gsl, gsh;   // element strides of dy
  int H, blocks;
};

struct QkArgs {
  QkSide s[2];
  const float* tab;   // [tab_rows][rot]: rot / 2 cosines, rot / 2 sines
  const void* pos;    // null: 0 .. L-1
  int64_t pos_sb;
  int pos64;
  int B, L, D, rot, tab_rows, lpr_log2;
  float eps;
};

template <typename T, int V>
struct QkVec {
  typedef T vec __attribute__((ext_vector_type(V)));
  struct __attribute__((packed, aligned(V * sizeof(T) < 16 ? V * sizeof(T) : 16))) mem { T e[V]; };
  static __device__ __forceinline__ void load(const T* p, float (&o)[V]) {
    const mem m = *reinterpret_cast<const mem*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = to_f32(m.e[i]);
  }
  static __device__ __forceinline__ void store(T* p, const float (&o)[V]) {
    mem m;
#pragma unroll
    for (int i = 0; i < V; ++i) m.e[i] = from_f32<T>(o[i]);
    *reinterpret_cast<mem*>(p) = m;
  }
};

// The two V-vectors of a lane's pairs p0 .. p0 + V - 1.  Split halves: (p, p + rot/2) in the rotated part, the rest paired likewise
// (its pairing is free).  Interleaved: 2 V consecutive values, taken apart in registers.
template <bool ILV>
__device__ __forceinline__ void qk_pair_offsets(int p0, int V, int D, int rot, int& lo, int& hi) {
  if (ILV) {
    lo = 2 * p0;
    hi = lo + V;
  } else if (2 * p0 < rot) {
    lo = p0;
    hi = p0 + rot / 2;
  } else {
    lo = rot / 2 + p0;
    hi = lo + (D - rot) / 2;
  }
}
template <bool ILV, int V>
__device__ __forceinline__ void qk_split(const float (&a)[V], const float (&b)[V], float (&u)[V], float (&w)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = 2 * i;
    u[i] = ILV ? (e < V ? a[e % V] : b[e % V]) : a[i];
    w[i] = ILV ? (e + 1 < V ? a[(e + 1) % V] : b[(e + 1) % V]) : b[i];
  }
}
template <bool ILV, int V>
__device__ __forceinline__ void qk_join(const float (&u)[V], const float (&w)[V], float (&a)[V], float (&b)[V]) {
#pragma unroll
  for (int e = 0; e < 2 * V; ++e) {
    const float v = ILV ? ((e & 1) ? w[e / 2] : u[e / 2]) : (e < V ? u[e % V] : w[e % V]);
    if (e < V) a[e % V] = v;
    else b[e % V] = v;
  }
}

__device__ __forceinline__ float qk_group_sum(float v, int lpr_log2) {
  for (int o = 0; o < lpr_log2; ++o) v += __shfl_xor(v, 1 << o);
  return v;
}

// angle of a row: its position, or -1 where the position is not in the table
__device__ __forceinline__ int qk_position(const QkArgs& a, int tok) {
  int64_t p;
  if (a.pos == nullptr) {
    p = tok % a.L;
  } else {
    const int64_t at = (int64_t)(tok / a.L) * a.pos_sb + tok % a.L;
    p = a.pos64 ? reinterpret_cast<const int64_t*>(a.pos)[at] : reinterpret_cast<const int32_t*>(a.pos)[at];
  }
  return p >= 0 && p < a.tab_rows ? (int)p : -1;
}

// CP: chunks of V pairs per lane (2 only for heads too odd for vectors and wider than 128)
template <typename T, typename W, int V, int CP, bool ILV, bool BWD>
__global__ __launch_bounds__(QKN_THREADS) void qk_norm_kernel(const QkArgs a) {
  __shared__ float red[BWD ? 16 * QKN_THREADS : 1];
  const int side = (int)blockIdx.x < a.s[0].blocks ? 0 : 1;
  const QkSide& s = a.s[side];
  const int blk = blockIdx.x - (side ? a.s[0].blocks : 0);
  const int lpr = 1 << a.lpr_log2, grp = threadIdx.x >> a.lpr_log2, li = threadIdx.x & (lpr - 1), rpb = QKN_THREADS >> a.lpr_log2;
  const int rows = a.B * a.L * s.H;
  int lo[CP], hi[CP];
  bool in[CP];
  float w0[CP][V], w1[CP][V], s0[CP][V], s1[CP][V];
#pragma unroll
  for (int c = 0; c < CP; ++c) {
    const int p0 = (li + c * lpr) * V;
    in[c] = 2 * p0 < a.D;
    qk_pair_offsets<ILV>(in[c] ? p0 : 0, V, a.D, a.rot, lo[c], hi[c]);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      w0[c][i] = s.w ? to_f32(reinterpret_cast<const W*>(s.w)[lo[c] + i]) : 1.f;
      w1[c][i] = s.w ? to_f32(reinterpret_cast<const W*>(s.w)[hi[c] + i]) : 1.f;
      s0[c][i] = s1[c][i] = 0.f;
    }
  }
  const float inv_d = 1.f / (float)a.D;
  // every lane group walks the same number of rows, so that the exchanges below always have all lanes of a wave
  for (int r0 = blk * rpb; r0 < rows; r0 += s.blocks * rpb) {
    const int row = min(r0 + grp, rows - 1);
    const bool live = r0 + grp < rows;
    const int tok = row / s.H, head = row - tok * s.H;
    const int bi = tok / a.L, l = tok - bi * a.L;
    const T* x = reinterpret_cast<const T*>(s.x) + bi * s.sb + l * s.sl + head * s.sh;
    float x0[CP][V], x1[CP][V], ss = 0.f;
#pragma unroll
    for (int c = 0; c < CP; ++c) {
      QkVec<T, V>::load(x + lo[c], x0[c]);
      QkVec<T, V>::load(x + hi[c], x1[c]);
#pragma unroll
      for (int i = 0; i < V; ++i) ss += in[c] ? x0[c][i] * x0[c][i] + x1[c][i] * x1[c][i] : 0.f;
    }
    float g0[CP][V], g1[CP][V];
    if (BWD) {
      const T* dy = reinterpret_cast<const T*>(s.dy) + bi * s.gsb + l * s.gsl + head * s.gsh;
#pragma unroll
      for (int c = 0; c < CP; ++c) {
        QkVec<T, V>::load(dy + lo[c], g0[c]);
        QkVec<T, V>::load(dy + hi[c], g1[c]);
      }
    }
    const int pos = a.rot ? qk_position(a, tok) : 0;
    float cs[CP][V], sn[CP][V];
#pragma unroll
    for (int c = 0; c < CP; ++c) {
      const int p0 = (li + c * lpr) * V;
      const bool turned = 2 * p0 < a.rot;
      if (turned && pos >= 0) {
        const float* t = a.tab + (int64_t)pos * a.rot + p0;
        QkVec<float, V>::load(t, cs[c]);
        QkVec<float, V>::load(t + a.rot / 2, sn[c]);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          cs[c][i] = pos < 0 ? __builtin_nanf("") : 1.f;   // a position that the table does not hold: the whole row becomes NaN
          sn[c][i] = 0.f;
        }
      }
    }
    const float rstd = 1.f / sqrtf(qk_group_sum(ss, a.lpr_log2) * inv_d + a.eps);
    if (!BWD) {
      T* y = reinterpret_cast<T*>(s.y) + (int64_t)row * a.D;
#pragma unroll
      for (int c = 0; c < CP; ++c) {
        float o0[V], o1[V], u[V], v[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          o0[i] = x0[c][i] * rstd * w0[c][i];
          o1[i] = x1[c][i] * rstd * w1[c][i];
        }
        qk_split<ILV, V>(o0, o1, u, v);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float uu = u[i] * cs[c][i] - v[i] * sn[c][i], vv = v[i] * cs[c][i] + u[i] * sn[c][i];
          u[i] = uu;
          v[i] = vv;
        }
        qk_join<ILV, V>(u, v, o0, o1);
        if (live && in[c]) {
          QkVec<T, V>::store(y + lo[c], o0);
          QkVec<T, V>::store(y + hi[c], o1);
        }
      }
    } else {
      float dot = 0.f;
#pragma unroll
      for (int c = 0; c < CP; ++c) {
        float u[V], v[V];
        qk_split<ILV, V>(g0[c], g1[c], u, v);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float uu = u[i] * cs[c][i] + v[i] * sn[c][i], vv = v[i] * cs[c][i] - u[i] * sn[c][i];
          u[i] = uu;
          v[i] = vv;
        }
        qk_join<ILV, V>(u, v, g0[c], g1[c]);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          x0[c][i] *= rstd;
          x1[c][i] *= rstd;
          s0[c][i] += live ? g0[c][i] * x0[c][i] : 0.f;
          s1[c][i] += live ? g1[c][i] * x1[c][i] : 0.f;
          g0[c][i] *= w0[c][i];
          g1[c][i] *= w1[c][i];
          dot += in[c] ? g0[c][i] * x0[c][i] + g1[c][i] * x1[c][i] : 0.f;
        }
      }
      dot = qk_group_sum(dot, a.lpr_log2) * inv_d;
      T* dx = reinterpret_cast<T*>(s.dx) + (int64_t)row * a.D;
#pragma unroll
      for (int c = 0; c < CP; ++c) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          g0[c][i] = rstd * (g0[c][i] - x0[c][i] * dot);
          g1[c][i] = rstd * (g1[c][i] - x1[c][i] * dot);
        }
        if (live && in[c]) {
          QkVec<T, V>::store(dx + lo[c], g0[c]);
          QkVec<T, V>::store(dx + hi[c], g1[c]);
        }
      }
    }
  }
  if (BWD && s.part != nullptr) {   // D / LPR <= 16: the lane groups' sums fit
#pragma unroll
    for (int c = 0; c < CP; ++c)
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (in[c]) {
          red[grp * a.D + lo[c] + i] = s0[c][i];
          red[grp * a.D + hi[c] + i] = s1[c][i];
        }
    __syncthreads();
    for (int d = threadIdx.x; d < a.D; d += QKN_THREADS) {
      float t = 0.f;
      for (int g = 0; g < rpb; ++g) t += red[g * a.D + d];
      s.part[(int64_t)blk * a.D + d] = t;
    }
  }
}

// dw[d] = sum over the workgroups' partials: 8 columns and 32 row slices a workgroup, each slice in order, the slices joined in order
template <typename W>
__global__ __launch_bounds__(256) void qk_norm_dw_kernel(const QkArgs a) {
  __shared__ float red[32][8];
  const QkSide& s = a.s[blockIdx.y];
  if (s.part == nullptr) return;
  const int col = threadIdx.x & 7, sl = threadIdx.x >> 3, d = blockIdx.x * 8 + col;
  float t = 0.f;
  if (d < a.D) {
#pragma unroll 8
    for (int r = sl; r < s.blocks; r += 32) t += s.part[(int64_t)r * a.D + d];
  }
  red[sl][col] = t;
  __syncthreads();
  if (sl == 0 && d < a.D) {
    for (int k = 1; k < 32; ++k) t += red[k][col];
    reinterpret_cast<W*>(s.dw)[d] = from_f32<W>(t);
  }
}

static bool qk_vec_ok(const QkArgs& a, int V, size_t es, bool bwd) {
  if ((a.rot / 2) % V || ((a.D - a.rot) / 2) % V) return false;
  const size_t al = std::min<size_t>(16, V * es);
  auto ptr_ok = [&](const void* p) { return reinterpret_cast<uintptr_t>(p) % al == 0; };
  if (a.rot && reinterpret_cast<uintptr_t>(a.tab) % 16) return false;
  for (const QkSide& s : a.s) {
    if (!s.H) continue;
    if (s.sb % V || s.sl % V || s.sh % V || !ptr_ok(s.x) || !ptr_ok(bwd ? s.dx : s.y)) return false;
    if (bwd && (s.gsb % V || s.gsl % V || s.gsh % V || !ptr_ok(s.dy))) return false;
  }
  return true;
}

// rows of partials a side needs: enough workgroups to fill the chip four times over, fewer where there are not that many rows
static int qk_bwd_blocks(int64_t rows, int D) {
  return (int)std::min<int64_t>(QKN_MAX_BLOCKS, (rows * std::max(D / 16, 1) + QKN_THREADS - 1) / QKN_THREADS);
}

template <typename T, typename W, int V, int CP>
static int qk_launch(const QkArgs& a, bool ilv, bool bwd, hipStream_t st) {
  const dim3 grid(a.s[0].blocks + a.s[1].blocks), blk(QKN_THREADS);
  ProfEvents pe(MMK_K_QK_NORM);
  auto go = [&](auto kern) { hipExtLaunchKernelGGL(kern, grid, blk, 0, st, pe.start, pe.stop, 0, a); };
  if (bwd) ilv ? go(qk_norm_kernel<T, W, V, CP, true, true>) : go(qk_norm_kernel<T, W, V, CP, false, true>);
  else ilv ? go(qk_norm_kernel<T, W, V, CP, true, false>) : go(qk_norm_kernel<T, W, V, CP, false, false>);
  MMK_LAUNCH_CHECK();
  if (bwd && (a.s[0].part || a.s[1].part)) {
    hipLaunchKernelGGL((qk_norm_dw_kernel<W>), dim3((a.D + 7) / 8, 2), dim3(256), 0, st, a);
    MMK_LAUNCH_CHECK();
  }
  return 0;
}

template <typename T, typename W>
static int qk_run(QkArgs& a, bool ilv, bool bwd, hipStream_t st) {
  const int V = qk_vec_ok(a, 8, sizeof(T), bwd) ? 8 : qk_vec_ok(a, 4, sizeof(T), bwd) ? 4 : 1;
  const int chunks = a.D / 2 / V;
  a.lpr_log2 = 0;
  while ((1 << a.lpr_log2) < chunks && a.lpr_log2 < 6) ++a.lpr_log2;
  const int rpb = QKN_THREADS >> a.lpr_log2;
  for (QkSide& s : a.s) {
    const int64_t need = ((int64_t)a.B * a.L * s.H + rpb - 1) / rpb;
    s.blocks = (int)std::min<int64_t>(need, bwd ? s.blocks : QKN_MAX_BLOCKS);
  }
  if (V == 8) return qk_launch<T, W, 8, 1>(a, ilv, bwd, st);
  if (V == 4) return qk_launch<T, W, 4, 1>(a, ilv, bwd, st);
  return chunks > 64 ? qk_launch<T, W, 1, 2>(a, ilv, bwd, st) : qk_launch<T, W, 1, 1>(a, ilv, bwd, st);
}

template <typename T>
static int qk_run_w(QkArgs& a, int dtype, int w_dtype, bool ilv, bool bwd, hipStream_t st) {
  return w_dtype == MMK_F32 && dtype != MMK_F32 ? qk_run<T, float>(a, ilv, bwd, st) : qk_run<T, T>(a, ilv, bwd, st);
}

static int qk_check(const QkArgs& a, int dtype, int w_dtype) {
  MMK_REQUIRE(a.B >= 0 && a.L >= 0 && a.s[0].H >= 0 && a.s[1].H >= 0, "negative size");
  MMK_REQUIRE(a.D >= 2 && a.D <= 256 && a.D % 2 == 0, "head dim must be even and at most 256");
  MMK_REQUIRE(a.rot >= 0 && a.rot <= a.D && a.rot % 2 == 0, "the rotated width must be even and at most the head dim");
  MMK_REQUIRE(a.rot == 0 || a.tab != nullptr, "a rotation needs its table");
  MMK_REQUIRE(a.rot == 0 || a.pos != nullptr || a.L <= a.tab_rows, "the table holds fewer positions than the sequence");
  MMK_REQUIRE((int64_t)a.B * a.L * std::max(a.s[0].H, a.s[1].H) < (int64_t(1) << 30), "too many rows");
  MMK_REQUIRE(w_dtype == MMK_F32 || w_dtype == dtype, "weights are f32 or of the operands' type");
  return 0;
}

static void qk_fill(QkArgs& a, const float* tab, int tab_rows, const void* pos, int pos64, int64_t pos_sb, int B, int L, int H, int Hk, int D,
                    int rot, float eps) {
  a.tab = tab;
  a.tab_rows = tab_rows;
  a.pos = pos;
  a.pos64 = pos64;
  a.pos_sb = pos_sb;
  a.B = B;
  a.L = L;
  a.D = D;
  a.rot = rot;
  a.eps = eps;
  a.s[0].H = H;
  a.s[1].H = Hk;
}

}  // namespace mmk

using namespace mmk;

extern "C" {

int mmk_qk_norm_rotary_fwd(const void* q, const void* k, const void* qw, const void* kw, const float* table, int table_rows,
                           const void* positions, int pos64, int64_t pos_sb, void* qo, void* ko, int B, int L, int H, int Hk, int D, int rot,
                           int interleaved, const int64_t* q_strides, const int64_t* k_strides, float eps, int dtype, int w_dtype, void* stream) {
  QkArgs a = {};
  qk_fill(a, table, table_rows, positions, pos64, pos_sb, B, L, H, Hk, D, rot, eps);
  if (int rc = qk_check(a, dtype, w_dtype)) return rc;
  if ((int64_t)B * L * (H + Hk) == 0) return 0;
  const void* x[2] = {q, k};
  const void* w[2] = {qw, kw};
  void* y[2] = {qo, ko};
  const int64_t* st[2] = {q_strides, k_strides};
  for (int i = 0; i < 2; ++i) {
    MMK_REQUIRE(st[i] && (a.s[i].H == 0 || (x[i] && y[i])), "missing operand");
    a.s[i].x = x[i];
    a.s[i].w = w[i];
    a.s[i].y = y[i];
    a.s[i].sb = st[i][0];
    a.s[i].sl = st[i][1];
    a.s[i].sh = st[i][2];
  }
  return MMK_DISPATCH_DTYPE(dtype, T, [&]() -> int { return qk_run_w<T>(a, dtype, w_dtype, interleaved != 0, false, (hipStream_t)stream); });
}

int mmk_qk_norm_rotary_part_rows(int64_t rows, int D) { return qk_bwd_blocks(rows, D); }

int mmk_qk_norm_rotary_bwd(const void* q, const void* k, const void* qw, const void* kw, const float* table, int table_rows,
                           const void* positions, int pos64, int64_t pos_sb, const void* dqo, const void* dko, void* dq, void* dk, void* dqw,
                           void* dkw, float* q_part, float* k_part, int B, int L, int H, int Hk, int D, int rot, int interleaved,
                           const int64_t* q_strides, const int64_t* k_strides, const int64_t* dq_strides, const int64_t* dk_strides, float eps,
                           int dtype, int w_dtype, void* stream) {
  QkArgs a = {};
  qk_fill(a, table, table_rows, positions, pos64, pos_sb, B, L, H, Hk, D, rot, eps);
  if (int rc = qk_check(a, dtype, w_dtype)) return rc;
  MMK_REQUIRE((q_part == nullptr) == (dqw == nullptr) && (k_part == nullptr) == (dkw == nullptr), "a weight gradient needs its partials");
  if ((int64_t)B * L * (H + Hk) == 0) return 0;   // (the caller's weight gradients of no rows: zeros it makes itself)
  const void* x[2] = {q, k};
  const void* w[2] = {qw, kw};
  const void* g[2] = {dqo, dko};
  void* dx[2] = {dq, dk};
  void* dw[2] = {dqw, dkw};
  float* part[2] = {q_part, k_part};
  const int64_t* st[2] = {q_strides, k_strides};
  const int64_t* gst[2] = {dq_strides, dk_strides};
  for (int i = 0; i < 2; ++i) {
    QkSide& s = a.s[i];
    MMK_REQUIRE(st[i] && gst[i] && (s.H == 0 || (x[i] && g[i] && dx[i])), "missing operand");
    s.x = x[i];
    s.w = w[i];
    s.dy = g[i];
    s.dx = dx[i];
    s.dw = dw[i];
    s.part = part[i];
    s.sb = st[i][0];
    s.sl = st[i][1];
    s.sh = st[i][2];
    s.gsb = gst[i][0];
    s.gsl = gst[i][1];
    s.gsh = gst[i][2];
    s.blocks = qk_bwd_blocks((int64_t)B * L * s.H, D);
  }
  return MMK_DISPATCH_DTYPE(dtype, T, [&]() -> int { return qk_run_w<T>(a, dtype, w_dtype, interleaved != 0, true, (hipStream_t)stream); });
}

}  // extern "C"
