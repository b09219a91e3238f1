// Orthogonalised update of a matrix (the step of a Muon-type optimizer), batched over matrices of one shape:
//
//   X_0 = G / (|G|_F + eps),   A = X X^T,   B = b A + c A^2,   X <- a X + B X,   `steps` times; short side first (G transposed if tall)
//
// which drives every singular value of G towards 1.  Compute-bound: m^2 n + m^3 + 2 m^2 n multiply-adds a step (A and A^2 are symmetric:
// tiles on and above the diagonal are computed, their mirror image is stored with them).
//
// Products run on v_mfma_f32_32x32x16_f16 with f32 accumulation.  f16, not bf16: all singular values stay below 1.3, so range is no
// matter, and its 11 bits leave 1.2e-3 to 1.7e-3 in the result where bf16 operands leave 1e-2.  X itself is kept in f32: a X enters a step
// unrounded, and only the correction B X passes through 16 bits -- with a rounded X the small singular values of a matrix with a few
// large ones drown in the large ones' rounding, amplified 3.4 times a step (measured: 2e-2 instead of 6e-4).  The f16 copies carry a
// power of two S ~ sqrt(max side), exact, which lifts the entries of large matrices (about 1 / S) out of f16's subnormals.
//
// Layout: rows and columns padded to 128 with zeros, which the iteration keeps.  All products have both operands contracted along their
// rows: A = X X^T reads X; A^2 reads A (symmetric); B X reads B and the transposed copy of X that the previous step's epilogue stored.
#include <hip/hip_ext.h>

#include <algorithm>

#include "attn_image.h"
#include "common.h"

namespace mmk {

typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

constexpr int NS_GROUP = 64;      // matrices of one launch (their addresses are kernel arguments)
constexpr int NS_PARTS = 1024;    // partial sums of squares per matrix: at one 64 x 64 tile each, enough workgroups to fill the chip
constexpr int NS_TILE = 128;

struct NsPtrs {
  const void* src[NS_GROUP];
  void* mom[NS_GROUP];
  void* dst[NS_GROUP];
};

struct NsArgs {
  int rows, cols, m, n, mp, np;   // m <= n: short and long side, padded
  int tall;                       // rows > cols: X = G^T
  int64_t rs, cs;                 // element strides of src
  float eps, S, inv_S;
  float ca, cb, cc;
  // workspace, all per matrix
  double* parts;   // [NS_PARTS]
  float* x32;      // [mp][np]
  f16_t* x16;      // [mp][np], times S
  f16_t* xt[2];    // [np][mp], times S: read and written by alternate steps
  f16_t* a16;      // [mp][mp], times S
  f16_t* b16;      // [mp][mp], times S
  // momentum
  float mu;
  int nesterov;
  // the step of the weights
  const float* lr_dev;
  float lr, adjust, weight_decay;
};

__device__ __forceinline__ int64_t ns_src_at(const NsArgs& a, int i, int j) {   // element (i, j) of X in G
  return a.tall ? (int64_t)j * a.rs + (int64_t)i * a.cs : (int64_t)i * a.rs + (int64_t)j * a.cs;
}

// Sum of squares of each matrix as NS_PARTS partials in f64 (no overflow for any f32 entries); with MOM the momentum is moved on first --
// M <- mu M + G, U = G + mu M (nesterov) or M -- and U goes to x32, not normalised yet (through LDS where X is G^T).
template <typename T, bool MOM>
__global__ __launch_bounds__(256) void ns_reduce_kernel(const NsArgs a, const NsPtrs p) {
  __shared__ float tile[MOM ? 64 : 1][65];
  __shared__ double red[256];
  const int mat = blockIdx.y, l = threadIdx.x & 63, w = threadIdx.x >> 6;
  const T* src = reinterpret_cast<const T*>(p.src[mat]);
  float* mom = MOM ? reinterpret_cast<float*>(p.mom[mat]) : nullptr;
  float* x32 = a.x32 + (int64_t)mat * a.mp * a.np;
  const int tr = (a.rows + 63) / 64, tc = (a.cols + 63) / 64;
  const bool by_col = MOM || a.cs <= a.rs;   // a wave reads along the axis that is contiguous in memory
  double sum = 0.0;
  for (int t = blockIdx.x; t < tr * tc; t += NS_PARTS) {
    const int r0 = 64 * (t / tc), c0 = 64 * (t % tc);
    float g[16], mv[16];   // all of a thread's values in flight at once
#pragma unroll
    for (int u = 0; u < 16; ++u) {
      const int k = w + 4 * u, r = r0 + (by_col ? k : l), c = c0 + (by_col ? l : k);
      const bool in = r < a.rows && c < a.cols;
      g[u] = in ? to_f32(src[(int64_t)r * a.rs + (int64_t)c * a.cs]) : 0.f;
      if (MOM) mv[u] = in ? mom[(int64_t)r * a.cols + c] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < 16; ++u) {
      if (MOM) {
        const int k = w + 4 * u, r = r0 + k, c = c0 + l;
        mv[u] = fmaf(a.mu, mv[u], g[u]);
        g[u] = a.nesterov ? fmaf(a.mu, mv[u], g[u]) : mv[u];
        if (a.tall) tile[k][l] = g[u];
        if (r < a.rows && c < a.cols) {
          mom[(int64_t)r * a.cols + c] = mv[u];
          if (!a.tall) x32[(int64_t)r * a.np + c] = g[u];
        }
      }
      sum += (double)g[u] * (double)g[u];
    }
    if (MOM && a.tall) {
      __syncthreads();
      for (int k = w; k < 64; k += 4)
        if (c0 + k < a.cols && r0 + l < a.rows) x32[(int64_t)(c0 + k) * a.np + r0 + l] = tile[l][k];
      __syncthreads();
    }
  }
  red[threadIdx.x] = sum;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if (threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) a.parts[mat * NS_PARTS + blockIdx.x] = red[0];
}

// X = G / (|G| + eps) into x32, x16 and xt[0], zero beyond the matrix.  64 x 64 tiles through LDS for the transposed copy.
template <typename T, bool MOM>
__global__ __launch_bounds__(256) void ns_prepare_kernel(const NsArgs a, const NsPtrs p) {
  __shared__ double red[256];
  __shared__ float tile[64][65];
  const int mat = blockIdx.y, tid = threadIdx.x, l = tid & 63, w = tid >> 6;
  const T* src = reinterpret_cast<const T*>(p.src[mat]);
  const int tn = a.np / 64, i0 = 64 * (blockIdx.x / tn), j0 = 64 * (blockIdx.x % tn);
  float* x32 = a.x32 + (int64_t)mat * a.mp * a.np;
  // read along the axis that is contiguous in memory: j of X, or i
  const bool by_j = MOM || (a.tall ? a.rs <= a.cs : a.cs <= a.rs);
  float v[16];
#pragma unroll
  for (int u = 0; u < 16; ++u) {
    const int k = w + 4 * u, i = i0 + (by_j ? k : l), j = j0 + (by_j ? l : k);
    v[u] = i < a.m && j < a.n ? (MOM ? x32[(int64_t)i * a.np + j] : to_f32(src[ns_src_at(a, i, j)])) : 0.f;
  }
  double sq = 0.0;
  for (int k = tid; k < NS_PARTS; k += 256) sq += a.parts[mat * NS_PARTS + k];
  red[tid] = sq;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if (tid < o) red[tid] += red[tid + o];
    __syncthreads();
  }
  const float inv = (float)(1.0 / (sqrt(red[0]) + (double)a.eps));
#pragma unroll
  for (int u = 0; u < 16; ++u) tile[by_j ? w + 4 * u : l][by_j ? l : w + 4 * u] = v[u] * inv;
  __syncthreads();
  f16_t* x16 = a.x16 + (int64_t)mat * a.mp * a.np;
  f16_t* xt = a.xt[0] + (int64_t)mat * a.mp * a.np;
  for (int k = w; k < 64; k += 4) {
    const float x = tile[k][l];
    x32[(int64_t)(i0 + k) * a.np + j0 + l] = x;
    x16[(int64_t)(i0 + k) * a.np + j0 + l] = (f16_t)(x * a.S);
    xt[(int64_t)(j0 + k) * a.mp + i0 + l] = (f16_t)(tile[l][k] * a.S);
  }
}

enum { NS_XXT = 0, NS_POLY = 1, NS_STEP = 2, NS_LAST = 3 };

// One 128 x 128 tile of P Q^T (contraction along rows of K values), and what the step does with it:
//   NS_XXT   A = P Q^T                      P = Q = X      NS_POLY  B = b A + c P Q^T               P = Q = A      (upper tiles + mirror)
//   NS_STEP  X = a X + P Q^T, f32 and both f16 copies      P = B, Q = X^T
//   NS_LAST  the same, rounded to bf16 into dst, or as the step of the f32 weights
// W: the weights' step instead of the bf16 result
template <int MODE, bool W>
__global__ __launch_bounds__(256, 2) void ns_gemm_kernel(const NsArgs a, const NsPtrs p, int xt_in) {
  extern __shared__ __attribute__((aligned(16))) char smem[];   // 2 stages of P and Q tiles, 16 KiB each
  constexpr int STAGE = 2 * 16384;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 31, hf = lane >> 5, wm = wave >> 1, wn = wave & 1;
  const int mat = blockIdx.y;
  const int64_t mn = (int64_t)a.mp * a.np, mm = (int64_t)a.mp * a.mp;
  int ti, tj;
  if (MODE == NS_XXT || MODE == NS_POLY) {   // tile number -> (ti <= tj)
    tj = (int)((sqrtf(8.f * blockIdx.x + 1.f) - 1.f) * 0.5f);
    while ((tj + 1) * (tj + 2) / 2 <= (int)blockIdx.x) ++tj;
    while (tj * (tj + 1) / 2 > (int)blockIdx.x) --tj;
    ti = blockIdx.x - tj * (tj + 1) / 2;
  } else {
    const int tiles_m = a.mp / NS_TILE;
    ti = blockIdx.x % tiles_m;
    tj = blockIdx.x / tiles_m;
  }
  const f16_t *P, *Q;
  int K;
  if (MODE == NS_XXT) {
    P = Q = a.x16 + mat * mn;
    K = a.np;
  } else if (MODE == NS_POLY) {
    P = Q = a.a16 + mat * mm;
    K = a.mp;
  } else {
    P = a.b16 + mat * mm;
    Q = a.xt[xt_in] + mat * mn;
    K = a.mp;
  }
  P += (int64_t)ti * NS_TILE * K;
  Q += (int64_t)tj * NS_TILE * K;

  uint32_t voff[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int row = 8 * (wave + 4 * u) + (lane >> 3);
    voff[u] = (uint32_t)(row * K + ((lane & 7) ^ img_swz(row & 15)) * 8) * 2u;
  }
  const uint32_t lds0 = lds_addr_of(smem);
  auto issue = [&](int kt) {
    const uint32_t at = lds0 + (uint32_t)((kt & 1) * STAGE);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      lds_dma16(P + 64 * kt, voff[u], at + (uint32_t)((wave + 4 * u) * 1024));
      lds_dma16(Q + 64 * kt, voff[u], at + 16384u + (uint32_t)((wave + 4 * u) * 1024));
    }
  };
  f32x16 acc[2][2];
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[x][y][e] = 0.f;
  const ImgLane il = img_lane(lane);
  const int nk = K / 64;
  issue(0);
  for (int kt = 0; kt < nk; ++kt) {
    __builtin_amdgcn_s_waitcnt(0x0F70);
    __syncthreads();
    if (kt + 1 < nk) issue(kt + 1);
    const char* sp = smem + (kt & 1) * STAGE + wm * 8192;
    const char* sq = smem + (kt & 1) * STAGE + 16384 + wn * 8192;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      f16x8 fp[2], fq[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        fp[x] = *reinterpret_cast<const f16x8*>(sp + x * 4096 + il.row[kk]);
        fq[x] = *reinterpret_cast<const f16x8*>(sq + x * 4096 + il.row[kk]);
      }
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[x], fq[y], acc[x][y], 0, 0, 0);
    }
  }
  // acc[x][y]: row i = 64 wm + 32 x + 8 (e >> 2) + 4 hf + (e & 3), column j = 64 wn + 32 y + r of the tile
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int i = ti * NS_TILE + 64 * wm + 32 * x + 8 * g + 4 * hf, j = tj * NS_TILE + 64 * wn + 32 * y + r;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[x][y][4 * g + e];
        if (MODE == NS_XXT || MODE == NS_POLY) {
          f16_t* out = (MODE == NS_XXT ? a.a16 : a.b16) + mat * mm;
          const f16_t* in = a.a16 + mat * mm;
          f16x4 o;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float t = MODE == NS_XXT ? v[e] * a.inv_S : fmaf(a.cb, (float)in[(int64_t)(i + e) * a.mp + j], v[e] * (a.cc * a.inv_S));
            o[e] = (f16_t)t;
            if (ti != tj) out[(int64_t)(i + e) * a.mp + j] = o[e];
          }
          *reinterpret_cast<f16x4*>(out + (int64_t)j * a.mp + i) = o;   // the mirror image (on the diagonal: the tile itself)
        } else {
          float* x32 = a.x32 + mat * mn;
          const float k2 = a.inv_S * a.inv_S;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = fmaf(a.ca, x32[(int64_t)(i + e) * a.np + j], v[e] * k2);
          if (MODE == NS_STEP) {
            f16x4 o;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              o[e] = (f16_t)(v[e] * a.S);
              x32[(int64_t)(i + e) * a.np + j] = v[e];
              a.x16[mat * mn + (int64_t)(i + e) * a.np + j] = o[e];
            }
            *reinterpret_cast<f16x4*>(a.xt[1 - xt_in] + mat * mn + (int64_t)j * a.mp + i) = o;
          } else if (j < a.n) {
            const float lr = W && a.lr_dev ? *a.lr_dev : a.lr;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (i + e < a.m) {
                const int64_t at = a.tall ? (int64_t)j * a.cols + i + e : (int64_t)(i + e) * a.cols + j;
                if (W) {
                  float* wt = reinterpret_cast<float*>(p.dst[mat]);
                  wt[at] = fmaf(-lr * a.adjust, v[e], wt[at] * (1.f - lr * a.weight_decay));
                } else {
                  reinterpret_cast<bf16_t*>(p.dst[mat])[at] = (bf16_t)v[e];
                }
              }
          }
        }
      }
}

// ------------------------------------------------------------------------------------------------ host
static int64_t ns_up(int64_t v) { return (v + NS_TILE - 1) / NS_TILE * NS_TILE; }
// bytes of one matrix in the workspace
static int64_t ns_bytes(int rows, int cols) {
  const int64_t mp = ns_up(std::min(rows, cols)), np = ns_up(std::max(rows, cols));
  return NS_PARTS * 8 + mp * np * (4 + 2 + 2 * 2) + mp * mp * (2 + 2);
}
// matrices of one pass: as many as 1 GiB of workspace holds, at least one
static int ns_group(int count, int rows, int cols) {
  const int64_t fit = (int64_t(1) << 30) / ns_bytes(rows, cols);
  return (int)std::max<int64_t>(1, std::min<int64_t>({(int64_t)count, (int64_t)NS_GROUP, fit}));
}

template <typename K>
static int ns_launch(K kern, dim3 grid, int lds, hipStream_t st, const NsArgs& a, const NsPtrs& p, int xt_in) {
  KernelSetup ks;
  if (int rc = kernel_setup(reinterpret_cast<const void*>(kern), 256, lds, &ks)) return rc;
  ProfEvents pe(MMK_K_NEWTON_SCHULZ);
  hipExtLaunchKernelGGL(kern, grid, dim3(256), lds, st, pe.start, pe.stop, 0, a, p, xt_in);
  MMK_LAUNCH_CHECK();
  return 0;
}

template <typename T>
static int ns_begin(const NsArgs& a, const NsPtrs& p, int count, bool mom, hipStream_t st) {
  const dim3 rg(NS_PARTS, count), pg((a.mp / 64) * (a.np / 64), count), blk(256);
  if (mom) {
    hipLaunchKernelGGL((ns_reduce_kernel<T, true>), rg, blk, 0, st, a, p);
    MMK_LAUNCH_CHECK();
    hipLaunchKernelGGL((ns_prepare_kernel<T, true>), pg, blk, 0, st, a, p);
  } else {
    hipLaunchKernelGGL((ns_reduce_kernel<T, false>), rg, blk, 0, st, a, p);
    MMK_LAUNCH_CHECK();
    hipLaunchKernelGGL((ns_prepare_kernel<T, false>), pg, blk, 0, st, a, p);
  }
  MMK_LAUNCH_CHECK();
  return 0;
}

static int ns_run(const mmk_newton_schulz_args* q, NsArgs a, const NsPtrs& p, int count, hipStream_t st) {
  const bool mom = q->momenta != nullptr;
  const int rc0 = MMK_DISPATCH_DTYPE(q->dtype, T, [&]() -> int { return ns_begin<T>(a, p, count, mom, st); });
  if (rc0) return rc0;
  const int tm = a.mp / NS_TILE, tn = a.np / NS_TILE, lds = 2 * 2 * 16384;
  const dim3 sym(tm * (tm + 1) / 2, count), full(tm * tn, count);
  for (int s = 0; s < q->steps; ++s) {
    if (int rc = ns_launch(ns_gemm_kernel<NS_XXT, false>, sym, lds, st, a, p, s & 1)) return rc;
    if (int rc = ns_launch(ns_gemm_kernel<NS_POLY, false>, sym, lds, st, a, p, s & 1)) return rc;
    const int rc = s + 1 < q->steps ? ns_launch(ns_gemm_kernel<NS_STEP, false>, full, lds, st, a, p, s & 1)
                   : q->weights     ? ns_launch(ns_gemm_kernel<NS_LAST, true>, full, lds, st, a, p, s & 1)
                                    : ns_launch(ns_gemm_kernel<NS_LAST, false>, full, lds, st, a, p, s & 1);
    if (rc) return rc;
  }
  return 0;
}

static int ns_check(int count, int rows, int cols) {
  MMK_REQUIRE(count >= 0 && rows >= 1 && cols >= 1, "bad sizes");
  MMK_REQUIRE(std::max(rows, cols) <= 32768, "sides up to 32768");   // a tile's rows are addressed by 32-bit byte offsets
  return 0;
}

}  // namespace mmk

using namespace mmk;

extern "C" {

int64_t mmk_newton_schulz_ws_bytes(int count, int rows, int cols) {
  if (ns_check(count, rows, cols)) return -1;
  return count == 0 ? 0 : ns_bytes(rows, cols) * ns_group(count, rows, cols);
}

int mmk_newton_schulz(const mmk_newton_schulz_args* q, void* ws, void* stream) {
  MMK_REQUIRE(q != nullptr, "no arguments");
  if (int rc = ns_check(q->count, q->rows, q->cols)) return rc;
  MMK_REQUIRE(q->steps >= 1 && q->steps <= 32, "1 to 32 steps");
  MMK_REQUIRE(!q->momenta || q->dtype == MMK_F32 || q->dtype == MMK_BF16 || q->dtype == MMK_F16, "unsupported dtype");
  if (q->count == 0) return 0;
  MMK_REQUIRE(q->src && q->dst && ws, "missing operand");
  NsArgs a = {};
  a.rows = q->rows;
  a.cols = q->cols;
  a.tall = q->rows > q->cols;
  a.m = std::min(q->rows, q->cols);
  a.n = std::max(q->rows, q->cols);
  a.mp = (int)ns_up(a.m);
  a.np = (int)ns_up(a.n);
  a.rs = q->row_stride;
  a.cs = q->col_stride;
  a.eps = q->eps;
  a.S = 1.f;
  while (a.S * a.S * 4.f <= (float)a.n) a.S *= 2.f;   // the power of two at or below sqrt(n)
  a.inv_S = 1.f / a.S;
  a.ca = q->coef[0];
  a.cb = q->coef[1];
  a.cc = q->coef[2];
  a.mu = q->momentum;
  a.nesterov = q->nesterov;
  a.lr_dev = q->lr_dev;
  a.lr = q->lr;
  a.adjust = q->adjust;
  a.weight_decay = q->weight_decay;
  const int group = ns_group(q->count, q->rows, q->cols);
  const int64_t mn = (int64_t)a.mp * a.np, mm = (int64_t)a.mp * a.mp;
  char* w = reinterpret_cast<char*>(ws);
  auto take = [&](int64_t bytes) {
    char* at = w;
    w += bytes * group;
    return at;
  };
  a.x32 = (float*)take(mn * 4);
  a.x16 = (f16_t*)take(mn * 2);
  a.xt[0] = (f16_t*)take(mn * 2);
  a.xt[1] = (f16_t*)take(mn * 2);
  a.a16 = (f16_t*)take(mm * 2);
  a.b16 = (f16_t*)take(mm * 2);
  a.parts = (double*)take(NS_PARTS * 8);
  for (int at = 0; at < q->count; at += group) {
    const int n = std::min(group, q->count - at);
    NsPtrs p = {};
    for (int i = 0; i < n; ++i) {
      p.src[i] = q->src[at + i];
      p.mom[i] = q->momenta ? q->momenta[at + i] : nullptr;
      p.dst[i] = q->dst[at + i];
    }
    if (int rc = ns_run(q, a, p, n, (hipStream_t)stream)) return rc;
  }
  return 0;
}

}  // extern "C"
