// Orthogonalised update of a matrix (the step of a Muon-type optimizer), batched over matrices of one shape:
//
//   X_0 = G / (|G|_F + eps),   A = X X^T,   B = b A + c A^2,   X <- a X + B X,   `steps` times; short side first (G transposed if tall)
//
// which drives every singular value of G towards 1.  Compute-bound: m^2 n + m^3 + 2 m^2 n multiply-adds a step (A and A^2 are symmetric:
// tiles on and above the diagonal are computed, their mirror image is stored with them).
//
// Products run on v_mfma_f32_32x32x16_f16 with f32 accumulation.  f16, not bf16: all singular values stay below 1.3, so range is no
// matter, and its 11 bits leave 5e-4 in the result where bf16 operands leave 1e-2.  X itself is kept in more: in f32 where it stays on chip, else
// in two f16 parts (layout below).  a X enters a step from there, and only the correction B X passes through 16 bits -- with a rounded X the
// small singular values of a matrix with a few large ones drown in the large ones' rounding, amplified 3.4 times a step (measured: 2e-2 instead of 6e-4).  The diagonals of A and B, which
// come to hold nearly all of them, are kept in f32 beside the operands and enter as A^2 = E^2 + D E + E D + D^2 and B X = E X + D X (with
// rounded diagonals the result is off by 1.5e-3 to 1.9e-3).  The f16 copies carry a
// power of two S ~ sqrt(max side), exact, which lifts the entries of large matrices (about 1 / S) out of f16's subnormals.
//
// Layout: sides padded with zeros, which the iteration keeps.  X is stored transposed, [n][m], as two f16 arrays: the operand S X rounded, and
// the rest S X - that, kept between steps: together 22 bits where the rest is a normal f16, else S X to 2^-25
// (about 19 bits of the first X of a 4096 x 4096 matrix, where S X is near 2^-6).  A step moves 8 bytes an element: the transposed copy serves
// both products
// -- B X takes its rows, X X^T contracts along its columns with transposed LDS reads -- and its epilogue is in place.
#include <float.h>
#include <hip/hip_ext.h>

#include <algorithm>

#include "attn_image.h"
#include "common.h"

namespace mmk {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

constexpr int NS_GROUP = 64;      // matrices of one launch (their addresses are kernel arguments)
constexpr int NS_PARTS = 1024;    // most partial sums of squares per matrix: a workgroup each, which takes one 64 x 64 tile or more

struct NsPtrs {
  const void* src[NS_GROUP];
  void* mom[NS_GROUP];
  void* dst[NS_GROUP];
};

struct NsArgs {
  int rows, cols, m, n, mp, np;   // m <= n: short and long side, padded
  int tall;                       // rows > cols: X = G^T
  int flat;                       // every src is a run of rows * cols values from an aligned address
  int64_t rs, cs;                 // element strides of src
  float eps, S, inv_S;
  float ca, cb, cc;
  // workspace, all per matrix
  double* parts;   // [NS_PARTS]
  float* u32;      // momentum: the update before it is normalised, [np][mp] (X^T); shares its memory with xt[1] and a16
  f16_t* xt[2];    // X^T [np][mp], times S, rounded: read and written by alternate steps
  f16_t* xl;       // what the rounding left
  f16_t* a16;      // [mp][mp], times S, the diagonal zero
  f16_t* b16;      // [mp][mp], times S, the diagonal zero
  float* diag_a;   // [mp] the diagonals, times S, in f32
  float* diag_b;
  // momentum
  float mu;
  int nesterov;
  // the step of the weights
  const float* lr_dev;
  float lr, adjust, weight_decay;
};

// moves the momentum on and returns the update
__device__ __forceinline__ float ns_momentum(const NsArgs& a, float& m, float g) {
  m = fmaf(a.mu, m, g);
  return a.nesterov ? fmaf(a.mu, m, g) : m;
}
// one weight's step; `lr` in f32 as it stands in the device word
__device__ __forceinline__ float ns_weight(const NsArgs& a, float lr, float w, float x) {
  return fmaf(-lr * a.adjust, x, w * (1.f - lr * a.weight_decay));
}

__device__ __forceinline__ int64_t ns_src_at(const NsArgs& a, int i, int j) {   // element (i, j) of X in G
  return a.tall ? (int64_t)j * a.rs + (int64_t)i * a.cs : (int64_t)i * a.rs + (int64_t)j * a.cs;
}

// how many partial sums a matrix has
__host__ __device__ __forceinline__ int ns_parts(const NsArgs& a) {
  const int tiles = ((a.rows + 63) / 64) * ((a.cols + 63) / 64);
  return tiles < NS_PARTS ? tiles : NS_PARTS;
}
// sum over a workgroup of four waves, the same in every thread; `red`: four doubles of LDS
__device__ __forceinline__ double ns_block_sum(double x, double* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

// Sum of squares of each matrix as ns_parts partials in f64 (no overflow for any f32 entries); with MOM the momentum is moved on first --
// M <- mu M + G, U = G + mu M (nesterov) or M -- and U^T goes to u32 in X^T's layout, not normalised yet (through LDS where that is U^T).
template <typename T, bool MOM>
__global__ __launch_bounds__(256) void ns_reduce_kernel(const NsArgs a, const NsPtrs p) {
  __shared__ float tile[MOM ? 64 : 1][65];
  __shared__ double red[4];
  const int mat = blockIdx.y, l = threadIdx.x & 63, w = threadIdx.x >> 6;
  const T* src = reinterpret_cast<const T*>(p.src[mat]);
  float* mom = MOM ? reinterpret_cast<float*>(p.mom[mat]) : nullptr;
  float* u32 = MOM ? a.u32 + (int64_t)mat * a.mp * a.np : nullptr;
  const int tr = (a.rows + 63) / 64, tc = (a.cols + 63) / 64;
  const bool by_col = MOM || a.cs <= a.rs;   // a wave reads along the axis that is contiguous in memory
  double sum = 0.0;
  if (!MOM && a.flat) {   // the order does not matter: 4096 values at a time, 16 bytes a lane (12 x 2304 x 768 f32: 15 us, tile by tile 36)
    constexpr int V = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(V)));
    const int64_t n = (int64_t)a.rows * a.cols;
    for (int64_t at = (int64_t)blockIdx.x * 4096 + threadIdx.x * V; at < n; at += (int64_t)gridDim.x * 4096) {
      vec g[16 / V];
#pragma unroll
      for (int u = 0; u < 16 / V; ++u) {
        const int64_t x = at + u * 256 * V;
        if (x + V <= n) {
          g[u] = *reinterpret_cast<const vec*>(src + x);
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) g[u][e] = x + e < n ? src[x + e] : (T)0.f;
        }
      }
#pragma unroll
      for (int u = 0; u < 16 / V; ++u)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const double v = (double)to_f32(g[u][e]);
          sum += v * v;
        }
    }
  } else for (int t = blockIdx.x; t < tr * tc; t += gridDim.x) {
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
        g[u] = ns_momentum(a, mv[u], g[u]);
        if (!a.tall) tile[k][l] = g[u];
        if (r < a.rows && c < a.cols) {
          mom[(int64_t)r * a.cols + c] = mv[u];
          if (a.tall) u32[(int64_t)r * a.mp + c] = g[u];
        }
      }
      sum += (double)g[u] * (double)g[u];
    }
    if (MOM && !a.tall) {
      __syncthreads();
      for (int k = w; k < 64; k += 4)
        if (c0 + k < a.cols && r0 + l < a.rows) u32[(int64_t)(c0 + k) * a.mp + r0 + l] = tile[l][k];
      __syncthreads();
    }
  }
  sum = ns_block_sum(sum, red);
  if (threadIdx.x == 0) a.parts[mat * NS_PARTS + blockIdx.x] = sum;
}

// values at any element's address as one vector of 16 bytes
template <typename T>
struct NsVec {
  static constexpr int V = 16 / sizeof(T);
  struct __attribute__((packed, aligned(sizeof(T)))) mem {
    T e[V];
  };
  static __device__ __forceinline__ mem load(const T* p) { return *reinterpret_cast<const mem*>(p); }
  static __device__ __forceinline__ void store(T* p, const mem& m) { *reinterpret_cast<mem*>(p) = m; }
};

// X^T = G^T / (|G| + eps) as xt[0] and xl, zero beyond the matrix.  64 x 64 tiles, through LDS where G is read along the other axis.  16-bit values of a
// unit stride are read 16 bytes a lane (3 x 1000 x 1777 bf16: 15 us, 18 one by one); f32 ones, whose lines are whole anyway, one by one (12 x
// 2304 x 768: 31 us, 34 in vectors).
template <typename T, bool MOM>
__global__ __launch_bounds__(256) void ns_prepare_kernel(const NsArgs a, const NsPtrs p) {
  __shared__ double red[4];
  __shared__ float tile[64][65];   // [j][i]
  const int mat = blockIdx.y, tid = threadIdx.x, l = tid & 63, w = tid >> 6;
  const T* src = reinterpret_cast<const T*>(p.src[mat]);
  const int64_t mn = (int64_t)a.mp * a.np;
  const int tm = a.mp / 64, j0 = 64 * (blockIdx.x / tm), i0 = 64 * (blockIdx.x % tm);
  // read along the axis that is contiguous in memory: i (the short side) or j
  const bool by_i = MOM || (a.tall ? a.cs <= a.rs : a.rs <= a.cs);
  const bool unit = !MOM && sizeof(T) == 2 && min(a.rs, a.cs) == 1;
  typedef NsVec<T> vec;
  constexpr int V = vec::V, LINE = 64 / V;   // lanes of a line of the tile
  float v[16];
#pragma unroll
  for (int u = 0; u < 16; ++u) {   // unit: vector u / V, element u % V
    const int line = unit ? tid / LINE + (u / V) * (256 / LINE) : w + 4 * u, at = unit ? tid % LINE * V : l;
    const int i = i0 + (by_i ? at : line), j = j0 + (by_i ? line : at);
    if (!unit) {
      v[u] = i < a.m && j < a.n ? (MOM ? a.u32[mat * mn + (int64_t)j * a.mp + i] : to_f32(src[ns_src_at(a, i, j)])) : 0.f;
    } else if (u % V == 0) {
      const bool in = i < a.m && j < a.n;
      const int left = by_i ? a.m - i : a.n - j;
      const T* p = src + (in ? ns_src_at(a, i, j) : 0);
      typename vec::mem x;
      if (in && left >= V) {
        x = vec::load(p);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) x.e[e] = in && e < left ? p[e] : (T)0.f;
      }
#pragma unroll
      for (int e = 0; e < V; ++e) v[u + e] = to_f32(x.e[e]);
    }
  }
  double sq = 0.0;
  for (int k = tid; k < ns_parts(a); k += 256) sq += a.parts[mat * NS_PARTS + k];
  sq = ns_block_sum(sq, red);
  const float inv = (float)(1.0 / (sqrt(sq) + (double)a.eps));
#pragma unroll
  for (int u = 0; u < 16; ++u) {
    const int line = unit ? tid / LINE + (u / V) * (256 / LINE) : w + 4 * u, at = unit ? tid % LINE * V + u % V : l;
    tile[by_i ? line : at][by_i ? at : line] = v[u] * inv * a.S;
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < 4; ++u) {   // four values a lane, four rows a wave
    const int k = 16 * u + 4 * w + (l >> 4), i = 4 * (l & 15);
    const int64_t at = mat * mn + (int64_t)(j0 + k) * a.mp + i0 + i;
    f16x4 hi, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = tile[k][i + e];
      hi[e] = (f16_t)x;
      lo[e] = (f16_t)(x - (float)hi[e]);
    }
    *reinterpret_cast<f16x4*>(a.xt[0] + at) = hi;
    *reinterpret_cast<f16x4*>(a.xl + at) = lo;
  }
}

enum { NS_XXT = 0, NS_POLY = 1, NS_STEP = 2, NS_LAST = 3, NS_WEIGHTS = 4 };

// s_waitcnt vmcnt(N) as a builtin; the loop below holds no other load than the LDS-DMA it counts
template <int N>
__device__ __forceinline__ void ns_wait_loads() {
  __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14));
}

// eight values of X at (row, col ..) of the result
template <int MODE>
__device__ __forceinline__ void ns_result(const NsArgs& a, void* dst, int row, int col, const float (&v)[8]) {
  if (row >= a.rows) return;
  const int64_t at = (int64_t)row * a.cols + col;
  if (MODE == NS_WEIGHTS) {
    const float lr = a.lr_dev ? *a.lr_dev : a.lr;
    float* w = reinterpret_cast<float*>(dst) + at;
    if (col + 8 <= a.cols) {
#pragma unroll
      for (int q = 0; q < 8; q += 4) {
        auto x = NsVec<float>::load(w + q);
#pragma unroll
        for (int e = 0; e < 4; ++e) x.e[e] = ns_weight(a, lr, x.e[e], v[q + e]);
        NsVec<float>::store(w + q, x);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (col + e < a.cols) w[e] = ns_weight(a, lr, w[e], v[e]);
    }
  } else {
    bf16_t* o = reinterpret_cast<bf16_t*>(dst) + at;
    if (col + 8 <= a.cols) {
      NsVec<bf16_t>::mem x;
#pragma unroll
      for (int e = 0; e < 8; ++e) x.e[e] = (bf16_t)v[e];
      NsVec<bf16_t>::store(o, x);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (col + e < a.cols) o[e] = (bf16_t)v[e];
    }
  }
}

// One TM x TN tile of a product, and what the step does with it:
//   NS_XXT      A = X X^T                 operands: columns of X^T             tiles with a block on or above the diagonal, and the mirror image
//   NS_POLY     B = b A + c A A^T         operands: rows of A                  the same
//   NS_STEP     X = a X + B X             rows of B, rows of X^T               X^T in place (the operand copy into the other buffer)
//   NS_LAST     the same, rounded to bf16 into dst;  NS_WEIGHTS  the same as the step of the f32 weights
// 2 x WN waves of 32 MB x 64 (MB x 2 accumulators of v_mfma_f32_32x32x16_f16): 128 x 128 tiles of four waves (MB = 2, WN = 2), or 256 x 256 of
// eight (4, 4).  K steps of 64 through NST LDS stages (one: no overlap within a workgroup) filled by LDS-DMA, 128-byte rows: what bounds these products is the L2
// side (rows of 64 bytes, twice the requests, made the step product of 4096 x 4096 161 us instead of 144), not latency (deeper
// rings and fragments read a step ahead changed nothing).  Consecutive tiles run on one XCD, so that a matrix is fetched into one L2 or two
// instead of eight.
// KG groups of waves take the K steps in turn, each with a ring of its own, and their accumulators are added in LDS on the way out (always in
// the same order): a workgroup that is alone on its CU then has two waves on each SIMD, and half the barriers.
// Step product of 4096 x 4096: 138 us, 995 TFLOP/s (its epilogue moves 134 MB, 27 us, with nothing to run under); X X^T: 92 us, 770.  The last step
// as the step of the weights: 158 us (12 x 2304 x 768: 90, and 57 without the weights); the momentum pass 56 us on average of the two.
// The accumulators leave through LDS as f32, 64 columns at a time, so that all global accesses of the epilogue are whole rows of 16 bytes a lane.
template <int MODE, int MB, int WN, int NST, int KG>
__global__ __launch_bounds__(128 * WN * KG, 2) void ns_gemm_kernel(const NsArgs a, const NsPtrs p, int xt_in, int tiles) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int NW = 2 * WN, NT = 64 * NW * KG, TM = 64 * MB, TN = 64 * WN, PB = TM * 128, STAGE = PB + TN * 128, PIECES = (TM + TN) / 8 / NW;
  constexpr bool SYM = MODE == NS_XXT || MODE == NS_POLY;
  static_assert(KG <= 2 && NT % (TM / 8) == 0 && TM / 8 % NW == 0 && TN / 8 % NW == 0 && (!SYM || TM == TN), "pieces divide evenly; symmetric products use square tiles");
  const int tid = threadIdx.x, lane = tid & 63, all_waves = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kg = all_waves / NW, wave = all_waves % NW;
  const int r = lane & 31, hf = lane >> 5, wm = wave / WN, wn = wave % WN;
  // blockIdx -> tile: consecutive tiles on one XCD
  const int per = gridDim.x >> 3, item = (int)blockIdx.x < per * 8 ? (blockIdx.x & 7) * per + (blockIdx.x >> 3) : blockIdx.x;
  const int mat = item / tiles, tile = item - mat * tiles;
  const int64_t mn = (int64_t)a.mp * a.np, mm = (int64_t)a.mp * a.mp;
  int ti, tj;
  if (SYM) {   // ti <= tj
    tj = (int)((sqrtf(8.f * tile + 1.f) - 1.f) * 0.5f);
    while ((tj + 1) * (tj + 2) / 2 <= tile) ++tj;
    while (tj * (tj + 1) / 2 > tile) --tj;
    ti = tile - tj * (tj + 1) / 2;
  } else {     // groups of eight tile rows, columns inside: the tiles in flight on an XCD share both operands
    const int tiles_m = a.mp / TM, tiles_n = a.np / TN;
    const int g = tile / (8 * tiles_n), rows = min(8, tiles_m - 8 * g), in = tile - g * 8 * tiles_n;
    ti = 8 * g + in % rows;
    tj = in / rows;
  }
  const f16_t *P, *Q;
  int K;
  int64_t step;   // elements between K steps
  if (MODE == NS_XXT) {
    P = a.xt[xt_in] + mat * mn + ti * TM;
    Q = a.xt[xt_in] + mat * mn + tj * TN;
    K = a.np;
    step = (int64_t)64 * a.mp;
  } else {
    P = (MODE == NS_POLY ? a.a16 : a.b16) + mat * mm + (int64_t)ti * TM * a.mp;
    Q = (MODE == NS_POLY ? a.a16 + mat * mm : a.xt[xt_in] + mat * mn) + (int64_t)tj * TN * a.mp;
    K = a.mp;
    step = 64;
  }
  // ---- LDS stages: attn_image.h images, rows of 64 values.  Rows of an operand: one image of TM (TN) rows.  Columns of X^T: images of
  // 64 rows x 64 columns, 8 KiB.  A DMA piece is 8 rows; the swizzle repeats every 16 rows, so pieces of one parity share their offsets.
  char* const ring = smem + kg * NST * STAGE;
  const uint32_t lds0 = lds_addr_of(ring);
  const int prow = 8 * (wave & 1) + (lane >> 3);   // (NW is even: all pieces of a wave have its parity)
  const uint32_t voff = (uint32_t)((lane >> 3) * a.mp + ((lane & 7) ^ img_swz(prow)) * 8) * 2u;
  auto issue = [&](int k, int stage) {
    const uint32_t at = lds0 + (uint32_t)(stage * STAGE);
#pragma unroll
    for (int u = 0; u < PIECES; ++u) {
      const bool is_p = u < TM / 8 / NW;
      const int pc = wave + NW * (is_p ? u : u - TM / 8 / NW);
      const f16_t* base = (is_p ? P : Q) + (k * KG + kg) * step;
      if (MODE == NS_XXT) base += (int64_t)(8 * (pc & 7)) * a.mp + 64 * (pc >> 3);
      else base += (int64_t)(8 * pc) * a.mp;
      lds_dma16(base, voff, at + (uint32_t)((is_p ? 0 : PB) + pc * 1024));
    }
  };
  const ImgLane il = img_lane(lane);
  // fragment of 32 rows (or columns) `blk` of an operand part, k quarter kk of 16
  auto frag = [&](const char* part, int blk, int kk) -> f16x8 {
    if (MODE == NS_XXT) return __builtin_bit_cast(f16x8, lds_tr_frag(part + (blk >> 1) * 8192, il, kk * 2048, blk & 1));
    return *reinterpret_cast<const f16x8*>(part + blk * 4096 + il.row[kk]);
  };

  f32x16 acc[MB][2];
#pragma unroll
  for (int x = 0; x < MB; ++x)
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[x][y][e] = 0.f;
  const int nk = K / 64 / KG;   // this group's steps: kg, kg + KG ..  (sides are padded to multiples of 128)
  for (int k = 0; k < min(max(NST - 1, 1), nk); ++k) issue(k, k);
  int stage = 0;
  for (int k = 0; k < nk; ++k) {
    if (NST > 1 && k + NST - 2 < nk) ns_wait_loads<(NST > 1 ? NST - 2 : 0) * PIECES>();
    else ns_wait_loads<0>();   // (nothing more is requested: the last stages arrive together)
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");   // the stage is here, and no wave still reads the one before it
    if (NST > 1 && k + NST - 1 < nk) issue(k + NST - 1, stage == 0 ? NST - 1 : stage - 1);
    const char* sp = ring + stage * STAGE;
    const char* sq = sp + PB;
    stage = stage == NST - 1 ? 0 : stage + 1;
    // the fragments of a quarter are read while the products of the one before run
    f16x8 fp[2][MB], fq[2][2];
    auto read = [&](int kk) {
#pragma unroll
      for (int y = 0; y < 2; ++y) fq[kk & 1][y] = frag(sq, 2 * wn + y, kk);
#pragma unroll
      for (int x = 0; x < MB; ++x) fp[kk & 1][x] = frag(sp, MB * wm + x, kk);
    };
    read(0);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      if (kk < 3) read(kk + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int x = 0; x < MB; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[kk & 1][x], fq[kk & 1][y], acc[x][y], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (NST == 1 && k + 1 < nk) {   // the one stage is free once all waves have read it
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      issue(k + 1, 0);
    }
  }
  // ---- epilogue: pass `pass` brings the 64 columns j of wave column wn = pass to LDS, each with the tile's TM rows i along it
  constexpr int PITCH = TM + 4;
  float* T = reinterpret_cast<float*>(smem);   // [64 j][PITCH]
  float d[8];   // of this thread's columns i, the same in every turn: the diagonal of A; a + that of B
  if (MODE != NS_XXT) {
    const float* from = (MODE == NS_POLY ? a.diag_a : a.diag_b) + (int64_t)mat * a.mp + ti * TM + 8 * (tid % (TM / 8));
#pragma unroll
    for (int e = 0; e < 8; ++e) d[e] = MODE == NS_POLY ? from[e] : fmaf(from[e], a.inv_S, a.ca);
  }
#pragma unroll
  for (int pass = 0; pass < WN; ++pass) {
    __syncthreads();
#pragma unroll
    for (int from = 0; from < KG; ++from) {
      if (wn == pass && kg == from) {
#pragma unroll
        for (int x = 0; x < MB; ++x)
#pragma unroll
          for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              float4* at = reinterpret_cast<float4*>(T + (32 * y + r) * PITCH + 32 * MB * wm + 32 * x + 8 * g + 4 * hf);
              float4 v = make_float4(acc[x][y][4 * g], acc[x][y][4 * g + 1], acc[x][y][4 * g + 2], acc[x][y][4 * g + 3]);
              if (from > 0) {
                const float4 o = *at;
                v = make_float4(o.x + v.x, o.y + v.y, o.z + v.z, o.w + v.w);
              }
              *at = v;
            }
      }
      __syncthreads();
    }
    const int j0 = tj * TN + 64 * pass, i0 = ti * TM;
#pragma unroll 2
    for (int c = tid; c < 8 * TM; c += NT) {
      const int row = c / (TM / 8), col = 8 * (c % (TM / 8)), j = j0 + row, i = i0 + col;
      float* t = T + row * PITCH + col;
      float v[8];
      *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(t);
      *reinterpret_cast<float4*>(v + 4) = *reinterpret_cast<const float4*>(t + 4);
      if (SYM) {
        const int64_t at = mat * mm + (int64_t)j * a.mp + i;
        // S A = the product / S;  S B = b S E + c ((S E)^2 + (d_i + d_j) S E) / S beside the diagonal, b d + c ((S E)^2 + d^2) / S on it
        const float k = MODE == NS_XXT ? a.inv_S : a.cc * a.inv_S;
        f16x8 a8, o;
        float dj = 0.f, y[8];
        if (MODE == NS_POLY) {
          a8 = *reinterpret_cast<const f16x8*>(a.a16 + at);
          dj = a.diag_a[(int64_t)mat * a.mp + j];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = MODE == NS_XXT ? 0.f : (float)a8[e];
          y[e] = MODE == NS_XXT ? v[e] * k : fmaf(a.cb, x, k * fmaf(d[e] + dj, x, v[e]));
        }
        if (ti == tj) {
          const int own = j - i;   // which of the eight stands on the diagonal
          float on = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            on = e == own ? v[e] : on;
            y[e] = e == own ? 0.f : y[e];
          }
          on = MODE == NS_XXT ? on * k : fmaf(a.cb, dj, k * fmaf(dj, dj, on));
          if (own >= 0 && own < 8) (MODE == NS_XXT ? a.diag_a : a.diag_b)[(int64_t)mat * a.mp + j] = on;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = (f16_t)y[e];
        *reinterpret_cast<f16x8*>((MODE == NS_XXT ? a.a16 : a.b16) + at) = o;
        *reinterpret_cast<f16x8*>(t) = o;   // (this thread's own place: for the mirror image below)
      } else {
        // S X' = (a + d / S) S X + (S B) (S X) / S with the diagonal d of S B
        const int64_t at = mat * mn + (int64_t)j * a.mp + i;
        const f16x8 h8 = *reinterpret_cast<const f16x8*>(a.xt[xt_in] + at), l8 = *reinterpret_cast<const f16x8*>(a.xl + at);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = fmaf(d[e], (float)h8[e] + (float)l8[e], v[e] * a.inv_S);
        if (MODE == NS_STEP) {
          f16x8 hi, lo;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            hi[e] = (f16_t)v[e];
            lo[e] = (f16_t)(v[e] - (float)hi[e]);
          }
          *reinterpret_cast<f16x8*>(a.xt[1 - xt_in] + at) = hi;
          *reinterpret_cast<f16x8*>(a.xl + at) = lo;
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] *= a.inv_S;
          if (a.tall) {
            ns_result<MODE>(a, p.dst[mat], j, i, v);
          } else {
            *reinterpret_cast<float4*>(t) = *reinterpret_cast<const float4*>(v);
            *reinterpret_cast<float4*>(t + 4) = *reinterpret_cast<const float4*>(v + 4);
          }
        }
      }
    }
    if (MODE == NS_STEP) continue;
    if (!SYM && a.tall) continue;
    __syncthreads();
    if (SYM) {   // the mirror image (a tile on the diagonal is its own): 8 x 8 blocks turned in registers; eight lanes store 64 columns j of a row i
      f16_t* out = (MODE == NS_XXT ? a.a16 : a.b16) + mat * mm;
      for (int c = tid; c < (ti == tj ? 0 : TM); c += NT) {
        const int j8 = 8 * (c & 7), i8 = 8 * (c >> 3);
        f16x8 in[8], o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) in[e] = *reinterpret_cast<const f16x8*>(T + (j8 + e) * PITCH + i8);
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int f = 0; f < 8; ++f) o[e][f] = in[f][e];
#pragma unroll
        for (int e = 0; e < 8; ++e) *reinterpret_cast<f16x8*>(out + (int64_t)(i0 + i8 + e) * a.mp + j0 + j8) = o[e];
      }
    } else {     // rows of the result are rows i
      for (int c = tid; c < 8 * TM; c += NT) {
        const int j8 = 8 * (c & 7), row = c >> 3;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = T[(j8 + e) * PITCH + row];
        ns_result<MODE>(a, p.dst[mat], i0 + row, j0 + j8, v);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ small matrices
// A matrix of at most 128 x 256 never leaves its CU: one workgroup of eight waves does the whole iteration (the launches alone cost 108 us
// for 201 x 65, this 41).  X^T is held twice: in f32 in the accumulator layout of the step product (wave w: rows 32 w .. of X^T on the
// lanes, 128 columns in 4 x 16 registers), which takes a X without any rounding, and rounded to f16 in LDS (two images of 256 rows x 64
// columns), whose rows serve B X and whose columns, read transposed, X X^T.  A and then B stand in a third place (two images of 128 x 64).
constexpr int NS_SMALL_M = 128, NS_SMALL_N = 256, NS_SMALL_PITCH = 129;
constexpr int NS_SMALL_X = 2 * 256 * 128, NS_SMALL_LDS = NS_SMALL_X + 128 * NS_SMALL_PITCH * 4;

// byte offset of column c (of 128) in row `row` of the images at distance `image` of each other
__device__ __forceinline__ int ns_img_at(int row, int c, int image) {
  return (c >> 6) * image + row * 128 + ((((c & 63) >> 3) ^ img_swz(row)) << 4) + (c & 7) * 2;
}

// MUON: the momentum is moved on first and the weights at last.  MB: blocks of 32 that hold anything of the short side (at least two): the rest
// is zero and not computed.  The k steps of a product are unrolled, so that their fragments are in flight together (201 x 65: 41 us; three blocks instead of four saved 5 of it, two at 64 x 256 11).
template <typename T, bool MUON, int MB>
__global__ __launch_bounds__(512, 2) void ns_small_kernel(const NsArgs a, const NsPtrs p, int steps) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  char* X = smem;
  char* A = smem + NS_SMALL_X;                          // 32 KiB, inside the staging area of the first and last phase
  float* stage = reinterpret_cast<float*>(A);           // [128 j][129]
  float* diag_a = reinterpret_cast<float*>(A + 32768);  // [128] the diagonals of A and B, times S; zero in the images
  float* diag_b = diag_a + 128;
  const int mat = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 31, hf = lane >> 5, fast = tid & 127, slow = tid >> 7;
  const T* src = reinterpret_cast<const T*>(p.src[mat]);
  float* mom = MUON ? reinterpret_cast<float*>(p.mom[mat]) : nullptr;
  const int halves = a.n > 128 ? 2 : 1;
  f32x16 x[MB];
  double sum = 0.0;
  // ---- G in halves of 128 rows j of X^T, read along the axis that is contiguous in memory
  const bool by_i = a.tall ? a.cs <= a.rs : a.rs <= a.cs;
  for (int half = 0; half < 2; ++half) {
    if (half < halves) {
#pragma unroll 8
      for (int k = slow; k < 128; k += 4) {
        const int i = by_i ? fast : k, jl = by_i ? k : fast, j = 128 * half + jl;
        float v = 0.f;
        if (i < a.m && j < a.n) {
          v = to_f32(src[ns_src_at(a, i, j)]);
          if (MUON) {
            float* at = mom + (a.tall ? (int64_t)j * a.cols + i : (int64_t)i * a.cols + j);
            float m = *at;
            v = ns_momentum(a, m, v);
            *at = m;
          }
        }
        sum += (double)v * (double)v;
        stage[jl * NS_SMALL_PITCH + i] = v;
      }
    }
    __syncthreads();
    if (wave >> 2 == half) {
#pragma unroll
      for (int b = 0; b < MB; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          x[b][e] = half < halves ? stage[(32 * (wave & 3) + r) * NS_SMALL_PITCH + 32 * b + (e & 3) + 8 * (e >> 2) + 4 * hf] : 0.f;
    }
    __syncthreads();
  }
  double* red = reinterpret_cast<double*>(stage);
  red[tid] = sum;
  __syncthreads();
  for (int o = 256; o > 0; o >>= 1) {
    if (tid < o) red[tid] += red[tid + o];
    __syncthreads();
  }
  const float inv = (float)(1.0 / (sqrt(red[0]) + (double)a.eps));
#pragma unroll
  for (int b = 0; b < MB; ++b)
#pragma unroll
    for (int e = 0; e < 16; ++e) x[b][e] = x[b][e] * inv * a.S;   // (in this order: inv S may be past f32's end)
  auto store_x = [&]() {
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f16x4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (f16_t)x[b][4 * g + e];
        *reinterpret_cast<f16x4*>(X + ns_img_at(32 * wave + r, 32 * b + 8 * g + 4 * hf, 32768)) = o;
      }
  };
  store_x();
  const ImgLane il = img_lane(lane);
  const int bi = wave >> 1, bc = 2 * (wave & 1);   // this wave's blocks of A: rows 32 bi .., columns 32 bc .. + 63
  const int k16 = (a.n + 15) / 16;
  const bool mine = bi < MB && bc < MB;   // (with three blocks a wave's second one may be the fourth: what it computes is not read)
  auto zero = [](f32x16& z) {
#pragma unroll
    for (int e = 0; e < 16; ++e) z[e] = 0.f;
  };
  for (int s = 0; s < steps; ++s) {
    __syncthreads();   // X is complete; nobody reads B any more
    f32x16 acc[MB];
    zero(acc[0]);
    zero(acc[1]);
    auto contract = [&](int k) {
      const f16x8 fp = __builtin_bit_cast(f16x8, lds_tr_frag(X + (bi >> 1) * 32768, il, k * 2048, bi & 1));
#pragma unroll
      for (int y = 0; y < 2; ++y)
        acc[y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp, __builtin_bit_cast(f16x8, lds_tr_frag(X + (bc >> 1) * 32768, il, k * 2048, y)), acc[y], 0, 0, 0);
    };
    if (mine) {
      int k = 0;
      for (; k + 4 <= k16; k += 4) {
#pragma unroll
        for (int u = 0; u < 4; ++u) contract(k + u);
      }
      for (; k < k16; ++k) contract(k);
    }
    // element (i, i') of the symmetric result stands in row i' (the lane) at columns i (four registers): its mirror image
    f16x4 av[2][4];
    // (the diagonal of a block on the diagonal: lane r of the half that holds its row, register `own`)
    const bool holds = ((r >> 2) & 1) == hf;
    const int own = (r & 3) + 4 * (r >> 3);
    auto on_diagonal = [&](f32x16& z) {
      float on = 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        on = e == own ? z[e] : on;
        z[e] = e == own && holds ? 0.f : z[e];
      }
      return on;
    };
    if (mine) {
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int ip = 32 * (bc + y) + r;
        if (bi == bc + y) {
          const float on = on_diagonal(acc[y]) * a.inv_S;
          if (holds) diag_a[ip] = on;
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
#pragma unroll
          for (int e = 0; e < 4; ++e) av[y][g][e] = (f16_t)(acc[y][4 * g + e] * a.inv_S);
          *reinterpret_cast<f16x4*>(A + ns_img_at(ip, 32 * bi + 8 * g + 4 * hf, 16384)) = av[y][g];
        }
      }
    }
    __syncthreads();
    zero(acc[0]);
    zero(acc[1]);
    float4 di[4];
    float djs[2];
#pragma unroll
    for (int g = 0; g < 4; ++g) di[g] = *reinterpret_cast<const float4*>(diag_a + 32 * bi + 8 * g + 4 * hf);
#pragma unroll
    for (int y = 0; y < 2; ++y) djs[y] = diag_a[32 * (bc + y) + r];
    if (mine) {
#pragma unroll
      for (int k = 0; k < 2 * MB; ++k) {
        const f16x8 fp = *reinterpret_cast<const f16x8*>(A + (k >> 2) * 16384 + bi * 4096 + il.row[k & 3]);
#pragma unroll
        for (int y = 0; y < 2; ++y)
          acc[y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp, *reinterpret_cast<const f16x8*>(A + (k >> 2) * 16384 + (bc + y) * 4096 + il.row[k & 3]), acc[y],
                                                          0, 0, 0);
      }
    }
    __syncthreads();   // all of A is read
    if (mine) {
      const float k = a.cc * a.inv_S;
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int ip = 32 * (bc + y) + r;
        const float dj = djs[y];
        if (bi == bc + y) {   // (E is zero there: what follows leaves the zero)
          const float on = on_diagonal(acc[y]);
          if (holds) diag_b[ip] = fmaf(a.cb, dj, k * fmaf(dj, dj, on));
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float d[4] = {di[g].x, di[g].y, di[g].z, di[g].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[y][4 * g + e] = fmaf(a.cb, (float)av[y][g][e], k * fmaf(d[e] + dj, (float)av[y][g][e], acc[y][4 * g + e]));
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          f16x4 o;
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = (f16_t)acc[y][4 * g + e];
          *reinterpret_cast<f16x4*>(A + ns_img_at(ip, 32 * bi + 8 * g + 4 * hf, 16384)) = o;
        }
      }
    }
    __syncthreads();
    if (32 * wave < a.n) {   // (rows past the matrix are zero and stay so)
#pragma unroll
      for (int b = 0; b < MB; ++b) zero(acc[b]);
#pragma unroll
      for (int k = 0; k < 2 * MB; ++k) {
        const f16x8 fq = *reinterpret_cast<const f16x8*>(X + (k >> 2) * 32768 + wave * 4096 + il.row[k & 3]);
#pragma unroll
        for (int b = 0; b < MB; ++b)
          acc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const f16x8*>(A + (k >> 2) * 16384 + b * 4096 + il.row[k & 3]), fq, acc[b], 0, 0, 0);
      }
#pragma unroll
      for (int b = 0; b < MB; ++b)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float4 d4 = *reinterpret_cast<const float4*>(diag_b + 32 * b + 8 * g + 4 * hf);
          const float d[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) x[b][4 * g + e] = fmaf(fmaf(d[e], a.inv_S, a.ca), x[b][4 * g + e], acc[b][4 * g + e] * a.inv_S);
        }
      if (s + 1 < steps) store_x();   // (a wave's rows are its own in this product)
    }
  }
  // ---- result, half by half through LDS
  const float lr = MUON && a.lr_dev ? *a.lr_dev : a.lr;
  for (int half = 0; half < halves; ++half) {
    __syncthreads();
    if (wave >> 2 == half) {
#pragma unroll
      for (int b = 0; b < MB; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          stage[(32 * (wave & 3) + r) * NS_SMALL_PITCH + 32 * b + (e & 3) + 8 * (e >> 2) + 4 * hf] = x[b][e] * a.inv_S;
    }
    __syncthreads();
#pragma unroll 8
    for (int k = slow; k < 128; k += 4) {   // rows of the result run along i if it is tall, else along j
      const int i = a.tall ? fast : k, jl = a.tall ? k : fast, j = 128 * half + jl;
      if (i < a.m && j < a.n) {
        const int64_t at = a.tall ? (int64_t)j * a.cols + i : (int64_t)i * a.cols + j;
        const float v = stage[jl * NS_SMALL_PITCH + i];
        if (MUON) {
          float* w = reinterpret_cast<float*>(p.dst[mat]) + at;
          *w = ns_weight(a, lr, *w, v);
        } else {
          reinterpret_cast<bf16_t*>(p.dst[mat])[at] = (bf16_t)v;
        }
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ host
static int64_t ns_up(int64_t v, int to) { return (v + to - 1) / to * to; }
// Tiles of 256 x 256 for the step product where they fill whole rounds of the CUs to three quarters (1 x 4096 x 4096, 256 tiles: 148 us a
// product against 160 with tiles of 128; 12 x 768 x 2304, 324 tiles, the second round almost empty: 75 and 61) and need no more padding, which
// all products would carry (whole iterations with 256 / 128: 64 x 640 x 640 1220 / 702 us, 16 x 896 x 1024 551 / 452, 1 x 3968 x 4096 1520 / 1381)
static bool ns_wide(int count, int rows, int cols) {
  const int64_t m = std::min(rows, cols), n = std::max(rows, cols);
  if (ns_up(m, 256) != ns_up(m, 128) || ns_up(n, 256) != ns_up(n, 128)) return false;
  const int64_t tiles = count * (ns_up(m, 256) / 256) * (ns_up(n, 256) / 256);
  return tiles * 4 >= (tiles + 255) / 256 * 256 * 3;
}
struct NsSize {
  int64_t mp, np, bytes;
};
// padded sides and bytes of one matrix in the workspace
static NsSize ns_size(int rows, int cols, bool wide) {
  NsSize s;
  s.mp = ns_up(std::min(rows, cols), wide ? 256 : 128);
  s.np = ns_up(std::max(rows, cols), wide ? 256 : 128);
  s.bytes = NS_PARTS * 8 + s.mp * 2 * 4 + s.mp * s.np * (2 * 2 + 2) + std::max(s.mp, s.np) * s.mp * 2 + s.mp * s.mp * 2;
  return s;
}
// matrices of one pass: as many as 1 GiB of workspace holds, at least one
static int ns_group(int count, int64_t bytes) {
  return (int)std::max<int64_t>(1, std::min<int64_t>({(int64_t)count, (int64_t)NS_GROUP, (int64_t(1) << 30) / bytes}));
}

template <int MODE, int MB, int WN, int NST, int KG>
static int ns_gemm(const NsArgs& a, const NsPtrs& p, int count, int tiles, int xt_in, hipStream_t st) {
  constexpr int TM = 64 * MB, TN = 64 * WN, LDS = std::max(KG * NST * (TM + TN) * 128, 64 * (TM + 4) * 4);
  auto kern = ns_gemm_kernel<MODE, MB, WN, NST, KG>;
  KernelSetup ks;
  if (int rc = kernel_setup(reinterpret_cast<const void*>(kern), 128 * WN * KG, LDS, &ks)) return rc;
  ProfEvents pe(MMK_K_NEWTON_SCHULZ);
  hipExtLaunchKernelGGL(kern, dim3(tiles * count), dim3(128 * WN * KG), LDS, st, pe.start, pe.stop, 0, a, p, xt_in, tiles);
  MMK_LAUNCH_CHECK();
  return 0;
}

template <typename T>
static int ns_begin(const NsArgs& a, const NsPtrs& p, int count, bool mom, hipStream_t st) {
  const dim3 rg(ns_parts(a), count), pg((a.mp / 64) * (a.np / 64), count), blk(256);
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

// Stages of the ring: with more than two workgroups for every CU one stage each (four share a CU, and the loads of one run under the products
// of the others: 12 x 768 x 2304, 1296 tiles, 57 us a step product against 61 with two stages; 4096 x 4096, 528 tiles, 101 us for X X^T
// against 114), else two (336 tiles, 1000 x 1000 x 1777: 23 us).  At most one workgroup a CU: two groups of waves along K (whole iterations of
// 1024 x 4096: 355 us against 422, 128 x 4096: 243 against 279, 1536 x 1536: 302 against 353; four groups of one stage were slower, and
// two groups of one stage for up to 512 tiles too)
template <int MODE>
static int ns_product(const NsArgs& a, const NsPtrs& p, int count, bool wide, int xt_in, hipStream_t st) {
  const int tm = a.mp / 128;
  int tiles = tm * (a.np / 128);
  if constexpr (MODE == NS_XXT || MODE == NS_POLY) tiles = tm * (tm + 1) / 2;
  else if (wide) return ns_gemm<MODE, 4, 4, 2, 1>(a, p, count, (a.mp / 256) * (a.np / 256), xt_in, st);
  const int64_t all = (int64_t)tiles * count;
  if (all <= 256) return ns_gemm<MODE, 2, 2, 2, 2>(a, p, count, tiles, xt_in, st);
  return all > 512 ? ns_gemm<MODE, 2, 2, 1, 1>(a, p, count, tiles, xt_in, st) : ns_gemm<MODE, 2, 2, 2, 1>(a, p, count, tiles, xt_in, st);
}

static int ns_steps(const mmk_newton_schulz_args* q, const NsArgs& a, const NsPtrs& p, int count, bool wide, hipStream_t st) {
  for (int s = 0; s < q->steps; ++s) {
    if (int rc = ns_product<NS_XXT>(a, p, count, wide, s & 1, st)) return rc;
    if (int rc = ns_product<NS_POLY>(a, p, count, wide, s & 1, st)) return rc;
    const int rc = s + 1 < q->steps ? ns_product<NS_STEP>(a, p, count, wide, s & 1, st)
                   : q->weights     ? ns_product<NS_WEIGHTS>(a, p, count, wide, s & 1, st)
                                    : ns_product<NS_LAST>(a, p, count, wide, s & 1, st);
    if (rc) return rc;
  }
  return 0;
}

static int ns_run(const mmk_newton_schulz_args* q, const NsArgs& a, const NsPtrs& p, int count, bool wide, hipStream_t st) {
  const bool mom = q->momenta != nullptr;
  const int rc = MMK_DISPATCH_DTYPE(q->dtype, T, [&]() -> int { return ns_begin<T>(a, p, count, mom, st); });
  if (rc) return rc;
  return ns_steps(q, a, p, count, wide, st);
}

static bool ns_small(int rows, int cols) { return std::min(rows, cols) <= NS_SMALL_M && std::max(rows, cols) <= NS_SMALL_N; }
template <typename T, int MB>
static int ns_small_go(const mmk_newton_schulz_args* q, const NsArgs& a, const NsPtrs& p, int count, hipStream_t st) {
  auto go = [&](auto kern) {
    KernelSetup ks;
    if (int rc = kernel_setup(reinterpret_cast<const void*>(kern), 512, NS_SMALL_LDS, &ks)) return rc;
    ProfEvents pe(MMK_K_NEWTON_SCHULZ);
    hipExtLaunchKernelGGL(kern, dim3(count), dim3(512), NS_SMALL_LDS, st, pe.start, pe.stop, 0, a, p, (int)q->steps);
    MMK_LAUNCH_CHECK();
    return 0;
  };
  return q->weights ? go(ns_small_kernel<T, true, MB>) : go(ns_small_kernel<T, false, MB>);
}
template <typename T>
static int ns_small_run(const mmk_newton_schulz_args* q, const NsArgs& a, const NsPtrs& p, int count, hipStream_t st) {
  return a.m <= 64 ? ns_small_go<T, 2>(q, a, p, count, st) : a.m <= 96 ? ns_small_go<T, 3>(q, a, p, count, st) : ns_small_go<T, 4>(q, a, p, count, st);
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
  if (count == 0 || ns_small(rows, cols)) return 0;
  const NsSize s = ns_size(rows, cols, ns_wide(count, rows, cols));
  return s.bytes * ns_group(count, s.bytes);
}

int mmk_newton_schulz(const mmk_newton_schulz_args* q, void* ws, void* stream) {
  MMK_REQUIRE(q != nullptr, "no arguments");
  if (int rc = ns_check(q->count, q->rows, q->cols)) return rc;
  MMK_REQUIRE(q->steps >= 1 && q->steps <= 32, "1 to 32 steps");
  MMK_REQUIRE(q->eps >= FLT_MIN, "eps must be a normal positive number");   // (1 / eps has to be finite: zeros are divided by it)
  MMK_REQUIRE((q->momenta != nullptr) == (q->weights != 0), "an optimizer's step has momenta and weights, an update neither");
  if (q->count == 0) return 0;
  const bool small = ns_small(q->rows, q->cols);
  MMK_REQUIRE(q->src && q->dst && (ws || small), "missing operand");
  MMK_REQUIRE(reinterpret_cast<uintptr_t>(ws) % 16 == 0, "the workspace must be 16-byte aligned");
  for (int i = 0; i < q->count; ++i) MMK_REQUIRE(q->src[i] && q->dst[i] && (!q->momenta || q->momenta[i]), "missing operand");
  NsArgs a = {};
  a.rows = q->rows;
  a.cols = q->cols;
  a.tall = q->rows > q->cols;
  a.m = std::min(q->rows, q->cols);
  a.n = std::max(q->rows, q->cols);
  const bool wide = ns_wide(q->count, q->rows, q->cols);
  const NsSize size = ns_size(q->rows, q->cols, wide);
  a.mp = (int)size.mp;
  a.np = (int)size.np;
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
  const int group = small ? NS_GROUP : ns_group(q->count, size.bytes);
  const int64_t mn = size.mp * size.np, mm = size.mp * size.mp;
  char* w = reinterpret_cast<char*>(ws);
  auto take = [&](int64_t bytes) {
    char* at = w;
    w += bytes * group;
    return at;
  };
  a.parts = (double*)take(NS_PARTS * 8);
  a.diag_a = (float*)take(size.mp * 4);
  a.diag_b = (float*)take(size.mp * 4);
  a.xt[0] = (f16_t*)take(mn * 2);
  a.xl = (f16_t*)take(mn * 2);
  // xt[1] and, behind it, a16: the un-normalised update of the momentum (4 bytes an element) is read before either is written
  a.u32 = (float*)w;
  a.xt[1] = (f16_t*)take(mn * 2);
  a.a16 = (f16_t*)take(std::max(mm, mn) * 2);
  a.b16 = (f16_t*)take(mm * 2);
  for (int at = 0; at < q->count; at += group) {
    const int n = std::min(group, q->count - at);
    NsPtrs p = {};
    a.flat = (q->col_stride == 1 && q->row_stride == q->cols) || (q->row_stride == 1 && q->col_stride == q->rows);
    for (int i = 0; i < n; ++i) {
      p.src[i] = q->src[at + i];
      p.mom[i] = q->momenta ? q->momenta[at + i] : nullptr;
      p.dst[i] = q->dst[at + i];
      a.flat &= reinterpret_cast<uintptr_t>(p.src[i]) % 16 == 0;
    }
    const int rc = small ? MMK_DISPATCH_DTYPE(q->dtype, T, [&]() -> int { return ns_small_run<T>(q, a, p, n, (hipStream_t)stream); })
                         : ns_run(q, a, p, n, wide, (hipStream_t)stream);
    if (rc) return rc;
  }
  return 0;
}

}  // extern "C"
