// Attention with a learned relative position bias by buckets, for any length:
//
//   s_ij = scale q_i . k_j + table[bucket(j - i - off), h],   P = softmax over the kept keys j,   o_i = sum_j P_ij v_j
//   backward:  dP = dO V^T,  delta_i = dO_i . o_i,  dS = P (dP - delta),  dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO,
//              dtable[c, h] = sum over all samples and all (i, j) with bucket c of dS
//
// The bias depends on the distance alone and is constant beyond max_distance, so it never exists as a matrix: a workgroup keeps one head's
// bias as a vector over the distances -max_distance .. max_distance in LDS, tiles that lie wholly beyond it take one scalar, and the
// backward sums dS of near tiles along their diagonals in LDS, of far tiles in registers.
//
// Matrix products run on v_mfma_f32_32x32x16 with the softmax axis across the accumulator registers: S^T = K Q^T has the query on the
// lane, so the running maximum, the sum and the rescale of O^T are lane-local, and the exponentiated accumulators are the B operand
// of O^T = V^T P^T as they stand (csrc/attention.hip uses the same forms for whole heads on chip; attn_image.h has the images).  K / V (or
// Q / dO) tiles of 64 rows go to LDS by LDS-DMA, double-buffered, one barrier a tile.  P and dS are rounded to the operands' type for their
// products -- the matrix unit takes 16-bit operands; statistics, sums, accumulators and the table's gradient stay in f32.
// delta decides how exact the table's gradient is: dS sums to zero along a row, and an error of delta is one of every dS of the row.  With
// o rounded (or summed from rounded P) dtable is off by 4e-3 at 512 keys, an f32 one too.  So a forward that will be differentiated sums
// o from P in two parts, rounded and the rest, and hands the backward what the rounding of o left: delta and dtable then hold to 1e-5.
// Where nothing will be differentiated the prompt kernel rounds P once -- o is then off by 2.3e-3 of its size in bf16 where its own rounding is
// 1.7e-3, and the second product would make it 40 % slower (233 us for 166) --; the few-rows kernel always takes both parts.
// f16's range is narrow for dS (P is about 1 / Lk, the incoming gradient of any size) and for P of far keys, so both go through their products
// times a power of two, which is exact and leaves with the accumulators: P times a constant, dS times one that follows its largest value.
#include <hip/hip_ext.h>
#include <limits.h>

#include <algorithm>

#include "attn_image.h"
#include "common.h"

namespace mmk {

typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int REL_MAX_BORDERS = 64;
constexpr int REL_MAX_BUCKETS = 256;
constexpr int REL_MAX_FAR = 512;
constexpr float REL_LOG2E = 1.4426950408889634f;

struct RelArgs {
  const void *q, *k, *v;
  int64_t q_sb, q_sh, q_sl, k_sb, k_sh, k_sl, v_sb, v_sh, v_sl;   // element strides of [B, H, L, D] views
  void* out;       // [B, Lq, H, D] contiguous
  void* out_lo;    // the same layout: what out's rounding left, for the backward; null: not wanted
  float* lse;      // [B, H, Lq], base 2 of the biased scores; +inf for a row without keys; may be null
  int B, H, Hk, G, Lq, Lk;   // G = H / Hk query heads share a key head
  float scale, sl2;          // sl2 = scale log2 e
  const void* table;         // [buckets][H]
  int table_f32, buckets, side, near, far, bidir, n_borders;
  int causal, off;
  const int32_t* off_ptr;    // per-sample offsets, or null
  const void* mask;
  int64_t mask_sb;
  int mask_kind;             // MMK_REL_MASK_*
  // backward
  const void* dout;          // [B, Lq, H, D] contiguous
  const void *o, *o_lo;
  void *dq, *dk, *dv;        // contiguous [B, L, heads, D]
  float *delta, *dtab_part;  // [B, H, Lq]; [workgroups of the dQ kernel][buckets] or null
  float* dkv_part;           // [splits][dK, dV][B, Lk, Hk, D]
  int dkv_splits;
  // split forward
  float* part;               // partial results of the key splits
  int splits;
  int borders[REL_MAX_BORDERS];   // smallest distance of the 2nd, 3rd, .. logarithmic bucket
};

template <typename T>
__device__ __forceinline__ f32x16 rel_mfma(s16x8 a, s16x8 b, f32x16 c);
template <>
__device__ __forceinline__ f32x16 rel_mfma<bf16_t>(s16x8 a, s16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x16 rel_mfma<f16_t>(s16x8 a, s16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// Per-lane offsets into an image (attn_image.h: ImgLane) held as two registers: the chunk index is XORed into bits 4 .. 6, so the offset of
// another k step, half or column block is one XOR away.
struct RelLane {
  int row0, tr0;
  __device__ __forceinline__ explicit RelLane(int lane) {
    const ImgLane il = img_lane(lane);
    row0 = il.row[0];
    tr0 = il.tr[0][0];
  }
  // the same offsets, formed anew where they are used: hoisted out of the loop they would pin a register each
  __device__ __forceinline__ RelLane fresh() const {
    RelLane o = *this;
    asm volatile("" : "+v"(o.row0), "+v"(o.tr0));
    return o;
  }
};
__device__ __forceinline__ s16x8 rel_row_frag(const char* img, const RelLane& il, int kk) {   // k step kk (16 columns) of the lane's row
  return *reinterpret_cast<const s16x8*>(img + (il.row0 ^ (kk << 5)));
}
__device__ __forceinline__ s16x8 rel_tr_frag(const char* img, const RelLane& il, int off, int ct) {   // transposed: rows from off / 128, column block ct
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(img + off + (il.tr0 ^ (ct << 6))));
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(img + off + 1024 + (il.tr0 ^ (ct << 6) ^ 16)));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}
// eight accumulator registers (one k step) as a B operand
template <typename T>
__device__ __forceinline__ s16x8 rel_operand(const f32x16& x, int s) {
  typedef T t8 __attribute__((ext_vector_type(8)));
  t8 o;
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = from_f32<T>(x[8 * s + e]);
  return __builtin_bit_cast(s16x8, o);
}
// two neighbouring values of an operand in f32 (bf16 taken apart by hand: through conversions of single values the packed ones get lost)
__device__ __forceinline__ float2 rel_pair(uint32_t w, bf16_t) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
__device__ __forceinline__ float2 rel_pair(uint32_t w, f16_t) {
  typedef f16_t f2 __attribute__((ext_vector_type(2)));
  const f2 v = __builtin_bit_cast(f2, w);
  return make_float2((float)v[0], (float)v[1]);
}
// what rel_operand's rounding left
template <typename T>
__device__ __forceinline__ s16x8 rel_operand_rest(const f32x16& x, int s, s16x8 rounded) {
  typedef T t8 __attribute__((ext_vector_type(8)));
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  const u4 w = __builtin_bit_cast(u4, rounded);
  t8 o;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 hi = rel_pair(w[e], T());
    o[2 * e] = from_f32<T>(x[8 * s + 2 * e] - hi.x);
    o[2 * e + 1] = from_f32<T>(x[8 * s + 2 * e + 1] - hi.y);
  }
  return __builtin_bit_cast(s16x8, o);
}
// The forward's P is relative to a maximum that is at most 2^8 too low; in f16 it is carried 2^7 higher, to 2^15 at most, so that keys far below
// the first one are still there when there are many of them: each is off by 2^-32 of the first at most, 2^20 of them by half a step of the
// result (the softmax's sum is of the same values; lse takes the factor out again).
template <typename T>
constexpr int REL_FWD_BITS = std::is_same<T, f16_t>::value ? 7 : 0;
// exp2(s - m + bits): where a backward follows, s - m by itself first, which is exactly 0 at the maximum -- a row with one key then has exactly the
// weight 2^bits there, o = v and dS = 0 (see rel_dq_kernel) --, else with the shift in m, one addition less
template <typename T, bool EXACT>
__device__ __forceinline__ float rel_weight(float s, float m) {
  return EXACT && REL_FWD_BITS<T> ? att_exp2((s - m) + REL_FWD_BITS<T>) : att_exp2(s - m);
}
// P's factor in the backward: P <= 1, and what f32 makes of a score may carry it a little above
template <typename T>
constexpr int REL_P_BITS = std::is_same<T, f16_t>::value ? 14 : 0;

// f16: the power of two that dS of a lane's row (key) goes through its product with, a running one like the maximum of a softmax: it falls
// when a value times it would pass 2^15, and the accumulators of that lane (and of the one 32 away, which holds the same row) fall with it.
// Values 2^-29 of the largest so far are still normal.  bf16 has f32's range and needs none.  (2 x 16 (on 4) x 4097 x 128 causal and back: 874 us,
// without it 830; 16 x 12 x 512 x 64: 152 both.)
struct RelRange {
  int bits = 60;   // (from here down f16 results of such dS are zero anyway)
  float factor = 0x1p60f;
  template <int N>
  __device__ __forceinline__ void follow(const f32x16& x, f32x16 (&acc)[N]) {
    float most = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) most = fmaxf(most, fabsf(x[e]));
    most = fmaxf(most, __shfl_xor(most, 32));
    const bool over = most * factor > 32768.f;
    if (__any(over)) {
      const int to = over ? min(bits, 15 - __builtin_amdgcn_frexp_expf(most)) : bits;   // (an infinity passes as it is)
      const float by = __builtin_ldexpf(1.f, to - bits);
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[n][e] *= by;
      bits = to;
      factor = __builtin_ldexpf(1.f, to);
    }
  }
  __device__ __forceinline__ float undo(float mul) const { return __builtin_ldexpf(mul, -bits); }
};
__device__ __forceinline__ f32x16 rel_zero() {
  f32x16 z;
#pragma unroll
  for (int e = 0; e < 16; ++e) z[e] = 0.f;
  return z;
}
// accumulator register e of a lane in half h is row (e & 3) + 8 (e >> 2) + 4 h of the tile
__device__ __forceinline__ constexpr int acc_row(int e) { return (e & 3) + 8 * (e >> 2); }

// the same value of the lane 32 away
__device__ __forceinline__ float rel_other_half(float v) { return __shfl_xor(v, 32); }

__device__ __forceinline__ int rel_bucket(const RelArgs& a, int rel) {
  const int dist = a.bidir ? abs(rel) : max(-rel, 0);
  const int base = a.bidir && rel > 0 ? a.side : 0;
  if (dist < a.near) return base + dist;
  int b = base + a.near;
  for (int t = 0; t < a.n_borders; ++t) b += dist >= a.borders[t];
  return b;
}
__device__ __forceinline__ float rel_table(const RelArgs& a, int bucket, int h, bf16_t) {
  const int64_t at = (int64_t)bucket * a.H + h;
  return a.table_f32 ? reinterpret_cast<const float*>(a.table)[at] : (float)reinterpret_cast<const bf16_t*>(a.table)[at];
}
__device__ __forceinline__ float rel_table(const RelArgs& a, int bucket, int h, f16_t) {
  const int64_t at = (int64_t)bucket * a.H + h;
  return a.table_f32 ? reinterpret_cast<const float*>(a.table)[at] : (float)reinterpret_cast<const f16_t*>(a.table)[at];
}
// bias[x] of the distance x - far - ext, in base-2 units; distances beyond `far` on either side (ext of them) repeat the last one, so that a
// tile that reaches beyond needs no clamp
template <typename T>
__device__ __forceinline__ void rel_bias_fill(const RelArgs& a, float* bias, int ext, int h, int tid, int nt) {
  const int n = 2 * (a.far + ext) + 1;
  for (int x = tid; x < n; x += nt) {
    const int rel = min(max(x - a.far - ext, -a.far), a.far);
    bias[x] = rel_table(a, rel_bucket(a, rel), h, T()) * REL_LOG2E;
  }
}

// (both are the same for the whole workgroup; read back into scalars, which keeps the branches on them scalar)
__device__ __forceinline__ int rel_offset(const RelArgs& a, int b) {
  const int o = a.off_ptr ? a.off_ptr[b] : a.off;
  return __builtin_amdgcn_readfirstlane(min(max(o, -(1 << 29)), 1 << 29));   // (distances stay within 32 bits; far beyond every bucket border)
}
// how many leading keys of the sample can be kept at all.  Causal: none behind the last query, whatever stands there (the places of a cache
// that are not filled yet)
__device__ __forceinline__ int rel_key_len(const RelArgs& a, int b, int off) {
  int64_t n = a.Lk;
  if (a.mask_kind == MMK_REL_MASK_LEN32) n = reinterpret_cast<const int32_t*>(a.mask)[b];
  if (a.mask_kind == MMK_REL_MASK_LEN64) n = reinterpret_cast<const int64_t*>(a.mask)[b];
  if (a.causal) n = min(n, (int64_t)a.Lq + off);
  return __builtin_amdgcn_readfirstlane((int)(n < 0 ? 0 : n < a.Lk ? n : a.Lk));
}
// whether the mask keeps key j (1 where there is no per-key mask); j may lie past the end
__device__ __forceinline__ int rel_mask_at(const RelArgs& a, int b, int j) {
  if (a.mask_kind < MMK_REL_MASK_8) return 1;
  const int64_t at = (int64_t)b * a.mask_sb + min(j, a.Lk - 1);
  if (a.mask_kind == MMK_REL_MASK_8) return reinterpret_cast<const uint8_t*>(a.mask)[at] != 0;
  if (a.mask_kind == MMK_REL_MASK_32) return reinterpret_cast<const int32_t*>(a.mask)[at] != 0;
  return reinterpret_cast<const int64_t*>(a.mask)[at] != 0;
}

// blockIdx -> head (of all samples) and rank among its `blocks` work items.  The heads are dealt to the eight XCDs in turn (samples of unequal
// length would load them unequally otherwise), all items of a head run on one XCD and share its L2, and there the heads go in groups of
// eight with the first rank of every head before the second: rank 0 is the longest item of a causal call, and a long one that started
// last would run alone at the end (causal forward of 2 x 16 x 4097 x 128: 181 us, head by head 207; 4 x 12 x 2048 x 64 and back: 204 and
// 253).  The last heads % 8 heads are spread over all XCDs, item by item.
struct RelPlace {
  int head, rank;
};
__device__ __forceinline__ RelPlace rel_place(int id, int blocks, int heads) {
  const int per = heads >> 3, whole = per * 8 * blocks;
  if (id >= whole) {
    const int rest = heads & 7, x = id - whole;
    return {per * 8 + x % rest, x / rest};
  }
  const int x = id >> 3, group = x / (8 * blocks), size = min(8, per - 8 * group), in = x - group * 8 * blocks;
  return {(8 * group + in % size) * 8 + (id & 7), in / size};
}

// One wave's share of a 64-row tile in LDS: CB column blocks of 64 of X, then of Y; of each image's 8 pieces of 8 rows, pieces `wave` and
// `wave` + 4 (32 rows further, where the swizzle is the same: one per-lane offset serves both)
template <typename T, int CB>
struct RelLoader {
  uint32_t vx, vy;
  __device__ __forceinline__ RelLoader(int64_t x_sl, int64_t y_sl, int wave, int lane) {
    const int row = 8 * wave + (lane >> 3), ch = (lane & 7) ^ img_swz(row & 15);
    vx = (uint32_t)(row * (int)x_sl + ch * 8) * 2u;
    vy = (uint32_t)(row * (int)y_sl + ch * 8) * 2u;
  }
  // rows row0 .. row0 + 63 of X and Y (rows past `rows - 1` repeat that row), to the stage at `lds`
  __device__ __forceinline__ void issue(const T* x, const T* y, int64_t x_sl, int64_t y_sl, int row0, int rows, uint32_t lds, int wave,
                                        int lane) const {
    auto each = [&](auto voff) {
#pragma unroll
      for (int im = 0; im < 2 * CB; ++im) {
        const int64_t sl = im < CB ? x_sl : y_sl;
        const T* base = (im < CB ? x : y) + (int64_t)row0 * sl + 64 * (im % CB);
#pragma unroll
        for (int u = 0; u < 2; ++u) voff(base, sl, im < CB, u, lds + (uint32_t)(im * 8192 + (wave + 4 * u) * 1024));
      }
    };
    if (row0 + 64 <= rows)
      each([&](const T* base, int64_t sl, bool is_x, int u, uint32_t at) { lds_dma16(base + 32 * u * sl, is_x ? vx : vy, at); });
    else
      each([&](const T* base, int64_t sl, bool, int u, uint32_t at) {
        const int row = 8 * (wave + 4 * u) + (lane >> 3), ch = (lane & 7) ^ img_swz(row & 15);
        lds_dma16(base, (uint32_t)(min(row, rows - 1 - row0) * (int)sl + ch * 8) * 2u, at);
      });
  }
};

// rows of `img` (CB images of 64 rows) whose bit in `word` is clear become zero: a masked key may hold anything, and 0 * NaN is NaN
template <int CB>
__device__ __forceinline__ void rel_zero_rows(char* img, uint64_t word, int wave, int lane) {
  const int row = 16 * wave + (lane >> 2);
  if (!((word >> row) & 1)) {
    const uint4 z = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
      uint4* p = reinterpret_cast<uint4*>(img + cb * 8192 + row * 128 + (lane & 3) * 32);
      p[0] = z;
      p[1] = z;
    }
  }
}

// a of the lower half's lanes and b of the upper half's stay; the other halves change places
__device__ __forceinline__ void rel_swap_halves(uint32_t& a, uint32_t& b) {
  typedef uint32_t u2 __attribute__((ext_vector_type(2)));
  const u2 r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0];
  b = r[1];
}
// D^T accumulators (lane = row, registers = columns) -> row `row` of a contiguous-row tensor, times mul; `rest`, if given, takes what the
// rounding left.  A lane holds four of each eight columns; the halves trade, so that each lane stores 16 bytes.
template <typename T, int D>
__device__ __forceinline__ void rel_store_row(T* row, T* rest, const f32x16 (&o)[D / 32], float mul, int h) {
  typedef T t4 __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; g += 2) {
      t4 hi[2], lo[2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = o[dt][4 * (g + u) + e] * mul;
          hi[u][e] = from_f32<T>(x);
          lo[u][e] = from_f32<T>(x - to_f32(hi[u][e]));
        }
      auto put = [&](T* to, t4 x, t4 y) {
        uint2 a = __builtin_bit_cast(uint2, x), b = __builtin_bit_cast(uint2, y);
        rel_swap_halves(a.x, b.x);
        rel_swap_halves(a.y, b.y);
        *reinterpret_cast<uint4*>(to + 32 * dt + 8 * (g + h)) = make_uint4(a.x, a.y, b.x, b.y);
      };
      put(row, hi[0], hi[1]);
      if (rest) put(rest, lo[0], lo[1]);
    }
}
template <int D>
__device__ __forceinline__ void rel_store_row(float* row, const f32x16 (&o)[D / 32], int h) {
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<float4*>(row + 32 * dt + 8 * g + 4 * h) = make_float4(o[dt][4 * g], o[dt][4 * g + 1], o[dt][4 * g + 2], o[dt][4 * g + 3]);
}
// four values of the output, and what their rounding left
template <typename T>
__device__ __forceinline__ void rel_store_out(const RelArgs& a, int64_t at, float4 v) {
  const float x[4] = {v.x, v.y, v.z, v.w};
  typedef T t4 __attribute__((ext_vector_type(4)));
  t4 hi, lo;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    hi[e] = from_f32<T>(x[e]);
    lo[e] = from_f32<T>(x[e] - to_f32(hi[e]));
  }
  *reinterpret_cast<t4*>(reinterpret_cast<T*>(a.out) + at) = hi;
  if (a.out_lo) *reinterpret_cast<t4*>(reinterpret_cast<T*>(a.out_lo) + at) = lo;
}

// ------------------------------------------------------------------------------------------------ forward
// Workgroup: 4 waves x 32 queries of one (sample, head); tiles of 64 keys.  (64 queries a wave would halve the LDS reads, but the vector
// unit -- exponential, bias, maximum, sum: twice the cycles of the products at D = 64 -- bounds it and finer workgroups fill the chip better:
// 4 x 12 x 512 x 64 20 us with 32 and 23 with 64, 2 x 12 x 8192 x 64 503 and 498.  At D = 128 the LDS reads take as long as the products:
// a fragment of 1 KiB for each, four waves, 128 bytes a cycle.)  Scores of the next tile formed under the exponentials of this one, in one
// wave: 5 to 15 % slower than two waves that do so by themselves.  2 x 16 x 4096 x 128: 281 us, 978 TFLOP/s (f16 298); 2 x 12 x 8192 x 64: 496 us, 831
// (f16 523); 256 x 12 x 77 x 64: 36 us, 3.4 TB/s.  LO: P V with P in two parts, 233 us for 2 x 16 x 4097 x 128 causal, 166 without.
template <typename T, int D, bool LO>
__global__ __launch_bounds__(256, 2) void rel_fwd_kernel(const RelArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int CB = D / 64, STAGE = 2 * CB * 8192, EXT = 96;
  float* bias = reinterpret_cast<float*>(smem + 2 * STAGE);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 31, hf = lane >> 5;
  const int nqb = (a.Lq + 127) / 128;
  const RelPlace pl = rel_place(blockIdx.x, nqb, a.B * a.H);
  const int bh = pl.head, b = bh / a.H, h = bh - b * a.H;
  const int qb = a.causal ? nqb - 1 - pl.rank : pl.rank;   // causal: the longest rows first
  const int off = rel_offset(a, b), klen = rel_key_len(a, b, off);
  const int i_wg = qb * 128, i_wave = i_wg + 32 * wave, i = i_wave + r;
  int nkt = (klen + 63) / 64;
  if (a.causal) {
    const int last = min(klen - 1, min(i_wg + 128, a.Lq) - 1 + off);
    nkt = last < 0 ? 0 : last / 64 + 1;
  }
  const T* kp = reinterpret_cast<const T*>(a.k) + b * a.k_sb + (h / a.G) * a.k_sh;
  const T* vp = reinterpret_cast<const T*>(a.v) + b * a.v_sb + (h / a.G) * a.v_sh;
  const RelLoader<T, CB> ld(a.k_sl, a.v_sl, wave, lane);
  const uint32_t lds0 = lds_addr_of(smem);
  int keep = 1;
  if (nkt > 0) {
    ld.issue(kp, vp, a.k_sl, a.v_sl, 0, a.Lk, lds0, wave, lane);
    keep = rel_mask_at(a, b, lane);
  }

  s16x8 qf[D / 16];
  f32x16 o[D / 32];
  float m = -INFINITY, l = 0.f;
  {
    const T* qp = reinterpret_cast<const T*>(a.q) + b * a.q_sb + h * a.q_sh + min(i, a.Lq - 1) * a.q_sl + 8 * hf;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) qf[kk] = *reinterpret_cast<const s16x8*>(qp + 16 * kk);
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) o[dt] = rel_zero();
  }
  rel_bias_fill<T>(a, bias, EXT, h, tid, 256);
  const RelLane il(lane);
  const int ip = i + off;   // this lane's query position
  for (int kt = 0; kt < nkt; ++kt) {
    wait_vmem_all();   // this tile and its mask are here
    __syncthreads();   // and nobody reads the one before it any more
    const int j0 = 64 * kt;
    const uint64_t word = __ballot(j0 + lane < klen && keep);
    if (kt + 1 < nkt) {
      ld.issue(kp, vp, a.k_sl, a.v_sl, j0 + 64, a.Lk, lds0 + ((kt + 1) & 1) * STAGE, wave, lane);
      keep = rel_mask_at(a, b, j0 + 64 + lane);
    }
    char* K = smem + (kt & 1) * STAGE;
    char* V = K + CB * 8192;
    if (word == 0) continue;
    if (~word) {
      rel_zero_rows<CB>(V, word, wave, lane);
      __syncthreads();
    }
    if (i_wave >= a.Lq || (a.causal && j0 > i_wave + 31 + off)) continue;   // no row, or no key of the tile, for this wave
    f32x16 s[2];
    s[0] = s[1] = rel_zero();
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
      for (int t = 0; t < 2; ++t) s[t] = rel_mfma<T>(rel_row_frag(K + (kk >> 2) * 8192 + t * 4096, il, kk & 3), qf[kk], s[t]);
    const int rel_hi = j0 + 63 - (i_wave + off), rel_lo = j0 - (i_wave + 31 + off);
    if (rel_hi <= -a.far || rel_lo >= a.far) {
      const float c = bias[rel_hi <= -a.far ? 0 : 2 * (a.far + EXT)];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[t][e] = fmaf(s[t][e], a.sl2, c);
    } else {
      const float* bp = bias + (a.far + EXT + j0 + 4 * hf - ip);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[t][e] = fmaf(s[t][e], a.sl2, bp[32 * t + acc_row(e)]);
    }
    if (~word || (a.causal && rel_hi > 0)) {
      const int jmax = a.causal ? ip - j0 - 4 * hf : INT_MAX;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint32_t w = (uint32_t)(word >> (32 * t)) >> (4 * hf);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (!((w >> acc_row(e)) & 1) || 32 * t + acc_row(e) > jmax) s[t][e] = -INFINITY;
      }
    }
    float mt = s[0][0];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) mt = fmaxf(mt, s[t][e]);
    mt = fmaxf(mt, rel_other_half(mt));
    // the running maximum moves only when it grows by more than 2^8: until then the sums stay exact enough in f32 and the
    // rescale of O is skipped for the whole wave
    if (__any(mt > m + 8.f)) {
      const float mn = fmaxf(m, mt);
      const float alpha = mn == m ? 1.f : att_exp2(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[dt][e] *= alpha;
    }
    const float top = m == -INFINITY ? 0.f : LO ? m : m - REL_FWD_BITS<T>;
    float lt = 0.f;   // (a tile's sum by itself: single keys far below the sum so far would not move it)
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[t][e] = rel_weight<T, LO>(s[t][e], top);
        lt += s[t][e];
      }
    l += lt;
#pragma unroll
    for (int st = 0; st < 4; ++st) {
      const s16x8 pf = rel_operand<T>(s[st >> 1], st & 1);
      s16x8 pl;
      if (LO) pl = rel_operand_rest<T>(s[st >> 1], st & 1, pf);
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) {
        const s16x8 vf = rel_tr_frag(V + (dt >> 1) * 8192, il, st * 2048, dt & 1);
        o[dt] = rel_mfma<T>(vf, pf, o[dt]);
        if (LO) o[dt] = rel_mfma<T>(vf, pl, o[dt]);
      }
    }
  }
  const float sum = l + rel_other_half(l);
  if (i < a.Lq) {
    const int64_t row = (((int64_t)b * a.Lq + i) * a.H + h) * D;
    rel_store_row<T, D>(reinterpret_cast<T*>(a.out) + row, LO ? reinterpret_cast<T*>(a.out_lo) + row : nullptr, o, sum > 0.f ? 1.f / sum : sum, hf);
    if (a.lse && hf == 0) a.lse[((int64_t)b * a.H + h) * a.Lq + i] = sum == 0.f ? INFINITY : m + (log2f(sum) - REL_FWD_BITS<T>);
  }
}

// ------------------------------------------------------------------------------------------------ forward, few rows
// One workgroup per (sample, key head, split of the keys).  Row = query head of the group x query, 32 at most; all of them
// share every key tile, so the keys are read once for the whole group.  The four waves walk tiles of 32 keys of their own, each through
// LDS of its own without barriers, and are joined at the end; splits are joined by rel_join_kernel.  Bound by the K / V bytes: 716 MB in
// 140 us, 5.1 TB/s.
template <typename T, int D>
__global__ __launch_bounds__(256, 1) void rel_split_kernel(const RelArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int CB = D / 64, IMG = 4096, STAGE = 2 * CB * IMG, EXT = 1;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 31, hf = lane >> 5;
  char* mine = smem + wave * 2 * STAGE;
  float* bias_all = reinterpret_cast<float*>(smem + 8 * STAGE);
  const int nb = 2 * (a.far + EXT) + 1;
  const int split = blockIdx.x % a.splits, bk = blockIdx.x / a.splits;
  const int b = bk / a.Hk, hk = bk - b * a.Hk;
  const int rows = a.G * a.Lq;
  const int rc = min(r, rows - 1), g = rc / a.Lq, i = rc - g * a.Lq, h = hk * a.G + g;
  const int off = rel_offset(a, b), klen = rel_key_len(a, b, off), ip = i + off;
  for (int gg = 0; gg < a.G; ++gg) rel_bias_fill<T>(a, bias_all + gg * nb, EXT, hk * a.G + gg, tid, 256);
  const float* bias = bias_all + g * nb + a.far + EXT;
  // tiles of this split: the sample's own length is divided, so that short samples do not leave splits idle
  const int tiles = (klen + 31) / 32, per = (tiles + a.splits - 1) / a.splits;
  const int t0 = split * per + wave, t1 = min((split + 1) * per, tiles);
  const T* kp = reinterpret_cast<const T*>(a.k) + b * a.k_sb + hk * a.k_sh;
  const T* vp = reinterpret_cast<const T*>(a.v) + b * a.v_sb + hk * a.v_sh;
  s16x8 qf[D / 16];
  f32x16 o[D / 32];
  {
    const T* qp = reinterpret_cast<const T*>(a.q) + b * a.q_sb + h * a.q_sh + i * a.q_sl + 8 * hf;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) qf[kk] = *reinterpret_cast<const s16x8*>(qp + 16 * kk);
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) o[dt] = rel_zero();
  }
  float m = -INFINITY, l = 0.f;
  const RelLane il(lane);
  const uint32_t lds0 = lds_addr_of(mine);
  auto issue = [&](int t, int stage) {
#pragma unroll
    for (int im = 0; im < 2 * CB; ++im) {
      const int64_t sl = im < CB ? a.k_sl : a.v_sl;
      const T* base = (im < CB ? kp : vp) + (int64_t)(32 * t) * sl + 64 * (im % CB);
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const int rw = 8 * p + (lane >> 3), ch = (lane & 7) ^ img_swz(rw & 15);
        lds_dma16(base, (uint32_t)(min(rw, a.Lk - 1 - 32 * t) * (int)sl + ch * 8) * 2u, lds0 + (uint32_t)(stage * STAGE + im * IMG + p * 1024));
      }
    }
  };
  __syncthreads();   // the bias vectors
  int keep = 1;
  if (t0 < t1) {
    issue(t0, 0);
    keep = rel_mask_at(a, b, 32 * t0 + r);
  }
  int stage = 0;
  for (int t = t0; t < t1; t += 4, stage ^= 1) {
    wait_vmem_all();
    asm volatile("" ::: "memory");
    const int j0 = 32 * t;
    const uint32_t word = (uint32_t)__ballot(j0 + r < klen && keep);
    if (t + 4 < t1) {
      issue(t + 4, stage ^ 1);
      keep = rel_mask_at(a, b, j0 + 128 + r);
    }
    if (word == 0) continue;
    char* K = mine + stage * STAGE;
    char* V = K + CB * IMG;
    if (~word && !((word >> r) & 1)) {   // (both halves of a lane pair clear one half of the row each)
      const uint4 z = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int cb = 0; cb < CB; ++cb)
#pragma unroll
        for (int c = 0; c < 4; ++c) *reinterpret_cast<uint4*>(V + cb * IMG + r * 128 + hf * 64 + c * 16) = z;
    }
    f32x16 s = rel_zero();
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) s = rel_mfma<T>(rel_row_frag(K + (kk >> 2) * IMG, il, kk & 3), qf[kk], s);
    const uint32_t w = word >> (4 * hf);
    const int rel0 = j0 + 4 * hf - ip, jmax = a.causal ? -rel0 : INT_MAX;
    float mt = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      s[e] = fmaf(s[e], a.sl2, bias[min(max(rel0 + acc_row(e), -a.far), a.far)]);
      if (!((w >> acc_row(e)) & 1) || acc_row(e) > jmax) s[e] = -INFINITY;
      mt = fmaxf(mt, s[e]);
    }
    mt = fmaxf(mt, rel_other_half(mt));
    if (__any(mt > m + 8.f)) {
      const float mn = fmaxf(m, mt);
      const float alpha = mn == m ? 1.f : att_exp2(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[dt][e] *= alpha;
    }
    const float top = m == -INFINITY ? 0.f : m;
    float lt = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      s[e] = rel_weight<T, true>(s[e], top);
      lt += s[e];
    }
    l += lt;
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const s16x8 pf = rel_operand<T>(s, st);
      const s16x8 pl = rel_operand_rest<T>(s, st, pf);   // (in two parts always: under the loads it costs less than 1 %)
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) {
        const s16x8 vf = rel_tr_frag(V + (dt >> 1) * IMG, il, st * 2048, dt & 1);
        o[dt] = rel_mfma<T>(vf, pf, o[dt]);
        o[dt] = rel_mfma<T>(vf, pl, o[dt]);
      }
    }
  }
  l += rel_other_half(l);
  // ---- join the waves: [wave][32 rows] of (m, l), then O row by row
  __syncthreads();
  float* ml = reinterpret_cast<float*>(smem);               // [4][2][32]
  float* ob = reinterpret_cast<float*>(smem + 1024);         // [4][32][D + 4]
  if (hf == 0) {
    ml[wave * 64 + r] = m;
    ml[wave * 64 + 32 + r] = l;
  }
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4)
      *reinterpret_cast<float4*>(ob + (wave * 32 + r) * (D + 4) + 32 * dt + 8 * q4 + 4 * hf) =
          make_float4(o[dt][4 * q4], o[dt][4 * q4 + 1], o[dt][4 * q4 + 2], o[dt][4 * q4 + 3]);
  __syncthreads();
  for (int x = tid; x < rows * (D / 4); x += 256) {
    const int rr = x / (D / 4), d = 4 * (x - rr * (D / 4));
    float mm = -INFINITY, ll = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int wv = 0; wv < 4; ++wv) mm = fmaxf(mm, ml[wv * 64 + rr]);
#pragma unroll
    for (int wv = 0; wv < 4; ++wv) {
      const float mw = ml[wv * 64 + rr];
      const float f = mw == -INFINITY ? 0.f : att_exp2(mw - mm);
      const float4 v4 = *reinterpret_cast<const float4*>(ob + (wv * 32 + rr) * (D + 4) + d);
      ll += f * ml[wv * 64 + 32 + rr];
      acc.x += f * v4.x;
      acc.y += f * v4.y;
      acc.z += f * v4.z;
      acc.w += f * v4.w;
    }
    const int64_t prow = (int64_t)bk * 32 + rr;
    if (a.splits > 1) {
      float* p = a.part + (prow * a.splits + split) * (D + 4);   // [.., D] sums, then (m, l)
      *reinterpret_cast<float4*>(p + d) = acc;
      if (d == 0) *reinterpret_cast<float2*>(p + D) = make_float2(mm, ll);
    } else {
      const int go = rr / a.Lq, io = rr - go * a.Lq, ho = hk * a.G + go;
      const float f = ll > 0.f ? 1.f / ll : ll;
      rel_store_out<T>(a, (((int64_t)b * a.Lq + io) * a.H + ho) * D + d, make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f));
      if (a.lse && d == 0) a.lse[((int64_t)b * a.H + ho) * a.Lq + io] = ll == 0.f ? INFINITY : mm + (log2f(ll) - REL_FWD_BITS<T>);
    }
  }
}

// one group of D / 4 threads per row
template <typename T, int D>
__global__ __launch_bounds__(256) void rel_join_kernel(const RelArgs a) {
  const int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int rows = a.G * a.Lq;
  const int64_t row = x / (D / 4);
  const int d = 4 * (int)(x - row * (D / 4));
  const int bk = (int)(row / rows), ro = (int)(row - (int64_t)bk * rows);
  if (bk >= a.B * a.Hk) return;
  const int b = bk / a.Hk, hk = bk - b * a.Hk, go = ro / a.Lq, io = ro - go * a.Lq, ho = hk * a.G + go;
  const float* p = a.part + ((int64_t)bk * 32 + ro) * a.splits * (D + 4);
  float mm = -INFINITY, ll = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = 0; s < a.splits; ++s) mm = fmaxf(mm, p[s * (D + 4) + D]);
  for (int s = 0; s < a.splits; ++s) {
    const float ms = p[s * (D + 4) + D];
    const float f = ms == -INFINITY ? 0.f : att_exp2(ms - mm);
    const float4 v4 = *reinterpret_cast<const float4*>(p + s * (D + 4) + d);
    ll += f * p[s * (D + 4) + D + 1];
    acc.x += f * v4.x;
    acc.y += f * v4.y;
    acc.z += f * v4.z;
    acc.w += f * v4.w;
  }
  const float f = ll > 0.f ? 1.f / ll : ll;
  rel_store_out<T>(a, (((int64_t)b * a.Lq + io) * a.H + ho) * D + d, make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f));
  if (a.lse && d == 0) a.lse[((int64_t)b * a.H + ho) * a.Lq + io] = ll == 0.f ? INFINITY : mm + (log2f(ll) - REL_FWD_BITS<T>);
}

// ------------------------------------------------------------------------------------------------ backward: dQ, delta, dtable
// Sums of a 32 x 32 tile of dS^T along its diagonals.  Register e of lane (row R of 16 lanes, c = lane & 15, half hf) is key
// 16 K + n + 4 hf (n = acc_row(e) & 15, K = e >> 3) and query 16 R + c.  Shifting the register by n lanes within its row of 16 puts equal
// distances into one lane: what stays in the row has distance 16 (K - R) + 4 hf - c, what leaves it on the other side 16 more.  With
// row shifts that fill with zeros both parts are one DPP add each.  d[k] of a lane: the sum at distance 16 (k - R) + 4 hf - c from the
// tile's corner.
template <int N>
__device__ __forceinline__ void rel_diag_add(float x, float& stay, float& leave) {
  if (N == 0) {
    stay += x;
  } else {
    const int xi = __builtin_bit_cast(int, x);
    stay += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, xi, 0x100 + (N & 15), 0xf, 0xf, true));           // lane c takes lane c + N
    leave += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, xi, 0x110 + ((16 - N) & 15), 0xf, 0xf, true));   // lane c takes lane c + N - 16
  }
}
__device__ __forceinline__ void rel_diagonals(const f32x16& s, float (&d)[3]) {
  d[0] = d[1] = d[2] = 0.f;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    rel_diag_add<0>(s[8 * k + 0], d[k], d[k + 1]);
    rel_diag_add<1>(s[8 * k + 1], d[k], d[k + 1]);
    rel_diag_add<2>(s[8 * k + 2], d[k], d[k + 1]);
    rel_diag_add<3>(s[8 * k + 3], d[k], d[k + 1]);
    rel_diag_add<8>(s[8 * k + 4], d[k], d[k + 1]);
    rel_diag_add<9>(s[8 * k + 5], d[k], d[k + 1]);
    rel_diag_add<10>(s[8 * k + 6], d[k], d[k + 1]);
    rel_diag_add<11>(s[8 * k + 7], d[k], d[k + 1]);
  }
}

// As the forward, with the query on the lane: dS^T needs lse and delta of the lane alone, and dQ^T += K^T dS^T takes it from the
// accumulators.  delta is the diagonal of O dO^T, formed by the instructions and in the order of dP = V dO^T, and what o's rounding left times dO:
// where one key has all of a row's weight (o = v), dP - delta is exactly zero, as dS is.
// dtable: rel_diagonals sums a near tile along its diagonals in registers, and each half wave adds the sums to a
// vector over the distances of its own (plain LDS reads and writes in a fixed order; LDS float atomics took 175 cycles a wave
// instruction, which made this kernel 3.5 times slower).  Tiles beyond max_distance add to two registers.
// D = 64 leaves room for three workgroups a CU, in registers and in LDS (16 documents of 512 rows, 12 heads: 41 us instead of 57
// with two, the dK / dV kernel below 42 instead of 61).  At D = 128 bound as the forward: 2 x 16 x 4097 x 128 causal 284 us, 725 TFLOP/s (f16 328).
constexpr int REL_DIAG = 8;   // vectors over the distances
template <typename T, int D>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void rel_dq_kernel(const RelArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int CB = D / 64, STAGE = 2 * CB * 8192, EXT = 96, VECS = REL_DIAG;
  constexpr bool F16 = std::is_same<T, f16_t>::value;
  float* bias = reinterpret_cast<float*>(smem + 2 * STAGE);
  const int nbias = (2 * (a.far + EXT) + 1 + 3) & ~3;
  float* diag = bias + nbias;   // [VECS][nbias], per half wave
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 31, hf = lane >> 5;
  const int nqb = (a.Lq + 127) / 128;
  const RelPlace pl = rel_place(blockIdx.x, nqb, a.B * a.H);
  const int bh = pl.head, b = bh / a.H, h = bh - b * a.H;
  const int qb = a.causal ? nqb - 1 - pl.rank : pl.rank;
  const int off = rel_offset(a, b), klen = rel_key_len(a, b, off);
  const int i_wg = qb * 128, i_wave = i_wg + 32 * wave, i = i_wave + r;
  int nkt = (klen + 63) / 64;
  if (a.causal) {
    const int last = min(klen - 1, min(i_wg + 128, a.Lq) - 1 + off);
    nkt = last < 0 ? 0 : last / 64 + 1;
  }
  const T* kp = reinterpret_cast<const T*>(a.k) + b * a.k_sb + (h / a.G) * a.k_sh;
  const T* vp = reinterpret_cast<const T*>(a.v) + b * a.v_sb + (h / a.G) * a.v_sh;
  const RelLoader<T, CB> ld(a.k_sl, a.v_sl, wave, lane);
  const uint32_t lds0 = lds_addr_of(smem);
  int keep = 1;
  if (nkt > 0) {
    ld.issue(kp, vp, a.k_sl, a.v_sl, 0, a.Lk, lds0, wave, lane);
    keep = rel_mask_at(a, b, lane);
  }

  s16x8 qf[D / 16], gf[D / 16];
  f32x16 dq[D / 32];
  RelRange range;
  float lse, delta = 0.f, far_l = 0.f, far_r = 0.f;
  {
    const int ic = min(i, a.Lq - 1);
    const T* qp = reinterpret_cast<const T*>(a.q) + b * a.q_sb + h * a.q_sh + ic * a.q_sl + 8 * hf;
    const int64_t orow = (((int64_t)b * a.Lq + ic) * a.H + h) * D + 8 * hf;
    const T* gp = reinterpret_cast<const T*>(a.dout) + orow;
    const T* op = reinterpret_cast<const T*>(a.o) + orow;
    const T* lp = reinterpret_cast<const T*>(a.o_lo) + orow;
    f32x16 od = rel_zero();
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      typedef T t8 __attribute__((ext_vector_type(8)));
      qf[kk] = *reinterpret_cast<const s16x8*>(qp + 16 * kk);
      gf[kk] = *reinterpret_cast<const s16x8*>(gp + 16 * kk);
      od = rel_mfma<T>(*reinterpret_cast<const s16x8*>(op + 16 * kk), gf[kk], od);
      const t8 g8 = __builtin_bit_cast(t8, gf[kk]), l8 = *reinterpret_cast<const t8*>(lp + 16 * kk);
#pragma unroll
      for (int e = 0; e < 8; ++e) delta = fmaf(to_f32(g8[e]), to_f32(l8[e]), delta);
    }
    const int own = ((r >> 2) & 1) == hf ? (r & 3) + 4 * (r >> 3) : -1;   // the register that holds (r, r)
#pragma unroll
    for (int e = 0; e < 16; ++e) delta += e == own ? od[e] : 0.f;
    delta += rel_other_half(delta);
    const int64_t at = ((int64_t)b * a.H + h) * a.Lq + ic;
    lse = i < a.Lq ? a.lse[at] : INFINITY;
    if (i < a.Lq && hf == 0) a.delta[at] = delta;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) dq[dt] = rel_zero();
  }
  rel_bias_fill<T>(a, bias, EXT, h, tid, 256);
  if (a.dtab_part)
    for (int x = tid; x < VECS * nbias; x += 256) diag[x] = 0.f;
  float* my_diag = diag + (tid >> 5) * nbias + 4 * hf - r;
  const RelLane il(lane);
  const int ip = i + off;
  for (int kt = 0; kt < nkt; ++kt) {
    wait_vmem_all();   // this tile and its mask are here
    __syncthreads();   // and nobody reads the one before it any more
    const int j0 = 64 * kt;
    const uint64_t word = __ballot(j0 + lane < klen && keep);
    if (kt + 1 < nkt) {
      ld.issue(kp, vp, a.k_sl, a.v_sl, j0 + 64, a.Lk, lds0 + ((kt + 1) & 1) * STAGE, wave, lane);
      keep = rel_mask_at(a, b, j0 + 64 + lane);
    }
    char* K = smem + (kt & 1) * STAGE;
    char* V = K + CB * 8192;
    if (word == 0) continue;
    if (~word) {
      rel_zero_rows<CB>(K, word, wave, lane);
      __syncthreads();
    }
    if (i_wave >= a.Lq || (a.causal && j0 > i_wave + 31 + off)) continue;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f32x16 s = rel_zero(), dp = rel_zero();
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        s = rel_mfma<T>(rel_row_frag(K + (kk >> 2) * 8192 + t * 4096, il, kk & 3), qf[kk], s);
        dp = rel_mfma<T>(rel_row_frag(V + (kk >> 2) * 8192 + t * 4096, il, kk & 3), gf[kk], dp);
      }
      const int jt = j0 + 32 * t;
      const int rel_hi = jt + 31 - (i_wave + off), rel_lo = jt - (i_wave + 31 + off);
      const bool left = rel_hi <= -a.far, right = rel_lo >= a.far;
      const uint32_t wt = (uint32_t)(word >> (32 * t));
      if (left || right) {
        const float c = bias[left ? 0 : 2 * (a.far + EXT)] - lse;
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = att_exp2(fmaf(s[e], a.sl2, c));
      } else {
        const float* bp = bias + (a.far + EXT + jt + 4 * hf - ip);
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = att_exp2(fmaf(s[e], a.sl2, bp[acc_row(e)]) - lse);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] *= dp[e] - delta;
      if (~wt || (a.causal && rel_hi > 0)) {
        const int jmax = a.causal ? ip - jt - 4 * hf : INT_MAX;
        const uint32_t w = wt >> (4 * hf);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (!((w >> acc_row(e)) & 1) || acc_row(e) > jmax) s[e] = 0.f;
      }
      if (a.dtab_part) {
        if (left || right) {
          float t4 = 0.f;
#pragma unroll
          for (int e = 0; e < 16; ++e) t4 += s[e];
          far_l += left ? t4 : 0.f;
          far_r += left ? 0.f : t4;
        } else {
          float d[3];
          rel_diagonals(s, d);
          float* at = my_diag + (a.far + EXT + jt - (i_wave + off));   // (r = 16 R + c)
          // the upper 16 lanes of a half stand where the lower ones were one k before: one after the other (LDS keeps a wave's order)
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            at[16 * k] += d[k];
            asm volatile("" ::: "memory");
          }
        }
      }
      if (F16) {
        range.follow(s, dq);
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] *= range.factor;
      }
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        const s16x8 df = rel_operand<T>(s, st);
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) dq[dt] = rel_mfma<T>(rel_tr_frag(K + (dt >> 1) * 8192, il, t * 4096 + st * 2048, dt & 1), df, dq[dt]);
      }
    }
  }
  if (i < a.Lq) rel_store_row<T, D>(reinterpret_cast<T*>(a.dq) + (((int64_t)b * a.Lq + i) * a.H + h) * D, nullptr, dq, F16 ? range.undo(a.scale) : a.scale, hf);
  if (!a.dtab_part) return;
  // ---- this workgroup's sums by bucket: the far sums join their wave's vectors at its ends, the vectors are added in order, and
  // a thread per (bucket, slice) collects its distances
  far_l = wave_sum(far_l);
  far_r = wave_sum(far_r);
  __syncthreads();
  if (lane == 0) {
    diag[VECS / 4 * wave * nbias] += far_l;
    diag[VECS / 4 * wave * nbias + 2 * (a.far + EXT)] += far_r;
  }
  __syncthreads();
  const int n = 2 * (a.far + EXT) + 1;
  int* which = reinterpret_cast<int*>(bias);
  for (int x = tid; x < n; x += 256) {
    float t = 0.f;
#pragma unroll
    for (int v = 0; v < VECS; ++v) t += diag[v * nbias + x];
    diag[x] = t;
    which[x] = rel_bucket(a, min(max(x - a.far - EXT, -a.far), a.far));
  }
  __syncthreads();
  const int slices = 256 / a.buckets;
  const int bucket = tid % a.buckets, sl = tid / a.buckets;
  float t = 0.f;
  if (sl < slices)
    for (int x = sl; x < n; x += slices) t += which[x] == bucket ? diag[x] : 0.f;
  float* red = diag + nbias;
  __syncthreads();
  red[tid] = t;
  __syncthreads();
  if (tid < a.buckets) {
    t = 0.f;
    for (int s = 0; s < slices; ++s) t += red[s * a.buckets + tid];
    a.dtab_part[((int64_t)bh * nqb + qb) * a.buckets + tid] = t;
  }
}

// dtable[c][h] = sum over samples and query blocks of the partials, in order.  One workgroup per head.
template <typename W>
__global__ __launch_bounds__(256) void rel_dtable_kernel(const float* part, W* dtable, int B, int H, int nqb, int buckets) {
  __shared__ float red[256];
  const int h = blockIdx.x, slices = 256 / buckets, c = threadIdx.x % buckets, sl = threadIdx.x / buckets;
  float t = 0.f;
  if (sl < slices)
    for (int x = sl; x < B * nqb; x += slices) {
      const int b = x / nqb, qb = x - b * nqb;
      t += part[(((int64_t)b * H + h) * nqb + qb) * buckets + c];
    }
  red[threadIdx.x] = t;
  __syncthreads();
  if (threadIdx.x < buckets) {
    t = 0.f;
    for (int s = 0; s < slices; ++s) t += red[s * buckets + threadIdx.x];
    dtable[(int64_t)threadIdx.x * H + h] = from_f32<W>(t);
  }
}

// ------------------------------------------------------------------------------------------------ backward: dK, dV
// The key on the lane: a wave keeps K and V of its 32 keys as operands, walks the query tiles of all heads of the group, and sums dK^T
// and dV^T of the group in its accumulators.  With few key blocks (few key heads) or unequal ones (causal: the first keys see all rows, the
// last few) the walk is divided among `dkv_splits` workgroups, whose f32 sums rel_dkv_join_kernel adds in order.
// 2 x 16 (on 4) x 4097 x 128 causal: 370 us, 743 TFLOP/s (f16 412), and 23 us for the join.
template <typename T, int D>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void rel_dkv_kernel(const RelArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int CB = D / 64, STAGE = 2 * CB * 8192 + 512, KB = 128, EXT = 96;
  constexpr bool F16 = std::is_same<T, f16_t>::value;
  constexpr int BITS = REL_P_BITS<T>;
  float* bias = reinterpret_cast<float*>(smem + 2 * STAGE);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 31, hf = lane >> 5;
  const int nkb = (a.Lk + KB - 1) / KB, S = a.dkv_splits;
  const RelPlace pl = rel_place(blockIdx.x, nkb * S, a.B * a.Hk);
  const int kb = pl.rank / S, split = pl.rank - kb * S, b = pl.head / a.Hk, hk = pl.head - b * a.Hk;
  const int off = rel_offset(a, b), klen = rel_key_len(a, b, off);
  const int j_wg = kb * KB, j_wave = j_wg + 32 * wave, j = j_wave + r;
  const bool kept = j < klen && rel_mask_at(a, b, j);
  f32x16 dk[D / 32], dv[D / 32];
  RelRange range;   // of 2^BITS dS
  s16x8 kf[D / 16], vf[D / 16];
  {
    const int jc = min(j, a.Lk - 1);
    const T* kp = reinterpret_cast<const T*>(a.k) + b * a.k_sb + hk * a.k_sh + jc * a.k_sl + 8 * hf;
    const T* vp = reinterpret_cast<const T*>(a.v) + b * a.v_sb + hk * a.v_sh + jc * a.v_sl + 8 * hf;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      kf[kk] = *reinterpret_cast<const s16x8*>(kp + 16 * kk);
      vf[kk] = *reinterpret_cast<const s16x8*>(vp + 16 * kk);
    }
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) dk[dt] = dv[dt] = rel_zero();
  }
  const bool wave_keeps = __any(kept), wave_whole = __all(kept);
  const bool wg_keeps = __builtin_amdgcn_readfirstlane(__syncthreads_or(kept));
  // query tiles: causal rows end before i + off = j
  const int nqt = (a.Lq + 63) / 64;
  const int first = a.causal ? max(0, j_wg - off) / 64 : 0;
  const int per = max(nqt - first, 0), all = wg_keeps ? per * a.G : 0;
  const int begin = (int)((int64_t)all * split / S), end = (int)((int64_t)all * (split + 1) / S);
  const RelLane il_(lane);
  const int64_t g_sl = (int64_t)a.H * D;
  const RelLoader<T, CB> ld(a.q_sl, g_sl, wave, lane);
  const uint32_t lds0 = lds_addr_of(smem);
  float rowv = 0.f;   // lanes of waves 0, 1: lse, delta of the next tile's rows
  auto issue = [&](int x) {
    const int h = hk * a.G + x / per, i0 = 64 * (first + x % per);
    const T* qp = reinterpret_cast<const T*>(a.q) + b * a.q_sb + h * a.q_sh;
    const T* gp = reinterpret_cast<const T*>(a.dout) + ((int64_t)b * a.Lq * a.H + h) * D;
    ld.issue(qp, gp, a.q_sl, g_sl, i0, a.Lq, lds0 + ((x - begin) & 1) * STAGE, wave, lane);
    if (wave < 2) {
      const int i = i0 + lane;
      const float* src = wave ? a.delta : a.lse;
      const float past = wave ? 0.f : INFINITY;   // rows past the end: P = 0
      rowv = i < a.Lq ? src[((int64_t)b * a.H + h) * a.Lq + i] : past;
    }
  };
  int head = -1;
  if (begin < end) issue(begin);
  for (int x = begin; x < end; ++x) {
    const int hg = x / per, i0 = 64 * (first + x % per);
    char* Q = smem + ((x - begin) & 1) * STAGE;
    char* Gr = Q + CB * 8192;
    float* rows = reinterpret_cast<float*>(Q + 2 * CB * 8192);   // [lse 64][delta 64]
    wait_vmem_all();
    if (wave < 2) rows[64 * wave + lane] = wave ? rowv : rowv - BITS;   // (P comes out times 2^BITS)
    if (hg != head) {   // (nobody reads the old bias any more once all are past this barrier)
      __syncthreads();
      rel_bias_fill<T>(a, bias, EXT, hk * a.G + hg, tid, 256);
      head = hg;
    }
    __syncthreads();
    if (x + 1 < end) issue(x + 1);
    if (!wave_keeps || (a.causal && i0 + 63 + off < j_wave)) continue;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int it = i0 + 32 * t;
      if (it >= a.Lq || (a.causal && it + 31 + off < j_wave)) continue;
      // phase by phase, P's product before dP is formed: with everything in flight at once D = 128 would not fit 256 registers
      const RelLane il = il_.fresh();
      f32x16 s = rel_zero();
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) s = rel_mfma<T>(rel_row_frag(Q + (kk >> 2) * 8192 + t * 4096, il, kk & 3), kf[kk], s);
      const int rel_hi = j_wave + 31 - (it + off), rel_lo = j_wave - (it + 31 + off);
      const bool left = rel_hi <= -a.far, right = rel_lo >= a.far;
      const bool masked = !wave_whole || (a.causal && rel_hi > 0);
      const int imin = a.causal ? j - off - it - 4 * hf : INT_MIN;
      const float* lr = rows + 32 * t + 4 * hf;
      if (left || right) {
        const float c = bias[left ? 0 : 2 * (a.far + EXT)];
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = fmaf(s[e], a.sl2, c);
      } else {
        const float* bp = bias + (a.far + EXT + j - (it + off) - 4 * hf);
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = fmaf(s[e], a.sl2, bp[-acc_row(e)]);
      }
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const float4 ls = *reinterpret_cast<const float4*>(lr + 8 * q4);
        const float lv[4] = {ls.x, ls.y, ls.z, ls.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) s[4 * q4 + e] = att_exp2(s[4 * q4 + e] - lv[e]);
      }
      if (masked) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = kept && acc_row(e) >= imin ? s[e] : 0.f;
      }
      if (D == 128) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        const s16x8 pf = rel_operand<T>(s, st);
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
          dv[dt] = rel_mfma<T>(rel_tr_frag(Gr + (dt >> 1) * 8192, il, t * 4096 + st * 2048, dt & 1), pf, dv[dt]);
      }
      if (D == 128) __builtin_amdgcn_sched_barrier(0);
      f32x16 dp = rel_zero();
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) dp = rel_mfma<T>(rel_row_frag(Gr + (kk >> 2) * 8192 + t * 4096, il, kk & 3), vf[kk], dp);
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const float4 de = *reinterpret_cast<const float4*>(lr + 64 + 8 * q4);
        const float dl[4] = {de.x, de.y, de.z, de.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) dp[4 * q4 + e] = s[4 * q4 + e] * (dp[4 * q4 + e] - dl[e]);
      }
      if (masked) {   // (what a masked value holds reached dP)
#pragma unroll
        for (int e = 0; e < 16; ++e) dp[e] = kept && acc_row(e) >= imin ? dp[e] : 0.f;
      }
      if (F16) {
        range.follow(dp, dk);
#pragma unroll
        for (int e = 0; e < 16; ++e) dp[e] *= range.factor;
      }
      if (D == 128) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        const s16x8 df = rel_operand<T>(dp, st);
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
          dk[dt] = rel_mfma<T>(rel_tr_frag(Q + (dt >> 1) * 8192, il, t * 4096 + st * 2048, dt & 1), df, dk[dt]);
      }
    }
  }
  if (j < a.Lk) {
    const int64_t at = (((int64_t)b * a.Lk + j) * a.Hk + hk) * D;
    if (!kept) {   // (a NaN in a row's gradient meets P = 0 here)
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) dk[dt] = dv[dt] = rel_zero();
    }
    if (S == 1) {
      rel_store_row<T, D>(reinterpret_cast<T*>(a.dk) + at, nullptr, dk, F16 ? range.undo(__builtin_ldexpf(a.scale, -BITS)) : a.scale, hf);
      rel_store_row<T, D>(reinterpret_cast<T*>(a.dv) + at, nullptr, dv, __builtin_ldexpf(1.f, -BITS), hf);
    } else {
      if (F16) {
        const float k1 = range.undo(__builtin_ldexpf(1.f, -BITS)), v1 = __builtin_ldexpf(1.f, -BITS);
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            dk[dt][e] *= k1;
            dv[dt][e] *= v1;
          }
      }
      const int64_t n = (int64_t)a.B * a.Lk * a.Hk * D;
      rel_store_row<D>(a.dkv_part + 2 * split * n + at, dk, hf);
      rel_store_row<D>(a.dkv_part + (2 * split + 1) * n + at, dv, hf);
    }
  }
}

// dK, dV of the splits' sums, in order; four values a thread
template <typename T>
__global__ __launch_bounds__(256) void rel_dkv_join_kernel(const RelArgs a, int64_t n) {
  const int64_t x = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (x >= n) return;
  float4 k = make_float4(0.f, 0.f, 0.f, 0.f), v = k;
  for (int s = 0; s < a.dkv_splits; ++s) {
    const float4 ks = *reinterpret_cast<const float4*>(a.dkv_part + 2 * s * n + x), vs = *reinterpret_cast<const float4*>(a.dkv_part + (2 * s + 1) * n + x);
    k.x += ks.x; k.y += ks.y; k.z += ks.z; k.w += ks.w;
    v.x += vs.x; v.y += vs.y; v.z += vs.z; v.w += vs.w;
  }
  Vec4<T>::store(reinterpret_cast<T*>(a.dk) + x, make_float4(k.x * a.scale, k.y * a.scale, k.z * a.scale, k.w * a.scale));
  Vec4<T>::store(reinterpret_cast<T*>(a.dv) + x, v);
}

// ------------------------------------------------------------------------------------------------ host
static int rel_dq_blocks(const mmk_rel_attn* p) { return (p->Lq + 127) / 128; }

constexpr int REL_LDS = 160 * 1024;
static int64_t rel_split_lds(const mmk_rel_attn* p) {   // four waves' double-buffered tiles and the bias vector of every head of the group
  return std::max(8 * 2 * (p->D / 64) * 4096 + (int64_t)(p->H / p->Hk) * (2 * (p->max_distance + 1) + 1) * 4, (int64_t)1024 + 4 * 32 * (p->D + 4) * 4);
}
// The few-rows kernel takes over where one block of 32 rows holds all queries of a group.
static bool rel_few_rows(const mmk_rel_attn* p) { return (int64_t)(p->H / p->Hk) * p->Lq <= 32 && rel_split_lds(p) <= REL_LDS; }
// splits of the keys: about two workgroups per CU, at least two tiles of 32 keys per wave
static int rel_splits(const mmk_rel_attn* p) {
  const int64_t groups = (int64_t)p->B * p->Hk;
  const int64_t want = (512 + groups - 1) / groups, most = std::max<int64_t>(1, ((int64_t)p->Lk + 255) / 256);
  return (int)std::min<int64_t>(std::min(want, most), 64);
}
// Workgroups that share one key block's walk: two a CU are wanted, four where causal leaves them unequal, each with 8 query tiles at least
static int rel_dkv_splits(const mmk_rel_attn* p) {
  const int64_t blocks = std::max<int64_t>(1, (int64_t)p->B * p->Hk * ((p->Lk + 127) / 128)), want = p->causal ? 1024 : 512;
  const int64_t tiles = (int64_t)(p->H / p->Hk) * ((p->Lq + 63) / 64);
  return (int)std::max<int64_t>(1, std::min<int64_t>({(want + blocks - 1) / blocks, tiles / 8, 16}));
}
static int64_t rel_dkv_floats(const mmk_rel_attn* p) {
  const int s = rel_dkv_splits(p);
  return s == 1 ? 0 : 2 * (int64_t)s * p->B * p->Lk * p->Hk * p->D;
}

static int rel_check(const mmk_rel_attn* p) {
  MMK_REQUIRE(p != nullptr, "no geometry");
  MMK_REQUIRE(p->dtype == MMK_BF16 || p->dtype == MMK_F16, "operands are bf16 or f16");
  MMK_REQUIRE(p->table_dtype == MMK_F32 || p->table_dtype == p->dtype, "the table is f32 or of the operands' type");
  MMK_REQUIRE(p->D == 64 || p->D == 128, "head dim must be 64 or 128");
  MMK_REQUIRE(p->B >= 0 && p->H >= 1 && p->Hk >= 1 && p->H % p->Hk == 0 && p->Lq >= 0 && p->Lk >= 0, "bad sizes");
  MMK_REQUIRE(p->Lq <= (1 << 28) && p->Lk <= (1 << 28), "sequence too long");
  // a launch holds 2^32 threads: the forward's workgroups take 128 queries of a head each, however many keys there are
  MMK_REQUIRE((int64_t)p->B * p->H * std::max<int64_t>(1, ((int64_t)p->Lq + 127) / 128) < (1 << 24), "too many query rows");
  MMK_REQUIRE(p->buckets >= 1 && p->buckets <= REL_MAX_BUCKETS && p->n_borders >= 0 && p->n_borders <= REL_MAX_BORDERS, "too many buckets");
  MMK_REQUIRE(p->n_borders == 0 || p->borders, "missing borders");
  MMK_REQUIRE(p->near_buckets >= 1 && p->near_buckets <= REL_MAX_BUCKETS, "1 to 256 single distances a side");
  MMK_REQUIRE(p->max_distance >= 1 && p->max_distance <= REL_MAX_FAR, "max_distance must be 1 .. 512");
  MMK_REQUIRE((p->bidirectional ? 2 : 1) * (p->near_buckets + p->n_borders + 1) == p->buckets, "near and logarithmic buckets do not add up");
  for (int i = 0; i < 3; ++i) {
    MMK_REQUIRE(p->q_strides[i] % 8 == 0 && p->k_strides[i] % 8 == 0 && p->v_strides[i] % 8 == 0, "strides must be multiples of 8 elements");
    MMK_REQUIRE(p->q_strides[i] >= 0 && p->k_strides[i] >= 0 && p->v_strides[i] >= 0, "negative strides");
  }
  // a tile's 64 rows are addressed by 32-bit byte offsets
  MMK_REQUIRE(p->q_strides[2] <= (1 << 23) && p->k_strides[2] <= (1 << 23) && p->v_strides[2] <= (1 << 23), "row stride too large");
  MMK_REQUIRE(p->mask_kind >= MMK_REL_MASK_NONE && p->mask_kind <= MMK_REL_MASK_64 && (p->mask_kind == 0) == (p->mask == nullptr), "bad mask");
  for (const void* x : {p->q, p->k, p->v}) MMK_REQUIRE(reinterpret_cast<uintptr_t>(x) % 16 == 0, "operands must be 16-byte aligned");
  return 0;
}

// the backward's, beside those, 128 keys of a key head (divided only where they are few)
static int rel_check_bwd(const mmk_rel_attn* p) {
  if (int rc = rel_check(p)) return rc;
  MMK_REQUIRE((int64_t)p->B * p->Hk * (((int64_t)p->Lk + 127) / 128) < (1 << 24), "too many key rows");
  return 0;
}

static RelArgs rel_args(const mmk_rel_attn* p) {
  RelArgs a = {};
  a.q = p->q;
  a.k = p->k;
  a.v = p->v;
  a.q_sb = p->q_strides[0];
  a.q_sh = p->q_strides[1];
  a.q_sl = p->q_strides[2];
  a.k_sb = p->k_strides[0];
  a.k_sh = p->k_strides[1];
  a.k_sl = p->k_strides[2];
  a.v_sb = p->v_strides[0];
  a.v_sh = p->v_strides[1];
  a.v_sl = p->v_strides[2];
  a.B = p->B;
  a.H = p->H;
  a.Hk = p->Hk;
  a.G = p->H / p->Hk;
  a.Lq = p->Lq;
  a.Lk = p->Lk;
  a.scale = p->scale;
  a.sl2 = p->scale * REL_LOG2E;
  a.table = p->table;
  a.table_f32 = p->table_dtype == MMK_F32;
  a.buckets = p->buckets;
  a.side = p->bidirectional ? p->buckets / 2 : p->buckets;
  a.near = p->near_buckets;
  a.far = p->max_distance;
  a.bidir = p->bidirectional != 0;
  a.n_borders = p->n_borders;
  a.causal = p->causal != 0;
  a.off = p->q_offset;
  a.off_ptr = p->q_offsets;
  a.mask = p->mask;
  a.mask_sb = p->mask_stride;
  a.mask_kind = p->mask_kind;
  for (int i = 0; i < p->n_borders; ++i) a.borders[i] = p->borders[i];
  return a;
}

// lds_most: the largest dynamic LDS any call of this kernel asks for (the opt-in is made once, at its first launch)
template <typename K>
static int rel_launch(K kern, int id, int64_t grid, int lds, int lds_most, const RelArgs& a, hipStream_t st) {
  KernelSetup ks;
  if (int rc = kernel_setup(reinterpret_cast<const void*>(kern), 256, lds_most, &ks)) return rc;
  ProfEvents pe(id);
  hipExtLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(256), lds, st, pe.start, pe.stop, 0, a);
  MMK_LAUNCH_CHECK();
  return 0;
}

// bytes of a vector over the distances -far - ext .. far + ext
static constexpr int rel_vec_bytes(int far, int ext) { return ((2 * (far + ext) + 1 + 3) & ~3) * 4; }

template <typename T, int D>
static int rel_forward(const mmk_rel_attn* p, RelArgs& a, hipStream_t st) {
  if (rel_few_rows(p)) {
    a.splits = rel_splits(p);
    if (int rc = rel_launch(rel_split_kernel<T, D>, MMK_K_REL_ATTN_FWD, (int64_t)a.B * a.Hk * a.splits, (int)rel_split_lds(p), REL_LDS, a, st))
      return rc;
    if (a.splits == 1) return 0;
    const int64_t n = (int64_t)a.B * a.H * a.Lq * (D / 4);
    return rel_launch(rel_join_kernel<T, D>, MMK_K_REL_ATTN_FWD, (n + 255) / 256, 0, 0, a, st);
  }
  constexpr int EXT = 96, TILES = 2 * 2 * (D / 64) * 8192;
  const int64_t grid = (int64_t)a.B * a.H * ((a.Lq + 127) / 128);
  return rel_launch(a.out_lo ? rel_fwd_kernel<T, D, true> : rel_fwd_kernel<T, D, false>, MMK_K_REL_ATTN_FWD, grid, TILES + rel_vec_bytes(a.far, EXT),
                    TILES + rel_vec_bytes(REL_MAX_FAR, EXT), a, st);
}

template <typename T, int D>
static int rel_backward(const mmk_rel_attn* p, RelArgs& a, void* dtable, hipStream_t st) {
  constexpr int TILES = 2 * 2 * (D / 64) * 8192;
  const int nqb = rel_dq_blocks(p);
  if (a.Lq > 0) {
    constexpr int EXT = 96;
    if (int rc = rel_launch(rel_dq_kernel<T, D>, MMK_K_REL_ATTN_BWD, (int64_t)a.B * a.H * nqb,
                            TILES + rel_vec_bytes(a.far, EXT) * (a.dtab_part ? 1 + REL_DIAG : 1),
                            TILES + (1 + REL_DIAG) * rel_vec_bytes(REL_MAX_FAR, EXT), a, st))
      return rc;
  }
  if (a.Lk > 0) {
    const int64_t grid = (int64_t)a.B * a.Hk * ((a.Lk + 127) / 128) * a.dkv_splits;
    if (int rc = rel_launch(rel_dkv_kernel<T, D>, MMK_K_REL_ATTN_BWD, grid, TILES + 1024 + rel_vec_bytes(a.far, 96),
                            TILES + 1024 + rel_vec_bytes(REL_MAX_FAR, 96), a, st))
      return rc;
    if (a.dkv_splits > 1) {
      const int64_t n = (int64_t)a.B * a.Lk * a.Hk * D;
      hipLaunchKernelGGL(rel_dkv_join_kernel<T>, dim3((unsigned)((n / 4 + 255) / 256)), dim3(256), 0, st, a, n);
      MMK_LAUNCH_CHECK();
    }
  }
  if (dtable) {   // (no queries: no partials, and no workspace for them)
    const int n = a.Lq > 0 ? nqb : 0;
    if (p->table_dtype == MMK_F32)
      hipLaunchKernelGGL(rel_dtable_kernel<float>, dim3(a.H), dim3(256), 0, st, a.dtab_part, (float*)dtable, a.B, a.H, n, a.buckets);
    else
      hipLaunchKernelGGL(rel_dtable_kernel<T>, dim3(a.H), dim3(256), 0, st, a.dtab_part, (T*)dtable, a.B, a.H, n, a.buckets);
    MMK_LAUNCH_CHECK();
  }
  return 0;
}

template <typename F>
static int rel_dispatch(const mmk_rel_attn* p, F f) {
  if (p->dtype == MMK_BF16) return p->D == 64 ? f(bf16_t(), std::integral_constant<int, 64>()) : f(bf16_t(), std::integral_constant<int, 128>());
  return p->D == 64 ? f(f16_t(), std::integral_constant<int, 64>()) : f(f16_t(), std::integral_constant<int, 128>());
}

}  // namespace mmk

using namespace mmk;

extern "C" {

int64_t mmk_rel_attn_fwd_ws_floats(const mmk_rel_attn* p) {
  if (rel_check(p)) return -1;
  if (!rel_few_rows(p) || (int64_t)p->B * p->Lq == 0) return 0;
  const int s = rel_splits(p);
  return s == 1 ? 0 : (int64_t)p->B * p->Hk * 32 * s * (p->D + 4);
}

int mmk_rel_attn_fwd(const mmk_rel_attn* p, void* out, void* out_lo, float* lse, float* ws, void* stream) {
  if (int rc = rel_check(p)) return rc;
  if ((int64_t)p->B * p->Lq == 0) return 0;
  MMK_REQUIRE(p->q && out && (p->Lk == 0 || (p->k && p->v)) && p->table, "missing operand");
  MMK_REQUIRE(mmk_rel_attn_fwd_ws_floats(p) == 0 || ws, "missing workspace");
  for (const void* x : {(const void*)out, (const void*)out_lo, (const void*)ws})
    MMK_REQUIRE(reinterpret_cast<uintptr_t>(x) % 16 == 0, "outputs and the workspace must be 16-byte aligned");
  RelArgs a = rel_args(p);
  a.out = out;
  a.out_lo = out_lo;
  a.lse = lse;
  a.part = ws;
  return rel_dispatch(p, [&](auto t, auto d) { return rel_forward<decltype(t), decltype(d)::value>(p, a, (hipStream_t)stream); });
}

int64_t mmk_rel_attn_bwd_ws_floats(const mmk_rel_attn* p, int want_dtable) {
  if (rel_check_bwd(p)) return -1;
  return rel_dkv_floats(p) + (int64_t)p->B * p->H * p->Lq + (want_dtable ? (int64_t)p->B * p->H * rel_dq_blocks(p) * p->buckets : 0);
}

int mmk_rel_attn_bwd(const mmk_rel_attn* p, const void* out, const void* out_lo, const float* lse, const void* dout, void* dq, void* dk, void* dv,
                     void* dtable, float* ws, void* stream) {
  if (int rc = rel_check_bwd(p)) return rc;
  MMK_REQUIRE(p->Lk == 0 || (dk && dv && p->k && p->v), "missing operand");
  MMK_REQUIRE(p->Lq == 0 || (p->q && out && out_lo && lse && dout && dq && p->table), "missing operand");
  MMK_REQUIRE(ws || mmk_rel_attn_bwd_ws_floats(p, dtable != nullptr) == 0, "missing workspace");
  for (const void* x : {out, out_lo, dout, (const void*)dq, (const void*)dk, (const void*)dv, (const void*)ws})
    MMK_REQUIRE(reinterpret_cast<uintptr_t>(x) % 16 == 0, "gradients and the workspace must be 16-byte aligned");
  if (p->B == 0) {
    if (!dtable) return 0;
    MMK_REQUIRE(false, "the table's gradient of no samples is the caller's zero");
  }
  RelArgs a = rel_args(p);
  a.o = out;
  a.o_lo = out_lo;
  a.lse = const_cast<float*>(lse);
  a.dout = dout;
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  a.dkv_part = ws;   // (first: its rows are read four floats at a time)
  a.dkv_splits = rel_dkv_splits(p);
  a.delta = ws + rel_dkv_floats(p);
  a.dtab_part = dtable ? a.delta + (int64_t)p->B * p->H * p->Lq : nullptr;
  return rel_dispatch(p, [&](auto t, auto d) { return rel_backward<decltype(t), decltype(d)::value>(p, a, dtable, (hipStream_t)stream); });
}

}  // extern "C"
