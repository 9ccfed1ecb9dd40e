// MX4: 4-bit microscaled floating point (OCP microscaling: e2m1 elements, one e8m0 scale per 32 columns) -- quantisation, its
// inverse, and the product y = act(x w^T + bias) [+ res] on v_mfma_scale_f32_16x16x128_f8f6f4, which multiplies the block scales
// in.  The step below the e4m3 convs (conv_f8.hip): a pointwise conv IS such a product over pixels.
//
// One block of 32 values v:  E = biased exponent of the largest |v|,  scale byte s = max(E - 2, 0),  X = 2^(s - 127),
// code = e2m1(v / X): magnitudes 0, 1/2, 1, 3/2, 2, 3, 4, 6 (codes 0..7), sign in bit 3, round to nearest even, saturating at 6
// (|v| / X < 8: a value in (7, 8) loses up to a quarter -- the definition's choice of the scale).  v / X is exact (a power of
// two), so the rounding to the code is the only one.  A block with a value that is not finite gets s = 255 and reads as NaN.
//
// Storage: codes[rows][ceil(cols / 32) * 16] bytes, two codes to a byte, the first in the low half; scales[rows][ceil(cols / 32)].
// Columns behind the last are zeros.  An MFMA operand of 16 rows x 128 columns is then, per lane (row = lane & 15, block
// g = lane >> 4), one aligned 16-byte load of codes and one scale byte: nothing is rearranged between memory and the pipe.
#include <algorithm>
#include <type_traits>

#include "conv_common.h"

namespace yl {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef int v4i __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------------------------------------ element access
template <typename T>
__device__ __forceinline__ float to_f32(T v) {
  return (float)v;
}
// eight values from p, the ones from `n` on as zeros; VEC: p is 16-byte aligned and all eight are there
template <typename T>
__device__ __forceinline__ void load8(const T* p, int n, bool vec, float (&v)[8]) {
  if (vec && n >= 8) {
    if constexpr (sizeof(T) == 4) {
      const f32x4 a = reinterpret_cast<const f32x4*>(p)[0], b = reinterpret_cast<const f32x4*>(p)[1];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] = a[j];
        v[4 + j] = b[j];
      }
    } else {
      typedef T t8 __attribute__((ext_vector_type(8)));
      const t8 a = *reinterpret_cast<const t8*>(p);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = (float)a[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? to_f32(p[j]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int n, bool vec, const float (&v)[8]) {
  if (vec && n >= 8) {
    if constexpr (sizeof(T) == 4) {
      reinterpret_cast<f32x4*>(p)[0] = f32x4{v[0], v[1], v[2], v[3]};
      reinterpret_cast<f32x4*>(p)[1] = f32x4{v[4], v[5], v[6], v[7]};
    } else {
      typedef T t8 __attribute__((ext_vector_type(8)));
      *reinterpret_cast<t8*>(p) = t8{(T)v[0], (T)v[1], (T)v[2], (T)v[3], (T)v[4], (T)v[5], (T)v[6], (T)v[7]};
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = (T)v[j];
  }
}

// the other lanes of a group of four: max over the 32 values of a block
__device__ __forceinline__ unsigned quad_max(unsigned m) {
  unsigned o = (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xF, 0xF, true);  // lanes 1 0 3 2
  m = m > o ? m : o;
  o = (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xF, 0xF, true);  // lanes 2 3 0 1
  return m > o ? m : o;
}

// the scale byte of a block from its largest magnitude, the bits of |v| (inf and NaN are the largest)
__device__ __forceinline__ unsigned scale_of(unsigned m) {
  const unsigned e = m >> 23;
  return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}
__device__ __forceinline__ unsigned codes8(const float (&v)[8], unsigned s) {
  const float x = __uint_as_float(s ? s << 23 : 0x00400000u);  // 2^(s - 127)
  unsigned c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], x, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], x, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], x, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], x, 3);
}
// Four lanes hold a block, eight values each: -> this lane's eight codes (4 bytes), the block's scale byte.
__device__ __forceinline__ unsigned quantize8(const float (&v)[8], unsigned* scale_byte) {
  unsigned m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const unsigned b = __float_as_uint(v[j]) & 0x7FFFFFFFu;
    m = m > b ? m : b;
  }
  *scale_byte = scale_of(quad_max(m));
  return codes8(v, *scale_byte);
}

// the float 2^(s - 127); NaN for 255.  (2^-127 is not a normal number: its own bit pattern.)
__device__ __forceinline__ float scale_value(unsigned s) {
  return __uint_as_float(s == 0 ? 0x00400000u : (s == 255u ? 0x7FC00000u : s << 23));
}

// item = (row, group of eight columns) of a [rows][per_row] list of fewer than 2^32
struct Item {
  long long row;
  int c8;
};
__device__ __forceinline__ Item item_of(unsigned i, unsigned per_row) {
  const unsigned q = i / per_row;
  return Item{q, (int)(i - q * per_row)};
}

// One lane holds a whole block: 32 values from p (zeros from the n-th on) -> the 16 bytes of codes, the scale byte.
template <typename T>
__device__ __forceinline__ v4i quantize32(const T* p, int n, bool vec, int* scale_byte) {
  float v[4][8];
  unsigned m = 0;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    load8(p + q * 8, n - q * 8, vec, v[q]);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const unsigned b = __float_as_uint(v[q][j]) & 0x7FFFFFFFu;
      m = m > b ? m : b;
    }
  }
  const unsigned s = scale_of(m);
  v4i c;
#pragma unroll
  for (int q = 0; q < 4; ++q) c[q] = (int)codes8(v[q], s);
  *scale_byte = (int)s;
  return c;
}

struct QuantArgs {
  const void* x;
  long long rows, stride;  // stride in elements
  int cols, kb;            // blocks per row
  int vec;                 // every group of eight starts on 16 bytes
  uint8_t* codes;
  uint8_t* scales;
};

// Four lanes to a block, eight values each: one 16-byte load of 16-bit values, one 4-byte store.  Bound by memory: 204800 x 384 bf16 (199 MB)
// 43 us, 4600 GB/s; its inverse 30 us (the codes come from cache there).
template <typename T>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(QuantArgs a) {
  const unsigned per_row = 4u * (unsigned)a.kb;
  const unsigned i = blockIdx.x * 256u + threadIdx.x;
  if (i >= (unsigned)a.rows * per_row) return;  // (whole groups of four lanes: the list's length is a multiple of 4)
  const Item t = item_of(i, per_row);
  float v[8];
  load8(static_cast<const T*>(a.x) + t.row * a.stride + t.c8 * 8, a.cols - t.c8 * 8, a.vec, v);
  unsigned s;
  const unsigned c = quantize8(v, &s);
  reinterpret_cast<unsigned*>(a.codes)[i] = c;
  if ((t.c8 & 3) == 0) a.scales[t.row * a.kb + (t.c8 >> 2)] = (uint8_t)s;
}

template <typename T>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(QuantArgs a, T* y) {
  const unsigned per_row = 4u * (unsigned)a.kb;
  const unsigned i = blockIdx.x * 256u + threadIdx.x;
  if (i >= (unsigned)a.rows * per_row) return;
  const Item t = item_of(i, per_row);
  const unsigned c = reinterpret_cast<const unsigned*>(a.codes)[i];
  const float x = scale_value(a.scales[t.row * a.kb + (t.c8 >> 2)]);
  float v[8];
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const f32x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 1);
  const f32x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 3);
  v[0] = p0[0] * x, v[1] = p0[1] * x, v[2] = p1[0] * x, v[3] = p1[1] * x;
  v[4] = p2[0] * x, v[5] = p2[1] * x, v[6] = p3[0] * x, v[7] = p3[1] * x;
  store8(y + t.row * a.stride + t.c8 * 8, a.cols - t.c8 * 8, a.vec, v);
}

// ------------------------------------------------------------------------------------------------ product
struct LinearArgs {
  const void* x;           // activations: codes (or, for few rows, values), row stride in elements of what it is
  long long x_stride;
  int xvec;                // values: every group of eight starts on 16 bytes
  const uint8_t* xs;       // scales
  const uint8_t *wc, *ws;  // weight
  long long rows;
  int n, k, kb;
  const float* bias;
  const void* res;
  long long res_stride;
  void* y;
  long long y_stride;
  int act;
  int vec;                         // every group of eight results (and residuals) starts on 16 bytes
  int ntiles, mtiles;              // tiled product: tiles along n and the rows, groups of 64 rows of the tiled scales
  int wgroups, xgroups;
};

__device__ __forceinline__ v8i widen(v4i v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1); }

// y[m][n .. n + 4): bias, SiLU, residual, one rounding.  What is added is asked for ahead of the product.
template <typename T>
struct Finish4 {
  typedef T t4 __attribute__((ext_vector_type(4)));
  float bias[4], res[4];
  __device__ __forceinline__ void load(const LinearArgs& a, long long m, int n) {
    const int left = a.n - n;
    const T* rp = static_cast<const T*>(a.res) + m * a.res_stride + n;
#pragma unroll
    for (int r = 0; r < 4; ++r) bias[r] = a.bias && r < left ? a.bias[n + r] : 0.f;
    if (a.res) {
      if (a.vec && left >= 4) {
        const t4 q = *reinterpret_cast<const t4*>(rp);
#pragma unroll
        for (int r = 0; r < 4; ++r) res[r] = (float)q[r];
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) res[r] = r < left ? (float)rp[r] : 0.f;
      }
    }
  }
  __device__ __forceinline__ void store(const LinearArgs& a, f32x4 v, long long m, int n) const {
    const int left = a.n - n;
    T* yp = static_cast<T*>(a.y) + m * a.y_stride + n;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      v[r] += bias[r];
      if (a.act) v[r] = silu_f(v[r]);
      if (a.res) v[r] += res[r];
    }
    if (a.vec && left >= 4) {
      *reinterpret_cast<t4*>(yp) = t4{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (r < left) yp[r] = (T)v[r];
    }
  }
};

// ------------------------------------------------------------------------------------------------ product, split over k
// Few rows: the product is the time it takes to read the weight (one row of x: 0.53 bytes per multiply-add), and a grid of large
// tiles would leave most of the chip idle.  A workgroup owns 16 WT weight rows x 16 XT rows of x; its NW waves take the k-steps in
// turn, operands straight from memory into registers, and the partial sums meet in LDS in a fixed order.
// X: what x is: codes (uint8_t), or the values themselves -- a lane's part of the operand is one row's block of 32, so each lane
// quantises its own, without a launch, a workspace or an exchange (16 rows and weights of up to 2^24 elements: see plan_linear).  Lanes of
// rows that x does not have quantise the last one's block once more: 614 vector instructions of a wave for one row of 4096, most of them that.
// Measured, one row: 4096 x 4096 values 8 us (cold caches 11), codes 5-6; 128000 x 4096 codes 63 us, 4400 GB/s.
template <typename T, typename X, int WT, int XT, int NW>
__global__ __launch_bounds__(64 * NW) void mx4_split_kernel(LinearArgs a) {
  __shared__ __attribute__((aligned(16))) f32x4 part[NW][WT * XT][64];
  const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int n0 = (int)(blockIdx.x % (unsigned)a.ntiles) * (16 * WT);
  const long long m0 = (long long)(blockIdx.x / (unsigned)a.ntiles) * (16 * XT);
  constexpr bool CODES = std::is_same_v<X, uint8_t>;
  const uint8_t *wp[WT], *wsp[WT], *xsp[XT];
  const X* xp[XT];
#pragma unroll
  for (int i = 0; i < WT; ++i) {  // rows behind the last: the last one's values, not stored
    const long long row = min(n0 + i * 16 + r, a.n - 1);
    wp[i] = a.wc + row * a.kb * 16;
    wsp[i] = a.ws + row * a.kb;
  }
#pragma unroll
  for (int j = 0; j < XT; ++j) {
    const long long row = min(m0 + j * 16 + r, a.rows - 1);
    xp[j] = static_cast<const X*>(a.x) + row * a.x_stride;
    xsp[j] = a.xs + row * a.kb;
  }
  f32x4 acc[WT][XT];
#pragma unroll
  for (int i = 0; i < WT; ++i)
#pragma unroll
    for (int j = 0; j < XT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  // the tile that this wave finishes
  static_assert(WT * XT <= NW, "a wave finishes one tile at most");
  const int fi = wave / XT, fj = wave % XT, fn = n0 + fi * 16 + 4 * g;
  const long long fm = m0 + fj * 16 + r;
  const bool finishes = wave < WT * XT && fm < a.rows;
  Finish4<T> fin;
  if (finishes) fin.load(a, fm, fn);
  const int nk = (a.kb + 3) >> 2;
  constexpr int U = WT * XT <= 2 ? 4 : 2;  // k-steps whose loads are in flight together
  for (int it0 = wave; it0 < nk; it0 += U * NW) {
    v4i w[U][WT], x[U][XT];
    int sw[U][WT], sx[U][XT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u && it0 + u * NW >= nk) break;  // (the same in every lane)
      const int b = (it0 + u * NW) * 4 + g;
      const bool in = b < a.kb;  // columns behind the last: zeros
      const int bb = in ? b : 0;
#pragma unroll
      for (int i = 0; i < WT; ++i) {
        w[u][i] = *reinterpret_cast<const v4i*>(wp[i] + (long long)bb * 16);
        sw[u][i] = wsp[i][bb];
        if (!in) w[u][i] = v4i{0, 0, 0, 0}, sw[u][i] = 127;
      }
#pragma unroll
      for (int j = 0; j < XT; ++j) {
        if constexpr (CODES) {
          x[u][j] = *reinterpret_cast<const v4i*>(xp[j] + (long long)bb * 16);
          sx[u][j] = in ? xsp[j][bb] : 127;
        } else {
          x[u][j] = quantize32(xp[j] + (long long)bb * 32, in ? a.k - bb * 32 : 0, a.xvec, &sx[u][j]);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u && it0 + u * NW >= nk) break;
#pragma unroll
      for (int i = 0; i < WT; ++i)
#pragma unroll
        for (int j = 0; j < XT; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(widen(w[u][i]), widen(x[u][j]), acc[i][j], 4, 4, 0, sw[u][i], 0, sx[u][j]);
    }
  }
#pragma unroll
  for (int i = 0; i < WT; ++i)
#pragma unroll
    for (int j = 0; j < XT; ++j) part[wave][i * XT + j][lane] = acc[i][j];
  __syncthreads();
  if (!finishes) return;
  f32x4 s = part[0][wave][lane];
#pragma unroll
  for (int w = 1; w < NW; ++w) s += part[w][wave][lane];
  fin.store(a, s, fm, fn);
}

// ------------------------------------------------------------------------------------------------ tiled product
// D = W X^T on 16 x 16 tiles: operand A = weight rows, so a lane's four results are consecutive columns of y.  Rows of two adjacent
// weight tiles interleave (row r of tile t is column (t / 2) 32 + (r / 4) 8 + (t & 1) 4 + r % 4): the two tiles of a lane are then 8
// consecutive columns, 16 bytes of a bf16 row.
__device__ __forceinline__ int weight_row(int t, int r) { return (t >> 1) * 32 + (r >> 2) * 8 + (t & 1) * 4 + (r & 3); }

// Scales in the order the pipe takes them: S[k4][group of 64 rows][lane][tile 0..3], a dword = the bytes of four successive k-steps
// (128 columns each) for the lane's row and block -- v_mfma_scale picks the byte by an immediate, so 16 bytes per lane feed four
// tiles through 512 columns and no instruction unpacks anything.
__device__ __forceinline__ unsigned scale_slot(int row64, int block16, bool weight) {
  // row64: row inside its group of 64; block16: block inside its group of 16 columns-blocks -> byte offset in the 1 KiB
  int t, r;
  if (weight) {  // inverse of weight_row
    const int q = row64 & 31;
    t = (row64 >> 5) * 2 + ((q >> 2) & 1);
    r = (q >> 3) * 4 + (q & 3);
  } else {
    t = row64 >> 4;
    r = row64 & 15;
  }
  return (unsigned)((((block16 & 3) * 16 + r) * 4 + t) * 4 + (block16 >> 2));
}

constexpr int GROUPS_Y = 32768;  // groups of 64 rows along y of the grid, the rest along z
struct TileArgs {
  QuantArgs q;         // x; q.codes nullptr: x comes quantised, q.scales are its scales
  uint8_t* xs;         // tiled scales of x
  const uint8_t* ws;   // the weight's scales [n][kb]
  uint8_t* wst;        // ... tiled
  int n, xgroups, wgroups;  // groups of 64 rows
};

// One workgroup: 64 rows x 512 columns of x -- codes and the 1 KiB of tiled scales -- or the scales of 64 weight rows.  16384 x 4096 bf16 and
// 4096 weight rows 35 us (4900 GB/s), 12800 x 768 9 us (latency: every load of the launch is in flight at once).
template <typename T>
__global__ __launch_bounds__(1024) void mx4_tile_kernel(TileArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t sm[1024];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int kb = a.q.kb;
  const int group = (int)(blockIdx.z * gridDim.y + blockIdx.y);  // (gridDim.y is at most GROUPS_Y)
  if (group >= a.xgroups + a.wgroups) return;
  const bool weight = group >= a.xgroups;
  const int rg = weight ? group - a.xgroups : group, k4 = blockIdx.x;
  sm[tid] = 0x7F;
  __syncthreads();
  if (weight || !a.q.codes) {
    const uint8_t* src = weight ? a.ws : a.q.scales;
    const long long rows = weight ? a.n : a.q.rows;
    const int row = tid >> 4, blk = tid & 15;
    const long long gr = (long long)rg * 64 + row;
    const int gb = k4 * 16 + blk;
    if (gr < rows && gb < kb) sm[scale_slot(row, blk, weight)] = src[gr * kb + gb];
  } else {
    const int c8 = k4 * 64 + lane;  // this lane's group of eight columns
    const bool live = c8 < 4 * kb;
    const T* x = static_cast<const T*>(a.q.x);
    float v[4][8];
#pragma unroll
    for (int u = 0; u < 4; ++u) {  // a wave's four rows are in flight together
      const long long row = (long long)rg * 64 + wave * 4 + u;
      const int left = live && row < a.q.rows ? a.q.cols - c8 * 8 : 0;
      load8(x + row * a.q.stride + c8 * 8, left, a.q.vec, v[u]);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int r64 = wave * 4 + u;
      const long long row = (long long)rg * 64 + r64;
      unsigned s;
      const unsigned c = quantize8(v[u], &s);
      if (live && row < a.q.rows) {
        reinterpret_cast<unsigned*>(a.q.codes)[row * (4 * kb) + c8] = c;
        if ((lane & 3) == 0) sm[scale_slot(r64, lane >> 2, false)] = (uint8_t)s;
      }
    }
  }
  __syncthreads();
  if (tid < 256) {
    unsigned* dst = reinterpret_cast<unsigned*>(weight ? a.wst : a.xs) + ((size_t)k4 * (weight ? a.wgroups : a.xgroups) + rg) * 256;
    dst[tid] = reinterpret_cast<const unsigned*>(sm)[tid];
  }
}

typedef __attribute__((address_space(3))) void lds_void_m;

// A workgroup of 2 x NWM waves owns 32 WT weight rows x 16 NWM XT activation rows; a wave WT x XT tiles.  Both operands pass through
// LDS by LDS-DMA in slices of KS k-steps (128 columns, 64 bytes of a row each) through a ring of NS; a 1 KiB piece is 16 / KS rows,
// neighbouring lanes on one row.  Measured, kernel alone: 16384 x 4096 x 4096 with bias, SiLU and residual 205 us, 2.7 PFLOP/s (8192^3, call:
// 3.2; bound by LDS reads of the fragments beside the MFMAs, and by the epilogue's 268 MB); 12800 x 768 x 768 15.7 us, 0.96 PFLOP/s (six
// k-steps to a tile: prologue and epilogue).  The 16-byte blocks of a row are permuted by xor with a function of the row, which makes the
// fragment reads (16 rows, one block) conflict-free although rows lie 64 or 128 bytes apart.
template <typename T, int WT, int XT, int NWM, int KS, int NS>
__global__ __launch_bounds__(128 * NWM, 2) void mx4_gemm_kernel(LinearArgs a) {
  constexpr int NW = 2 * NWM;
  constexpr int TN = 32 * WT, TM = 16 * NWM * XT;
  constexpr int TILE = KS * 1024;                                // bytes of a 16-row tile in a slice
  constexpr int NPA = TN / 16 * KS, NP = NPA + TM / 16 * KS, PW = NP / NW;  // 1 KiB pieces of a slice; per wave
  constexpr int STAGE = NP * 1024;
  constexpr int LB = 2 + (KS == 2), LM = (1 << LB) - 1;          // lanes per row of a piece: 4 KS
  static_assert(NP % NW == 0 && NPA % NW == 0 && NW % KS == 0, "pieces divide over the waves");
  extern __shared__ __attribute__((aligned(16))) unsigned char gsm[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, r = lane & 15;
  const int wn = wave / NWM, wm = wave % NWM;
  // tiles: groups of eight activation tiles walk the weight tiles together, consecutive workgroups of an XCD share both
  const int tile = xcd_remap((int)blockIdx.x, (int)gridDim.x);
  const int per = 8 * a.ntiles, grp = tile / per, first = grp * 8;
  const int gm = min(8, a.mtiles - first), rest = tile - grp * per;
  const int tm = first + rest % gm, tn = rest / gm;
  const long long m0 = (long long)tm * TM;
  const int n0 = tn * TN;
  const int pitch = a.kb * 16;
  const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(a.wc + (long long)n0 * pitch), (short)0, (unsigned)min(TN, a.n - n0) * (unsigned)pitch, 0x00020000);
  const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(static_cast<const uint8_t*>(a.x) + m0 * pitch), (short)0, (unsigned)min((long long)TM, a.rows - m0) * (unsigned)pitch, 0x00020000);
  const int nk = (a.kb + 3) >> 2;            // k-steps
  // the permutation of a row's blocks, and this lane's part of a piece: row lane / (4 KS), block (lane mod 4 KS) permuted
  auto swz = [](int row) { return KS == 1 ? -(row >> 2) & 3 : (row >> 1) & 7; };
  const int pr = lane >> LB;
  unsigned src[PW];  // byte offset in the operand, without the slice
  int blk = 0;       // (the same for every piece of a wave: its pieces cover the same half of a tile)
#pragma unroll
  for (int i = 0; i < PW; ++i) {
    const int p = wave + NW * i, t = p / KS, row = (p % KS) * (16 / KS) + pr;
    const int b = (lane & LM) ^ swz(row);
    src[i] = (unsigned)(p < NPA ? weight_row(t, row) : (t - NPA / KS) * 16 + row) * (unsigned)pitch + (unsigned)b * 16u;
    blk = b;
  }
  auto issue = [&](int sl, int slot) __attribute__((always_inline)) {
    const unsigned past = sl * (4 * KS) + blk < a.kb ? (unsigned)sl * (64u * KS) : OOB_LANE;  // columns behind the last: zeros
#pragma unroll
    for (int i = 0; i < PW; ++i) {
      const int p = wave + NW * i;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(i < NPA / NW ? rw : rx, (lds_void_m*)(gsm + slot * STAGE + p * 1024), 16,
                                               (int)(past == OOB_LANE ? OOB_LANE : src[i] + past), 0, 0, 0);
    }
  };
  // tiled scales of this wave's tiles: four tiles' bytes for four slices are 16 bytes of a lane
  struct Scales {
    v4i w[WT / 4], x[XT / 4];
  };
  const v4i* wsp = reinterpret_cast<const v4i*>(a.ws) + ((size_t)(n0 >> 6) + wn * (WT / 4)) * 64 + lane;
  const v4i* xsp = reinterpret_cast<const v4i*>(a.xs) + ((size_t)(m0 >> 6) + wm * (XT / 4)) * 64 + lane;
  const size_t wstep = (size_t)a.wgroups * 64, xstep = (size_t)a.xgroups * 64;
  const int wleft = a.wgroups - ((n0 >> 6) + wn * (WT / 4)), xleft = a.xgroups - (int)((m0 >> 6) + wm * (XT / 4));
  const int k4n = (nk + 3) >> 2;
  auto scales = [&](int k4, Scales& s) __attribute__((always_inline)) {
    const v4i one = {0x7F7F7F7F, 0x7F7F7F7F, 0x7F7F7F7F, 0x7F7F7F7F};
    const int k = min(k4, k4n - 1);
#pragma unroll
    for (int i = 0; i < WT / 4; ++i) s.w[i] = i < wleft ? wsp[k * wstep + i * 64] : one;
#pragma unroll
    for (int i = 0; i < XT / 4; ++i) s.x[i] = i < xleft ? xsp[k * xstep + i * 64] : one;
  };

  f32x4 acc[WT][XT];
#pragma unroll
  for (int i = 0; i < WT; ++i)
#pragma unroll
    for (int j = 0; j < XT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  const unsigned char* ap = gsm + wn * WT * TILE + r * (64 * KS);
  const unsigned char* bp = gsm + (NPA * 1024) + wm * XT * TILE + r * (64 * KS);
  struct Frags {
    v4i w[WT], x[XT];
  };
  auto load = [&](int slot, int ks, Frags& f) __attribute__((always_inline)) {
    const unsigned o = (unsigned)slot * STAGE + (unsigned)(((ks * 4 + g) ^ swz(r)) * 16);
#pragma unroll
    for (int j = 0; j < XT; ++j) f.x[j] = *reinterpret_cast<const v4i*>(bp + o + j * TILE);
#pragma unroll
    for (int i = 0; i < WT; ++i) f.w[i] = *reinterpret_cast<const v4i*>(ap + o + i * TILE);
  };
  auto mma = [&](const Frags& f, const Scales& s, auto tag) __attribute__((always_inline)) {
    constexpr int S = decltype(tag)::value;
#pragma unroll
    for (int i = 0; i < WT; ++i)
#pragma unroll
      for (int j = 0; j < XT; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(widen(f.w[i]), widen(f.x[j]), acc[i][j], 4, 4, S, s.w[i >> 2][i & 3], S,
                                                                     s.x[j >> 2][j & 3]);
  };
  // my pieces of the oldest slice in flight have landed, my reads are done; behind the barrier so have everybody's
  auto enter = [&]() __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NS - 2) * PW) : "memory");
    __builtin_amdgcn_s_barrier();
  };
  Scales sc, sn;
  scales(0, sn);
#pragma unroll
  for (int s = 0; s < NS - 1; ++s) issue(s, s);
  int slot = 0, sl = 0;
  for (int k4 = 0; k4 < k4n; ++k4) {
    sc = sn;
    scales(k4 + 1, sn);
    auto step = [&](auto tag) __attribute__((always_inline)) {
      constexpr int S = decltype(tag)::value;
      if (k4 * 4 + S >= nk) return;
      if constexpr (S % KS == 0) {
        enter();
        issue(sl + NS - 1, slot == 0 ? NS - 1 : slot - 1);
      }
      Frags f;
      load(slot, S % KS, f);
      mma(f, sc, tag);
      if constexpr ((S + 1) % KS == 0) {
        ++sl;
        slot = slot + 1 == NS ? 0 : slot + 1;
      }
    };
    step(std::integral_constant<int, 0>{});
    step(std::integral_constant<int, 1>{});
    step(std::integral_constant<int, 2>{});
    step(std::integral_constant<int, 3>{});
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the last refills, all out of range)

  // epilogue, a row of y at a time: a lane's pieces of it are 64 bytes apart, so a row's stores (and residual loads) complete lines
  float bias[WT / 2][8];
#pragma unroll
  for (int i = 0; i < WT / 2; ++i)
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int n = n0 + (wn * (WT / 2) + i) * 32 + g * 8 + q;
      bias[i][q] = a.bias && n < a.n ? a.bias[n] : 0.f;
    }
#pragma unroll
  for (int j = 0; j < XT; ++j) {
    const long long m = m0 + (wm * XT + j) * 16 + r;
    if (m < a.rows) {
      float rv[WT / 2][8];
      if (a.res) {
#pragma unroll
        for (int i = 0; i < WT / 2; ++i) {
          const int n = n0 + (wn * (WT / 2) + i) * 32 + g * 8;
          load8(static_cast<const T*>(a.res) + m * a.res_stride + n, a.n - n, a.vec, rv[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < WT / 2; ++i) {
        const int n = n0 + (wn * (WT / 2) + i) * 32 + g * 8;
        float v[8];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          v[q] = acc[2 * i][j][q] + bias[i][q];
          v[4 + q] = acc[2 * i + 1][j][q] + bias[i][4 + q];
        }
        if (a.act) silu8(v);
        if (a.res) {
#pragma unroll
          for (int q = 0; q < 8; ++q) v[q] += rv[i][q];
        }
        store8(static_cast<T*>(a.y) + m * a.y_stride + n, a.n - n, a.vec, v);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ host
static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
static int elem_bytes(int dtype) { return dtype == YL_F32 ? 4 : 2; }
static bool value_type(int dtype) { return dtype == YL_BF16 || dtype == YL_F16 || dtype == YL_F32; }

// the shape checks the entry points share; `who` names the call in the message
static int check_matrix(const char* who, long long rows, long long cols, long long stride) {
  if (rows < 0 || cols < 1) return fail(-1, std::string(who) + ": rows >= 0 and columns >= 1 are needed");
  if (cols > (1LL << 22)) return fail(-3, std::string(who) + ": more than 4194304 columns");
  if (rows > (1LL << 40) / ((cols + 31) / 32)) return fail(-3, std::string(who) + ": more than 2^40 blocks");
  if (rows > 1 && stride < cols) return fail(-1, std::string(who) + ": the row stride is smaller than a row");
  return 0;
}

template <typename F>
static int by_type(int dtype, F f) {
  if (dtype == YL_BF16) return f((__bf16*)nullptr);
  if (dtype == YL_F16) return f((_Float16*)nullptr);
  return f((float*)nullptr);
}

// four threads to a block of 32; a launch has fewer than 2^32 threads (a larger one is cut off, without an error)
static int grid_of(const char* who, long long rows, int kb, unsigned* grid) {
  if (rows > (0xFFFFFF00LL / 4) / kb) return fail(-3, std::string(who) + ": more than 2^30 blocks of 32 columns in one call");
  *grid = (unsigned)((rows * 4 * kb + 255) / 256);
  return 0;
}

static int quantize_launch(const void* x, int dtype, long long rows, long long cols, long long stride, uint8_t* codes,
                           uint8_t* scales, hipStream_t s) {
  QuantArgs a{};
  a.x = x, a.rows = rows, a.stride = stride, a.cols = (int)cols, a.kb = (int)((cols + 31) / 32);
  a.vec = aligned16(x) && (rows == 1 || stride * elem_bytes(dtype) % 16 == 0);
  a.codes = codes, a.scales = scales;
  unsigned grid;
  if (int rc = grid_of("mx4_quantize", rows, a.kb, &grid)) return rc;
  return by_type(dtype, [&](auto* t) {
    hipLaunchKernelGGL(mx4_quantize_kernel<std::remove_pointer_t<decltype(t)>>, dim3(grid), dim3(256), 0, s, a);
    YL_HIP(hipGetLastError());
    return 0;
  });
}

}  // namespace yl

using namespace yl;

extern "C" int yl_mx4_quantize(const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t x_stride, uint8_t* codes,
                               uint8_t* scales, void* stream) {
  if (!value_type(x_dtype)) return fail(-1, "mx4_quantize: bf16, fp16 or fp32 values");
  if (int rc = check_matrix("mx4_quantize", rows, cols, x_stride)) return rc;
  if (rows == 0) return 0;
  if (!x || !codes || !scales) return fail(-1, "mx4_quantize: null pointer");
  if (!aligned16(codes)) return fail(-1, "mx4_quantize: codes must be 16-byte aligned");
  return quantize_launch(x, x_dtype, rows, cols, x_stride, codes, scales, static_cast<hipStream_t>(stream));
}

extern "C" int yl_mx4_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t cols, void* y, int y_dtype,
                                 int64_t y_stride, void* stream) {
  if (!value_type(y_dtype)) return fail(-1, "mx4_dequantize: bf16, fp16 or fp32 values");
  if (int rc = check_matrix("mx4_dequantize", rows, cols, y_stride)) return rc;
  if (rows == 0) return 0;
  if (!y || !codes || !scales) return fail(-1, "mx4_dequantize: null pointer");
  if (!aligned16(codes)) return fail(-1, "mx4_dequantize: codes must be 16-byte aligned");
  QuantArgs a{};
  a.rows = rows, a.stride = y_stride, a.cols = (int)cols, a.kb = (int)((cols + 31) / 32);
  a.vec = aligned16(y) && (rows == 1 || y_stride * elem_bytes(y_dtype) % 16 == 0);
  a.codes = const_cast<uint8_t*>(codes), a.scales = const_cast<uint8_t*>(scales);
  unsigned grid;
  if (int rc = grid_of("mx4_dequantize", rows, a.kb, &grid)) return rc;
  return by_type(y_dtype, [&](auto* t) {
    typedef std::remove_pointer_t<decltype(t)> T;
    hipLaunchKernelGGL(mx4_dequantize_kernel<T>, dim3(grid), dim3(256), 0, static_cast<hipStream_t>(stream), a, static_cast<T*>(y));
    YL_HIP(hipGetLastError());
    return 0;
  });
}

// ---- how a product runs: a wave per 16 x 16 tile for few rows, else tiles through LDS on the pipe's own order of the scales
struct Plan {
  bool tiled, big, inplace;
  int wt, xt;                    // split over k: 16-row tiles of a workgroup
  long long ntiles, mtiles;
  long long codes, xs, ws, all;  // bytes: codes of x, scales of x, tiled scales of the weight, the workspace
  long long xgroups, wgroups, k4;
};

static Plan plan_linear(int x_dtype, long long rows, long long n, long long k) {
  Plan p{};
  const long long kb = (k + 31) / 32;
  p.codes = x_dtype == YL_MX4 ? 0 : (rows * kb * 16 + 255) / 256 * 256;
  const long long tiles128 = ((n + 127) / 128) * ((rows + 127) / 128), tiles256 = ((n + 255) / 256) * ((rows + 255) / 256);
  // Measured, kernel alone, tiles of 128 against the split form: 64 x 768 x 768 6.8 / 5.4 us, 400 x 768 x 768 (24 tiles) 7.0 / 5.8,
  // 256 x 1024 x 4096 (16 tiles) 15.2 / 14.8, 33 x 8192 x 8192 25 / 20; 128 x 4096 x 4096 (32 tiles) 15.6 / 15.1,
  // 1600 x 768 x 768 (78) 7.5 / 11, 512 x 4096 x 4096 (128) 16.5 / 48.
  p.tiled = rows > 64 && tiles128 >= 32;
  if (p.tiled) {
    // tiles of 128: three workgroups on a CU hide each other's prologue and epilogue, tiles of 256 move half the bytes.  Measured,
    // tiles of 128 / 256: 204800 x 384 x 384 53 / 81 us, 51200 x 384 x 768 24 / 32; 4096^3 50 / 41, 16384 x 4096 x 4096 232 / 191.
    p.big = tiles256 >= 192 && kb >= 32;
    const int tile = p.big ? 256 : 128;
    p.ntiles = (n + tile - 1) / tile, p.mtiles = (rows + tile - 1) / tile;
    p.k4 = (kb + 15) / 16, p.xgroups = (rows + 63) / 64, p.wgroups = (n + 63) / 64;
    p.xs = p.k4 * p.xgroups * 1024, p.ws = p.k4 * p.wgroups * 1024;
  } else {
    // 32 weight rows x 64 rows of x to a workgroup, 16 x 32 where that makes few workgroups (whole call: 300 x 96 x 16384 (15 of the
    // large) 44 / 23 us, 64 x 4096 x 4096 (128) 13.4 / 12.9; 33 x 8192 x 8192 (256) 19 / 33)
    const bool small = rows <= 32 || (n + 31) / 32 * ((rows + 63) / 64) <= 128;
    p.xt = rows <= 16 ? 1 : (small ? 2 : 4);
    // Up to 16 rows of values are quantised where they are read, by every workgroup again: what that costs grows with the weight, a launch
    // of its own does not.  In place / two launches: 1 x 4096 x 4096 11.4 / 6.1 + 4.7 us with a gap between (kernels alone, cold caches),
    // 1 x 11008 x 4096 18.6 / 11.7, 1 x 32000 x 4096 59 / 21 (whole call).
    p.inplace = x_dtype != YL_MX4 && p.xt == 1 && n * k <= 1 << 24;
    // two weight tiles share a workgroup's codes where there are many (16 x 32000 x 4096 30 / 23 us, 1 x 8192 x 4096 no difference)
    p.wt = small ? (p.xt == 1 && !p.inplace && n >= 16384 ? 2 : 1) : 2;
    p.ntiles = (n + 16 * p.wt - 1) / (16 * p.wt), p.mtiles = (rows + 16 * p.xt - 1) / (16 * p.xt);
    if (p.inplace) p.codes = 0;
    p.xs = x_dtype == YL_MX4 || p.inplace ? 0 : (rows * kb + 255) / 256 * 256;
  }
  p.all = p.codes + p.xs + p.ws;
  return p;
}

template <typename T, int WT, int XT, int NWM, int KS, int NS>
static int gemm_launch(const LinearArgs& a, hipStream_t s) {
  auto kern = mx4_gemm_kernel<T, WT, XT, NWM, KS, NS>;
  const int lds = NS * KS * (2 * WT + NWM * XT) * 1024;
  if (int rc = allow_big_lds(reinterpret_cast<const void*>(kern), lds)) return rc;
  hipLaunchKernelGGL(kern, dim3((unsigned)a.ntiles * (unsigned)a.mtiles), dim3(128 * NWM), lds, s, a);
  YL_HIP(hipGetLastError());
  return 0;
}

template <typename T, typename X, int WT, int XT, int NW>
static int split_launch(const LinearArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((mx4_split_kernel<T, X, WT, XT, NW>), dim3((unsigned)a.ntiles * (unsigned)a.mtiles), dim3(64 * NW), 0, s, a);
  YL_HIP(hipGetLastError());
  return 0;
}

// the sizes and the activations' type: what the call and the size of its workspace refuse alike
static int check_linear(int x_dtype, long long rows, long long n, long long k, Plan* p) {
  if (!value_type(x_dtype) && x_dtype != YL_MX4) return fail(-1, "mx4_linear: activations are bf16, fp16, fp32 or MX4");
  if (int rc = check_matrix("mx4_linear", rows, k, k)) return rc;
  if (int rc = check_matrix("mx4_linear", n, k, k)) return rc;
  if (n < 1 || n > (1 << 22)) return fail(n < 1 ? -1 : -3, "mx4_linear: 1 to 4194304 output columns");
  if (rows == 0) return 0;
  *p = plan_linear(x_dtype, rows, n, k);
  if (p->ntiles * p->mtiles > 0xFFFFFFFFLL / (p->tiled && !p->big ? 256 : 512))  // (threads of a grid: below 2^32)
    return fail(-3, "mx4_linear: more rows than one launch covers");
  return 0;
}

extern "C" int64_t yl_mx4_linear_workspace_bytes(int x_dtype, int64_t rows, int64_t n, int64_t k) {
  Plan p{};
  return check_linear(x_dtype, rows, n, k, &p) ? -1 : p.all;
}

extern "C" int yl_mx4_linear(const void* x, const uint8_t* x_scales, int x_dtype, int64_t rows, int64_t x_stride,
                             const uint8_t* w_codes, const uint8_t* w_scales, int64_t n, int64_t k, const float* bias, int act,
                             const void* res, int64_t res_stride, void* y, int y_dtype, int64_t y_stride, void* work,
                             int64_t work_bytes, void* stream) {
  hipStream_t s = static_cast<hipStream_t>(stream);
  Plan p{};
  if (int rc = check_linear(x_dtype, rows, n, k, &p)) return rc;
  if (!value_type(y_dtype)) return fail(-1, "mx4_linear: bf16, fp16 or fp32 results");
  if (rows == 0) return 0;
  if (x_dtype != YL_MX4)
    if (int rc = check_matrix("mx4_linear", rows, k, x_stride)) return rc;
  if (rows > 1 && (y_stride < n || (res && res_stride < n))) return fail(-1, "mx4_linear: a row stride is smaller than a row");
  if (!x || !w_codes || !w_scales || !y) return fail(-1, "mx4_linear: null pointer");
  if (x_dtype == YL_MX4 && !x_scales) return fail(-1, "mx4_linear: MX4 activations come with their scales");
  if (!aligned16(w_codes) || (x_dtype == YL_MX4 && !aligned16(x))) return fail(-1, "mx4_linear: codes must be 16-byte aligned");
  if (p.all > 0 && (!work || work_bytes < p.all || !aligned16(work)))
    return fail(-1, "mx4_linear: workspace missing, too small or not 16-byte aligned");
  LinearArgs a{};
  a.rows = rows, a.n = (int)n, a.k = (int)k, a.kb = (int)((k + 31) / 32);
  a.wc = w_codes, a.ws = w_scales, a.bias = bias, a.act = act;
  a.res = res, a.res_stride = res_stride, a.y = y, a.y_stride = y_stride;
  const int ye = elem_bytes(y_dtype);
  a.vec = aligned16(y) && (rows == 1 || y_stride * ye % 16 == 0) && (!res || (aligned16(res) && (rows == 1 || res_stride * ye % 16 == 0)));
  a.ntiles = (int)p.ntiles, a.mtiles = (int)p.mtiles, a.xgroups = (int)p.xgroups, a.wgroups = (int)p.wgroups;
  uint8_t* const codes = static_cast<uint8_t*>(work);
  uint8_t* const xs = codes + p.codes;
  const bool packed = x_dtype == YL_MX4;
  const int xvec = !packed && aligned16(x) && (rows == 1 || x_stride * elem_bytes(x_dtype) % 16 == 0);
  a.x = packed ? x : codes, a.x_stride = 16LL * a.kb;
  if (!p.tiled) {
    a.xs = packed ? x_scales : xs;
    if (p.inplace) {
      a.x = x, a.x_stride = x_stride, a.xvec = xvec;
      return by_type(y_dtype, [&](auto* t) {
        return by_type(x_dtype, [&](auto* u) {
          return split_launch<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(u)>, 1, 1, 8>(a, s);
        });
      });
    }
    if (!packed)
      if (int rc = quantize_launch(x, x_dtype, rows, k, x_stride, codes, xs, s)) return rc;
    return by_type(y_dtype, [&](auto* t) {
      typedef std::remove_pointer_t<decltype(t)> T;
      if (p.xt == 1) return p.wt == 1 ? split_launch<T, uint8_t, 1, 1, 8>(a, s) : split_launch<T, uint8_t, 2, 1, 8>(a, s);
      return p.xt == 2 ? split_launch<T, uint8_t, 1, 2, 8>(a, s) : split_launch<T, uint8_t, 2, 4, 8>(a, s);
    });
  }
  TileArgs ta{};
  ta.q.x = x, ta.q.rows = rows, ta.q.stride = x_stride, ta.q.cols = (int)k, ta.q.kb = a.kb;
  ta.q.vec = xvec;
  ta.q.codes = packed ? nullptr : codes, ta.q.scales = const_cast<uint8_t*>(x_scales);
  ta.xs = xs, ta.ws = w_scales, ta.wst = xs + p.xs, ta.n = (int)n, ta.xgroups = a.xgroups, ta.wgroups = a.wgroups;
  if (int rc = by_type(packed ? YL_BF16 : x_dtype, [&](auto* t) {
        const unsigned groups = (unsigned)(p.xgroups + p.wgroups), gy = std::min<unsigned>(groups, GROUPS_Y);
        hipLaunchKernelGGL(mx4_tile_kernel<std::remove_pointer_t<decltype(t)>>, dim3((unsigned)p.k4, gy, (groups + gy - 1) / gy), dim3(1024), 0, s, ta);
        YL_HIP(hipGetLastError());
        return 0;
      }))
    return rc;
  a.xs = ta.xs, a.ws = ta.wst;
  return by_type(y_dtype, [&](auto* t) {
    typedef std::remove_pointer_t<decltype(t)> T;
    return p.big ? gemm_launch<T, 8, 4, 4, 2, 2>(a, s) : gemm_launch<T, 4, 4, 2, 1, 3>(a, s);
  });
}
